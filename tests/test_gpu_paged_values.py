"""Paged attention where values leave the ordinary range: NaN and infinite scores, weights below the pages' type."""
import math

import pytest
import torch

from minfer_b200 import ops
import paged_ref as ref

pytestmark = pytest.mark.gpu
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
TYPES = pytest.mark.parametrize("dtype", [F32, F16, BF16], ids=["f32", "f16", "bf16"])

# single tokens in one range of tiles and in many, chunks of both, both kinds in one batch
BATCHES = pytest.mark.parametrize("seqs", [[(1, 50), (1, 20000)], [(1, 300)] * 40, [(70, 5000)], [(130, 16000)], [(200, 333)] * 3, [(1, 9000), (90, 2000)]],
                                  ids=["long", "many", "chunk", "late chunk", "chunks", "mixed"])


@pytest.fixture(autouse=True)
def _device(gpu):
    return gpu


def run(b, q, **kw):
    out = torch.full((b.total, b.hq, b.d), 77.0, dtype=b.dtype, device="cuda")
    n = ops.paged_attention_workspace_bytes(b.total, b.hq, b.hkv, b.d, b.dtype)
    ws = torch.full((n,), 255, dtype=torch.uint8, device="cuda")
    ops.paged_attention(out, q, *b.args(), workspace=ws, **kw)
    return out


@TYPES
@BATCHES
def test_nan_queries_stay_nan(dtype, seqs):
    """A NaN anywhere in a query makes its row NaN, however the keys are shared out, and no other row."""
    b = ref.Batch(seqs, 8, 2, 128, 16, dtype, seed=1)
    q = b.q()
    want = run(b, q)
    bad = torch.zeros(b.total, b.hq, dtype=torch.bool, device="cuda")
    bad[::3, 1], bad[b.total - 1, 6], bad[b.total // 2, 4] = True, True, True
    q[bad, 5] = math.nan
    out = run(b, q)
    assert out[bad].isnan().all()
    assert torch.equal(out[~bad], want[~bad])
