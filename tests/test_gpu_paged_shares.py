"""In how many shares the chunk kernel works on the keys: as many as its row tiles leave SMs idle, none where they
fill the GPU by themselves."""
import pytest
import torch

from minfer_b200 import ops
import paged_ref as ref

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _device(gpu):
    return gpu


def shares(b, **kw):
    """Shares of a call, by what it wrote into its workspace behind the part of the kernels for few rows (which is all
    that a call of very many rows has): a sum for every row of every share, behind the rows of D values."""
    size = lambda n: ops.paged_attention_workspace_bytes(n, b.hq, b.hkv, b.d, b.dtype)  # noqa: E731
    few = size(1 << 20)
    ws = torch.full((size(b.total),), 255, dtype=torch.uint8, device="cuda")
    out = torch.empty(b.total, b.hq, b.d, dtype=b.dtype, device="cuda")
    q = b.q()
    ops.paged_attention(out, q, *b.args(), workspace=ws, **kw)
    want, bound = ref.attention(b, q)
    assert ((out.double() - want).abs() <= bound).all()
    written = (ws[few:].view(torch.int32) != -1).sum().item()
    row = b.hq * b.total * (b.d + 2)
    assert written % row == 0
    return max(written // row, 1)


def test_many_short_sequences_fill_the_gpu():
    """64 sequences of 5 tokens, 8 heads a group: 40 rows each, a tile of its own for every sequence and KV head."""
    b = ref.Batch([(5, 4096)] * 64, 64, 8, 128, 64, torch.bfloat16, seed=1)
    assert shares(b, max_new=5, max_len=4096) == 1


def test_sixteen_sequences_fill_it_once():
    b = ref.Batch([(5, 4096)] * 16, 64, 8, 128, 64, torch.bfloat16, seed=2)
    assert shares(b, max_new=5, max_len=4096) == 1


def test_few_tiles_are_shared_out():
    """One chunk, alone and among single tokens, and few short sequences."""
    b = ref.Batch([(64, 4096)], 64, 8, 128, 64, torch.bfloat16, seed=3)
    alone = shares(b, max_new=64, max_len=4096)
    assert alone > 4
    b = ref.Batch([(5, 4096)] * 3, 64, 8, 128, 64, torch.bfloat16, seed=4)
    assert shares(b, max_new=5, max_len=4096) > 3
