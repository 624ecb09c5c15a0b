"""Rotary append and attention on pages whose offsets pass 2^32 elements: the same rows as on a small cache."""
import pytest
import torch

from minfer_b200 import ops
import paged_ref as ref

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _device(gpu):
    return gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
def test_append_writes_every_row_and_head_there(dtype):
    b = ref.Batch([(1, 150), (70, 200)], 4, 2, 128, 64, dtype, seed=13)
    qkv = torch.randn(b.total, 8 * 128, device="cuda")
    f = ops.rope_freqs(128, 1e6)[0].cuda()
    weights = dict(q_norm_w=1 + 0.1 * torch.randn(128, device="cuda"), k_norm_w=1 + 0.1 * torch.randn(128, device="cuda"))
    n_pages = 5 * 2 ** 30 // (2 * 64 * 128)
    k = torch.zeros(n_pages, 2, 64, 128, dtype=dtype, device="cuda")
    v = torch.zeros_like(k)
    table = b.table.clone()
    used = []
    for s in range(2):
        for i in range(b.max_pages):
            page = int(b.table[s, i])
            if 0 <= page < b.n_pages:
                table[s, i] = n_pages - 1 - page
                used.append(page)
    used = torch.tensor(used, device="cuda")
    b.k.zero_()
    b.v.zero_()
    q, want_q = (torch.empty(b.total, 4, 128, dtype=dtype, device="cuda") for _ in range(2))
    ops.paged_rope_append(want_q, b.k, b.v, b.table, qkv, b.q_start, b.lens, f, **weights)
    ops.paged_rope_append(q, k, v, table, qkv, b.q_start, b.lens, f, **weights)
    assert torch.equal(q, want_q)
    at = n_pages - 1 - used
    assert (b.k[used] != 0).any() and torch.equal(k[at], b.k[used]) and torch.equal(v[at], b.v[used])
    k[at], v[at] = 0, 0  # and nothing anywhere else
    assert all(not x[i:i + 65536].any() for x in (k, v) for i in range(0, n_pages, 65536))
