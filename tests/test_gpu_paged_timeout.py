"""Paged attention with a limit of a millisecond on its waits, in calls that take several: blocks give up, and every
row is either finished or as it was."""
import pytest
import torch

from minfer_b200 import ops

pytestmark = pytest.mark.gpu
SENTINEL = 77.0


@pytest.fixture(autouse=True)
def _device(gpu):
    yield gpu
    ops.paged_status(clear=True)


# (sequences, new tokens of each, keys, query heads, KV heads): single tokens, chunks whole and in shares, both
CASES = {"tokens": ([1] * 250, 32768, 64, 8), "chunk": ([16384], 131072, 16, 2), "shares": ([256], 1 << 23, 1, 1),
         "mixed": ([16384] + [1] * 30, 131072, 16, 2)}


@pytest.mark.parametrize("name", list(CASES))
def test_rows_are_finished_or_untouched(monkeypatch, name):
    new, keys, hq, hkv = CASES[name]
    g = torch.Generator(device="cuda")
    g.manual_seed(1)
    r = lambda *s: torch.randn(*s, generator=g, device="cuda", dtype=torch.bfloat16)  # noqa: E731
    n, n_pages = sum(new), min(keys // 64, 2048)
    k, v, q = r(n_pages, hkv, 64, 128), r(n_pages, hkv, 64, 128), r(n, hq, 128)
    table = (torch.arange(keys // 64, device="cuda", dtype=torch.int32) % n_pages).repeat(len(new), 1)  # pages are shared
    start = torch.tensor([0] + new, device="cuda").cumsum(0).to(torch.int32)
    lens = torch.full((len(new),), keys, dtype=torch.int32, device="cuda")
    want = torch.empty_like(q)
    ops.paged_attention(want, q, k, v, table, start, lens, max_new=max(new), max_len=keys)
    assert ops.paged_status() == 0 and torch.isfinite(want).all()
    monkeypatch.setenv("MF_PREFILL_TIMEOUT_MS", "1")
    ws = torch.full((ops.paged_attention_workspace_bytes(n, hq, hkv, 128, torch.bfloat16),), 255, dtype=torch.uint8, device="cuda")
    for _ in range(3):  # the workspace holds the parts of the calls before
        out = torch.full_like(q, SENTINEL)
        ops.paged_attention(out, q, k, v, table, start, lens, max_new=max(new), max_len=keys, workspace=ws)
        status = ops.paged_status()
        same, left = (out == want).all(-1), (out == SENTINEL).all(-1)
        print(name, "gave up" if status else "finished", f"{int(left.sum())} of {n * hq} rows left")
        assert (same | left).all()
        assert status == (2 if left.any() else 0)
    monkeypatch.delenv("MF_PREFILL_TIMEOUT_MS")
    out = torch.full_like(q, SENTINEL)
    ops.paged_attention(out, q, k, v, table, start, lens, max_new=max(new), max_len=keys, workspace=ws)
    assert torch.equal(out, want) and ops.paged_status() == 0
