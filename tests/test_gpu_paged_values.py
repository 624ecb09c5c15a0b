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


@TYPES
@BATCHES
@pytest.mark.parametrize("what", ["nan", "inf"])
def test_nan_and_infinite_scores_show(dtype, seqs, what):
    """One key whose score is NaN, or +inf (softmax of it is inf - inf), makes NaN of every row that sees it, at any
    place of its group of keys."""
    if what == "inf" and dtype == F16:
        pytest.skip("no finite fp16 operands have an infinite score")
    b = ref.Batch(seqs, 8, 2, 128, 16, dtype, seed=2)
    q = b.q()
    q[:, :, 3] = 9.0
    want = run(b, q)
    for at in range(8):
        pages = [(b.table[s, 0], (at + s) % 8) for s in range(len(seqs))]
        saved = [b.k[p, 0, r].clone() for p, r in pages]
        for p, r in pages:
            b.k[p, 0, r] = 0
            b.k[p, 0, r, 3] = math.nan if what == "nan" else 3e38
        out = run(b, q)
        for s, (n, length) in enumerate(seqs):
            sees = torch.arange(length - n, length, device="cuda") >= (at + s) % 8
            rows = out[b.start[s]:b.start[s] + n, :4]
            assert rows[sees].isnan().all() and torch.isfinite(rows[~sees]).all()
        assert torch.equal(out[:, 4:], want[:, 4:])
        for (p, r), x in zip(pages, saved):
            b.k[p, 0, r] = x


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@BATCHES
def test_scores_of_minus_infinity_weigh_nothing(dtype, seqs):
    """Scores that overflow to -inf are as if masked: alone they leave a row 0, beside others they add nothing."""
    b = ref.Batch(seqs, 8, 2, 128, 16, dtype, seed=3)
    q = torch.full((b.total, 8, 128), 1e20, dtype=dtype, device="cuda")
    keys = [(b.table[s, i // 16], i % 16) for s in range(len(seqs)) for i in range(seqs[s][1])]
    pages, rows = (torch.tensor(x, device="cuda") for x in zip(*[(int(p), r) for p, r in keys]))
    b.k[pages, :, rows] = torch.full((), -1e20, dtype=dtype, device="cuda")
    assert (run(b, q) == 0).all()
    for s in range(len(seqs)):  # one key of each sequence that counts
        b.k[b.table[s, 0], :, 2] = 0
    out = run(b, q)
    for s, (n, length) in enumerate(seqs):
        v = b.v[b.table[s, 0], :, 2].repeat_interleave(4, 0)
        sees = torch.arange(length - n, length, device="cuda") >= 2
        rows = out[b.start[s]:b.start[s] + n]
        assert torch.equal(rows[sees], v.expand_as(rows)[sees]) and (rows[~sees] == 0).all()


@pytest.mark.parametrize("seqs", [[(1, 4096)] * 64, [(64, 4096)], [(300, 6000)] * 8], ids=["tokens", "chunk", "chunks"])
def test_small_weights_of_fp16(seqs):
    """Thousands of keys, each 2^-25.5 as likely as the first: below what fp16 holds, a 1000th of the row together.

    P carries a factor 2^7, so its rounding is off by 2^-12 of P, or by 2^-25 in its subnormal range, 2^-32 of the
    largest weight; the sum of weights is rounded nowhere near that, and v is 1: error <= n 2^-32 + 2^-11 o (the
    output's rounding and P's) + 2^-18 o (exponentials, sums)."""
    b = ref.Batch(seqs, 8, 2, 128, 16, F16, seed=4)
    s0 = -17.6875  # 2^-25.52
    for s, (n, length) in enumerate(seqs):
        pages = b.table[s, :-(-length // 16)].long()
        b.k[pages] = 0
        b.k[pages, :, :, 7] = s0
        b.v[pages] = 1
        b.k[pages[0], :, 0, 7] = 0
        b.v[pages[0], :, 0] = 0
    q = torch.zeros(b.total, 8, 128, dtype=F16, device="cuda")
    q[:, :, 7] = 1
    out = run(b, q, scale=1.0)
    for s, (n, length) in enumerate(seqs):
        small = torch.arange(length - n, length, dtype=torch.float64, device="cuda") * math.exp(s0)
        want = (small / (1 + small))[:, None, None]
        err = (out[b.start[s]:b.start[s] + n].double() - want).abs()
        assert (err <= length * 2.0 ** -32 + want * (2.0 ** -11 + 2.0 ** -18)).all(), (err / want).max()


class WithAbsoluteValues:
    """A batch whose V is |V|: its attention is sum p |v|."""

    def __init__(self, b):
        self.__dict__ = {**b.__dict__, "v": b.v.abs()}


@pytest.mark.parametrize("dtype", [F16, BF16], ids=["f16", "bf16"])
@pytest.mark.parametrize("heads", [(32, 8), (8, 8), (5, 1), (8, 1)], ids=str)
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("max_new", [0, 1], ids=["", "hint"])
def test_decode_rounds_only_its_output(dtype, heads, d, max_new):
    """Up to 8 rows: P is kept in two parts, so where the reference's bound allows twice a rounding of P to the pages'
    type (2 u sum p |v|), two roundings of its second part are all that is left: the first leaves at most 2^-8 P, the
    second 2^-8 of that (fp16: less), 2^-15 sum p |v| for both."""
    b = ref.Batch([(1, n) for n in (1, 17, 300, 4096, 9000, 2500)], *heads, d, 16, dtype, seed=6)
    q = b.q()
    out = run(b, q, max_new=max_new).double()
    want, bound = ref.attention(b, q)
    a = ref.attention(WithAbsoluteValues(b), q)[0]
    bound = bound + a * (2.0 ** -15 - torch.finfo(dtype).eps)
    assert ((out - want).abs() <= bound).all()
