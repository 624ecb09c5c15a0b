"""The paged-cache operators against their definitions in 64 bits: rotary append and attention, every type, head
layout and page size where they can go wrong, empty rows, dropped pages, poisoned rows, strides, streams and graphs."""
import math

import pytest
import torch

from minfer_b200 import ops
from minfer_b200._lib import MinferError
import paged_ref as ref
from test_gpu_sample_batch import rule as sampling_rule_64

pytestmark = pytest.mark.gpu
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
SENTINEL = 77.0


@pytest.fixture(autouse=True)
def _device(gpu):
    return gpu


def run_attention(b, q, **kw):
    out = torch.full((b.total, b.hq, b.d), SENTINEL, dtype=b.dtype, device="cuda")
    n = ops.paged_attention_workspace_bytes(b.total, b.hq, b.hkv, b.d, b.dtype)
    ws = torch.full((n,), 255, dtype=torch.uint8, device="cuda")  # NaN wherever it is read unwritten
    ops.paged_attention(out, q, *b.args(), workspace=ws, **kw)
    return out


def check_attention(b, q=None, window=0, scale=None, **kw):
    q = b.q() if q is None else q
    out = run_attention(b, q, window=window, **({} if scale is None else {"scale": scale}), **kw)
    want, bound = ref.attention(b, q, window, scale)
    lo, hi = b.start[0], b.start[-1]
    assert (out[:lo] == SENTINEL).all() and (out[hi:] == SENTINEL).all()
    err = (out[lo:hi].double() - want[lo:hi]).abs()
    over = err / bound[lo:hi]
    assert torch.isfinite(out[lo:hi]).all()
    assert over.numel() == 0 or over.max() <= 1, f"error {over.max():.3g} times the bound"
    return out


TYPES = [(F32, "f32"), (F16, "f16"), (BF16, "bf16")]
HEADS = [(1, 1), (4, 2), (6, 2), (8, 1), (5, 5), (10, 2), (32, 2), (32, 1)]


@pytest.mark.parametrize("dtype", [t for t, _ in TYPES], ids=[n for _, n in TYPES])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("hq,hkv", HEADS)
def test_single_tokens(dtype, d, hq, hkv):
    """Decode: one new token of each sequence, lengths from one key to several tiles, one of them without keys."""
    b = ref.Batch([(1, 1), (1, 2), (1, 63), (1, 64), (1, 65), (0, 9), (1, 0), (1, 700)], hq, hkv, d, 16, dtype, seed=hq + d)
    check_attention(b, max_new=1)


@pytest.mark.parametrize("dtype", [t for t, _ in TYPES], ids=[n for _, n in TYPES])
@pytest.mark.parametrize("page", [8, 16, 24, 64, 80, 128, 256])
def test_page_sizes(dtype, page):
    b = ref.Batch([(1, 333), (3, 129), (40, 200)], 8, 2, 128, page, dtype, seed=page)
    check_attention(b)


@pytest.mark.parametrize("dtype", [t for t, _ in TYPES], ids=[n for _, n in TYPES])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("hq,hkv", HEADS)
def test_chunks(dtype, d, hq, hkv):
    """Chunks of new tokens: whole prompts, late chunks, odd sizes, mixed with single tokens."""
    b = ref.Batch([(65, 65), (130, 517), (1, 300), (7, 7), (0, 0), (129, 1000)], hq, hkv, d, 32, dtype, seed=hq * 3 + d)
    check_attention(b)


@pytest.mark.parametrize("dtype", [t for t, _ in TYPES], ids=[n for _, n in TYPES])
@pytest.mark.parametrize("window", [1, 5, 64, 100, 129, 5000])
def test_window(dtype, window):
    b = ref.Batch([(1, 400), (1, 3), (70, 70), (50, 613)], 8, 2, 128, 16, dtype, seed=window)
    check_attention(b, window=window)


@pytest.mark.parametrize("dtype", [t for t, _ in TYPES], ids=[n for _, n in TYPES])
def test_window_drops_pages(dtype):
    """Pages behind every row's window may be given away: their ids are bad, or their rows hold anything."""
    b = ref.Batch([(1, 400), (20, 420), (90, 610)], 8, 2, 128, 16, dtype, seed=3)
    q = b.q()
    want = check_attention(b, q, window=64)
    for s, (n, length) in enumerate(b.seqs):
        first = (length - n - 64 + 1) // 16  # page of the first position that any row sees
        for i in range(first):
            if i % 2:
                b.table[s, i] = [-1, b.n_pages, 2 ** 31 - 1, -2 ** 31][i // 2 % 4]
            else:
                b.k[b.table[s, i]] = math.nan
                b.v[b.table[s, i]] = math.inf
        row = (length - n - 64 + 1) % 16
        b.k[b.table[s, first], :, :row] = math.inf
        b.v[b.table[s, first], :, :row] = math.nan
    got = run_attention(b, q, window=64)
    assert torch.equal(got, want)


@pytest.mark.parametrize("dtype", [t for t, _ in TYPES], ids=[n for _, n in TYPES])
def test_dropped_pages(dtype):
    """A bad page id masks its positions: in the middle, at the ends, all of a sequence's."""
    b = ref.Batch([(1, 200), (1, 33), (80, 300), (1, 16), (33, 33)], 8, 2, 128, 16, dtype, seed=5)
    bad = [-1, b.n_pages, -2 ** 31]
    for s, pages in ((0, (0, 3, 12)), (1, (2,)), (2, (0, 1, 2, 3, 9, 14)), (3, (0,)), (4, (0, 1, 2))):
        for i in pages:
            b.table[s, i] = bad[i % 3]
    out = check_attention(b)
    assert (out[b.start[3]:b.start[5]] == 0).all()


@pytest.mark.parametrize("dtype", [t for t, _ in TYPES], ids=[n for _, n in TYPES])
def test_rows_without_keys(dtype):
    """Tokens before position 0 (more new tokens than positions) see nothing: zeros."""
    b = ref.Batch([(5, 2), (3, 0), (40, 1), (100, 30), (1, 1)], 4, 2, 128, 16, dtype, seed=6)
    out = check_attention(b)
    assert (out[:3] == 0).all() and (out[5:8] == 0).all() and (out[8:47] == 0).all()


@pytest.mark.parametrize("dtype", [t for t, _ in TYPES], ids=[n for _, n in TYPES])
def test_foreign_rows_and_layouts(dtype):
    """Rows of nobody stay; pages as [n_pages, page, heads, d], q and out as slices of wider rows, a table inside another."""
    b = ref.Batch([(1, 90), (66, 200)], 8, 2, 128, 16, dtype, seed=7, nhd=True, gap=(3, 5))
    q = b.q()
    want = check_attention(b, q)
    wide = torch.full((b.total, 12, 128), math.nan, dtype=dtype, device="cuda")
    wide[:, 2:10] = q
    out = torch.full((b.total, 10, 128), SENTINEL, dtype=dtype, device="cuda")
    table = torch.full((2, b.max_pages + 3), -5, dtype=torch.int32, device="cuda")
    table[:, :b.max_pages] = b.table
    ops.paged_attention(out[:, 1:9], wide[:, 2:10], b.k, b.v, table[:, :b.max_pages], b.q_start, b.lens)
    assert torch.equal(out[:, 1:9], want) and (out[:, 0] == SENTINEL).all() and (out[:, 9] == SENTINEL).all()
    flat = torch.full((b.total, 8 * 128), SENTINEL, dtype=dtype, device="cuda")
    ops.paged_attention(flat, q.view(b.total, -1), *b.args())
    assert torch.equal(flat.view_as(want), want)


@pytest.mark.parametrize("dtype", [t for t, _ in TYPES], ids=[n for _, n in TYPES])
@pytest.mark.parametrize("hints", [dict(), dict(max_new=1), dict(max_new=1, max_len=1), dict(max_new=300, max_len=100000), dict(max_len=2)])
def test_hints_change_nothing(dtype, hints):
    b = ref.Batch([(1, 1500), (9, 40), (200, 900)], 8, 2, 128, 16, dtype, seed=8)
    check_attention(b, **hints)


@pytest.mark.parametrize("dtype", [F16, BF16], ids=["f16", "bf16"])
@pytest.mark.parametrize("scale", [1.0, 0.01, -0.3])
def test_scale_and_large_scores(dtype, scale):
    """Scores of a few hundred, maxima that keep moving along the keys."""
    b = ref.Batch([(1, 1000), (64, 600)], 4, 2, 128, 16, dtype, seed=9)
    q = b.q()
    for s in range(2):  # later keys score higher: the running maximum moves in every tile
        for i in range(b.seqs[s][1]):
            page = b.table[s, i // 16]
            b.k[page, :, i % 16] = (b.k[page, :, i % 16].float() * (0.2 + i / 400)).to(dtype)
    check_attention(b, q, scale=scale)


def test_long_context():
    """32768 positions split over the whole GPU, against the definition."""
    b = ref.Batch([(1, 32768), (1, 5), (2, 20001)], 8, 2, 128, 64, BF16, seed=10)
    check_attention(b, max_new=2)
    b = ref.Batch([(130, 16000)], 8, 2, 128, 64, BF16, seed=11)
    check_attention(b)


@pytest.mark.parametrize("dtype", [t for t, _ in TYPES], ids=[n for _, n in TYPES])
def test_k_and_v_in_one_tensor(dtype):
    """K and V interleaved page by page in one allocation, V before K, and the same pages for both."""
    b = ref.Batch([(1, 150), (40, 90)], 8, 2, 128, 16, dtype, seed=14)
    q = b.q()
    want = check_attention(b, q)
    both = torch.stack([b.v, b.k], 1)  # [n_pages, 2, heads, page, d]
    b.v, b.k = both[:, 0], both[:, 1]
    assert torch.equal(run_attention(b, q), want)
    b.v = b.k
    check_attention(b, q)


def test_many_sequences():
    seqs = [((i % 3 == 0) + (i % 50 == 7) * 20, 1 + (i * 37) % 300) for i in range(600)]
    seqs = [(min(n, length), length) for n, length in seqs]
    b = ref.Batch(seqs, 4, 2, 64, 16, F16, seed=12)
    check_attention(b)


def test_offsets_past_32_bits():
    """Pages whose byte and element offsets pass 2^32."""
    need = 5 * 2 ** 30  # elements of K: 10 GB
    n_pages = need // (2 * 64 * 128)
    b = ref.Batch([(1, 150), (70, 200)], 4, 2, 128, 64, BF16, seed=13)
    q = b.q()
    want = run_attention(b, q)
    k = torch.empty(n_pages, 2, 64, 128, dtype=BF16, device="cuda")
    v = torch.empty_like(k)
    table = b.table.clone()
    for s in range(2):
        for i in range(b.max_pages):
            if 0 <= b.table[s, i] < b.n_pages:
                at = n_pages - 1 - int(b.table[s, i])
                k[at], v[at] = b.k[b.table[s, i]], b.v[b.table[s, i]]
                table[s, i] = at
    b.k, b.v, b.table, b.n_pages = k, v, table, n_pages
    assert torch.equal(run_attention(b, q), want)
    qkv = torch.randn(b.total, 8 * 128, device="cuda")
    f = ops.rope_freqs(128, 1e6)[0].cuda()
    ops.paged_rope_append(q, *b.args()[:3], qkv, b.q_start, b.lens, f)
    assert torch.equal(k[table[0, 149 // 64], 1, 149 % 64] * 0 + v[table[0, 149 // 64], 1, 149 % 64], qkv[0].view(8, 128)[7].to(BF16))


# ---------------------------------------------------------------- rotary append

def check_rope(b, x_dtype, d_rot, interleaved=False, norm=True, scaling="none", positions=None, seed=0, x_pad=0):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    width = (b.hq + 2 * b.hkv) * b.d
    qkv = (r(b.total, width + x_pad) * 2).to(x_dtype)[:, :width]
    f, m = ops.rope_freqs(d_rot, 1e6, scaling, 4.0, 32768) if d_rot else (torch.empty(0, dtype=torch.float64), 1.0)
    f = f.cuda()
    qw, kw = (1 + 0.3 * r(b.d), 1 + 0.3 * r(b.d)) if norm else (None, None)
    q = torch.full((b.total, b.hq, b.d), SENTINEL, dtype=b.dtype, device="cuda")
    b.k.fill_(SENTINEL)
    b.v.fill_(SENTINEL)
    want = ref.rope(b, qkv, f, interleaved, m, qw, kw, 1e-6, positions)
    ops.paged_rope_append(q, *b.args()[:3], qkv, b.q_start, b.lens, f, interleaved=interleaved, mscale=m, q_norm_w=qw,
                          k_norm_w=kw, eps=1e-6, positions=positions)
    # Norm: a sum of d squares, root, quotient and two products, below (d/2 + 8) 2^-24; the angle is rounded to a float
    # of at most pi (2^-23 absolute with the sine's own error), each product and sum adds 2^-24 of the pair's length.
    u, f24 = torch.finfo(b.dtype).eps / 2, 2.0 ** -24
    for got, w in zip((q, b.k, b.v), want):
        untouched = torch.isnan(w)
        assert (got[untouched] == SENTINEL).all()
        pair = w.abs().nan_to_num().amax(-1, keepdim=True) * 2 ** 0.5  # no pair is longer than twice the largest element's square
        bound = u * w.abs() + (b.d / 2 + 24) * f24 * pair + 2.0 ** -25 * (b.dtype == F16) + 1e-30
        assert ((got.double() - w).abs() <= bound)[~untouched].all()
        if got is b.v:
            assert torch.equal(got[~untouched].double(), w[~untouched].to(b.dtype).double())


@pytest.mark.parametrize("x_dtype", [F32, F16, BF16], ids=["xf32", "xf16", "xbf16"])
@pytest.mark.parametrize("dtype", [F32, F16, BF16], ids=["f32", "f16", "bf16"])
@pytest.mark.parametrize("d", [64, 128])
def test_rope_types(x_dtype, dtype, d):
    b = ref.Batch([(1, 1), (3, 40), (0, 5), (20, 20), (1, 17)], 6, 2, d, 16, dtype, seed=1)
    check_rope(b, x_dtype, d)


@pytest.mark.parametrize("d,d_rot", [(64, 64), (64, 8), (64, 56), (128, 128), (128, 64), (128, 112), (128, 8), (128, 0)])
@pytest.mark.parametrize("interleaved", [False, True], ids=["half", "pairs"])
@pytest.mark.parametrize("norm", [False, True], ids=["plain", "norm"])
def test_rope_layouts(d, d_rot, interleaved, norm):
    b = ref.Batch([(2, 9), (5, 4000)], 4, 4, d, 24, F32, seed=2)
    check_rope(b, F32, d_rot, interleaved, norm)


@pytest.mark.parametrize("scaling", ["none", "linear", "ntk", "yarn"])
def test_rope_far_positions(scaling):
    """Positions up to 2^31: the angles stay as exact as near zero."""
    b = ref.Batch([(4, 500)], 4, 2, 128, 16, F32, seed=3)
    pos = torch.tensor([131071, 1_000_003, 2 ** 24 + 1, 2 ** 31 - 1], dtype=torch.int32, device="cuda")
    check_rope(b, F32, 128, False, True, scaling, positions=pos)
    check_rope(b, F32, 128, True, True, scaling)


def test_rope_strides_foreign_rows_and_bad_pages():
    b = ref.Batch([(3, 50), (2, 1), (9, 90), (1, 40)], 8, 2, 128, 16, BF16, seed=4, nhd=True, gap=(2, 3))
    b.table[2, 5] = -1  # the last rows of sequence 2 have no page
    b.table[3, 2] = b.n_pages
    check_rope(b, F32, 128, x_pad=64)
    b.lens[0] = 10 ** 6  # past the table: nothing appended, the queries rotated
    b.seqs[0] = (3, b.max_pages * 16)  # lengths are clamped to what the table holds
    b.table[0] = -7
    check_rope(b, F32, 128)


@pytest.mark.parametrize("n", [1, 7, 300, 5000])
def test_rope_many_rows(n):
    """Few and many rows: one head a warp, and many."""
    b = ref.Batch([(n, n + 3)], 16, 2, 128, 64, BF16, seed=5)
    qkv = torch.randn(n, 20 * 128, device="cuda")
    f = ops.rope_freqs(128, 1e6)[0].cuda()
    q = torch.empty(n, 16, 128, dtype=BF16, device="cuda")
    ops.paged_rope_append(q, *b.args()[:3], qkv, b.q_start, b.lens, f)
    ang = 2 * math.pi * torch.fmod(torch.arange(3, n + 3, device="cuda").double()[:, None] * f, 1.0)
    x = qkv.view(n, 20, 128)[:, :18].double()
    lo, hi = x[..., :64], x[..., 64:]
    c, s = torch.cos(ang)[:, None], torch.sin(ang)[:, None]
    w = torch.cat([lo * c - hi * s, hi * c + lo * s], -1)
    key = torch.arange(3, n + 3, device="cuda")
    k = b.k[b.table[0, key // 64].long(), :, key % 64]
    bound = 2.0 ** -8 * w.abs() + 32 * 2.0 ** -24 * x.abs().amax(-1, keepdim=True)
    assert ((q.double() - w[:, :16]).abs() <= bound[:, :16]).all() and ((k.double() - w[:, 16:]).abs() <= bound[:, 16:]).all()


# ---------------------------------------------------------------- how they are called

def test_python_refusals_on_gpu():
    b = ref.Batch([(1, 20)], 4, 2, 128, 16, BF16)
    q = b.q()
    out = torch.empty_like(q)
    bad = [dict(q=q.float()), dict(out=out[:, :2]), dict(q=q[:, :, ::2]), dict(page_table=b.table.long()), dict(kv_lens=b.lens[:0]),
           dict(v_pages=b.v[:-1]), dict(q_start=b.q_start[:1]), dict(v_pages=b.v.float()), dict(page_table=b.table.cpu())]
    good = dict(out=out, q=q, k_pages=b.k, v_pages=b.v, page_table=b.table, q_start=b.q_start, kv_lens=b.lens)
    for change in bad:
        with pytest.raises(ValueError):
            ops.paged_attention(**{**good, **change})
    with pytest.raises(MinferError):
        ops.paged_attention(**good, workspace=torch.empty(256, dtype=torch.uint8, device="cuda"))
    ops.paged_attention(**good)


def test_expanded_tensors_are_refused():
    """A stride of 0 must not be read as "contiguous"."""
    b = ref.Batch([(1, 20), (1, 30)], 4, 2, 128, 16, BF16)
    q, out = b.q(), torch.empty(2, 4, 128, dtype=BF16, device="cuda")
    good = dict(out=out, q=q, k_pages=b.k, v_pages=b.v, page_table=b.table, q_start=b.q_start, kv_lens=b.lens)
    one = b.k[:1].expand(b.n_pages, -1, -1, -1)
    head = b.k[:, :1].expand(-1, 2, -1, -1)
    row = b.k[:, :, :1].expand(-1, -1, 16, -1)
    for change in (dict(q=q[:1].expand(2, -1, -1)), dict(out=out[:1].expand(2, -1, -1)), dict(k_pages=one, v_pages=one), dict(k_pages=head, v_pages=head),
                   dict(k_pages=row, v_pages=row), dict(page_table=b.table[:1].expand(2, -1)), dict(q=torch.zeros(2, 128, 4, dtype=BF16, device="cuda").transpose(1, 2))):
        with pytest.raises(ValueError):
            ops.paged_attention(**{**good, **change})
    with pytest.raises(ValueError):
        ops.paged_rope_append(q, b.k, b.v, b.table, torch.zeros(1, 8 * 128, device="cuda").expand(2, -1), b.q_start, b.lens, torch.zeros(64, dtype=torch.float64, device="cuda"))


@pytest.mark.parametrize("dtype", [t for t, _ in TYPES], ids=[n for _, n in TYPES])
def test_extents_of_one(dtype):
    """One page, one head, one sequence, one token: whatever strides torch gives them."""
    for nhd in (False, True):
        b = ref.Batch([(1, 13)], 3, 1, 64, 16, dtype, nhd=nhd, spare=0)
        assert b.n_pages == 1
        check_attention(b)
        b.k, b.v = (x.as_strided(x.shape, (5, 7, *x.stride()[2:])) for x in (b.k, b.v))
        check_attention(b)
    b = ref.Batch([(1, 100)], 2, 2, 128, 8, dtype, nhd=True, spare=0)
    check_attention(b)


def test_nothing_to_do():
    """No tokens, or no sequences: no error, nothing written."""
    b = ref.Batch([(1, 20)], 4, 2, 128, 16, BF16, gap=(0, 2))
    f = ops.rope_freqs(128, 1e6)[0].cuda()
    k = b.k.clone()
    none = torch.empty(0, 4, 128, dtype=BF16, device="cuda")
    ops.paged_attention(none, none, *b.args())
    ops.paged_rope_append(none, *b.args()[:3], torch.empty(0, 8 * 128, device="cuda"), b.q_start, b.lens, f)
    out = torch.full((3, 4, 128), SENTINEL, dtype=BF16, device="cuda")
    empty = (b.k, b.v, b.table[:0], b.q_start[:1], b.lens[:0])
    ops.paged_attention(out, torch.zeros_like(out), *empty)
    ops.paged_rope_append(out, *empty[:3], torch.zeros(3, 8 * 128, device="cuda"), *empty[3:], f)
    assert (out == SENTINEL).all() and torch.equal(b.k.nan_to_num(), k.nan_to_num())
    # sequences without new tokens, rows of nobody
    ops.paged_attention(out, torch.zeros_like(out), b.k, b.v, b.table, torch.zeros(2, dtype=torch.int32, device="cuda"), b.lens)
    assert (out == SENTINEL).all()


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
def test_starts_and_lengths_out_of_range(dtype):
    """Starts past the call's rows and lengths past the table are clamped; a start that decreases gives no rows."""
    b = ref.Batch([(2, 48), (50, 90), (1, 7)], 4, 2, 128, 16, dtype, seed=30)  # the first fills its pages
    q = b.q()
    want = run_attention(b, q)
    b.q_start[-1] = 10 ** 6
    assert torch.equal(run_attention(b, q), want)
    b.q_start[-1] = -5  # the last sequence has no rows
    got = run_attention(b, q)
    assert torch.equal(got[:52], want[:52]) and (got[52] == SENTINEL).all()
    b.q_start[-1] = 53
    b.lens[0] = 2 ** 31 - 1  # clamped to the table's capacity: positions without a page hold no keys
    b.seqs[0] = (2, b.max_pages * b.page)
    check_attention(b, q)
    b.lens[0] = -7
    b.seqs[0] = (2, 0)
    check_attention(b, q)


@pytest.mark.parametrize("window", [2 ** 31 - 1, 2 ** 30, 400])
def test_windows_longer_than_everything(window):
    b = ref.Batch([(1, 90), (60, 200), (5, 3)], 4, 2, 128, 16, BF16, seed=31)
    q = b.q()
    assert torch.equal(run_attention(b, q, window=window), run_attention(b, q))


def step(b, qkv, f, q, out, ws, **kw):
    ops.paged_rope_append(q, b.k, b.v, b.table, qkv, b.q_start, b.lens, f)
    ops.paged_attention(out, q, *b.args(), workspace=ws, **kw)


@pytest.mark.parametrize("dtype", [t for t, _ in TYPES], ids=[n for _, n in TYPES])
def test_append_then_attend(dtype):
    """The two together: what is appended is attended, and the result is that of the definitions in turn."""
    b = ref.Batch([(1, 77), (33, 33), (70, 333)], 8, 2, 128, 16, dtype, seed=20)
    qkv = torch.randn(b.total, 12 * 128, device="cuda")
    f = ops.rope_freqs(128, 1e6)[0].cuda()
    q, out = torch.empty(b.total, 8, 128, dtype=dtype, device="cuda"), torch.empty(b.total, 8, 128, dtype=dtype, device="cuda")
    for s, (n, length) in enumerate(b.seqs):  # the new tokens' rows hold nothing yet
        for pos in range(length - n, length):
            b.k[b.table[s, pos // 16], :, pos % 16] = math.nan
            b.v[b.table[s, pos // 16], :, pos % 16] = math.nan
    step(b, qkv, f, q, out, None)
    want, bound = ref.attention(b, q)
    assert ((out.double() - want).abs() <= bound).all()


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
def test_graph_replays_with_new_lengths(dtype):
    """One captured step serves a growing batch, on a side stream; two graphs with workspaces of their own."""
    b = ref.Batch([(1, 300), (1, 64), (1, 1)], 8, 2, 128, 16, dtype, seed=21)
    qkv = torch.randn(3, 12 * 128, device="cuda")
    f = ops.rope_freqs(128, 1e6)[0].cuda()
    n = ops.paged_attention_workspace_bytes(3, 8, 2, 128, dtype)
    side = torch.cuda.Stream()
    graphs, outs = [], []
    b.lens -= 20
    for _ in range(2):
        q, out = (torch.zeros(3, 8, 128, dtype=dtype, device="cuda") for _ in range(2))
        ws = torch.empty(n, dtype=torch.uint8, device="cuda")  # lives as long as its graph
        with torch.cuda.stream(side):
            step(b, qkv, f, q, out, ws, max_new=1)
        side.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            step(b, qkv, f, q, out, ws, max_new=1)
        graphs.append(graph)
        outs.append((q, out, ws))
    for lens in ([280, 44, 0], [299, 64, 1], [300, 1, 1]):
        b.lens.copy_(torch.tensor(lens, dtype=torch.int32))
        b.seqs = [(1, x) for x in lens]
        qkv.normal_()
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for q, out, _ in outs:
            want, bound = ref.attention(b, q)
            assert ((out.double() - want).abs() <= bound).all()


def test_same_call_same_bits():
    b = ref.Batch([(1, 5000), (1, 200), (200, 900)], 8, 2, 128, 16, BF16, seed=22)
    q = b.q()
    first = run_attention(b, q)
    for _ in range(5):
        assert torch.equal(run_attention(b, q), first)


def test_batched_decoding_with_sampling():
    """The three operators as a batch is served: prompts of three sequences in one call, then single tokens, each id
    sampled from the logits of the last position; against the same steps in 64 bits."""
    g = torch.Generator(device="cuda")
    g.manual_seed(40)
    r = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    vocab, hq, hkv, d, page = 997, 4, 2, 64, 16
    emb, wqkv, wo = r(vocab, 96), r(96, (hq + 2 * hkv) * d) / 10, r(hq * d, vocab) / 4
    qw, kw = 1 + 0.1 * r(d), 1 + 0.1 * r(d)
    f, m = ops.rope_freqs(d, 1e4, "yarn", 2.0, 512)
    f = f.cuda()
    prompts = [torch.randint(0, vocab, (n,), generator=g, device="cuda").tolist() for n in (5, 40, 17)]
    k, v = (torch.full((20, hkv, page, d), math.nan, device="cuda") for _ in range(2))
    table = torch.randperm(20, generator=g, device="cuda").to(torch.int32)[:15].view(3, 5).contiguous()
    temp, top_k = torch.tensor([0.0, 0.8, 1.2], device="cuda"), torch.tensor([0, 50, 0], dtype=torch.int32, device="cuda")
    top_p, min_p = torch.tensor([1.0, 0.9, 0.95], device="cuda"), torch.tensor([0.0, 0.0, 0.02], device="cuda")
    lens = [0, 0, 0]
    seqs = [list(p) for p in prompts]
    for n_step in range(6):
        new = [s[n:] for s, n in zip(seqs, lens)]
        lens = [len(s) for s in seqs]
        start = [0]
        for n in new:
            start.append(start[-1] + len(n))
        tok = torch.tensor(sum(new, []), device="cuda")
        q_start, kv_lens = (torch.tensor(x, dtype=torch.int32, device="cuda") for x in (start, lens))
        qkv = emb[tok] @ wqkv
        q, out = torch.empty(len(tok), hq, d, device="cuda"), torch.empty(len(tok), hq, d, device="cuda")
        ops.paged_rope_append(q, k, v, table, qkv, q_start, kv_lens, f, mscale=m, q_norm_w=qw, k_norm_w=kw)
        ops.paged_attention(out, q, k, v, table, q_start, kv_lens)
        last = q_start[1:].long() - 1
        logits = out[last].view(3, -1) @ wo
        draws, ids, probs = torch.rand(3, generator=g, device="cuda"), torch.empty(3, dtype=torch.int32, device="cuda"), torch.empty(3, device="cuda")
        ops.sample_batch(ids, logits, draws, temp, top_k, top_p, min_p, probs=probs)
        for b in range(3):  # the whole sequence from its ids, in 64 bits
            x = (emb[torch.tensor(seqs[b], device="cuda")].double() @ wqkv.double()).view(-1, hq + 2 * hkv, d)
            y = x[:, :hq + hkv]
            y = y / torch.sqrt((y ** 2).mean(-1, keepdim=True) + 1e-6) * torch.cat([qw.double().expand(hq, d), kw.double().expand(hkv, d)])
            ang = 2 * math.pi * torch.arange(len(y), device="cuda").double()[:, None, None] * f
            a, z = y[..., :d // 2], y[..., d // 2:]
            y = m * torch.cat([a * torch.cos(ang) - z * torch.sin(ang), z * torch.cos(ang) + a * torch.sin(ang)], -1)
            kk, vv = y[:, hq:].repeat_interleave(hq // hkv, 1), x[:, hq + hkv:].repeat_interleave(hq // hkv, 1)
            p = torch.softmax(torch.einsum("hd,khd->hk", y[-1, :hq], kk) / math.sqrt(d), -1)
            lg = torch.einsum("hk,khd->hd", p, vv).reshape(-1) @ wo.double()
            assert (logits[b].double() - lg).abs().max() < 1e-4 * lg.abs().max()  # fp32 products of 96 and 256 terms
            want, prob = sampling_rule_64(lg.float().cpu().numpy(), draws[b].item(), temp[b].item(), top_k[b].item(), top_p[b].item(), min_p[b].item())
            assert ids[b].item() == want and abs(probs[b].item() - prob) < 1e-3
            seqs[b].append(want)
    assert ops.paged_status() == 0


def test_no_wait_gave_up():
    assert ops.paged_status(clear=False) == 0
