"""Refusals of the paged-cache and batch-sampling entry points, and the rotary frequencies: no GPU needed (every check
is made before a launch)."""
import ctypes as C
import math

import pytest
import torch

from minfer_b200 import _lib as L
from minfer_b200 import ops

lib = L.cuda_lib()
A = 0x10000  # an aligned address that no refused call touches


def kv(**change):
    c = dict(k_pages=A, v_pages=A, page_stride=0, head_stride=0, row_stride=0, page_table=A, q_start=A, kv_lens=A,
             table_stride=0, max_pages=4, n_pages=8, page_size=16, n_seqs=2, n_kv_heads=2, d_head=128, dtype=L.MF_BF16)
    c.update(change)
    return L.mf_paged_kv(*[c[n] for n, _ in L.mf_paged_kv._fields_])


def rope(**change):
    c = dict(q_out=A, q_stride=0, qkv=A, x_stride=0, x_dtype=L.MF_F32, n_tokens=3, n_heads=4, d_rot=128, interleaved=0,
             mscale=1.0, eps=1e-6, freqs=A, q_norm_w=None, k_norm_w=None, positions=None)
    c.update(change)
    return L.mf_paged_rope_desc(*[c[n] for n, _ in L.mf_paged_rope_desc._fields_])


def attn(**change):
    c = dict(out=A, out_stride=0, q=A, q_stride=0, n_tokens=3, n_heads=4, scale=0.0, window=0, max_new=0, max_len=0,
             workspace=A, workspace_bytes=1 << 40)
    c.update(change)
    return L.mf_paged_attn_desc(*[c[n] for n, _ in L.mf_paged_attn_desc._fields_])


BAD_KV = [(dict(k_pages=None), L.MF_E_INVALID), (dict(v_pages=None), L.MF_E_INVALID), (dict(page_table=None), L.MF_E_INVALID),
          (dict(q_start=None), L.MF_E_INVALID), (dict(kv_lens=None), L.MF_E_INVALID), (dict(dtype=3), L.MF_E_INVALID),
          (dict(n_seqs=-1), L.MF_E_INVALID), (dict(n_pages=0), L.MF_E_INVALID), (dict(max_pages=0), L.MF_E_INVALID),
          (dict(n_kv_heads=0), L.MF_E_INVALID), (dict(table_stride=3), L.MF_E_INVALID), (dict(d_head=96), L.MF_E_UNSUPPORTED),
          (dict(page_size=12), L.MF_E_UNSUPPORTED), (dict(page_size=0), L.MF_E_UNSUPPORTED), (dict(k_pages=A + 8), L.MF_E_INVALID),
          (dict(row_stride=64), L.MF_E_INVALID), (dict(row_stride=132), L.MF_E_INVALID), (dict(head_stride=2049), L.MF_E_INVALID),
          (dict(page_stride=-4096), L.MF_E_INVALID), (dict(q_start=A + 2), L.MF_E_INVALID)]


@pytest.mark.parametrize("change,code", BAD_KV, ids=lambda c: str(c)[:40])
def test_bad_cache(change, code):
    assert lib.mf_paged_rope_append(C.byref(kv(**change)), C.byref(rope()), None) == code
    assert lib.mf_paged_attention(C.byref(kv(**change)), C.byref(attn()), None) == code
    assert L.last_error()


@pytest.mark.parametrize("change,code", [
    (dict(q_out=None), L.MF_E_INVALID), (dict(qkv=None), L.MF_E_INVALID), (dict(freqs=None), L.MF_E_INVALID), (dict(x_dtype=7), L.MF_E_INVALID),
    (dict(n_tokens=-1), L.MF_E_INVALID), (dict(n_heads=3), L.MF_E_INVALID), (dict(n_heads=0), L.MF_E_INVALID), (dict(d_rot=130), L.MF_E_INVALID),
    (dict(d_rot=20), L.MF_E_INVALID), (dict(d_rot=-8), L.MF_E_INVALID), (dict(eps=-1.0), L.MF_E_INVALID), (dict(eps=math.nan), L.MF_E_INVALID),
    (dict(q_stride=500), L.MF_E_INVALID), (dict(x_stride=1026), L.MF_E_INVALID), (dict(qkv=A + 4), L.MF_E_INVALID), (dict(freqs=A + 4), L.MF_E_INVALID),
], ids=lambda c: str(c)[:40])
def test_bad_rope(change, code):
    assert lib.mf_paged_rope_append(C.byref(kv()), C.byref(rope(**change)), None) == code


@pytest.mark.parametrize("change,code", [
    (dict(out=None), L.MF_E_INVALID), (dict(q=None), L.MF_E_INVALID), (dict(n_heads=3), L.MF_E_INVALID), (dict(n_tokens=-2), L.MF_E_INVALID),
    (dict(window=-1), L.MF_E_INVALID), (dict(max_new=-1), L.MF_E_INVALID), (dict(max_len=-1), L.MF_E_INVALID), (dict(scale=math.inf), L.MF_E_INVALID),
    (dict(q_stride=8), L.MF_E_INVALID), (dict(out_stride=516), L.MF_E_INVALID), (dict(q=A + 2), L.MF_E_INVALID), (dict(workspace=None), L.MF_E_INVALID),
    (dict(workspace=A + 16), L.MF_E_INVALID), (dict(workspace_bytes=64), L.MF_E_INVALID), (dict(n_tokens=1 << 30), L.MF_E_UNSUPPORTED),
], ids=lambda c: str(c)[:40])
def test_bad_attention(change, code):
    assert lib.mf_paged_attention(C.byref(kv()), C.byref(attn(**change)), None) == code


def test_null_and_empty():
    assert lib.mf_paged_rope_append(None, C.byref(rope()), None) == L.MF_E_INVALID
    assert lib.mf_paged_rope_append(C.byref(kv()), None, None) == L.MF_E_INVALID
    assert lib.mf_paged_attention(C.byref(kv()), None, None) == L.MF_E_INVALID
    for k, n in ((kv(), 0), (kv(n_seqs=0), 3)):  # nothing to do
        assert lib.mf_paged_rope_append(C.byref(k), C.byref(rope(n_tokens=n)), None) == L.MF_OK
        assert lib.mf_paged_attention(C.byref(k), C.byref(attn(n_tokens=n)), None) == L.MF_OK


def sample(**change):
    c = dict(ids=A, probs=None, logits=A, dtype=L.MF_F32, ld=1000, n_rows=2, vocab=1000, draws=A, temp=A, top_k=A, top_p=A, min_p=A)
    c.update(change)
    return lib.mf_sample_batch(*c.values(), None)


@pytest.mark.parametrize("change,code", [
    (dict(ids=None), L.MF_E_INVALID), (dict(logits=None), L.MF_E_INVALID), (dict(draws=None), L.MF_E_INVALID), (dict(temp=None), L.MF_E_INVALID),
    (dict(top_k=None), L.MF_E_INVALID), (dict(top_p=None), L.MF_E_INVALID), (dict(min_p=None), L.MF_E_INVALID), (dict(n_rows=-1), L.MF_E_INVALID),
    (dict(vocab=0), L.MF_E_INVALID), (dict(ld=999), L.MF_E_INVALID), (dict(dtype=5), L.MF_E_INVALID), (dict(vocab=(1 << 18) + 1, ld=1 << 20), L.MF_E_UNSUPPORTED),
    (dict(logits=A + 2), L.MF_E_INVALID), (dict(ids=A + 1), L.MF_E_INVALID), (dict(n_rows=0), L.MF_OK),
], ids=lambda c: str(c)[:40])
def test_bad_sample(change, code):
    assert sample(**change) == code


def test_workspace_bytes():
    assert ops.paged_attention_workspace_bytes(5, 8, 2, 128, torch.bfloat16) > 0
    assert lib.mf_paged_attention_workspace_bytes(0, 8, 2, 128, L.MF_BF16) == 0
    assert lib.mf_paged_attention_workspace_bytes(5, 8, 2, 80, L.MF_BF16) == 0


def test_python_refusals():
    cpu = torch.zeros(4, 2, 16, 128)
    t = torch.zeros(1, 4, dtype=torch.int32)
    with pytest.raises(ValueError, match="CUDA"):
        ops.paged_attention(cpu[0], cpu[0], cpu, cpu, t, t[0], t[0])
    with pytest.raises(ValueError, match="CUDA"):
        ops.sample_batch(t[0], torch.zeros(1, 9), *[torch.zeros(1)] * 5)
    with pytest.raises(ValueError, match="scaling"):
        ops.rope_freqs(128, 1e6, "dynamic")


@pytest.mark.parametrize("d_rot,base", [(128, 1e6), (64, 1e4), (8, 500.0), (2, 10.0)])
def test_rope_freqs(d_rot, base):
    plain = [base ** (-2 * j / d_rot) for j in range(d_rot // 2)]
    turns = lambda f: f / (2 * math.pi)  # noqa: E731
    close = lambda got, want: max(abs(g / turns(w) - 1) for g, w in zip(got.tolist(), want)) < 1e-12  # noqa: E731
    f, m = ops.rope_freqs(d_rot, base)
    assert m == 1.0 and f.dtype == torch.float64 and close(f, plain)
    f, m = ops.rope_freqs(d_rot, base, "linear", 8.0)
    assert m == 1.0 and close(f, [x / 8 for x in plain])
    if d_rot > 2:
        f, m = ops.rope_freqs(d_rot, base, "ntk", 4.0)
        stretched = base * 4.0 ** (d_rot / (d_rot - 2))
        assert m == 1.0 and close(f, [stretched ** (-2 * j / d_rot) for j in range(d_rot // 2)])
    f, m = ops.rope_freqs(d_rot, base, "yarn", 4.0, orig_ctx=32768)
    assert m == pytest.approx(0.1 * math.log(4) + 1, rel=1e-6)
    for j, (got, w) in enumerate(zip(f.tolist(), plain)):
        turned = 32768 * turns(w)  # turns of pair j over the original context
        assert turns(w) / 4 * (1 - 1e-12) <= got <= turns(w) * (1 + 1e-12)
        if turned > 32 * base ** (2 / d_rot):  # a whole pair beyond the ramp's start
            assert got == pytest.approx(turns(w), rel=1e-12)
        if turned < base ** (-2 / d_rot):
            assert got == pytest.approx(turns(w) / 4, rel=1e-12)


@pytest.mark.parametrize("args", [(0, 1e6, "none"), (7, 1e6, "none"), (128, 1.0, "none"), (128, math.inf, "none"), (128, 1e6, "linear", 0.5),
                                  (128, 1e6, "yarn", 4.0), (2, 1e6, "ntk", 2.0), (128, 1e6, "yarn", 4.0, 32768, 1.0, 32.0)])
def test_bad_freqs(args):
    with pytest.raises(L.MinferError):
        ops.rope_freqs(*args)


def test_packed_descriptions_match_the_structures():
    """ops.py packs the C structures itself: same sizes and offsets as their ctypes declarations."""
    for packed, struct in ((ops._KV, L.mf_paged_kv), (ops._ROPE, L.mf_paged_rope_desc), (ops._ATTN, L.mf_paged_attn_desc)):
        assert packed.size == C.sizeof(struct)
        values = [0.5 if t is C.c_float else i + 1 for i, (_, t) in enumerate(struct._fields_)]
        got = struct.from_buffer_copy(packed.pack(*values))
        assert [getattr(got, n) for n, _ in struct._fields_] == values
