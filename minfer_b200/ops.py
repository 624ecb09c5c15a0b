"""The reference's CPU op interface (include/minfer/ops/kernels.hpp:13-32) and the
fused token-loop ops, on CUDA tensors, through libmfcuda's C ABI.

Arguments follow the reference's names and meaning (`out` first, then
inputs); tensors must be contiguous CUDA tensors (activations fp32, weights
fp32 / fp16 / bf16 — bf16 may also be passed as raw uint16 bit patterns).
Every call raises MinferError on a non-zero status.
"""
from __future__ import annotations

import ctypes as C
import functools
from struct import Struct

import torch

from ._lib import (MF_BF16, MF_F16, MF_F32, MF_ROPE_LINEAR, MF_ROPE_NTK, MF_ROPE_PLAIN, MF_ROPE_YARN, check, cuda_lib,
                   mf_attn_desc)

_lib = cuda_lib()


def _ptr(t: torch.Tensor | None) -> int | None:
    if t is None:
        return None
    if not t.is_cuda:
        raise ValueError("expected a CUDA tensor")
    if not t.is_contiguous():
        raise ValueError("expected a contiguous tensor")
    return t.data_ptr()


_CUDA_STREAM_LEGACY = 1  # cudaStreamLegacy: the C ABI reads a NULL stream as "manager stream"


def _stream() -> int:
    """torch's current stream as a cudaStream_t for the C ABI."""
    s = torch.cuda.current_stream().cuda_stream
    return s if s else _CUDA_STREAM_LEGACY


def dtype_code(w: torch.Tensor, dtype: str | None = None) -> int:
    if dtype is not None:
        return {"f32": MF_F32, "f16": MF_F16, "bf16": MF_BF16}[dtype]
    if w.dtype == torch.float32:
        return MF_F32
    if w.dtype == torch.float16:
        return MF_F16
    if w.dtype in (torch.bfloat16, torch.uint16, torch.int16):
        return MF_BF16
    raise ValueError(f"unsupported weight dtype {w.dtype}")


# ---------------------------------------------------------------- single ops

def matmul(out, x, weight, offset: int, d_out: int, d_in: int, dtype: str | None = None):
    """kernels.hpp `matmul`: out[i] = sum_j W[offset + i*d_in + j] * x[j]."""
    check(_lib.mf_matmul(_ptr(out), _ptr(x), _ptr(weight), dtype_code(weight, dtype), offset, d_out, d_in,
                         _stream()))


def rmsnorm(out, x, weight, dim: int, eps: float, n_rows: int = 1):
    check(_lib.mf_rmsnorm(_ptr(out), _ptr(x), _ptr(weight), dim, eps, n_rows, _stream()))


def softmax(out, x, size: int, n_rows: int = 1):
    check(_lib.mf_softmax(_ptr(out), _ptr(x), size, n_rows, _stream()))


def silu(out, x, n: int):
    check(_lib.mf_silu(_ptr(out), _ptr(x), n, _stream()))


def neox_rope(out, x, head_idx: int, d_head: int, d_rotary: int, freq_base: float, pos: int):
    check(_lib.mf_neox_rope(_ptr(out), _ptr(x), head_idx, d_head, d_rotary, freq_base, pos, _stream()))


def il_rope(out, x, head_idx: int, d_head: int, d_rotary: int, freq_base: float, pos: int):
    check(_lib.mf_il_rope(_ptr(out), _ptr(x), head_idx, d_head, d_rotary, freq_base, pos, _stream()))


def attn(att_scores, att_out, q_head, kh, vh, seq_len: int, d_head: int, kv_dim: int):
    check(_lib.mf_attn(_ptr(att_scores), _ptr(att_out), _ptr(q_head), _ptr(kh), _ptr(vh), seq_len, d_head, kv_dim,
                       _stream()))


def route(x_norm, active_experts, active_experts_weights, moe_scores, w_router, d_model: int, n_experts: int,
          n_active: int):
    check(_lib.mf_route(_ptr(x_norm), _ptr(active_experts), _ptr(active_experts_weights), _ptr(moe_scores),
                        _ptr(w_router), d_model, n_experts, n_active, _stream()))


def embed(out, weight, token_id: int, d_in: int, dtype: str | None = None):
    check(_lib.mf_embed(_ptr(out), _ptr(weight), dtype_code(weight, dtype), token_id, d_in, _stream()))


def argmax(logits, n: int, out):
    check(_lib.mf_argmax(_ptr(logits), n, _ptr(out), _stream()))


# ---------------------------------------------------------------- fused ops

def rope_table(n_pos: int, d_rot: int, base: float) -> torch.Tensor:
    """[n_pos, d_rot/2, 2] (cos, sin) in float (host tensor)."""
    out = torch.empty(n_pos, d_rot // 2, 2, dtype=torch.float32)
    check(_lib.mf_rope_table(C.c_void_p(out.data_ptr()), n_pos, d_rot, base))
    return out


def embed_step(x, emb, vocab: int, d_model: int, step_state, dtype: str | None = None):
    check(_lib.mf_embed_step(_ptr(x), _ptr(emb), dtype_code(emb, dtype), vocab, d_model, _ptr(step_state),
                             _stream()))


def rmsnorm_matmul(y, x, norm_w, eps: float, w, d_out: int, d_in: int, dtype: str | None = None):
    check(_lib.mf_rmsnorm_matmul(_ptr(y), _ptr(x), _ptr(norm_w), eps, _ptr(w), dtype_code(w, dtype), d_out, d_in,
                                 _stream()))


def matmul_residual(x, a, w, d_out: int, d_in: int, dtype: str | None = None):
    check(_lib.mf_matmul_residual(_ptr(x), _ptr(a), _ptr(w), dtype_code(w, dtype), d_out, d_in, _stream()))


def swiglu_matmul(h, x, norm_w, eps: float, w_gate_up, d_ff: int, d_in: int, dtype: str | None = None):
    check(_lib.mf_swiglu_matmul(_ptr(h), _ptr(x), _ptr(norm_w), eps, _ptr(w_gate_up), dtype_code(w_gate_up, dtype),
                                d_ff, d_in, _stream()))


def attn_workspace_bytes(n_heads: int, n_kv_heads: int, d_head: int, n_split: int) -> int:
    return int(_lib.mf_attn_workspace_bytes(n_heads, n_kv_heads, d_head, n_split))


def attn_default_split(n_kv_heads: int, max_seq: int) -> int:
    return int(_lib.mf_attn_default_split(n_kv_heads, max_seq))


def attn_decode(qkv, q_norm_w, k_norm_w, eps: float, rope_table, k_cache, v_cache, max_seq: int, step_state, out,
                n_heads: int, n_kv_heads: int, d_head: int, n_split: int, workspace):
    """The cache element type follows k_cache's dtype (float32 or bfloat16)."""
    d = mf_attn_desc(_ptr(qkv), _ptr(q_norm_w), _ptr(k_norm_w), eps, _ptr(rope_table), _ptr(k_cache), _ptr(v_cache),
                     max_seq, _ptr(step_state), _ptr(out), n_heads, n_kv_heads, d_head, n_split, _ptr(workspace),
                     dtype_code(k_cache))
    check(_lib.mf_attn_decode(C.byref(d), _stream()))


def router_topk(ids, weights, scores, x, norm_w, eps: float, w_router, d_model: int, n_experts: int, k: int):
    check(_lib.mf_router_topk(_ptr(ids), _ptr(weights), _ptr(scores), _ptr(x), _ptr(norm_w), eps, _ptr(w_router),
                              d_model, n_experts, k, _stream()))


def moe_swiglu(h, x, norm_w, eps: float, w_gate_up_exps, ids, k: int, d_ff: int, d_in: int,
               dtype: str | None = None):
    check(_lib.mf_moe_swiglu(_ptr(h), _ptr(x), _ptr(norm_w), eps, _ptr(w_gate_up_exps),
                             dtype_code(w_gate_up_exps, dtype), _ptr(ids), k, d_ff, d_in, _stream()))


def moe_down_residual(x, h, w_down_exps, ids, weights, k: int, d_model: int, d_ff: int, dtype: str | None = None):
    check(_lib.mf_moe_down_residual(_ptr(x), _ptr(h), _ptr(w_down_exps), dtype_code(w_down_exps, dtype), _ptr(ids),
                                    _ptr(weights), k, d_model, d_ff, _stream()))


def moe_ffn(x, h, norm_w, eps: float, w_router, w_gate_up_exps, w_down_exps, scores, ids, weights, d_model: int,
            d_ff: int, n_experts: int, k: int, dtype: str | None = None):
    """router_topk + moe_swiglu + moe_down_residual as one launch chain."""
    check(_lib.mf_moe_ffn(_ptr(x), _ptr(h), _ptr(norm_w), eps, _ptr(w_router), _ptr(w_gate_up_exps),
                          _ptr(w_down_exps), dtype_code(w_gate_up_exps, dtype), _ptr(scores), _ptr(ids), _ptr(weights),
                          d_model, d_ff, n_experts, k, _stream()))


def lm_head_workspace_bytes() -> int:
    return int(_lib.mf_lm_head_workspace_bytes())


def lm_head(logits, x, norm_w, eps: float, w, vocab: int, d_model: int, step_state=None, workspace=None,
            vocab_offset: int = 0, dtype: str | None = None):
    check(_lib.mf_lm_head(_ptr(logits), _ptr(x), _ptr(norm_w), eps, _ptr(w), dtype_code(w, dtype), vocab, d_model,
                          vocab_offset, _ptr(step_state), _ptr(workspace), _stream()))


# ---------------------------------------------------------------- a batch of sequences over a paged KV cache

_CODES = {torch.float32: MF_F32, torch.float16: MF_F16, torch.bfloat16: MF_BF16}
_SCALINGS = {"none": MF_ROPE_PLAIN, "linear": MF_ROPE_LINEAR, "ntk": MF_ROPE_NTK, "yarn": MF_ROPE_YARN}

# The descriptions (mf_paged_kv, mf_paged_rope_desc, mf_paged_attn_desc) as packed bytes, native layout: a decode step
# is short enough for the time of filling ctypes structures to count.
_KV = Struct("@PPqqqPPPiiiiiiii")
_ROPE = Struct("@PqPqiiiiiffPPPP0P")
_ATTN = Struct("@PqPqiifiiiPN")
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)  # absent on builds without CUDA
_current_device = getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device)


def _refuse(t: torch.Tensor, name: str, want: str):
    raise ValueError(f"{name}: expected {want}, got {tuple(t.shape)} {t.dtype} with strides {t.stride()} on {t.device}")


def _vector(t: torch.Tensor | None, name: str, dtype, device: int, n: int) -> int:
    """Address of n contiguous elements (0 for None)."""
    if t is None:
        return 0
    if t.dtype is not dtype or t.get_device() != device or t.shape != (n,) or not t.is_contiguous():
        _refuse(t, name, f"{n} contiguous {dtype} elements on cuda:{device}")
    return t.data_ptr()


def _rows(t: torch.Tensor, name: str, dtype, device: int, n: int, width: int) -> tuple[int, int]:
    """Address and row stride of n rows of `width` contiguous elements: [n, width], or [n, heads, d_head]."""
    shape = t.shape
    dims = len(shape)
    if (t.dtype is dtype and t.get_device() == device and 2 <= dims <= 3 and shape[0] == n
            and (shape[1] if dims == 2 else shape[1] * shape[2]) == width):
        if t.is_contiguous():
            return t.data_ptr(), width
        stride = t.stride()
        if stride[-1] == 1 and (dims == 2 or stride[1] == shape[2] or shape[1] == 1) and (n <= 1 or stride[0] >= width):
            return t.data_ptr(), stride[0] if n > 1 else width
    _refuse(t, name, f"{n} rows of {width} contiguous {dtype} elements on cuda:{device}")


def _width(t: torch.Tensor) -> int:
    shape = t.shape
    return shape[1] if len(shape) == 2 else shape[1] * shape[2] if len(shape) == 3 else -1


def _paged_kv(k_pages, v_pages, page_table, q_start, kv_lens) -> tuple[bytes, int, int, int, int]:
    """The cache's packed description, its device, KV heads, head width and dtype code."""
    dtype, device, shape, strides = k_pages.dtype, k_pages.get_device(), k_pages.shape, k_pages.stride()
    code = _CODES.get(dtype)
    if code is None or len(shape) != 4 or device < 0 or strides[3] != 1:
        _refuse(k_pages, "k_pages", "a CUDA tensor [n_pages, n_kv_heads, page_size, d_head] of float32, float16 or bfloat16, heads contiguous")
    if v_pages.dtype is not dtype or v_pages.get_device() != device or v_pages.shape != shape or v_pages.stride() != strides:
        _refuse(v_pages, "v_pages", "the dtype, device, shape and strides of k_pages")
    n_pages, heads, size, d = shape
    # the stride of an extent of one says nothing (0: the default); otherwise 0 is an expanded tensor
    page_stride = strides[0] if n_pages > 1 else 0
    head_stride = strides[1] if heads > 1 else 0
    if (n_pages > 1 and page_stride <= 0) or (heads > 1 and head_stride <= 0) or strides[2] <= 0:
        _refuse(k_pages, "k_pages", "pages, heads and rows that are not expanded")
    table_shape, table_strides = page_table.shape, page_table.stride()
    if (page_table.dtype is not torch.int32 or page_table.get_device() != device or len(table_shape) != 2
            or (table_shape[1] > 1 and table_strides[1] != 1) or (table_shape[0] > 1 and table_strides[0] < table_shape[1])):
        _refuse(page_table, "page_table", f"int32 rows on cuda:{device}, each contiguous, that do not overlap")
    n_seqs, max_pages = table_shape
    return _KV.pack(k_pages.data_ptr(), v_pages.data_ptr(), page_stride, head_stride, strides[2], page_table.data_ptr(),
                    _vector(q_start, "q_start", torch.int32, device, n_seqs + 1),
                    _vector(kv_lens, "kv_lens", torch.int32, device, n_seqs),
                    table_strides[0] if n_seqs > 1 else max_pages, max_pages, n_pages, size, n_seqs, heads, d, code), device, heads, d, code


def _on(device: int, fn, *args) -> None:
    """fn(*args, stream) on torch's current stream of CUDA device `device`."""
    if _current_device() == device:
        rc = fn(*args, _raw_stream(device) or _CUDA_STREAM_LEGACY)
    else:
        with torch.cuda.device(device):
            rc = fn(*args, _raw_stream(device) or _CUDA_STREAM_LEGACY)
    if rc < 0:
        check(rc)


def rope_freqs(d_rot: int, base: float, scaling: str = "none", factor: float = 1.0, orig_ctx: float = 0.0,
               beta_fast: float = 32.0, beta_slow: float = 1.0) -> tuple[torch.Tensor, float]:
    """Frequencies for paged_rope_append, in turns per position (host tensor, float64 [d_rot / 2]), and the magnitude
    (mscale). scaling: "none", "linear", "ntk" or "yarn" (which needs orig_ctx)."""
    if scaling not in _SCALINGS:
        raise ValueError(f"unknown scaling {scaling!r}")
    out = torch.empty(max(d_rot, 0) // 2, dtype=torch.float64)
    mscale = C.c_float()
    check(_lib.mf_rope_freqs(C.c_void_p(out.data_ptr()), d_rot, base, _SCALINGS[scaling], factor, orig_ctx, beta_fast,
                             beta_slow, C.byref(mscale)))
    return out, mscale.value


def paged_rope_append(q_out, k_pages, v_pages, page_table, qkv, q_start, kv_lens, freqs, *, interleaved: bool = False,
                      mscale: float = 1.0, q_norm_w=None, k_norm_w=None, eps: float = 1e-6, positions=None):
    """Q/K norm (where weights are given), rotary positions and the append to the paged cache, for the new tokens of a
    batch: rows [q_start[b], q_start[b+1]) of qkv are the last tokens of sequence b, kv_lens[b] long with them.

    k_pages / v_pages: [n_pages, n_kv_heads, page_size, d_head] (any strides with contiguous heads, e.g. a transposed
    view of [n_pages, page_size, n_kv_heads, d_head]); page_table: int32 [n_seqs, max_pages]; q_out: [n_tokens,
    n_heads, d_head] in the pages' dtype; qkv: [n_tokens, (n_heads + 2 n_kv_heads) * d_head]; freqs: float64
    [d_rot / 2] in turns per position (rope_freqs). Rows of no sequence, and the rest of the pages, stay as they are."""
    kv, device, heads, d, _ = _paged_kv(k_pages, v_pages, page_table, q_start, kv_lens)
    n, half = qkv.shape[0], freqs.shape[0]
    q_width = _width(q_out)
    x_code = _CODES.get(qkv.dtype)
    if x_code is None:
        raise ValueError(f"qkv: unsupported dtype {qkv.dtype}")
    q, q_stride = _rows(q_out, "q_out", k_pages.dtype, device, n, q_width)
    x, x_stride = _rows(qkv, "qkv", qkv.dtype, device, n, q_width + 2 * heads * d)
    if q_width % d:
        raise ValueError("q_out: expected whole heads")
    desc = _ROPE.pack(q, q_stride, x, x_stride, x_code, n, q_width // d, 2 * half, interleaved, mscale, eps,
                      _vector(freqs, "freqs", torch.float64, device, half), _vector(q_norm_w, "q_norm_w", torch.float32, device, d),
                      _vector(k_norm_w, "k_norm_w", torch.float32, device, d), _vector(positions, "positions", torch.int32, device, n))
    _on(device, _lib.mf_paged_rope_append, kv, desc)


@functools.lru_cache(maxsize=1024)
def _workspace_bytes(device: int, *sizes: int) -> int:
    with torch.cuda.device(device):
        return int(_lib.mf_paged_attention_workspace_bytes(*sizes))


def paged_attention_workspace_bytes(n_tokens: int, n_heads: int, n_kv_heads: int, d_head: int, dtype: torch.dtype) -> int:
    return int(_lib.mf_paged_attention_workspace_bytes(n_tokens, n_heads, n_kv_heads, d_head, _CODES[dtype]))


def paged_attention(out, q, k_pages, v_pages, page_table, q_start, kv_lens, *, scale: float = 0.0, window: int = 0,
                    max_new: int = 0, max_len: int = 0, workspace=None):
    """out = attention of the new tokens over the cached positions up to their own (the last `window` of them, 0: all);
    arguments as in paged_rope_append, out and q [n_tokens, n_heads, d_head]. scale 0 means 1 / sqrt(d_head). max_new
    and max_len are hints: the most new tokens and the longest length of a sequence. workspace: a uint8 tensor of
    paged_attention_workspace_bytes, 256-byte aligned, not shared by overlapping calls; None takes one from torch."""
    kv, device, heads, d, code = _paged_kv(k_pages, v_pages, page_table, q_start, kv_lens)
    n = q.shape[0]
    width = _width(q)
    qp, q_stride = _rows(q, "q", k_pages.dtype, device, n, width)
    op, o_stride = _rows(out, "out", k_pages.dtype, device, n, width)
    if width % d:
        raise ValueError("q: expected whole heads")
    if workspace is None:
        workspace = torch.empty(_workspace_bytes(device, n, width // d, heads, d, code), dtype=torch.uint8, device=k_pages.device)
    size = workspace.numel()
    desc = _ATTN.pack(op, o_stride, qp, q_stride, n, width // d, scale, window, max_new, max_len,
                      _vector(workspace, "workspace", torch.uint8, device, size), size)
    _on(device, _lib.mf_paged_attention, kv, desc)


def paged_status(clear: bool = True) -> int:
    """Status bits of paged_attention's kernels on the current device since the last clear (2: a wait gave up)."""
    status = C.c_int()
    check(_lib.mf_paged_status(C.byref(status), int(clear)))
    return status.value


def sample_batch(ids, logits, draws, temp, top_k, top_p, min_p, probs=None):
    """One id per row of logits [n_rows, vocab] (float32, float16 or bfloat16; rows may be strided): the reference
    Sampler's filters with row's own temp, top_k, top_p and min_p, and draws[row] in [0, 1) as its random number. ids and
    top_k are int32, the others float32 vectors of n_rows. probs (optional, float32) receives the ids' probabilities."""
    device, code = logits.get_device(), _CODES.get(logits.dtype)
    if code is None or logits.dim() != 2 or device < 0:
        raise ValueError("logits: expected a 2-d CUDA tensor of float32, float16 or bfloat16")
    n, vocab = logits.shape
    stride, inner = logits.stride()
    if vocab > 1 and inner != 1:
        raise ValueError("logits: expected contiguous rows")
    f, i = torch.float32, torch.int32
    _on(device, _lib.mf_sample_batch, _vector(ids, "ids", i, device, n), _vector(probs, "probs", f, device, n),
        logits.data_ptr(), code, stride if n > 1 else vocab, n, vocab, _vector(draws, "draws", f, device, n),
        _vector(temp, "temp", f, device, n), _vector(top_k, "top_k", i, device, n),
        _vector(top_p, "top_p", f, device, n), _vector(min_p, "min_p", f, device, n))
