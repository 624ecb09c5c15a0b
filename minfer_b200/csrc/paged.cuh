// One step of a batch of sequences over a paged KV cache: what the paged
// kernels share (paged_rope.cuh, paged_attn.cuh, paged_fa.cuh).
//
// The batch is ragged: sequence b owns the rows [q_start[b], q_start[b + 1])
// of the call's tokens, the last n_b of its kv_lens[b] positions. Lengths and
// tables are read on the device only, so one captured launch serves every
// step. Nothing in them is trusted: starts are clamped to the call's rows,
// lengths to what the table can hold, and a page id outside [0, n_pages)
// holds no keys (its positions are neither read nor written).
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "mf_common.cuh"

#define MF_HOST_DEVICE __host__ __device__ __forceinline__  // counting that tests run on the CPU

namespace mf {

// Copy of mf_paged_kv with the strides resolved.
struct PagedKv {
    void* k;
    void* v;
    long long page_stride, head_stride, row_stride;  // elements
    const int* table;                                // [n_seqs][table_stride]
    const int* q_start;                              // [n_seqs + 1]
    const int* kv_lens;                              // [n_seqs]
    int table_stride, max_pages, n_pages, page_size, n_seqs, n_kv_heads;
    int n_tokens;  // rows of the call
};

// One sequence of the batch: its first row, its new tokens and the position of the first of them.
struct PagedSeq {
    int row, n, first;
};
MF_DEVICE PagedSeq paged_seq(const PagedKv& p, int b) {
    const int s0 = min(max(__ldg(p.q_start + b), 0), p.n_tokens);
    const int s1 = min(max(__ldg(p.q_start + b + 1), 0), p.n_tokens);
    const long long cap = (long long)p.max_pages * p.page_size;
    const int len = (int)min((long long)max(__ldg(p.kv_lens + b), 0), min(cap, (long long)0x7fffff00));
    PagedSeq s;
    s.row = s0;
    s.n = max(s1 - s0, 0);
    s.first = len - s.n;  // may be negative: those tokens have no position and see nothing
    return s;
}

// Page of position `pos` of sequence b, or -1.
MF_DEVICE int paged_page(const PagedKv& p, int b, int pos) {
    const int i = pos / p.page_size;
    if (pos < 0 || i >= p.max_pages) return -1;
    const int pg = __ldg(p.table + (long long)b * p.table_stride + i);
    return (unsigned)pg < (unsigned)p.n_pages ? pg : -1;
}

// The sequence that owns row t: the last b with q_start[b] <= t, or -1 for a
// row before the first or behind the last. One warp together: 32 probes a round.
MF_DEVICE int paged_owner(const PagedKv& p, int t) {
    const int lane = threadIdx.x & 31;
    int b = -1, left = p.n_seqs + 1;  // entries [b + 1, b + 1 + left) are undecided
    while (left > 0) {
        const int step = (left + 31) >> 5;
        const int at = b + (lane + 1) * step;
        const bool in = (lane + 1) * step <= left && __ldg(p.q_start + at) <= t;
        const int c = __popc(__ballot_sync(0xffffffffu, in));
        b += c * step;
        left = min(step - 1, left - c * step);
    }
    return b < p.n_seqs ? b : -1;
}

template <typename T> MF_DEVICE float to_f(T v);
template <> MF_DEVICE float to_f<float>(float v) { return v; }
template <> MF_DEVICE float to_f<__half>(__half v) { return __half2float(v); }
template <> MF_DEVICE float to_f<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T> MF_DEVICE T from_f(float v);
template <> MF_DEVICE float from_f<float>(float v) { return v; }
template <> MF_DEVICE __half from_f<__half>(float v) { return __float2half_rn(v); }
template <> MF_DEVICE __nv_bfloat16 from_f<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// V values of type T, as one access
template <typename T, int V>
struct alignas(sizeof(T) * V) PackV {
    T e[V];
};

}  // namespace mf
