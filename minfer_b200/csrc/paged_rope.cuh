// Q/K norm, rotary positions and the append to the paged cache, for the new
// tokens of a batch: per token t at position pos and head h of its row
// [Hq | Hkv | Hkv] x D of the fused projection
//   x' = x / sqrt(mean(x^2) + eps) * w                    (q and k heads, optional)
//   (y_a, y_b) = m (x'_a cos - x'_b sin, x'_b cos + x'_a sin), angle = 2 pi pos f_j
// over the pairs (a, b) = (j, j + d_rot/2) or (2j, 2j + 1); the elements from
// d_rot on pass through. q goes to q_out, k and v to row pos % page_size of
// the page of pos, in the cache's type.
//
// f_j is in turns per position and 64 bits: a float angle at position 10^6 is
// off by up to 0.03 rad. pos * f_j is reduced to (-1/2, 1/2] turns in double
// and only then rounded, so the angle's error is that of one float rounding
// at every position. The two doubles per pair are computed once per token and
// kept in registers over the warp's heads.
//
// Bound by memory: every value is read and written once. One warp takes a
// token and `hpw` heads, D/32 neighbouring elements per lane; the partner of
// the half layout sits in lane +- d_rot/2 / (D/32) (hence d_rot % 8 == 0).
#pragma once

#include "paged.cuh"

namespace mf {

struct PagedRope {
    void* q_out;       // [n_tokens][q_stride]
    long long q_stride;
    const void* qkv;   // [n_tokens][x_stride]
    long long x_stride;
    const double* freqs;  // [d_rot / 2]
    const float* q_norm_w;
    const float* k_norm_w;
    const int* positions;  // rotary positions per row, or null: the cache positions
    float eps, mscale;
    int n_heads, d_rot, interleaved;
    int hpw;  // heads of one warp
};

constexpr int ROPE_WARPS = 8;
constexpr int ROPE_HB = 4;  // heads in flight per warp

template <typename X, typename T, int D>
__global__ void __launch_bounds__(ROPE_WARPS * 32) paged_rope_kernel(const PagedKv p, const PagedRope r) {
    constexpr int V = D / 32;
    pdl_launch_dependents();
    pdl_wait();
    const int lane = threadIdx.x & 31;
    const int Hq = r.n_heads, Hk = p.n_kv_heads, H = Hq + 2 * Hk;
    const int chunks = (H + r.hpw - 1) / r.hpw;
    const long long unit = (long long)blockIdx.x * ROPE_WARPS + (threadIdx.x >> 5);
    const int t = (int)(unit / chunks);
    if (t >= p.n_tokens) return;
    const int b = paged_owner(p, t);
    if (b < 0) return;  // rows behind the last sequence stay as they are
    const PagedSeq s = paged_seq(p, b);
    const int pos = s.first + (t - s.row);
    const int h0 = (int)(unit % chunks) * r.hpw, h1 = min(h0 + r.hpw, H);

    // cos and signed sin of this lane's elements
    float c[V], sn[V];
    const int half = r.d_rot >> 1;
#pragma unroll
    for (int i = 0; i < V; ++i) {
        const int e = lane * V + i;
        c[i] = 1.f;
        sn[i] = 0.f;
        if (e < r.d_rot && h0 < Hq + Hk) {
            const int j = r.interleaved ? e >> 1 : (e < half ? e : e - half);
            const bool first = r.interleaved ? (e & 1) == 0 : e < half;
            const double turns = (double)(r.positions ? __ldg(r.positions + t) : pos) * __ldg(r.freqs + j);
            float sv, cv;
            sincospif(2.0f * (float)(turns - rint(turns)), &sv, &cv);
            c[i] = cv * r.mscale;
            sn[i] = (first ? -sv : sv) * r.mscale;
        }
    }
    const int shift = half / V;
    const int from = lane * V < half ? lane + shift : lane - shift;  // partner lane of the half layout
    const int page = paged_page(p, b, pos);
    const long long kv_row = page >= 0 ? page * p.page_stride + (pos - pos / p.page_size * p.page_size) * p.row_stride : 0;
    const X* x0 = reinterpret_cast<const X*>(r.qkv) + t * r.x_stride + lane * V;

    for (int hb = h0; hb < h1; hb += ROPE_HB) {
        PackV<X, V> in[ROPE_HB];
#pragma unroll
        for (int u = 0; u < ROPE_HB; ++u)
            if (hb + u < h1) in[u] = *reinterpret_cast<const PackV<X, V>*>(x0 + (long long)(hb + u) * D);
#pragma unroll
        for (int u = 0; u < ROPE_HB; ++u) {
            const int h = hb + u;
            if (h >= h1) break;
            float x[V], y[V];
#pragma unroll
            for (int i = 0; i < V; ++i) x[i] = to_f<X>(in[u].e[i]);
            if (h < Hq + Hk) {
                const float* w = h < Hq ? r.q_norm_w : r.k_norm_w;
                if (w) {
                    float ss = 0.f;
#pragma unroll
                    for (int i = 0; i < V; ++i) ss = fmaf(x[i], x[i], ss);
                    const float inv = 1.0f / sqrtf(warp_sum(ss) / (float)D + r.eps);
#pragma unroll
                    for (int i = 0; i < V; ++i) x[i] = x[i] * inv * __ldg(w + lane * V + i);
                }
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    const float other = r.interleaved ? x[i ^ 1] : __shfl_sync(0xffffffffu, x[i], from & 31);
                    // past d_rot: passed through, whatever the other lane holds
                    y[i] = lane * V + i < r.d_rot ? fmaf(x[i], c[i], other * sn[i]) : x[i];
                }
            } else {
#pragma unroll
                for (int i = 0; i < V; ++i) y[i] = x[i];
            }
            PackV<T, V> out;
#pragma unroll
            for (int i = 0; i < V; ++i) out.e[i] = from_f<T>(y[i]);
            if (h < Hq) {
                *reinterpret_cast<PackV<T, V>*>(reinterpret_cast<T*>(r.q_out) + t * r.q_stride + (long long)h * D + lane * V) = out;
            } else if (page >= 0) {
                const bool is_k = h < Hq + Hk;
                T* base = reinterpret_cast<T*>(is_k ? p.k : p.v) + kv_row + (long long)(h - Hq - (is_k ? 0 : Hk)) * p.head_stride;
                *reinterpret_cast<PackV<T, V>*>(base + lane * V) = out;
            }
        }
    }
}

}  // namespace mf
