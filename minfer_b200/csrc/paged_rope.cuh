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
// off by up to 0.03 rad. pos * f_j is reduced to about (-1/2, 1/2] turns in
// double, with the product's own rounding error (up to 2^-25 turns at 2^31)
// added back from a second product, and only then rounded: for a given f_j the
// angle's error is that of one float rounding at every position. (f_j itself
// is rounded to 64 bits, which at position p is p f_j 2^-53 turns.) The angles
// are computed once per token and kept in registers over the warp's heads.
//
// Bound by memory: every value is read and written once. Eight lanes take a
// head, a warp four heads at a time and `hpw` heads of one token in all. A lane
// holds whole pairs: of the half layout's 4-element blocks, block s together
// with block s + d_rot/8 (s = lane, lane + 8), and the blocks behind d_rot two
// by two; so rotating needs no exchange, and the norm three shuffles for four
// heads. (With a head across the warp the sums and exchanges took 90
// instructions a head, more time than its 768 bytes: 42 us for the chunk below.)
// Measured: 156 MB (fp32 rows of 80 heads to bf16) in 29 us on inputs that are
// partly in L2, 31 on new ones (0.76 of the copy rate); one token 3.2 us.
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
constexpr int ROPE_HEADS = 4;  // heads of a warp at a time

template <typename X, typename T, int D>
__global__ void __launch_bounds__(ROPE_WARPS * 32, 3) paged_rope_kernel(const PagedKv p, const PagedRope r) {
    constexpr int NS = D / 64;  // pairs of blocks per lane
    constexpr int NA = 4 * NS;  // angles per lane
    pdl_launch_dependents();
    pdl_wait();
    const int lane = threadIdx.x & 31, sub = lane >> 3, l = lane & 7;
    const int Hq = r.n_heads, Hk = p.n_kv_heads, H = Hq + 2 * Hk;
    const int chunks = (H + r.hpw - 1) / r.hpw;
    const long long unit = (long long)blockIdx.x * ROPE_WARPS + (threadIdx.x >> 5);
    const int t = (int)(unit / chunks);
    if (t >= p.n_tokens) return;
    const int h0 = (int)(unit % chunks) * r.hpw, h1 = min(h0 + r.hpw, H);

    // the blocks of this lane (4 elements each)
    const int hb = r.d_rot >> 3;  // blocks of half of the rotated part
    int blk[NS][2];
#pragma unroll
    for (int u = 0; u < NS; ++u) {
        const int i = l + 8 * u;
        blk[u][0] = i < hb ? i : 2 * hb + 2 * (i - hb);
        blk[u][1] = i < hb ? i + hb : blk[u][0] + 1;
    }
    // Four heads at a time; the next four are on their way while these are turned, the first while the token's
    // sequence, page and angles are found.
    const X* x0 = reinterpret_cast<const X*>(r.qkv) + t * r.x_stride;
    PackV<X, 4> next[NS][2];
    auto fetch = [&](int h) {
        if (h < h1) {
#pragma unroll
            for (int u = 0; u < NS; ++u)
#pragma unroll
                for (int w = 0; w < 2; ++w) next[u][w] = *reinterpret_cast<const PackV<X, 4>*>(x0 + (long long)h * D + 4 * blk[u][w]);
        }
    };
    fetch(h0 + sub);
    const int b = paged_owner(p, t);
    if (b < 0) return;  // rows behind the last sequence stay as they are
    const PagedSeq s = paged_seq(p, b);
    const int pos = s.first + (t - s.row);

    // cos and sin of this lane's pairs (1 and 0 behind d_rot); the four heads' lanes share the work
    float c[NA], sn[NA];
    if (h0 < Hq + Hk) {
        float cv[NS], sv[NS];
#pragma unroll
        for (int v = 0; v < NS; ++v) {
            const int q = sub * NS + v, u = q >> 2, e = q & 3;  // angle q: pair e of the lane's blocks u
            const int i = l + 8 * u;
            cv[v] = 1.f;
            sv[v] = 0.f;
            if (i < hb) {
                // half layout: (4 i + e, and half on); pairs: two of each block
                const int j = !r.interleaved ? 4 * i + e : 2 * (e < 2 ? i : i + hb) + (e & 1);
                const double at = r.positions ? __ldg(r.positions + t) : pos, f = __ldg(r.freqs + j);
                const double turns = at * f, rest = fma(at, f, -turns);
                sincospif(2.0f * (float)((turns - rint(turns)) + rest), &sv[v], &cv[v]);
                cv[v] *= r.mscale;
                sv[v] *= r.mscale;
            }
        }
#pragma unroll
        for (int q = 0; q < NA; ++q) {
            c[q] = __shfl_sync(0xffffffffu, cv[q % NS], q / NS * 8 + l);
            sn[q] = __shfl_sync(0xffffffffu, sv[q % NS], q / NS * 8 + l);
        }
    }
    const int page = paged_page(p, b, pos);
    const long long kv_row = page >= 0 ? page * p.page_stride + (long long)(pos % p.page_size) * p.row_stride : 0;

    for (int hg = h0; hg < h1; hg += ROPE_HEADS) {
        const int h = hg + sub;
        PackV<X, 4> in[NS][2];
#pragma unroll
        for (int u = 0; u < NS; ++u)
#pragma unroll
            for (int w = 0; w < 2; ++w) in[u][w] = next[u][w];
        fetch(h + ROPE_HEADS);
        const bool live = h < h1, is_q = h < Hq, is_v = h >= Hq + Hk;
        float x[NS][2][4];
#pragma unroll
        for (int u = 0; u < NS; ++u)
#pragma unroll
            for (int w = 0; w < 2; ++w)
#pragma unroll
                for (int e = 0; e < 4; ++e) x[u][w][e] = live ? to_f<X>(in[u][w].e[e]) : 0.f;
        const float* nw = is_q ? r.q_norm_w : r.k_norm_w;
        if ((r.q_norm_w || r.k_norm_w) && hg < Hq + Hk) {  // the whole warp
            float ss = 0.f;
#pragma unroll
            for (int u = 0; u < NS; ++u)
#pragma unroll
                for (int w = 0; w < 2; ++w)
#pragma unroll
                    for (int e = 0; e < 4; ++e) ss = fmaf(x[u][w][e], x[u][w][e], ss);
#pragma unroll
            for (int o = 4; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
            if (nw && !is_v) {
                const float inv = rsqrtf(ss / (float)D + r.eps);
#pragma unroll
                for (int u = 0; u < NS; ++u)
#pragma unroll
                    for (int w = 0; w < 2; ++w)
#pragma unroll
                        for (int e = 0; e < 4; ++e) x[u][w][e] = x[u][w][e] * inv * __ldg(nw + 4 * blk[u][w] + e);
            }
        }
        if (!is_v) {
#pragma unroll
            for (int u = 0; u < NS; ++u) {
                if (l + 8 * u >= hb) continue;  // behind d_rot: as it is
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    auto turn = [&](float& a, float& z) {
                        const float xa = a, xz = z;
                        a = fmaf(xa, c[4 * u + e], -xz * sn[4 * u + e]);
                        z = fmaf(xz, c[4 * u + e], xa * sn[4 * u + e]);
                    };
                    if (r.interleaved) turn(x[u][e >> 1][2 * (e & 1)], x[u][e >> 1][2 * (e & 1) + 1]);
                    else turn(x[u][0][e], x[u][1][e]);
                }
            }
        }
        if (!live || (!is_q && page < 0)) continue;
        T* dst = is_q ? reinterpret_cast<T*>(r.q_out) + t * r.q_stride + (long long)h * D
                      : reinterpret_cast<T*>(is_v ? p.v : p.k) + kv_row + (long long)(h - Hq - (is_v ? Hk : 0)) * p.head_stride;
#pragma unroll
        for (int u = 0; u < NS; ++u)
#pragma unroll
            for (int w = 0; w < 2; ++w) {
                PackV<T, 4> y;
#pragma unroll
                for (int e = 0; e < 4; ++e) y.e[e] = from_f<T>(x[u][w][e]);
                *reinterpret_cast<PackV<T, 4>*>(dst + 4 * blk[u][w]) = y;
            }
    }
}

}  // namespace mf
