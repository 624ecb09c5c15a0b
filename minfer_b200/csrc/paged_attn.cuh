// Attention of new tokens over a paged cache on the CUDA cores, in fp32:
// o = sum_s softmax_s(scale q.k_s) v_s over the positions s in
// (pos - window, pos] that lie on a page, one pass with the running maximum
// and sum of each row.
//
// A CTA takes a range of the batch's key tiles (paged_work.cuh). Per tile of
// 64 keys: S = Q K^T in registers (4 rows x 4 keys a thread), softmax by the
// threads of a row, O += P V (4 rows x D/16 columns a thread). K and V tiles
// come by cp.async, each while the other is used; rows past the item's last
// key and rows without a page are filled with zeros and never read.
//   RT = 64 rows: 256 threads cover the 64 x 64 scores.
//   RT = 16 rows (a few tokens): four groups of 64 threads share D for S and
//   the keys for P V, so that a thread's tile stays 4 x 4 and shared memory
//   is not what bounds it; their sums are added at the end of an item.
// Tiles are stored without padding, 16-byte pieces c of row r at c ^ (r & 7)
// (no bank conflicts in either direction), so that two CTAs fit an SM and one
// computes while the other's softmax waits at a barrier (298 -> 217 us for
// chunks of 65 and single tokens over 4096 keys, 16/8 heads; 206 with items of
// nearly equal rows). Bound by instruction issue: about a quarter of the FMA
// rate in useful products, the rest are loads, exponentials and unused rows.
#pragma once

#include "paged_work.cuh"

namespace mf {

constexpr int PA_SIMT_KT = 64;
constexpr int PA_SIMT_THREADS = 256;

// Q, K, V, the partial scores, and alpha per row
template <int RT, int D> constexpr int paged_simt_smem() {
    return (RT * D + 2 * PA_SIMT_KT * D + 64 * PA_SIMT_KT + RT) * 4;
}

// Element c of row r of a tile whose rows have W elements.
template <int W> MF_DEVICE int pa_at(int r, int c) { return r * W + (((c >> 2) ^ (r & 7)) << 2) + (c & 3); }

// Rows [k0, k0 + 64) of one head of sequence b into shared memory; rows outside
// [lo, hi) or without a page become zeros. Returns which rows have a page (the same in every thread).
template <int D>
MF_DEVICE unsigned long long paged_simt_load(float* dst, const float* base, const PagedKv& p, int b, int h, int k0, int lo, int hi) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    constexpr int C = D / 4, RPI = 32 / C;  // pieces of a row, rows per access of a warp
    // each lane looks up two rows of the tile, and the warp shares them
    long long off[2];
    unsigned have[2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
        const int key = k0 + 32 * u + lane;
        const int page = key >= lo && key < hi ? paged_page(p, b, key) : -1;
        off[u] = page < 0 ? -1 : page * p.page_stride + (long long)h * p.head_stride + (long long)(key % p.page_size) * p.row_stride;
        have[u] = __ballot_sync(0xffffffffu, page >= 0);
    }
#pragma unroll
    for (int i = 0; i < PA_SIMT_KT / 8 / RPI; ++i) {
        const int row = (i * 8 + warp) * RPI + lane / C, c = lane % C * 4;
        const long long o0 = __shfl_sync(0xffffffffu, off[0], row & 31), o1 = __shfl_sync(0xffffffffu, off[1], row & 31);
        const long long o = row < 32 ? o0 : o1;
        const uint32_t s = (uint32_t)__cvta_generic_to_shared(dst + pa_at<D>(row, c));
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(s), "l"(base + (o < 0 ? 0 : o + c)), "r"(o < 0 ? 0 : 16) : "memory");
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
    return (unsigned long long)have[1] << 32 | have[0];
}

template <int D, int RT>
__global__ void __launch_bounds__(PA_SIMT_THREADS, 2) paged_simt_kernel(const PagedKv p, const PagedAttn a) {
    constexpr int KT = PA_SIMT_KT, NG = 64 / RT, GT = PA_SIMT_THREADS / NG;
    constexpr int NC = D / 64;            // float4 columns of O per thread
    constexpr int TPR = PA_SIMT_THREADS / RT, KPT = KT / TPR;  // softmax: threads per row, keys per thread
    extern __shared__ __align__(16) float paged_smem[];
    float* Qs = paged_smem;
    float* Ks = Qs + RT * D;
    float* Vs = Ks + KT * D;
    float* Ss = Vs + KT * D;             // [NG][RT][KT]
    float* alpha_s = Ss + NG * RT * KT;  // [RT]
    paged_begin(a);

    PagedItem it;
    long long share;
    const long long total = paged_find<RT, KT>(p, a, blockIdx.x, gridDim.x, reinterpret_cast<long long*>(Ks), share, it);
    const long long w0 = blockIdx.x * share, w1 = min(w0 + share, total);
    if (w0 >= w1) {
        paged_end(a);
        return;
    }
    const int tid = threadIdx.x, grp = tid / GT, tg = tid % GT;
    const int ty = tg / 16, tx = tg % 16;  // rows 4 ty .., keys tx + 16 j, columns 4 tx + 64 j
    const int srow = tid / TPR, sk = tid % TPR;
    const float* kb = reinterpret_cast<const float*>(p.k);
    const float* vb = reinterpret_cast<const float*>(p.v);

    for (long long w = w0; w < w1;) {
        const int j0 = (int)max(w - it.start, 0ll), j1 = (int)min((long long)it.tiles, w1 - it.start);
        if (j1 <= 0) break;  // only the item's first unit is in this range
        const int rows = min(it.step, it.s.n * a.G - it.r0);
        const int kt0 = it.k.lo / KT;
        __syncthreads();
        unsigned long long pages = paged_simt_load<D>(Ks, kb, p, it.b, it.h, (kt0 + j0) * KT, it.k.lo, it.k.hi);
        for (int i = tid; i < RT * D / 4; i += PA_SIMT_THREADS) {
            const int r = i / (D / 4), c = i % (D / 4) * 4, row = it.r0 + r;
            float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
            if (r < rows) v = *reinterpret_cast<const float4*>(reinterpret_cast<const float*>(a.q) + (long long)(it.s.row + row / a.G) * a.q_stride +
                                                                 (long long)(it.h * a.G + row % a.G) * D + c);
            *reinterpret_cast<float4*>(Qs + pa_at<D>(r, c)) = make_float4(v.x * a.scale2, v.y * a.scale2, v.z * a.scale2, v.w * a.scale2);
        }
        float o[4][4 * NC];
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int e = 0; e < 4 * NC; ++e) o[i][e] = 0.f;
        float m = -INFINITY, l = 0.f;  // of row srow (the same in its threads)
        const bool busy = 8 * (ty >> 1) < rows;  // a warp has rows of the item: the others skip the products
        const int my_pos = it.s.first + (it.r0 + srow) / a.G;
        const int my_lo = a.window > 0 ? my_pos - a.window + 1 : 0;

        for (int j = j0; j < j1; ++j) {
            const int k0 = (kt0 + j) * KT;
            const unsigned long long have = pages;
            paged_simt_load<D>(Vs, vb, p, it.b, it.h, k0, it.k.lo, it.k.hi);
            asm volatile("cp.async.wait_group 1;" ::: "memory");
            __syncthreads();  // K (and Q) are there
            float acc[4][4] = {};
#pragma unroll 4
            for (int d = grp * (D / NG); d < (busy ? (grp + 1) * (D / NG) : 0); d += 4) {
                float4 qv[4], kv[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) qv[i] = *reinterpret_cast<const float4*>(Qs + pa_at<D>(4 * ty + i, d));
#pragma unroll
                for (int i = 0; i < 4; ++i) kv[i] = *reinterpret_cast<const float4*>(Ks + pa_at<D>(tx + 16 * i, d));
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        acc[i][k] = fmaf(qv[i].x, kv[k].x, acc[i][k]);
                        acc[i][k] = fmaf(qv[i].y, kv[k].y, acc[i][k]);
                        acc[i][k] = fmaf(qv[i].z, kv[k].z, acc[i][k]);
                        acc[i][k] = fmaf(qv[i].w, kv[k].w, acc[i][k]);
                    }
            }
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int k = 0; k < 4; ++k) Ss[pa_at<KT>(grp * RT + 4 * ty + i, tx + 16 * k)] = acc[i][k];
            __syncthreads();
            // softmax of row srow over its KPT keys sk, sk + TPR, ...
            float sv[KPT], mx = m;
#pragma unroll
            for (int k = 0; k < KPT; ++k) {
                const int kk = sk + TPR * k, key = k0 + kk;
                float x = 0.f;
#pragma unroll
                for (int g = 0; g < NG; ++g) x += Ss[pa_at<KT>(g * RT + srow, kk)];
                sv[k] = key <= my_pos && key >= my_lo && (have >> kk & 1) ? x : -INFINITY;
                mx = fmaxf(mx, sv[k]);
            }
#pragma unroll
            for (int off = TPR / 2; off > 0; off >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, off));
            const float base = mx == -INFINITY ? 0.f : mx;  // nothing seen yet: every p is 0
            const float al = exp2f(m - base);
            float sum = 0.f;
#pragma unroll
            for (int k = 0; k < KPT; ++k) {
                const float e = exp2f(sv[k] - base);
                sum += e;
                Ss[pa_at<KT>(srow, sk + TPR * k)] = e;  // group 0's plane: only this thread reads or writes the entry
            }
#pragma unroll
            for (int off = TPR / 2; off > 0; off >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
            l = fmaf(l, al, sum);
            m = mx;
            if (sk == 0) alpha_s[srow] = al;
            asm volatile("cp.async.wait_group 0;" ::: "memory");
            __syncthreads();  // P, alpha and V are there; K is free
            if (j + 1 < j1) pages = paged_simt_load<D>(Ks, kb, p, it.b, it.h, k0 + KT, it.k.lo, it.k.hi);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float al4 = alpha_s[4 * ty + i];
#pragma unroll
                for (int e = 0; e < 4 * NC; ++e) o[i][e] *= al4;
            }
#pragma unroll 2
            for (int k = grp * (KT / NG); k < (busy ? (grp + 1) * (KT / NG) : 0); k += 4) {
                float4 pv[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) pv[i] = *reinterpret_cast<const float4*>(Ss + pa_at<KT>(4 * ty + i, k));
#pragma unroll
                for (int kk = 0; kk < 4; ++kk)
#pragma unroll
                    for (int n = 0; n < NC; ++n) {
                        const float4 v = *reinterpret_cast<const float4*>(Vs + pa_at<D>(k + kk, 4 * tx + 64 * n));
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const float pr = reinterpret_cast<const float*>(&pv[i])[kk];
                            o[i][4 * n] = fmaf(pr, v.x, o[i][4 * n]);
                            o[i][4 * n + 1] = fmaf(pr, v.y, o[i][4 * n + 1]);
                            o[i][4 * n + 2] = fmaf(pr, v.z, o[i][4 * n + 2]);
                            o[i][4 * n + 3] = fmaf(pr, v.w, o[i][4 * n + 3]);
                        }
                    }
            }
            __syncthreads();  // V and P are free
        }
        // the groups' sums of O, in order, in the K tile's place; m and l per row in the scores'
        if constexpr (NG > 1) {
            float* Os = Ks;  // [NG][RT][D] <= KT * D
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int n = 0; n < NC; ++n)
                    *reinterpret_cast<float4*>(Os + (grp * RT + 4 * ty + i) * D + 4 * tx + 64 * n) =
                        make_float4(o[i][4 * n], o[i][4 * n + 1], o[i][4 * n + 2], o[i][4 * n + 3]);
        }
        float* l_s = Ss;
        float* m_s = Ss + RT;
        if (sk == 0) {
            l_s[srow] = l;
            m_s[srow] = m;
        }
        __syncthreads();
        const bool whole = j0 == 0 && j1 == it.tiles;
        const long long slot = 2ll * blockIdx.x + (j0 > 0 ? 0 : 1);
        float* part = a.part + slot * RT * D;
        float* ml = a.part + 2ll * gridDim.x * RT * D + slot * RT * 2;
        auto store = [&](int r, int c, float4 v) {
            if (r >= rows) return;
            if (whole) {
                const float inv = l_s[r] == 0.f ? 0.f : 1.0f / l_s[r];
                const int row = it.r0 + r;
                *reinterpret_cast<float4*>(reinterpret_cast<float*>(a.out) + (long long)(it.s.row + row / a.G) * a.out_stride +
                                           (long long)(it.h * a.G + row % a.G) * D + c) = make_float4(v.x * inv, v.y * inv, v.z * inv, v.w * inv);
            } else {
                *reinterpret_cast<float4*>(part + r * D + c) = v;
                if (c == 0) {
                    ml[2 * r] = m_s[r];
                    ml[2 * r + 1] = l_s[r];
                }
            }
        };
        if constexpr (NG > 1) {
            for (int i = tid; i < RT * D / 4; i += PA_SIMT_THREADS) {
                const int r = i / (D / 4), c = i % (D / 4) * 4;
                float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
                for (int g = 0; g < NG; ++g) {
                    const float4 x = *reinterpret_cast<const float4*>(Ks + (g * RT + r) * D + c);
                    v.x += x.x;
                    v.y += x.y;
                    v.z += x.z;
                    v.w += x.w;
                }
                store(r, c, v);
            }
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int n = 0; n < NC; ++n) store(4 * ty + i, 4 * tx + 64 * n, make_float4(o[i][4 * n], o[i][4 * n + 1], o[i][4 * n + 2], o[i][4 * n + 3]));
        }
        w = it.start + j1;
        if (w < w1) paged_next<RT, KT>(p, a, it);
    }
    paged_end(a);
}

}  // namespace mf
