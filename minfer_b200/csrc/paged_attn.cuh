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
#pragma once

#include "paged_work.cuh"

namespace mf {

constexpr int PA_SIMT_KT = 64;
constexpr int PA_SIMT_THREADS = 256;

template <int RT, int D> constexpr int paged_simt_smem() {
    // Q, K, V (padded rows), S partials, alpha and l per row
    return (RT * (D + 4) + 2 * PA_SIMT_KT * (D + 4) + (64 / RT) * RT * (PA_SIMT_KT + 4) + 2 * RT) * 4 + PA_SIMT_KT * 4;
}

// D-element rows [k0, k0 + 64) of one head of sequence b into shared memory as
// fp32; rows outside [lo, hi) or without a page become zeros. `valid` (with K) notes which rows hold keys.
template <typename T, int D>
MF_DEVICE void paged_simt_load(float* dst, const T* base, const PagedKv& p, int b, int h, int k0, int lo, int hi, int* valid) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    constexpr int V = D / 32;
#pragma unroll 4
    for (int i = warp; i < PA_SIMT_KT; i += PA_SIMT_THREADS / 32) {
        const int key = k0 + i;
        const int page = key >= lo && key < hi ? paged_page(p, b, key) : -1;
        if (valid && lane == 0) valid[i] = page >= 0;
        float* d = dst + i * (D + 4) + lane * V;
        const T* src = base + (page >= 0 ? page * p.page_stride + (long long)h * p.head_stride + (key % p.page_size) * p.row_stride + lane * V : 0);
        if constexpr (sizeof(T) == 4) {
            const uint32_t s = (uint32_t)__cvta_generic_to_shared(d);
            if constexpr (V == 4) {
                asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(s), "l"(src), "r"(page >= 0 ? 16 : 0) : "memory");
            } else {
                asm volatile("cp.async.ca.shared.global [%0], [%1], 8, %2;" ::"r"(s), "l"(src), "r"(page >= 0 ? 8 : 0) : "memory");
            }
        } else {
            PackV<T, V> x = {};
            if (page >= 0) x = *reinterpret_cast<const PackV<T, V>*>(src);
#pragma unroll
            for (int e = 0; e < V; ++e) d[e] = to_f<T>(x.e[e]);
        }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
}

template <typename T, int D, int RT>
__global__ void __launch_bounds__(PA_SIMT_THREADS) paged_simt_kernel(const PagedKv p, const PagedAttn a) {
    constexpr int KT = PA_SIMT_KT, NG = 64 / RT, GT = PA_SIMT_THREADS / NG, LD = D + 4, LS = KT + 4;
    constexpr int NC = D / 64;            // float4 columns of O per thread
    constexpr int TPR = PA_SIMT_THREADS / RT, KPT = KT / TPR;  // softmax: threads per row, keys per thread
    extern __shared__ __align__(16) float paged_smem[];
    float* Qs = paged_smem;
    float* Ks = Qs + RT * LD;
    float* Vs = Ks + KT * LD;
    float* Ss = Vs + KT * LD;
    float* alpha_s = Ss + NG * RT * LS;
    float* l_s = alpha_s + RT;
    int* valid = reinterpret_cast<int*>(l_s + RT);
    __shared__ long long sh[34];
    pdl_wait();
    pdl_launch_dependents();  // after the wait: see paged_join_kernel

    PagedItem it;
    long long share;
    const long long total = paged_find<RT, KT>(p, a, blockIdx.x, gridDim.x, sh, share, it);
    const long long w0 = blockIdx.x * share, w1 = min(w0 + share, total);
    if (w0 >= w1) return;

    const int tid = threadIdx.x, grp = tid / GT, tg = tid % GT;
    const int ty = tg / 16, tx = tg % 16;  // rows 4 ty .., keys tx + 16 j, columns 4 tx + 64 j
    const int srow = tid / TPR, sk = tid % TPR;
    const T* kb = reinterpret_cast<const T*>(p.k);
    const T* vb = reinterpret_cast<const T*>(p.v);

    for (long long w = w0; w < w1;) {
        const int j0 = (int)max(w - it.start, 0ll), j1 = (int)min((long long)it.tiles, w1 - it.start);
        if (j1 <= 0) break;  // only the item's first unit is in this range
        const int rows = min(RT, it.s.n * a.G - it.r0);
        const int kt0 = it.k.lo / KT;
        __syncthreads();
        paged_simt_load<T, D>(Ks, kb, p, it.b, it.h, (kt0 + j0) * KT, it.k.lo, it.k.hi, valid);
        for (int i = tid; i < RT * D; i += PA_SIMT_THREADS) {
            const int r = i / D, row = it.r0 + r;
            Qs[r * LD + i % D] = r < rows ? to_f<T>(reinterpret_cast<const T*>(a.q)[(long long)(it.s.row + row / a.G) * a.q_stride +
                                                                                   (long long)(it.h * a.G + row % a.G) * D + i % D]) * a.scale2
                                          : 0.f;
        }
        float o[4][4 * NC];
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int e = 0; e < 4 * NC; ++e) o[i][e] = 0.f;
        float m = -INFINITY, l = 0.f;  // of row srow (the same in its threads)
        const int my_pos = it.s.first + (it.r0 + srow) / a.G;
        const int my_lo = a.window > 0 ? my_pos - a.window + 1 : 0;

        for (int j = j0; j < j1; ++j) {
            const int k0 = (kt0 + j) * KT;
            paged_simt_load<T, D>(Vs, vb, p, it.b, it.h, k0, it.k.lo, it.k.hi, nullptr);
            asm volatile("cp.async.wait_group 1;" ::: "memory");
            __syncthreads();  // K (and Q) are there
            float acc[4][4] = {};
#pragma unroll 4
            for (int d = grp * (D / NG); d < (grp + 1) * (D / NG); d += 4) {
                float4 qv[4], kv[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) qv[i] = *reinterpret_cast<const float4*>(Qs + (4 * ty + i) * LD + d);
#pragma unroll
                for (int i = 0; i < 4; ++i) kv[i] = *reinterpret_cast<const float4*>(Ks + (tx + 16 * i) * LD + d);
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
                for (int k = 0; k < 4; ++k) Ss[(grp * RT + 4 * ty + i) * LS + tx + 16 * k] = acc[i][k];
            __syncthreads();
            // softmax of row srow over its KPT keys sk, sk + TPR, ...
            float sv[KPT], mx = m;
#pragma unroll
            for (int k = 0; k < KPT; ++k) {
                const int kk = sk + TPR * k, key = k0 + kk;
                float x = 0.f;
#pragma unroll
                for (int g = 0; g < NG; ++g) x += Ss[(g * RT + srow) * LS + kk];
                sv[k] = key <= my_pos && key >= my_lo && valid[kk] ? x : -INFINITY;
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
                Ss[srow * LS + sk + TPR * k] = e;  // group 0's plane: only this thread reads or writes the entry
            }
#pragma unroll
            for (int off = TPR / 2; off > 0; off >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
            l = fmaf(l, al, sum);
            m = mx;
            if (sk == 0) alpha_s[srow] = al;
            asm volatile("cp.async.wait_group 0;" ::: "memory");
            __syncthreads();  // P, alpha and V are there; K is free
            if (j + 1 < j1) paged_simt_load<T, D>(Ks, kb, p, it.b, it.h, k0 + KT, it.k.lo, it.k.hi, valid);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float al4 = alpha_s[4 * ty + i];
#pragma unroll
                for (int e = 0; e < 4 * NC; ++e) o[i][e] *= al4;
            }
#pragma unroll 2
            for (int k = grp * (KT / NG); k < (grp + 1) * (KT / NG); k += 4) {
                float4 pv[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) pv[i] = *reinterpret_cast<const float4*>(Ss + (4 * ty + i) * LS + k);
#pragma unroll
                for (int kk = 0; kk < 4; ++kk)
#pragma unroll
                    for (int n = 0; n < NC; ++n) {
                        const float4 v = *reinterpret_cast<const float4*>(Vs + (k + kk) * LD + 4 * tx + 64 * n);
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
        // the groups' sums of O, in order, in the K tile's place
        if constexpr (NG > 1) {
            float* Os = Ks;  // [NG][RT][D] <= 2 * KT * LD
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int n = 0; n < NC; ++n)
                    *reinterpret_cast<float4*>(Os + (grp * RT + 4 * ty + i) * D + 4 * tx + 64 * n) =
                        make_float4(o[i][4 * n], o[i][4 * n + 1], o[i][4 * n + 2], o[i][4 * n + 3]);
        }
        if (sk == 0) {
            l_s[srow] = l;
            alpha_s[srow] = m;
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
                PackV<T, 4> y;
                y.e[0] = from_f<T>(v.x * inv);
                y.e[1] = from_f<T>(v.y * inv);
                y.e[2] = from_f<T>(v.z * inv);
                y.e[3] = from_f<T>(v.w * inv);
                *reinterpret_cast<PackV<T, 4>*>(reinterpret_cast<T*>(a.out) + (long long)(it.s.row + row / a.G) * a.out_stride +
                                                (long long)(it.h * a.G + row % a.G) * D + c) = y;
            } else {
                *reinterpret_cast<float4*>(part + r * D + c) = v;
                if (c == 0) {
                    ml[2 * r] = alpha_s[r];
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
}

}  // namespace mf
