// Attention of a few new tokens of each sequence over a paged cache (fp16 or
// bf16 pages): the decode step of a batch. o = softmax(scale q.k) v over the
// positions (pos - window, pos].
//
// Bound by memory: each K and V row is read once per KV head and meets the
// RT <= 32 query rows of its group. A CTA takes a range of the batch's key
// tiles of 32 KB (paged_work.cuh), so that lengths need not match. One warp
// keeps a ring of tiles in flight (two CTAs per SM, about 190 KB of copies
// outstanding), one TMA box per run of R keys of a page; four warps take a
// quarter of the keys of every tile each (64-wide heads: 32 keys, since with
// 16 a warp's fixed cost per tile outweighed its copies: 75 instead of 60 us
// for 64 sequences), with their own running maximum, sum and O (mma.sync
// m16n8k16, rows padded to 16: at two flops per byte and row the tensor pipe is
// far from its limit, and a 16-row tile of tcgen05 does not exist). They meet
// only at the end of an item, to join the four parts through shared memory. As
// in the chunk kernel the maximum moves only when it grows by more than 2^8;
// runs that no row sees are not read, and of a run that is seen in part the
// other rows are masked (scores) and zeroed (V, in registers).
// Measured: 32 sequences to 32768 keys, 64/8 heads, 354 us (2.28 GB, 0.98 of the
// copy rate); 64 sequences to 2048 keys, 16 heads of 64, 57 us (0.68); one
// sequence of 4096 keys 14 us with the join, a chain of latencies.
#pragma once

#include "paged_fa.cuh"

namespace mf {

template <int D> constexpr int pw_kt() { return D == 128 ? 64 : 128; }  // keys per tile: 32 KB of K and V either way
constexpr int PW_WARPS = 4;                       // consumers
constexpr int PW_THREADS = (PW_WARPS + 1) * 32;   // and the producer
constexpr int PW_COLS = 32;                       // columns of O joined at a time
constexpr int PW_LD = PW_COLS + 8;
template <int MT> constexpr int pw_stages() { return MT == 1 ? 3 : 2; }  // two CTAs fit an SM
template <int D> constexpr int pw_tile() { return pw_kt<D>() * D * 2; }
template <int D, int MT> constexpr int pw_smem() {
    return pw_stages<MT>() * 2 * pw_tile<D>() + PW_WARPS * 16 * MT * (PW_LD + 2) * 4 + (MT > 1 ? 16 * MT * D * 2 : 0) + 1024;
}

MF_DEVICE void ldsm4(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}
MF_DEVICE void ldsm4t(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}
template <typename T> MF_DEVICE void mma16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1);
template <> MF_DEVICE void mma16<__nv_bfloat16>(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <> MF_DEVICE void mma16<__half>(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

template <typename T> MF_DEVICE float2 pw_unpack(uint32_t v);
template <> MF_DEVICE float2 pw_unpack<__nv_bfloat16>(uint32_t v) { return make_float2(bf16_lo(v), bf16_hi(v)); }
template <> MF_DEVICE float2 pw_unpack<__half>(uint32_t v) { return f16x2_to_f2(v); }

// MT: 16-row tiles of query rows (RT = 16 MT).
template <typename T, int D, int MT>
__global__ void __launch_bounds__(PW_THREADS, 2)
    paged_few_kernel(const __grid_constant__ CUtensorMap tk, const __grid_constant__ CUtensorMap tv, const PagedKv p,
                     const PagedAttn a, const int run, const int at) {
    constexpr int RT = 16 * MT, ST = pw_stages<MT>(), KT = pw_kt<D>(), TILE = pw_tile<D>(), HALF = KT * 128;
    constexpr int KW = KT / PW_WARPS;  // keys of one warp: 16 or 32
    extern __shared__ uint8_t pw_smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(pw_smem_raw) + 1023) & ~(uintptr_t)1023);
    float* join = reinterpret_cast<float*>(smem + ST * 2 * TILE);  // [warp][RT][PW_LD]
    float2* ml_s = reinterpret_cast<float2*>(join + PW_WARPS * RT * PW_LD);  // [warp][RT]
    uint8_t* q_s = reinterpret_cast<uint8_t*>(ml_s + PW_WARPS * RT);  // MT > 1: [RT][D], rows of D * 2 bytes, swizzled
    __shared__ __align__(8) uint64_t full[ST], free_[ST];
    __shared__ uint32_t pages_s[ST];  // which 8-key runs of the stage have a page
    __shared__ long long sh[34];

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        for (int s = 0; s < ST; ++s) {
            mbar_init(&full[s], 1);
            mbar_init(&free_[s], PW_WARPS);
        }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    paged_begin(a);
    __syncthreads();
    PagedItem it;
    long long share;
    const long long total = paged_find<RT, KT>(p, a, blockIdx.x, gridDim.x, sh, share, it);
    const long long w0 = blockIdx.x * share, w1 = min(w0 + share, total);
    if (w0 >= w1) {
        paged_end(a);
        return;
    }
    const unsigned long long deadline = globaltimer_ns() + a.timeout_ns;
    bool failed = false;

    if (warp == PW_WARPS) {
        const int R = run, nr = KT / R;
        int n = 0;  // tiles issued
        for (long long w = w0; w < w1 && !failed;) {
            const int j0 = (int)max(w - it.start, 0ll), j1 = (int)min((long long)it.tiles, w1 - it.start);
            if (j1 <= 0) break;  // only the item's first unit is in this range
            const int key0 = it.k.lo / KT * KT;
            for (int j = j0; j < j1; ++j, ++n) {
                const int st = n % ST;
                const int c0 = key0 + j * KT + lane * R;  // this lane's run: keys [c0, c0 + R)
                const int page = lane < nr && c0 < it.k.hi && c0 + R > it.k.lo ? paged_page(p, it.b, c0) : -1;
                const int off = c0 % p.page_size;
                const unsigned boxes = __ballot_sync(0xffffffffu, page >= 0);
                if (n >= ST) mbar_wait(&free_[st], ((uint32_t)(n / ST) & 1u) ^ 1u, deadline, failed);
                failed = __any_sync(0xffffffffu, failed);
                if (failed) break;
                uint8_t* kd = smem + st * 2 * TILE;
                uint8_t* vd = kd + TILE;
                if (lane == 0) {
                    uint32_t ok = 0;  // per 8 keys
                    for (int i = 0; i < KT / 8; ++i) ok |= (boxes >> (8 * i / R) & 1u) << i;
                    pages_s[st] = ok;
                    mbar_expect_tx(&full[st], (uint32_t)__popc(boxes) * R * D * 4);
                }
                __syncwarp();
                if (page >= 0) {
#pragma unroll
                    for (int x = 0; x < D / 64; ++x) {
                        tma_load_page(kd + x * HALF + lane * R * 128, &tk, &full[st], 64 * x, off, it.h, page, at & 1);
                        tma_load_page(vd + x * HALF + lane * R * 128, &tv, &full[st], 64 * x, off, it.h, page, at >> 1);
                    }
                }
            }
            w = it.start + j1;
            if (w < w1 && !failed) paged_next<RT, KT>(p, a, it);
        }
        // the copies in flight land before shared memory goes away, also those that a consumer gave up on
        bool f2 = false;
        const unsigned long long d2 = globaltimer_ns() + a.timeout_ns;
        for (int j = max(0, n - ST); j < n; ++j) mbar_wait(&full[j % ST], (uint32_t)(j / ST) & 1u, d2, f2);
    } else {
        const float c2 = fabsf(a.scale2);
        const uint32_t flip = a.scale2 < 0.f ? 0x80008000u : 0u;  // a negative scale goes into Q's sign
        int n = 0;
        for (long long w = w0; w < w1;) {
            const int j0 = (int)max(w - it.start, 0ll), j1 = (int)min((long long)it.tiles, w1 - it.start);
            if (j1 <= 0) break;  // only the item's first unit is in this range
            const int rows = min(it.step, it.s.n * a.G - it.r0);
            const int key0 = it.k.lo / KT * KT;
            // Rows r and r + 8 of a 16-row tile are one thread's. An item of up to 8 rows has each in both places, and P
            // rounded to the pages' type in the first and what that left of it in the second: the products are the same in
            // number, and the two halves of O, added at the end, hold P exact to 2^-16 (fp16: 2^-22). (For more rows the second
            // part would be as many products again: 32 rows of 64 x 4 tokens at 4096 keys 245 us in place of 222.)
            const bool twice = rows <= 8;
            auto row_at = [&](int r) { return min(twice ? r & 7 : r, rows - 1); };  // rows past the end repeat the last
            const T* qb = reinterpret_cast<const T*>(a.q) + (long long)it.s.row * a.q_stride + (long long)it.h * a.G * D;
            auto q_row = [&](int r) { return qb + (long long)((it.r0 + r) / a.G) * a.q_stride + (long long)((it.r0 + r) % a.G) * D; };
            uint32_t qf[MT == 1 ? D / 16 : 1][4];
            if constexpr (MT == 1) {
                const int r = lane >> 2, c = (lane & 3) * 2;
                const T* q0 = q_row(row_at(r));
                const T* q1 = q_row(row_at(r + 8));
#pragma unroll
                for (int k = 0; k < D / 16; ++k) {
                    qf[k][0] = *reinterpret_cast<const uint32_t*>(q0 + 16 * k + c) ^ flip;
                    qf[k][1] = *reinterpret_cast<const uint32_t*>(q1 + 16 * k + c) ^ flip;
                    qf[k][2] = *reinterpret_cast<const uint32_t*>(q0 + 16 * k + c + 8) ^ flip;
                    qf[k][3] = *reinterpret_cast<const uint32_t*>(q1 + 16 * k + c + 8) ^ flip;
                }
            } else {
                named_bar_sync(1, PW_WARPS * 32);  // the last item's rows are done with
                for (int e = threadIdx.x; e < RT * (D / 8); e += PW_WARPS * 32) {
                    const int r = e / (D / 8), cc = e % (D / 8);
                    uint4 v = *reinterpret_cast<const uint4*>(q_row(row_at(r)) + cc * 8);
                    v = make_uint4(v.x ^ flip, v.y ^ flip, v.z ^ flip, v.w ^ flip);
                    *reinterpret_cast<uint4*>(q_s + r * (D * 2) + ((cc ^ (r & 7)) << 4)) = v;
                }
                named_bar_sync(1, PW_WARPS * 32);
            }
            // this lane's rows: lane / 4 (+ 8) of each 16-row tile; repeated ones are not stored
            int pos[MT][2], lo[MT][2];
            int hi_all = 0x7fffffff, lo_all = 0;
#pragma unroll
            for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    pos[mt][e] = it.s.first + (it.r0 + row_at(16 * mt + 8 * e + (lane >> 2))) / a.G;
                    lo[mt][e] = a.window > 0 ? pos[mt][e] - a.window + 1 : 0;
                    hi_all = min(hi_all, pos[mt][e]);
                    lo_all = max(lo_all, lo[mt][e]);
                }
            hi_all = __reduce_min_sync(0xffffffffu, hi_all);
            lo_all = __reduce_max_sync(0xffffffffu, lo_all);
            float o[MT][D / 8][4];
            float m[MT][2], l[MT][2];
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) {
                m[mt][0] = m[mt][1] = -INFINITY;
                l[mt][0] = l[mt][1] = 0.f;
#pragma unroll
                for (int d = 0; d < D / 8; ++d) o[mt][d][0] = o[mt][d][1] = o[mt][d][2] = o[mt][d][3] = 0.f;
            }

            for (int j = j0; j < j1; ++j, ++n) {
                const int st = n % ST;
                mbar_wait(&full[st], (uint32_t)(n / ST) & 1u, deadline, failed);
                failed = __any_sync(0xffffffffu, failed);
                if (failed) break;  // without an arrival: the producer refills nothing that another warp still reads
                const uint32_t kd = smem_u32(smem + st * 2 * TILE), vd = kd + TILE;
                const int kw = KW * warp, k0 = key0 + j * KT + kw;  // this warp's keys
                float s[MT][KW / 8][4];
#pragma unroll
                for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                    for (int t = 0; t < KW / 8; ++t) s[mt][t][0] = s[mt][t][1] = s[mt][t][2] = s[mt][t][3] = 0.f;
#pragma unroll
                for (int k = 0; k < D / 16; ++k) {
                    uint32_t qa[MT][4];
#pragma unroll
                    for (int mt = 0; mt < MT; ++mt) {
                        if constexpr (MT == 1) {
                            qa[0][0] = qf[k][0], qa[0][1] = qf[k][1], qa[0][2] = qf[k][2], qa[0][3] = qf[k][3];
                        } else {
                            const int r = 16 * mt + (lane & 15), cq = 2 * k + (lane >> 4);
                            ldsm4(qa[mt], smem_u32(q_s) + r * (D * 2) + ((cq ^ (r & 7)) << 4));
                        }
                    }
#pragma unroll
                    for (int kk = 0; kk < KW / 16; ++kk) {
                        const int key = kw + 16 * kk + ((lane >> 4) << 3) + (lane & 7), c = 2 * k + ((lane >> 3) & 1);
                        uint32_t b[4];
                        ldsm4(b, kd + key * 128 + (c >> 3) * HALF + (((c & 7) ^ (key & 7)) << 4));
#pragma unroll
                        for (int mt = 0; mt < MT; ++mt) {
                            mma16<T>(s[mt][2 * kk], qa[mt], b[0], b[1]);
                            mma16<T>(s[mt][2 * kk + 1], qa[mt], b[2], b[3]);
                        }
                    }
                }
                constexpr uint32_t ALL = (1u << (KW / 8)) - 1;
                const uint32_t ok = pages_s[st] >> (KW / 8 * warp) & ALL;
                if (!(k0 + KW - 1 <= hi_all && k0 >= lo_all && ok == ALL)) {
#pragma unroll
                    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                        for (int t = 0; t < KW / 8; ++t)
#pragma unroll
                            for (int e = 0; e < 4; ++e) {
                                const int key = k0 + 8 * t + (lane & 3) * 2 + (e & 1);
                                if (!(ok >> t & 1u) || key > pos[mt][e >> 1] || key < lo[mt][e >> 1]) s[mt][t][e] = -INFINITY;
                            }
                }
                uint32_t pa[MT][KW / 16][4];
#pragma unroll
                for (int mt = 0; mt < MT; ++mt) {
                    float alpha[2];
                    bool bump = false;
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        float mx = fmaxf(s[mt][0][2 * e], s[mt][0][2 * e + 1]);
#pragma unroll
                        for (int t = 1; t < KW / 8; ++t) mx = fmaxf(mx, fmaxf(s[mt][t][2 * e], s[mt][t][2 * e + 1]));
                        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
                        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2)) * c2;
                        const bool up = mx > m[mt][e] + 8.f;
                        const float mu = up ? mx : m[mt][e];
                        const float base = mu == -INFINITY ? 0.f : mu;
                        const float off = pf_lift<T>() - base;
                        alpha[e] = up ? ex2_approx(m[mt][e] - base) : 1.f;
                        bump |= up;
                        m[mt][e] = mu;
                        float sum = 0.f;
#pragma unroll
                        for (int t = 0; t < KW / 8; ++t)
#pragma unroll
                            for (int u = 0; u < 2; ++u) {
                                const float x = ex2_approx(fmaf(s[mt][t][2 * e + u], c2, off));
                                s[mt][t][2 * e + u] = x;
                                sum += x;
                            }
                        l[mt][e] = fmaf(l[mt][e], alpha[e], sum);  // of this lane's keys
                    }
                    if (__any_sync(0xffffffffu, bump)) {
#pragma unroll
                        for (int d = 0; d < D / 8; ++d) {
                            o[mt][d][0] *= alpha[0];
                            o[mt][d][1] *= alpha[0];
                            o[mt][d][2] *= alpha[1];
                            o[mt][d][3] *= alpha[1];
                        }
                    }
#pragma unroll
                    for (int kk = 0; kk < KW / 16; ++kk) {
                        pa[mt][kk][0] = pf_pack<T>(s[mt][2 * kk][0], s[mt][2 * kk][1]);
                        pa[mt][kk][2] = pf_pack<T>(s[mt][2 * kk + 1][0], s[mt][2 * kk + 1][1]);
                        if (twice) {
                            const float2 h0 = pw_unpack<T>(pa[mt][kk][0]), h1 = pw_unpack<T>(pa[mt][kk][2]);
                            s[mt][2 * kk][2] -= h0.x;
                            s[mt][2 * kk][3] -= h0.y;
                            s[mt][2 * kk + 1][2] -= h1.x;
                            s[mt][2 * kk + 1][3] -= h1.y;
                        }
                        pa[mt][kk][1] = pf_pack<T>(s[mt][2 * kk][2], s[mt][2 * kk][3]);
                        pa[mt][kk][3] = pf_pack<T>(s[mt][2 * kk + 1][2], s[mt][2 * kk + 1][3]);
                    }
                }
                // V rows that no row of the item sees are zeros, whatever the tile holds there (a register holds
                // the rows of two neighbouring keys, 2 (lane % 4) and the next, of a run of 8)
                uint32_t keep[KW / 8];
                const bool cut = k0 < it.k.lo || k0 + KW > it.k.hi || ok != ALL;
                if (cut) {
#pragma unroll
                    for (int t = 0; t < KW / 8; ++t) {
                        const int key = k0 + 8 * t + (lane & 3) * 2;
                        keep[t] = !(ok >> t & 1u) ? 0u
                                                  : (key >= it.k.lo && key < it.k.hi ? 0xffffu : 0u) |
                                                        (key + 1 >= it.k.lo && key + 1 < it.k.hi ? 0xffff0000u : 0u);
                    }
                }
#pragma unroll
                for (int kk = 0; kk < KW / 16; ++kk) {
                    const int key = kw + 16 * kk + (((lane >> 3) & 1) << 3) + (lane & 7);
#pragma unroll
                    for (int d = 0; d < D / 16; ++d) {
                        const int c = 2 * d + (lane >> 4);
                        uint32_t b[4];
                        ldsm4t(b, vd + key * 128 + (c >> 3) * HALF + (((c & 7) ^ (key & 7)) << 4));
                        if (cut) {
                            b[0] &= keep[2 * kk];
                            b[1] &= keep[2 * kk + 1];
                            b[2] &= keep[2 * kk];
                            b[3] &= keep[2 * kk + 1];
                        }
#pragma unroll
                        for (int mt = 0; mt < MT; ++mt) {
                            mma16<T>(o[mt][2 * d], pa[mt][kk], b[0], b[1]);
                            mma16<T>(o[mt][2 * d + 1], pa[mt][kk], b[2], b[3]);
                        }
                    }
                }
                __syncwarp();
                if (lane == 0) mbar_arrive(&free_[st]);
            }

            if (twice) {
#pragma unroll
                for (int d = 0; d < D / 8; ++d) {
                    o[0][d][0] += o[0][d][2];
                    o[0][d][1] += o[0][d][3];
                }
            }
            // join the four warps' parts, PW_COLS columns at a time
#pragma unroll
            for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    l[mt][e] += __shfl_xor_sync(0xffffffffu, l[mt][e], 1);
                    l[mt][e] += __shfl_xor_sync(0xffffffffu, l[mt][e], 2);
                    if ((lane & 3) == 0) ml_s[warp * RT + 16 * mt + 8 * e + (lane >> 2)] = make_float2(m[mt][e], failed ? PAGED_GAVE_UP : l[mt][e]);
                }
            const bool whole = j0 == 0 && j1 == it.tiles;
            const long long slot = 2ll * blockIdx.x + (j0 > 0 ? 0 : 1);
            float* part = a.part + slot * RT * D;
            float* part_ml = a.part + 2ll * gridDim.x * RT * D + slot * RT * 2;
            bool stop = false;
#pragma unroll
            for (int c0 = 0; c0 < D; c0 += PW_COLS) {
#pragma unroll
                for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                    for (int d = 0; d < PW_COLS / 8; ++d) {
                        float* x = join + (warp * RT + 16 * mt + (lane >> 2)) * PW_LD + 8 * d + (lane & 3) * 2;
                        *reinterpret_cast<float2*>(x) = make_float2(o[mt][c0 / 8 + d][0], o[mt][c0 / 8 + d][1]);
                        *reinterpret_cast<float2*>(x + 8 * PW_LD) = make_float2(o[mt][c0 / 8 + d][2], o[mt][c0 / 8 + d][3]);
                    }
                named_bar_sync(1, PW_WARPS * 32);
#pragma unroll
                for (int u = 0; u < MT; ++u) {
                    const int r = 16 * u + (threadIdx.x >> 3), c = (threadIdx.x & 7) * 4;
                    float mm = -INFINITY, ll = 0.f;
#pragma unroll
                    for (int i = 0; i < PW_WARPS; ++i) mm = fmaxf(mm, ml_s[i * RT + r].x);
                    float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
                    for (int i = 0; i < PW_WARPS; ++i) {
                        const float2 y = ml_s[i * RT + r];
                        const float wt = y.y != 0.f ? ex2_approx(y.x - mm) : 0.f;
                        const float4 v = *reinterpret_cast<const float4*>(join + (i * RT + r) * PW_LD + c);
                        stop |= y.y == PAGED_GAVE_UP;  // of every row, so all four warps know
                        ll = fmaf(y.y, wt, ll);
                        x.x = fmaf(v.x, wt, x.x);
                        x.y = fmaf(v.y, wt, x.y);
                        x.z = fmaf(v.z, wt, x.z);
                        x.w = fmaf(v.w, wt, x.w);
                    }
                    if (r < rows && !stop) {
                        if (whole) {
                            const float inv = ll == 0.f ? 0.f : 1.0f / ll;
                            T* out = reinterpret_cast<T*>(a.out) + (long long)(it.s.row + (it.r0 + r) / a.G) * a.out_stride +
                                     (long long)(it.h * a.G + (it.r0 + r) % a.G) * D + c0 + c;
                            *reinterpret_cast<uint2*>(out) = make_uint2(pf_pack<T>(x.x * inv, x.y * inv), pf_pack<T>(x.z * inv, x.w * inv));
                        } else {
                            *reinterpret_cast<float4*>(part + r * D + c0 + c) = x;
                            if (c0 == 0 && c == 0) *reinterpret_cast<float2*>(part_ml + 2 * r) = make_float2(mm, ll);
                        }
                    }
                }
                named_bar_sync(1, PW_WARPS * 32);
            }
            if (stop) {
                // nothing of this item or the next ones is written, and neither are the divided ones joined
                float2* ml = reinterpret_cast<float2*>(a.part + 2ll * gridDim.x * RT * D) + 2ll * blockIdx.x * RT;
                if (threadIdx.x < 2 * RT) ml[threadIdx.x] = make_float2(0.f, PAGED_GAVE_UP);
                break;
            }
            w = it.start + j1;
            if (w < w1) paged_next<RT, KT>(p, a, it);
        }
    }
    if (failed) atomicOr(a.status, 2);
    paged_end(a);
}

}  // namespace mf
