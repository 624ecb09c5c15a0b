// Attention of chunks of new tokens over a paged cache on the 5th-generation
// tensor cores (fp16 or bf16 pages): o = softmax(scale q.k) v over the
// positions (pos - window, pos], one pass with the running maximum and sum of
// each row.
//
// CTA = 256 query rows (row r of a sequence = token r / G, head r % G of one
// KV head's group) as two tiles of 128, and the 128-key tiles that they see
// (or this split's share of them). Both tiles use every K and V tile, and
// while the softmax of one runs the tensor core works for the other:
//   warps 0-3, 4-7  softmax of tile 0, 1: one thread per row. Q into shared
//                   memory first; per key tile: the row's 128 scores from
//                   TMEM, mask, maximum, exponentials, P as 16 bits back over
//                   the scores. The maximum moves only when it grows by more
//                   than 2^8 (a stale one changes rounding only, and P stays
//                   below 2^8, or 2^15: pf_lift); then the thread rescales its
//                   row of O.
//   warp 8          issues S_i = Q_i K^T (M128 N128) and O_i += P_i V (A = P
//                   from TMEM, B = V as it lies in the page: the key rows are
//                   the K extent, d is contiguous).
//   warps 9, 10     bring in K and V: one TMA box per run of R keys of a page
//                   (R = the power of two in page_size, 8 .. 64). Runs that no
//                   row sees or that have no page are not read: their scores
//                   are masked, their V rows zeroed, so nothing in them (NaN
//                   included) reaches a result; a run that is seen in part is
//                   copied row by row.
// TMEM: S_0, S_1 (P over them), O_0, O_1: 512 columns.
// One thread issues all MMAs, and they execute in order: S_i of the next tile
// may overwrite P_i once O_i += P_i V has been issued, and a thread that sees
// the commit of S_i knows that O_i holds every tile before.
//
// At D = 128 a pair of 128 x 128 score tiles costs 2048 cycles of the tensor
// core and as many of the special-function unit (1536 with a quarter of the
// exponentials on the FMA units). A tile's softmax (2200 cycles) and its MMAs
// with their barriers (1200) follow each other, so a pair takes about 3450.
// Measured: 4096 x 4096 causal, 32/8 heads, 142 us at 1965 MHz and 163 in a long
// loop, where the power cap takes the clock to 1750 (0.59 and 0.51 of the cuBLAS
// bf16 rate, diagonal tiles counted by their halves); of the 142 the pairs take
// 100 and the CTAs' beginnings, ends and last round the rest. 512 tokens after
// 28672, 64/8 heads, 413-440 and 478 us (1.10-1.18 and 1.02 PFLOP/s on the 128
// SMs that have a tile).
// Slower: two buffers of 64-key scores (159 / 513 us: an MMA of 64 keys takes
// 55 cycles, not 32), four groups of 64 columns (158 / 444), exponentials before
// the maximum is known (154 / 470).
#pragma once

#include <type_traits>

#include "paged_work.cuh"
#include "prefill_fa.cuh"

namespace mf {

constexpr int PF_ROWS = 256;  // query rows of a CTA
constexpr int PF_KT = 128;    // keys per tile
constexpr int PF_THREADS = 384;
constexpr int PF_STAGES = 2;  // K and V rings
constexpr int PF_HALF = PF_KT * 128;  // 128 rows x 64 elements (16 KB)
template <int D> constexpr int pf_tile() { return D / 64 * PF_HALF; }
template <int D> constexpr int pf_smem() { return (2 * PF_STAGES + 2) * pf_tile<D>() + 1024; }

struct PagedFa {
    int run;        // R: keys per TMA box
    int at;         // K's index along the maps' last extent, and V's in bit 1
    int min_rows;   // sequences of at most this many rows are another kernel's
    int n_split;    // gridDim.y: shares of the key tiles
    float* part_o;  // n_split > 1: [split][n_tokens * n_heads][D], unnormalised
    float2* part_ml;  // [split][n_tokens * n_heads]
};

// Shared-memory descriptors of 128-byte-swizzled tiles. Their upper words are
// constants and the address is the lowest field, so an operand a few 16-byte
// units on is one 32-bit addition: a descriptor built anew for every MMA cost
// as long as the MMA.
//   PF_DESC_MN: rows run along the M or N extent (sw128_kmajor_desc): the next 8 rows 1024 bytes on.
//   PF_DESC_K:  rows run along K: the next 8 rows 1024 bytes on, the next 64 elements of N PF_HALF bytes on.
constexpr uint32_t PF_DESC_HI = (1024u >> 4) | (1u << 14) | (2u << 29);
MF_DEVICE uint32_t pf_desc_mn(uint32_t saddr) { return saddr >> 4; }
MF_DEVICE uint32_t pf_desc_k(uint32_t saddr) { return saddr >> 4 | ((uint32_t)(PF_HALF >> 4) << 16); }

// D (TMEM) (+)= A * B with B from shared memory and A from shared memory or TMEM; lower words of the descriptors.
MF_DEVICE void pf_mma_ss(uint32_t d, uint32_t a_lo, uint32_t b_lo, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t.reg .b64 a, b;\n\t"
        "mov.b64 a, {%1, %5};\n\t"
        "mov.b64 b, {%2, %5};\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, p;\n\t}" ::"r"(d),
        "r"(a_lo), "r"(b_lo), "r"(idesc), "r"(accumulate), "n"(PF_DESC_HI)
        : "memory");
}
MF_DEVICE void pf_mma_ts(uint32_t d, uint32_t a, uint32_t b_lo, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t.reg .b64 b;\n\t"
        "mov.b64 b, {%2, %5};\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], b, %3, p;\n\t}" ::"r"(d),
        "r"(a), "r"(b_lo), "r"(idesc), "r"(accumulate), "n"(PF_DESC_HI)
        : "memory");
}
// One thread of the warp, known to the compiler as one: what it computes stays in uniform registers.
MF_DEVICE bool pf_elect() {
    uint32_t p;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(p));
    return p != 0;
}

// One box of the pages' map (d, row of the page, head, page, tensor).
MF_DEVICE void tma_load_page(void* dst, const CUtensorMap* tm, uint64_t* bar, int d, int row, int head, int page, int which) {
    asm volatile(
        "cp.async.bulk.tensor.5d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6, %7}], [%2];" ::
            "r"(smem_u32(dst)),
        "l"(reinterpret_cast<uint64_t>(tm)), "r"(smem_u32(bar)), "r"(d), "r"(row), "r"(head), "r"(page), "r"(which)
        : "memory");
}

// Two floats as one 64-bit operand of the packed fp32 instructions.
typedef unsigned long long f32x2;
MF_DEVICE f32x2 pf_two(float a, float b) {
    f32x2 r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
MF_DEVICE float2 pf_each(f32x2 v) {
    float2 r;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
    return r;
}
MF_DEVICE f32x2 pf_fma2(f32x2 a, f32x2 b, f32x2 c) {
    f32x2 r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
MF_DEVICE f32x2 pf_add2(f32x2 a, f32x2 b) {
    f32x2 r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
// Maxima that are NaN where an argument is.
MF_DEVICE float pf_max3(float a, float b, float c) {
    float r;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}
MF_DEVICE float pf_max(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
// 2^y of two finite y on the FMA units: y = n + r, |r| <= 1/2, a polynomial of
// degree 5 for 2^r, n added to its exponent. Its coefficients have the least
// maximum of the relative error beside a constant term of 1, found by linear
// programming, each rounded to a float before the next was fitted: 2^-23.3 in
// exact arithmetic, 2^-22.6 with every step rounded (P has 8 or 11 bits).
// Below 2^-126 the result is a tiny number instead of zero, and NaN is lost.
MF_DEVICE float2 pf_exp2_fma(f32x2 y) {
    const float2 c = pf_each(y);
    y = pf_two(fmaxf(c.x, -126.f), fmaxf(c.y, -126.f));
    const f32x2 magic = pf_two(12582912.f, 12582912.f);  // 1.5 * 2^23: the low bits of the sum are n
    const f32x2 t = pf_add2(y, magic);
    const f32x2 n = pf_add2(t, pf_two(-12582912.f, -12582912.f));
    const f32x2 r = pf_fma2(n, pf_two(-1.f, -1.f), y);
    f32x2 q = pf_two(1.32695213e-3f, 1.32695213e-3f);
    q = pf_fma2(q, r, pf_two(9.67129134e-3f, 9.67129134e-3f));
    q = pf_fma2(q, r, pf_two(5.55071086e-2f, 5.55071086e-2f));
    q = pf_fma2(q, r, pf_two(2.40222469e-1f, 2.40222469e-1f));
    q = pf_fma2(q, r, pf_two(6.93147004e-1f, 6.93147004e-1f));
    q = pf_fma2(q, r, pf_two(1.f, 1.f));
    const float2 ti = pf_each(t), qi = pf_each(q);
    return make_float2(__int_as_float(__float_as_int(qi.x) + (__float_as_int(ti.x) << 23)),
                       __int_as_float(__float_as_int(qi.y) + (__float_as_int(ti.y) << 23)));
}

// P = 2^(score - m + pf_lift): P is rounded to the pages' type, and fp16 holds
// nothing below 2^-25. With the maximum m up to 2^8 behind, 2^15 is the most
// that P may be lifted to; weights down to 2^-21 of the largest then keep fp16's
// 11 bits and smaller ones are off by at most 2^-32 of it, so 2^20 of them by
// at most 2^-12. (Without: 4096 keys 2^-25.5 as likely as the first were in the
// sum but not in O.) bf16 has the exponents of a float. The factor is in
// O and in the sum, and leaves with their quotient.
template <typename T> constexpr float pf_lift() { return std::is_same<T, __half>::value ? 7.f : 0.f; }

template <typename T> MF_DEVICE uint32_t pf_pack(float a, float b);
template <> MF_DEVICE uint32_t pf_pack<__nv_bfloat16>(float a, float b) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&v);
}
template <> MF_DEVICE uint32_t pf_pack<__half>(float a, float b) {
    const __half2 v = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&v);
}

// 16 columns of this warp's lanes
MF_DEVICE void pf_ld16(uint32_t taddr, uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr));
    tmem_wait_ld();
}
MF_DEVICE void pf_st16(uint32_t taddr, const uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(taddr),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
        "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
        : "memory");
}

// The row tile `tile` of the batch: sequences of more than min_rows rows, in
// order, each with its last rows (the most keys) first. One warp together.
struct PfTile {
    int b, r0;
};
MF_DEVICE PfTile pf_find(const PagedKv& p, int G, int min_rows, int tile) {
    const int lane = threadIdx.x & 31;
    PfTile f;
    f.b = -1;
    f.r0 = 0;
    for (int b0 = 0, base = 0; b0 < p.n_seqs; b0 += 32) {
        int rows = 0;
        if (b0 + lane < p.n_seqs) rows = paged_seq(p, b0 + lane).n * G;
        const int n = rows > min_rows ? (rows + PF_ROWS - 1) / PF_ROWS : 0;
        int inc = n;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int v = __shfl_up_sync(0xffffffffu, inc, o);
            if (lane >= o) inc += v;
        }
        const unsigned hit = __ballot_sync(0xffffffffu, tile < base + inc);
        if (hit) {
            const int src = __ffs(hit) - 1;
            f.b = b0 + src;
            f.r0 = (__shfl_sync(0xffffffffu, base + inc, src) - 1 - tile) * PF_ROWS;
            return f;
        }
        base += __shfl_sync(0xffffffffu, inc, 31);
    }
    return f;
}

template <typename T, int D>
__global__ void __launch_bounds__(PF_THREADS, 1)
    paged_fa_kernel(const __grid_constant__ CUtensorMap tk, const __grid_constant__ CUtensorMap tv, const PagedKv p,
                    const PagedAttn a, const PagedFa f) {
    constexpr int TILE = pf_tile<D>();
    constexpr bool BF = std::is_same<T, __nv_bfloat16>::value;
    extern __shared__ uint8_t pf_smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(pf_smem_raw) + 1023) & ~(uintptr_t)1023);
    uint8_t* ks = smem;
    uint8_t* vs = smem + PF_STAGES * TILE;
    uint8_t* qs = vs + PF_STAGES * TILE;
    __shared__ __align__(8) uint64_t k_full[PF_STAGES], k_free[PF_STAGES], v_full[PF_STAGES], v_free[PF_STAGES];
    __shared__ __align__(8) uint64_t q_full[2], s_full[2], p_full[2][2], o_full[2], drain;
    __shared__ uint32_t tmem_base_s;

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        for (int s = 0; s < PF_STAGES; ++s) {
            mbar_init(&k_full[s], 1);
            mbar_init(&k_free[s], 1);
            mbar_init(&v_full[s], 1);
            mbar_init(&v_free[s], 1);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(&q_full[i], 128);
            mbar_init(&s_full[i], 1);
            mbar_init(&p_full[i][0], 128);
            mbar_init(&p_full[i][1], 128);
            mbar_init(&o_full[i], 1);
        }
        mbar_init(&drain, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    pdl_wait();

    const int h = blockIdx.x % p.n_kv_heads;
    const PfTile pt = pf_find(p, a.G, f.min_rows, blockIdx.x / p.n_kv_heads);
    if (pt.b < 0) return;  // past the last tile: the whole CTA leaves, no TMEM taken yet
    const PagedSeq s = paged_seq(p, pt.b);
    const int rows = min(s.n * a.G - pt.r0, PF_ROWS);
    const bool two = rows > 128;
    const PagedSpan span = paged_span(s, a, pt.r0, PF_ROWS);
    const int kt0 = span.lo / PF_KT;
    const int nt_all = span.hi > span.lo ? (span.hi + PF_KT - 1) / PF_KT - kt0 : 0;
    const int j0 = (int)((long long)nt_all * blockIdx.y / f.n_split), j1 = (int)((long long)nt_all * (blockIdx.y + 1) / f.n_split);
    const int nt = j1 - j0;
    const int key0 = (kt0 + j0) * PF_KT;  // first key of tile 0 of this CTA

    if (warp == 8) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_base_s)), "r"(512)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = tmem_base_s;
    pdl_launch_dependents();  // only now: a dependent kernel may take TMEM before its wait
    const unsigned long long deadline = globaltimer_ns() + a.timeout_ns;
    bool failed = false;

    if (warp >= 8) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 88;");
        if (warp == 9 || warp == 10) {
            const bool is_k = warp == 9;
            const CUtensorMap* tm = is_k ? &tk : &tv;
            const int which = is_k ? f.at & 1 : f.at >> 1;
            uint8_t* ring = is_k ? ks : vs;
            uint64_t* full = is_k ? k_full : v_full;
            uint64_t* free_ = is_k ? k_free : v_free;
            const int R = f.run, nr = PF_KT / R;  // at most 16 runs of a tile, one per lane
            int issued = 0;
            for (int j = 0; j < nt; ++j) {
                const int st = j % PF_STAGES;
                // the page of this lane's run; its keys [c0, c0 + R)
                const int c0 = key0 + j * PF_KT + lane * R;
                const bool any = lane < nr && c0 < span.hi && c0 + R > span.lo;
                const int page = any ? paged_page(p, pt.b, c0) : -1;
                // V rows that no row sees are zeroed, so a run that is seen in part is not one box
                const bool whole = page >= 0 && (is_k || (c0 >= span.lo && c0 + R <= span.hi));
                const unsigned boxes = __ballot_sync(0xffffffffu, whole);
                unsigned rest = is_k ? 0u : __ballot_sync(0xffffffffu, lane < nr && !whole);
                if (j >= PF_STAGES) mbar_wait(&free_[st], ((uint32_t)(j / PF_STAGES) & 1u) ^ 1u, deadline, failed);
                if (__any_sync(0xffffffffu, failed)) {
                    failed = true;
                    break;
                }
                uint8_t* dst = ring + st * TILE;
                while (rest) {
                    const int i = __ffs(rest) - 1;
                    rest &= rest - 1;
                    const int pg = __shfl_sync(0xffffffffu, page, i), k0 = __shfl_sync(0xffffffffu, c0, i);
                    const T* src = reinterpret_cast<const T*>(p.v) + (pg < 0 ? 0 : pg * p.page_stride + (long long)h * p.head_stride + (long long)(k0 % p.page_size) * p.row_stride);
#pragma unroll 8
                    for (int e = lane; e < R * (D / 8); e += 32) {
                        const int r = e / (D / 8), c = e % (D / 8), key = k0 + r;
                        uint4 v = make_uint4(0, 0, 0, 0);
                        if (pg >= 0 && key >= span.lo && key < span.hi) v = __ldg(reinterpret_cast<const uint4*>(src + r * p.row_stride + c * 8));
                        const int row = i * R + r;
                        *reinterpret_cast<uint4*>(dst + (c >> 3) * PF_HALF + row * 128 + (((c & 7) ^ (row & 7)) << 4)) = v;
                    }
                }
                if (!is_k) asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                __syncwarp();
                if (lane == 0) mbar_expect_tx(&full[st], (uint32_t)__popc(boxes) * R * D * 2);
                __syncwarp();
                if (whole) {
                    const int off = c0 % p.page_size;
#pragma unroll
                    for (int x = 0; x < D / 64; ++x) tma_load_page(dst + x * PF_HALF + lane * R * 128, tm, &full[st], 64 * x, off, h, page, which);
                }
                issued = j + 1;
            }
            // the copies in flight land before shared memory goes away, also those that another warp gave up on
            bool f2 = false;
            const unsigned long long d2 = globaltimer_ns() + a.timeout_ns;
            for (int j = max(0, issued - PF_STAGES); j < issued; ++j) mbar_wait(&full[j % PF_STAGES], (uint32_t)(j / PF_STAGES) & 1u, d2, f2);
        } else if (warp == 8 && nt > 0 && pf_elect()) {
            constexpr uint32_t idesc_s = fa_idesc(128, PF_KT, BF);
            constexpr uint32_t idesc_o = fa_idesc(128, D, BF) | (1u << 16);  // B's rows run along K
            bool any = false;
            const uint32_t k_lo = pf_desc_mn(smem_u32(ks)), q_lo = pf_desc_mn(smem_u32(qs)), v_lo = pf_desc_k(smem_u32(vs));
            auto issue_s = [&](int i, int j) {  // S_i = Q_i K_j^T
                const uint32_t kb = k_lo + (uint32_t)(j % PF_STAGES) * (TILE >> 4), qb = q_lo + (uint32_t)i * (TILE >> 4);
#pragma unroll
                for (int k = 0; k < D / 16; ++k) {
                    const uint32_t off = ((uint32_t)(k >> 2) * PF_HALF + (uint32_t)(k & 3) * 32) >> 4;
                    pf_mma_ss(tmem + 128u * i, qb + off, kb + off, idesc_s, k > 0 ? 1u : 0u);
                }
                umma_commit(&s_full[i]);
                any = true;
            };
            auto issue_o = [&](int i, int j, int half) {  // O_i += P_i V_j, 64 keys
                const uint32_t vb = v_lo + (uint32_t)(j % PF_STAGES) * (TILE >> 4) + half * (PF_KT / 2 * 128 >> 4);
                const uint32_t pb = tmem + 128u * i + 32u * half;
#pragma unroll
                for (int k = 0; k < PF_KT / 32; ++k)
                    pf_mma_ts(tmem + 256u + 128u * i, pb + 8u * k, vb + (2048u * k >> 4), idesc_o, (j > 0 || half > 0 || k > 0) ? 1u : 0u);
            };
            for (int i = 0; i < (two ? 2 : 1); ++i) mbar_wait(&q_full[i], 0, deadline, failed);
            mbar_wait(&k_full[0], 0, deadline, failed);
            tc_fence_after();
            if (!failed) {
                issue_s(0, 0);
                if (two) issue_s(1, 0);
                umma_commit(&k_free[0]);
            }
            for (int j = 0; j < nt && !failed; ++j) {
                const bool more = j + 1 < nt;
                mbar_wait(&v_full[j % PF_STAGES], (uint32_t)(j / PF_STAGES) & 1u, deadline, failed);
                for (int i = 0; i < (two ? 2 : 1); ++i) {
                    if (!mbar_wait(&p_full[i][0], (uint32_t)j & 1u, deadline, failed)) break;
                    tc_fence_after();
                    issue_o(i, j, 0);
                    if (!mbar_wait(&p_full[i][1], (uint32_t)j & 1u, deadline, failed)) break;
                    tc_fence_after();
                    issue_o(i, j, 1);
                    if (more) {
                        if (i == 0 && !mbar_wait(&k_full[(j + 1) % PF_STAGES], (uint32_t)((j + 1) / PF_STAGES) & 1u, deadline, failed)) break;
                        tc_fence_after();
                        issue_s(i, j + 1);
                    } else {
                        umma_commit(&o_full[i]);
                    }
                }
                if (failed) break;
                umma_commit(&v_free[j % PF_STAGES]);
                if (more) umma_commit(&k_free[(j + 1) % PF_STAGES]);
            }
            if (any) {
                // the MMAs already issued finish before TMEM is freed, also where the softmax gave up on the last ones
                umma_commit(&drain);
                bool f2 = false;
                mbar_wait(&drain, 0, globaltimer_ns() + a.timeout_ns, f2);
            }
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 208;");
        const int i = warp >> 2;  // row tile
        const int r = threadIdx.x & 127;
        const int row = pt.r0 + 128 * i + r;  // of the sequence
        const bool live = row < s.n * a.G;
        const int tok = row / a.G, g = row % a.G;
        const uint32_t trow = tmem + ((uint32_t)((warp & 3) * 32) << 16);
        if (i == 0 || two) {
            // this row of Q, 16 bytes at a time into the swizzled tile (rows past the end: zeros);
            // a negative scale goes into Q's sign, so that the largest score stays the largest
            const uint32_t flip = a.scale2 < 0.f ? 0x80008000u : 0u;
            const float c2 = fabsf(a.scale2);
            const T* src = reinterpret_cast<const T*>(a.q) + (long long)(s.row + tok) * a.q_stride + (long long)(h * a.G + g) * D;
            uint8_t* dst = qs + i * TILE;
#pragma unroll
            for (int c = 0; c < D / 8; ++c) {
                uint4 v = make_uint4(0, 0, 0, 0);
                if (live) v = *reinterpret_cast<const uint4*>(src + c * 8);
                v = make_uint4(v.x ^ flip, v.y ^ flip, v.z ^ flip, v.w ^ flip);
                *reinterpret_cast<uint4*>(dst + (c >> 3) * PF_HALF + r * 128 + (((c & 7) ^ (r & 7)) << 4)) = v;
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            mbar_arrive(&q_full[i]);

            const int my_pos = live ? s.first + tok : -1;
            const int my_lo = a.window > 0 ? my_pos - a.window + 1 : 0;
            // keys that every row of this warp sees, for tiles that need no mask
            const int hi_all = __reduce_min_sync(0xffffffffu, live ? my_pos : 0x7fffffff);
            const int lo_all = __reduce_max_sync(0xffffffffu, live ? my_lo : 0);
            float m = -INFINITY, l = 0.f;
            for (int j = 0; j < nt; ++j) {
                const int k0 = key0 + j * PF_KT;
                // which runs of 8 keys have a page
                const int c0 = k0 + 8 * (lane & 15);
                const unsigned ok = __ballot_sync(0xffffffffu, c0 < span.hi && paged_page(p, pt.b, c0) >= 0) & 0xffffu;
                mbar_wait(&s_full[i], (uint32_t)j & 1u, deadline, failed);
                failed = __any_sync(0xffffffffu, failed);
                if (failed) break;  // without an arrival: no product of a tile whose P is not there
                tc_fence_after();
                uint32_t sr[128];
#pragma unroll
                for (int q = 0; q < 4; ++q) tmem_ld32_nowait(trow + 128u * i + 32 * q, *reinterpret_cast<uint32_t(*)[32]>(sr + 32 * q));
                tmem_wait_ld();
                const bool plain = k0 + PF_KT - 1 <= hi_all && k0 >= lo_all && ok == 0xffffu;
                if (!plain) {
#pragma unroll
                    for (int c = 0; c < 128; ++c)
                        if (!(k0 + c <= my_pos && k0 + c >= my_lo && (ok >> (c >> 3) & 1))) sr[c] = 0xff800000u;  // -inf
                }
                float m4[4];
#pragma unroll
                for (int c = 0; c < 4; ++c) m4[c] = __uint_as_float(sr[c]);
#pragma unroll
                for (int c = 4; c < 124; c += 8)
#pragma unroll
                    for (int u = 0; u < 4; ++u) m4[u] = pf_max3(m4[u], __uint_as_float(sr[c + u]), __uint_as_float(sr[c + 4 + u]));
#pragma unroll
                for (int u = 0; u < 4; ++u) m4[u] = pf_max(m4[u], __uint_as_float(sr[124 + u]));
                const float mx = pf_max(pf_max3(m4[0], m4[1], m4[2]), m4[3]) * c2;
                // Also the first keys of a row (m = -inf), and a NaN or infinite score: m is then NaN (inf - inf), and with
                // it every exponential of the special-function unit and the sum. The FMA units' alone would hide a NaN.
                const bool bump = !(mx <= m + 8.f);
                const float mu = bump ? mx + (mx - mx) : m;
                const float base = mu == -INFINITY ? 0.f : mu;
                const float alpha = bump ? ex2_approx(m - base) : 1.f;
                m = mu;
                // O_i holds the tiles before j (S_i was issued after them): rescale where the maximum moved
                if (j > 0 && __any_sync(0xffffffffu, bump)) {
#pragma unroll 1
                    for (int c = 0; c < D; c += 16) {
                        uint32_t o[16];
                        pf_ld16(trow + 256u + 128u * i + c, o);
#pragma unroll
                        for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * alpha);
                        pf_st16(trow + 256u + 128u * i + c, o);
                    }
                }
                // P in two halves of 64 keys: the tensor core starts on the first while the second is made. One pair of
                // every four takes its exponentials on the FMA units, since the special-function unit alone would need
                // as long as the tensor core for the whole tile.
                const float off = pf_lift<T>() - base;
                const f32x2 c2c2 = pf_two(c2, c2), bb = pf_two(off, off);
                f32x2 s2[2] = {pf_two(0.f, 0.f), pf_two(0.f, 0.f)};
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    uint32_t pk[32];
                    if (plain) {
#pragma unroll
                        for (int c = 0; c < 64; c += 2) {
                            const f32x2 y = pf_fma2(pf_two(__uint_as_float(sr[64 * half + c]), __uint_as_float(sr[64 * half + c + 1])), c2c2, bb);
                            float2 e;
                            if ((c & 6) == 6) {
                                e = pf_exp2_fma(y);
                            } else {
                                e = pf_each(y);
                                e.x = ex2_approx(e.x);
                                e.y = ex2_approx(e.y);
                            }
                            s2[c >> 1 & 1] = pf_add2(s2[c >> 1 & 1], pf_two(e.x, e.y));
                            pk[c >> 1] = pf_pack<T>(e.x, e.y);
                        }
                    } else {
#pragma unroll
                        for (int c = 0; c < 64; c += 2) {
                            const float e0 = ex2_approx(fmaf(__uint_as_float(sr[64 * half + c]), c2, off));
                            const float e1 = ex2_approx(fmaf(__uint_as_float(sr[64 * half + c + 1]), c2, off));
                            s2[c >> 1 & 1] = pf_add2(s2[c >> 1 & 1], pf_two(e0, e1));
                            pk[c >> 1] = pf_pack<T>(e0, e1);
                        }
                    }
                    tmem_st32(trow + 128u * i + 32 * half, pk);
                    tmem_wait_st();
                    tc_fence_before();
                    mbar_arrive(&p_full[i][half]);
                }
                const float2 sum = pf_each(pf_add2(s2[0], s2[1]));
                // scores that are all -inf add nothing (the FMA units make 2^-126 of them)
                l = fmaf(l, alpha, mu == -INFINITY ? 0.f : sum.x + sum.y);
            }
            if (nt > 0) mbar_wait(&o_full[i], 0, deadline, failed);
            tc_fence_after();
            const float inv = l == 0.f ? 0.f : 1.0f / l;
            const long long orow = (long long)(s.row + tok) * a.n_heads + h * a.G + g;
            const long long prow = (long long)blockIdx.y * p.n_tokens * a.n_heads + orow;
            T* out = reinterpret_cast<T*>(a.out) + (long long)(s.row + tok) * a.out_stride + (long long)(h * a.G + g) * D;
            if (f.n_split > 1 && live) f.part_ml[prow] = failed ? make_float2(0.f, PAGED_GAVE_UP) : make_float2(m, l);
#pragma unroll 1
            for (int c = 0; c < D; c += 32) {
                uint32_t o[32];
                if (nt > 0) {
                    tmem_ld32(trow + 256u + 128u * i + c, o);
                } else {
#pragma unroll
                    for (int e = 0; e < 32; ++e) o[e] = 0;
                }
                if (!live || failed) continue;
                if (f.n_split > 1) {
#pragma unroll
                    for (int e = 0; e < 32; e += 4)
                        *reinterpret_cast<uint4*>(f.part_o + prow * D + c + e) = make_uint4(o[e], o[e + 1], o[e + 2], o[e + 3]);
                } else {
#pragma unroll
                    for (int e = 0; e < 32; e += 8) {
                        uint4 v;
                        uint32_t* w = &v.x;
#pragma unroll
                        for (int u = 0; u < 4; ++u)  // a row that saw nothing is 0, whatever O holds
                            w[u] = l == 0.f ? 0u : pf_pack<T>(__uint_as_float(o[e + 2 * u]) * inv, __uint_as_float(o[e + 2 * u + 1]) * inv);
                        *reinterpret_cast<uint4*>(out + c + e) = v;
                    }
                }
            }
        }
    }
    if (failed) atomicOr(a.status, 2);
    tc_fence_before();
    __syncthreads();
    if (warp == 8) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
    }
}

// Joins the splits of paged_fa_kernel: one warp per (token, head) of the
// sequences that kernel served.
template <typename T, int D>
__global__ void __launch_bounds__(256) paged_fa_join_kernel(const PagedKv p, const PagedAttn a, const PagedFa f) {
    constexpr int V = D / 32;
    pdl_launch_dependents();
    pdl_wait();
    const int lane = threadIdx.x & 31;
    const long long rows = (long long)p.n_tokens * a.n_heads;
    const long long orow = (long long)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5);
    if (orow >= rows) return;
    const int t = (int)(orow / a.n_heads), hd = (int)(orow % a.n_heads);
    const int b = paged_owner(p, t);
    if (b < 0 || paged_seq(p, b).n * a.G <= f.min_rows) return;
    float2 ml = make_float2(-INFINITY, 0.f);
    if (lane < f.n_split) ml = __ldcg(f.part_ml + (long long)lane * rows + orow);
    if (__any_sync(0xffffffffu, ml.y == PAGED_GAVE_UP)) return;
    const float m = warp_max(ml.x);
    const float w_mine = ml.y != 0.f ? exp2f(ml.x - m) : 0.f;  // NaN stays
    const float l = warp_sum(ml.y * w_mine);
    float o[V] = {};
    for (int i = 0; i < f.n_split; ++i) {
        const float w = __shfl_sync(0xffffffffu, w_mine, i);
        if (w != 0.f) {
            const PackV<float, V> x = *reinterpret_cast<const PackV<float, V>*>(f.part_o + ((long long)i * rows + orow) * D + lane * V);
#pragma unroll
            for (int e = 0; e < V; ++e) o[e] = fmaf(x.e[e], w, o[e]);
        }
    }
    const float inv = l == 0.f ? 0.f : 1.0f / l;
    PackV<T, V> y;
#pragma unroll
    for (int e = 0; e < V; ++e) y.e[e] = from_f<T>(o[e] * inv);
    *reinterpret_cast<PackV<T, V>*>(reinterpret_cast<T*>(a.out) + (long long)t * a.out_stride + (long long)hd * D + lane * V) = y;
}

}  // namespace mf
