// One id per row of logits: top-k, top-p, min-p, temperature and a draw, each
// row with its own parameters and its own random number.
//
// The filters are those of the reference's Sampler (src/base/sampler.cpp:
// 40-117) in its order, over the candidates sorted by value (equal values:
// the lower index first; NaN counts as -inf): the top_k first; of those the
// shortest prefix whose softmax mass reaches top_p; of those the ones at least
// min_p as likely as the first; then the first whose cumulative softmax(x / T)
// reaches the draw. Every filter keeps a prefix of that order, so a row is
// never sorted: each stage looks for one border, the first candidate at which
// a running sum (of ones, of exp(x - top), of exp((x - top) / T)) reaches a
// target.
//
// A row lives in the shared memory of one thread-block cluster: the logits are
// read from memory once, and every later pass runs on chip.
//   top_k: the threads' maxima bound the k-th candidate; what is above goes to
//   the row's first block, which finds every border among it (sb_pick).
//   Otherwise: one pass adds up the exact weights and, coarsely, 512 bins of
//   1/16 below the top, which tell the border's bin; another adds up exactly
//   what lies before that bin and sends the bin to the first block.
//   Where a bin holds too many candidates, or the coarse sums named the wrong
//   one (the exact sums tell): by descent over the cluster (sb_find), the bin
//   that holds the border cut into 512 ranges of keys, and so on, until a few
//   candidates are left, or one value, whose ties are counted out by index.
//
// Sums: weights are exp() in 64 bits, rounded to multiples of 2^-45 and added
// as whole numbers, so a sum does not depend on the order of its terms and is
// off by at most 2^-46 per term. In floats a vocabulary of 10^5 would move the
// border of every hundredth draw.
//
// Measured, 151936 fp32 logits, times per call: one row 16 us with top_k 50, 48
// with top_p 0.9 alone; 64 rows 47 and 129 us (the floor, one read, is 6; the
// maximum alone takes 18, of one row 7.5). Bound by latencies (an exchange over the cluster is about a
// microsecond, and there are five to nine) and, without top_k, by shared-memory
// atomics and 64-bit arithmetic. Exact bins took three atomics per logit more
// (147 us for a mixed batch of 64 rows, now 79), a bitonic sort of the
// candidates 14 us more per border.
#pragma once

#include "mf_common.cuh"
#include "paged.cuh"

namespace mf {

constexpr int SB_THREADS = 512;
constexpr int SB_BINS = 512;        // one per thread
constexpr int SB_LIST = 64;         // candidates left to one warp (two per lane)
constexpr int SB_FEW = 2048;        // candidates that one block orders: four per thread
constexpr int SB_MAX_CLUSTER = 8;
constexpr int SB_MAX_VOCAB = 1 << 18;  // 2^18 weights of at most 2^45: sums of at most 2^63, unsigned
constexpr double SB_ONE = 35184372088832.0;  // 2^45

struct SampleBatch {
    const void* logits;  // [rows][ld]
    long long ld;
    const float* draws;
    const float* temp;
    const int* top_k;
    const float* top_p;
    const float* min_p;
    int* ids;
    float* probs;  // or null
    int vocab, slice;  // slice: logits per block, cluster rank r holds [r * slice, (r + 1) * slice)
};

typedef unsigned long long u64;

// Logits as they are compared: NaN is -inf, -0 is 0.
MF_DEVICE float sb_clean(float x) { return x != x ? -INFINITY : x + 0.0f; }
// Order-preserving whole number of a clean value, and back.
MF_DEVICE uint32_t sb_key(float x) {
    const uint32_t u = __float_as_uint(x);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}
MF_DEVICE float sb_value(uint32_t key) { return __uint_as_float(key & 0x80000000u ? key & 0x7fffffffu : ~key); }

// Level-1 bin of a value, sixteenths below the top: never decreases as x falls.
// (Rounded by the sum with 2^23, whose low bits are the whole number: a
// conversion costs four times as much.)
MF_DEVICE int sb_bin(float top, float x) {
    const float d = x == top ? 0.f : fminf(top - x, 31.95f);  // top may be infinite
    return __float_as_int(fmaf(d, 16.f, 8388608.f)) - 0x4b000000;
}

MF_DEVICE uint32_t sb_remote(const void* local, int rank) {
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"((uint32_t)__cvta_generic_to_shared(local)), "r"(rank));
    return r;
}
MF_DEVICE uint32_t sb_ld32(const uint32_t* local, int rank) {
    uint32_t v;
    asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(sb_remote(local, rank)) : "memory");
    return v;
}
MF_DEVICE u64 sb_ld64(const u64* local, int rank) {
    u64 v;
    asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(v) : "r"(sb_remote(local, rank)) : "memory");
    return v;
}

// Sum and maximum of a word over the blocks of the cluster. All loads are
// issued before the first is used: one after the other costs a remote latency each.
template <typename T> MF_DEVICE T sb_ld(const T* local, int rank) {
    if constexpr (sizeof(T) == 8) return sb_ld64(local, rank);
    else return sb_ld32(local, rank);
}
template <typename T> MF_DEVICE void sb_ld_all(const T* local, int size, T (&v)[SB_MAX_CLUSTER]) {
#pragma unroll
    for (int q = 0; q < SB_MAX_CLUSTER; ++q) v[q] = q < size ? sb_ld(local, q) : 0;
}
template <typename T> MF_DEVICE T sb_sum_all(const T* local, int size) {
    T v[SB_MAX_CLUSTER], s = 0;
    sb_ld_all(local, size, v);
#pragma unroll
    for (int q = 0; q < SB_MAX_CLUSTER; ++q) s += v[q];
    return s;
}

// The last kept candidate of a prefix of the order.
struct SbBorder {
    uint32_t key, idx;
    MF_DEVICE bool keeps(uint32_t k, uint32_t i) const { return k > key || (k == key && i <= idx); }
    MF_DEVICE bool before(const SbBorder& o) const { return key > o.key || (key == o.key && idx < o.idx); }
};

struct SbShared {
    uint32_t cnt[SB_BINS];
    uint32_t part[3][SB_BINS];  // weights in three parts of 16 bits: 32-bit shared atomics, no overflow below 2^16 terms
    union {
        u64 wsum[SB_BINS];                   // their sum, what the other blocks read
        float queue[SB_THREADS / 32][64];    // sb_scan_slice
    };
    double table[256];          // 2^(-i / 256)
    u64 cand[SB_FEW];          // (key, ~index) of the block's candidates
    u64 best;                   // (key, ~index) of the block's largest
    u64 scan[34];
    u64 found[4];
    uint32_t list_n;
    uint32_t list_key[SB_LIST], list_idx[SB_LIST];
    uint32_t ties;
    uint32_t first;             // smallest position asked for
    u64 sum[2];                 // the block's share of two sums, read by the others
    u64 told[4];                // what the row's first block found
};

struct SbRow {
    const float* vals;  // this block's slice
    int n, base;           // its length and first index
    int rank, size;        // of the cluster
    float top;
    SbShared* sh;
};

enum SbMode { SB_COUNT, SB_WEIGHT };

// exp((x - top) / T) in multiples of 2^-45, rounded to nearest. With z = top -
// x and n = rint(256 z / (T ln 2)): exp(-z/T) = 2^-(n >> 8) * 2^-(n & 255)/256 *
// e^t, t = n ln2/256 - z/T, |t| < 1.4e-3, where the series up to t^4/24 leaves
// 4e-17 (a table and a short polynomial, Tang 1989). About half the 64-bit
// operations of exp(); rows that keep most of the vocabulary spend their time here.
struct SbTemp {
    double inv_t, inv_step;  // 1 / T, 256 / (T ln 2)
    float inv_f;
};
MF_DEVICE SbTemp sb_temp(double t) {
    SbTemp s;
    s.inv_t = 1.0 / t;
    s.inv_step = 369.3299304675746 * s.inv_t;  // 256 / ln 2
    s.inv_f = (float)s.inv_t;
    return s;
}
MF_DEVICE u64 sb_weight(float x, float top, const SbTemp& s, const double* table) {
    if (x == top) return (u64)SB_ONE;
    if (!((top - x) * s.inv_f < 32.25f)) return 0;  // below half of 2^-45 (with room for the float's error)
    const double z = (double)top - (double)x, e = z * s.inv_t;
    const double magic = 6755399441055744.0;  // 1.5 * 2^52: the low bits of the sum are a whole number
    const double kk = fma(z, s.inv_step, magic);
    const int n = __double2loint(kk);
    const double t = fma(kk - magic, 0.0027076061740622863, -e);  // ln 2 / 256
    double p = fma(t, 1.0 / 24, 1.0 / 6);
    p = fma(t, p, 0.5);
    p = fma(t, p, 1.0);
    p = fma(t, p, 1.0);
    const double v = p * table[n & 255];  // in [0.49, 1.01)
    const double w = __hiloint2double(__double2hiint(v) + (45 - (n >> 8)) * 1048576, __double2loint(v));
    return (u64)__double_as_longlong(w + 4503599627370496.0) & 0xfffffffffffffull;  // + 2^52
}

// Block-wide inclusive scan of one u64 per thread.
MF_DEVICE u64 sb_scan(u64 v, SbShared* sh, u64& total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const u64 u = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v += u;
    }
    __syncthreads();
    if (lane == 31) sh->scan[warp] = v;
    __syncthreads();
    u64 base = 0;
    total = 0;
    for (int w = 0; w < SB_THREADS / 32; ++w) {
        const u64 s = sh->scan[w];
        if (w < warp) base += s;
        total += s;
    }
    return v + base;
}

// Smallest key of level-1 bin `bin` or below it in the order (monotone search).
MF_DEVICE uint32_t sb_bin_low(float top, int bin) {
    uint32_t lo = sb_key(-INFINITY), hi = sb_key(top);  // bin(hi) = 0 <= bin
    while (lo < hi) {
        const uint32_t mid = lo + ((hi - lo) >> 1);
        if (sb_bin(top, sb_value(mid)) <= bin) hi = mid;
        else lo = mid + 1;
    }
    return lo;
}

// The block's bins at zero (in step before the first use).
MF_DEVICE void sb_clear(SbShared* sh) {
    const int tid = threadIdx.x;
    sh->cnt[tid] = 0;
    sh->part[0][tid] = sh->part[1][tid] = 0;
    if (tid == 0) sh->first = ~0u;
}

// The first thread with `hit` (SB_THREADS if none has); sh->first must be ~0 and in step. One call per use.
MF_DEVICE int sb_first_thread(bool hit, SbShared* sh) {
    const unsigned hits = __ballot_sync(0xffffffffu, hit);
    if ((threadIdx.x & 31) == 0 && hits) atomicMin(&sh->first, threadIdx.x + __ffs(hits) - 1);
    __syncthreads();
    return min(sh->first, (uint32_t)SB_THREADS);
}

// A bin that ends at or behind the want-th candidate. For few it is the bin of
// the want-th largest of the threads' maxima, since as many candidates are at
// least that large: one atomic per thread instead of one per logit, and up to a
// quarter of the threads (1000 of 4096) hardly more than `want` candidates lie
// above its end. For more it is the bin of the want-th candidate itself (89 rows
// of 7430 logits, top_k 1000 among them: 55 us by the maxima of 1024 threads,
// which let nearly all logits through, 34 so).
MF_DEVICE int sb_top_bin(const SbRow& r, bool has, float thread_max, uint32_t want) {
    SbShared* sh = r.sh;
    const int tid = threadIdx.x;
    if (want <= (uint32_t)(r.size * SB_THREADS / 4)) {
        if (has) atomicAdd(&sh->cnt[sb_bin(r.top, thread_max)], 1u);
    } else {
#pragma unroll 4
        for (int i = tid; i < r.n; i += SB_THREADS) atomicAdd(&sh->cnt[sb_bin(r.top, r.vals[i])], 1u);
    }
    cluster_sync_all();
    const uint32_t c = sb_sum_all(&sh->cnt[tid], r.size);
    u64 total;
    const u64 inc = sb_scan(c, sh, total);
    const int bin = sb_first_thread(inc >= want, sh);
    cluster_sync_all();  // every block has read these bins
    return min(bin, SB_BINS - 1);
}

// Relative weight of a value within its bin, exp(-(z - (bin - 1/2)/16) / T), in 16
// bits: sums of these tell (nearly always) in which bin an exact running sum
// reaches its target, at one 32-bit atomic each instead of three exact ones.
MF_DEVICE uint32_t sb_coarse(float top, float x, int bin, float c) {
    const float d = x == top ? 0.f : top - x;
    float e;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(fminf(fmaf(-d, 16.f, (float)bin - 0.5f), 0.f) * c));
    return (uint32_t)__float_as_int(fmaf(e, 65535.f, 8388608.f)) & 0x7fffffu;  // as in sb_bin
}
// The coarse weight of this thread's bin over the whole row, in multiples of
// 2^-45 of the top's, from the blocks' sums in part[which].
MF_DEVICE u64 sb_coarse_bin(const SbRow& r, int which, float c) {
    uint32_t v[SB_MAX_CLUSTER];
    sb_ld_all(&r.sh->part[which][threadIdx.x], r.size, v);
    u64 w = 0;
#pragma unroll
    for (int q = 0; q < SB_MAX_CLUSTER; ++q) w += v[q];
    return (u64)((double)w * exp2(-((double)threadIdx.x - 0.5) * c) * (SB_ONE / 65535.0));
}

// Notes a candidate for sb_fetch (sh->list_n counts on past the end).
MF_DEVICE void sb_note(SbShared* sh, uint32_t key, uint32_t idx) {
    const uint32_t at = atomicAdd(&sh->list_n, 1u);
    if (at < SB_FEW) sh->cand[at] = (u64)key << 32 | (uint32_t)~idx;
}

// Walks the block's slice: `note` gets every value between lo and hi (both
// included) with its index, `add` every value above hi, a full warp of them at
// a time: few of many are above, and `add` is dear. Four values per load.
template <typename Note, typename Add> MF_DEVICE void sb_scan_slice(const SbRow& r, float lo, float hi, Note note, Add add) {
    const int lane = threadIdx.x & 31;
    float* queue = r.sh->queue[threadIdx.x >> 5];
    int n = 0;
    auto drain = [&] {  // the last 32
        __syncwarp();
        const int k = min(n, 32);
        if (lane < k) add(queue[n - k + lane]);
        n -= k;
        __syncwarp();
    };
    const int n4 = r.n / 4;
    for (int i0 = threadIdx.x & ~31; i0 < n4; i0 += SB_THREADS) {
        const int i = i0 + lane;
        const float4 v = i < n4 ? *reinterpret_cast<const float4*>(r.vals + 4 * i) : make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
        const bool in = i < n4;
        if (!__any_sync(0xffffffffu, in && fmaxf(fmaxf(v.x, v.y), fmaxf(v.z, v.w)) >= lo)) continue;
        const float x[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const bool above = in && x[e] > hi;
            const unsigned who = __ballot_sync(0xffffffffu, above);
            if (above) queue[n + __popc(who & ((1u << lane) - 1))] = x[e];
            n += __popc(who);
            if (in && !above && x[e] >= lo) note(x[e], r.base + 4 * i + e);
            if (n >= 32) drain();
        }
    }
    // the last values of a slice that is no multiple of four
    {
        const int i = 4 * n4 + (int)threadIdx.x;
        const bool in = i < r.n;
        const float x = in ? r.vals[i] : 0.f;
        const bool above = in && x > hi;
        const unsigned who = __ballot_sync(0xffffffffu, above);
        if (above) queue[n + __popc(who & ((1u << lane) - 1))] = x;
        n += __popc(who);
        if (in && !above && x >= lo) note(x, r.base + i);
    }
    while (n > 0) drain();
}

// Number of noted candidates of each block and of all. The blocks are in step before.
MF_DEVICE uint32_t sb_noted(const SbRow& r, uint32_t (&nq)[SB_MAX_CLUSTER]) {
    sb_ld_all(&r.sh->list_n, r.size, nq);
    uint32_t n = 0;
#pragma unroll
    for (int q = 0; q < SB_MAX_CLUSTER; ++q) n += nq[q];  // at most 2^18
    return n;
}

// Row's first block: the n <= SB_FEW noted candidates of all blocks, four per
// thread (0: none). The blocks may leave after the next cluster barrier.
constexpr int SB_E = SB_FEW / SB_THREADS;
MF_DEVICE void sb_fetch(const SbRow& r, const uint32_t (&nq)[SB_MAX_CLUSTER], uint32_t n, u64 (&v)[SB_E]) {
    SbShared* sh = r.sh;
#pragma unroll
    for (int e = 0; e < SB_E; ++e) {
        uint32_t i = threadIdx.x + e * SB_THREADS;  // candidate i of all: i - (those of the blocks before) of block q
        const bool in = i < n;
        int q = 0;
#pragma unroll
        for (; q < SB_MAX_CLUSTER - 1; ++q) {
            if (i < nq[q]) break;
            i -= nq[q];
        }
        v[e] = in ? sb_ld64(&sh->cand[i], q) : 0;
    }
}

// sb_find among the fetched candidates of at least `cut`, by one block: the
// first at which before + (running sum) reaches the target, `want` ones or
// share * total (total 0: before + the sum over them, and set to that).
// Candidates are distinct words (key, ~index), so the descent needs no rule
// for ties. `right`: the border lies among them; the result counts only then.
template <int MODE>
MF_DEVICE u64 sb_pick(const SbRow& r, const u64 (&v)[SB_E], u64 cut, const SbTemp& t, u64 before, u64 want, double share,
                      u64& total, bool& right) {
    SbShared* sh = r.sh;
    const int tid = threadIdx.x, lane = tid & 31;
    u64 w[SB_E], lo = ~0ull, hi = 0;
#pragma unroll
    for (int e = 0; e < SB_E; ++e) {
        const bool in = v[e] >= cut && v[e] != 0;
        w[e] = !in ? 0 : MODE == SB_COUNT ? 1 : sb_weight(sb_value((uint32_t)(v[e] >> 32)), r.top, t, sh->table);
        if (in) {
            lo = min(lo, v[e]);
            hi = max(hi, v[e]);
        }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        lo = min(lo, __shfl_xor_sync(0xffffffffu, lo, o));
        hi = max(hi, __shfl_xor_sync(0xffffffffu, hi, o));
    }
    __syncthreads();
    if (tid == 0) {
        sh->found[0] = ~0ull;
        sh->found[1] = 0;
    }
    __syncthreads();
    if (lane == 0) {
        atomicMin(&sh->found[0], lo);
        atomicMax(&sh->found[1], hi);
    }
    __syncthreads();
    lo = sh->found[0];
    hi = sh->found[1];
    right = lo <= hi;
    if (!right) return 0;
    double target = (double)want;
    for (int level = 0;; ++level) {
        const int shift = max(64 - __clzll(hi - lo) - 9, 0);
        sh->cnt[tid] = 0;
        if (MODE == SB_WEIGHT) sh->part[0][tid] = sh->part[1][tid] = sh->part[2][tid] = 0;
        if (tid == 0) {
            sh->first = ~0u;
            sh->list_n = 0;
        }
        __syncthreads();
#pragma unroll
        for (int e = 0; e < SB_E; ++e) {
            if (v[e] < lo || v[e] > hi || v[e] < cut || v[e] == 0) continue;
            const int bin = (int)((hi - v[e]) >> shift);
            atomicAdd(&sh->cnt[bin], 1u);
            if (MODE == SB_WEIGHT && w[e]) {
                atomicAdd(&sh->part[0][bin], (uint32_t)(w[e] & 0xffff));
                atomicAdd(&sh->part[1][bin], (uint32_t)((w[e] >> 16) & 0xffff));
                atomicAdd(&sh->part[2][bin], (uint32_t)(w[e] >> 32));
            }
        }
        __syncthreads();
        const uint32_t c = sh->cnt[tid];
        const u64 mine = MODE == SB_COUNT ? c : (u64)sh->part[0][tid] + ((u64)sh->part[1][tid] << 16) + ((u64)sh->part[2][tid] << 32);
        u64 all;
        const u64 inc = sb_scan(mine, sh, all);
        if (level == 0) {
            if (MODE == SB_WEIGHT) {
                if (total == 0) total = before + all;
                target = share * (double)total;
            }
            right = (before == 0 || (double)before < target) && (double)(before + all) >= target;
            if (!right) return 0;
        }
        const int bin = sb_first_thread(c > 0 && (double)(before + inc) >= target, sh);
        if (tid == bin) {
            sh->found[1] = before + inc - mine;
            sh->found[2] = c;
        }
        __syncthreads();
        before = sh->found[1];
        const uint32_t left = (uint32_t)sh->found[2];
        hi -= (u64)bin << shift;
        const u64 width = (1ull << shift) - 1;
        if (hi - lo > width) lo = hi - width;
        if (left <= 32) {
            // one warp orders them: the largest at which the sum over those not below it reaches the target
#pragma unroll
            for (int e = 0; e < SB_E; ++e)
                if (v[e] >= lo && v[e] <= hi && v[e] >= cut && v[e] != 0) {
                    const uint32_t at = atomicAdd(&sh->list_n, 1u);
                    sh->cand[at] = v[e];
                    sh->wsum[at] = w[e];
                }
            __syncthreads();
            if (tid < 32) {
                const u64 x = lane < left ? sh->cand[lane] : 0, y = lane < left ? sh->wsum[lane] : 0;
                u64 run = before;
                for (uint32_t o = 0; o < left; ++o) {
                    const u64 ox = __shfl_sync(0xffffffffu, x, o), oy = __shfl_sync(0xffffffffu, y, o);
                    if (ox >= x) run += oy;
                }
                u64 best = lane < left && (double)run >= target ? x : 0;
#pragma unroll
                for (int o = 16; o > 0; o >>= 1) best = max(best, __shfl_xor_sync(0xffffffffu, best, o));
                if (lane == 0) sh->found[3] = best;
            }
            __syncthreads();
            return sh->found[3];
        }
        __syncthreads();
    }
}

// First candidate of the prefix `in` at which the running sum reaches the
// target: target = want (SB_COUNT: want ones; share < 0), or share * (sum over
// the prefix) for weights. Sets `sum` to the whole sum. Every block of the
// cluster calls it and gets the same answer. If rounding leaves the target
// above the sum the last candidate with weight is taken.
template <int MODE>
MF_DEVICE SbBorder sb_find(const SbRow& r, const SbBorder& in, const SbTemp& t, u64 want, double share, u64& sum) {
    SbShared* sh = r.sh;
    const int tid = threadIdx.x, lane = tid & 31;
    uint32_t lo = sb_key(-INFINITY), hi = sb_key(r.top);
    u64 before = 0;
    double target = (double)want;
    for (int level = 0;; ++level) {
        // level 0: bins by value below the top; then 512 ranges of the keys in [lo, hi], largest first
        int shift = 0;
        if (level > 0) {
            const int bits = 32 - __clz(hi - lo);
            shift = max(bits - 9, 0);
        }
        sh->cnt[tid] = 0;
        if (MODE == SB_WEIGHT) sh->part[0][tid] = sh->part[1][tid] = sh->part[2][tid] = 0;
        __syncthreads();
        for (int i = tid; i < r.n; i += SB_THREADS) {
            const float x = r.vals[i];
            const uint32_t k = sb_key(x);
            if (k < lo || k > hi || !in.keeps(k, r.base + i)) continue;
            const int bin = level == 0 ? sb_bin(r.top, x) : (int)((hi - k) >> shift);
            atomicAdd(&sh->cnt[bin], 1u);
            if (MODE == SB_WEIGHT) {
                const u64 w = sb_weight(x, r.top, t, sh->table);
                if (w) {
                    atomicAdd(&sh->part[0][bin], (uint32_t)(w & 0xffff));
                    atomicAdd(&sh->part[1][bin], (uint32_t)((w >> 16) & 0xffff));
                    atomicAdd(&sh->part[2][bin], (uint32_t)(w >> 32));
                }
            }
        }
        __syncthreads();
        if (MODE == SB_WEIGHT)
            sh->wsum[tid] = (u64)sh->part[0][tid] + ((u64)sh->part[1][tid] << 16) + ((u64)sh->part[2][tid] << 32);
        cluster_sync_all();
        const uint32_t c = sb_sum_all(&sh->cnt[tid], r.size);
        const u64 w = MODE == SB_WEIGHT ? sb_sum_all(&sh->wsum[tid], r.size) : c;
        u64 total;
        const u64 inc = sb_scan(w, sh, total);
        cluster_sync_all();  // every block has read these bins
        if (level == 0) {
            sum = total;
            if (share >= 0.0) target = share * (double)total;
        }
        // the first bin with candidates whose running sum reaches the target, else the last one with any sum
        if (tid == 0) sh->found[0] = ~0ull;
        __syncthreads();
        const bool hit = c > 0 && (double)(before + inc) >= target;
        u64 key = hit ? (u64)tid : ~0ull;
        for (int o = 16; o > 0; o >>= 1) key = min(key, __shfl_xor_sync(0xffffffffu, key, o));
        if (lane == 0 && key != ~0ull) atomicMin(&sh->found[0], key);
        __syncthreads();
        if (sh->found[0] == ~0ull) {
            __syncthreads();
            if (tid == 0) sh->found[0] = 0;
            __syncthreads();
            if (w > 0) atomicMax(&sh->found[0], (u64)tid);
            __syncthreads();
        }
        const int bin = (int)sh->found[0];
        if (tid == bin) {
            sh->found[1] = before + inc - w;
            sh->found[2] = c;
        }
        __syncthreads();
        before = sh->found[1];
        const uint32_t left = (uint32_t)sh->found[2];
        if (level == 0) {
            const uint32_t l2 = sb_bin_low(r.top, bin);
            if (bin > 0) hi = sb_bin_low(r.top, bin - 1) - 1;
            lo = l2;
        } else {
            hi = hi - ((uint32_t)bin << shift);
            const u64 width = (1ull << shift) - 1;
            lo = hi - lo > width ? hi - (uint32_t)width : lo;
        }
        __syncthreads();
        if (left <= SB_LIST || lo == hi) {
            SbBorder out;
            if (left <= SB_LIST) {
                // few: every block collects its own, warp 0 of each orders all of them
                if (tid == 0) sh->list_n = 0;
                __syncthreads();
                for (int i = tid; i < r.n; i += SB_THREADS) {
                    const uint32_t k = sb_key(r.vals[i]);
                    if (k < lo || k > hi || !in.keeps(k, r.base + i)) continue;
                    const uint32_t at = atomicAdd(&sh->list_n, 1u);
                    sh->list_key[at] = k;
                    sh->list_idx[at] = r.base + i;
                }
                cluster_sync_all();
                if (tid < 32) {
                    uint32_t k[2] = {0, 0}, ix[2] = {~0u, ~0u};
                    bool has[2] = {false, false};
                    uint32_t off = 0;
                    for (int q = 0; q < r.size; ++q) {
                        const uint32_t nq = sb_ld32(&sh->list_n, q);
                        for (int s = 0; s < 2; ++s) {
                            const uint32_t at = lane + 32 * s;
                            if (at >= off && at < off + nq) {
                                k[s] = sb_ld32(&sh->list_key[at - off], q);
                                ix[s] = sb_ld32(&sh->list_idx[at - off], q);
                                has[s] = true;
                            }
                        }
                        off += nq;
                    }
                    u64 w2[2], run[2] = {0, 0};
                    uint32_t rank[2] = {0, 0};
                    for (int s = 0; s < 2; ++s)
                        w2[s] = !has[s] ? 0 : MODE == SB_COUNT ? 1 : sb_weight(sb_value(k[s]), r.top, t, sh->table);
                    for (int o = 0; o < 64; ++o) {  // rank and running sum by comparison with every candidate
                        const int src = o & 31, z = o >> 5;
                        const uint32_t ok = __shfl_sync(0xffffffffu, k[z], src), oi = __shfl_sync(0xffffffffu, ix[z], src);
                        const u64 ow = __shfl_sync(0xffffffffu, w2[z], src);
                        const bool oh = __shfl_sync(0xffffffffu, (int)has[z], src);
                        for (int s = 0; s < 2; ++s)
                            if (oh && (ok > k[s] || (ok == k[s] && oi <= ix[s]))) {
                                run[s] += ow;
                                ++rank[s];
                            }
                    }
                    // the first that reaches the target; if none does, the last with weight
                    uint32_t best = ~0u, last = 0;
                    for (int s = 0; s < 2; ++s)
                        if (has[s]) {
                            if ((double)(before + run[s]) >= target) best = min(best, rank[s]);
                            if (w2[s] > 0) last = max(last, rank[s]);
                        }
                    best = __reduce_min_sync(0xffffffffu, best);
                    last = __reduce_max_sync(0xffffffffu, last);
                    const uint32_t pick = best != ~0u ? best : max(last, 1u);
                    for (int s = 0; s < 2; ++s)
                        if (has[s] && rank[s] == pick) sh->found[3] = (u64)k[s] << 32 | ix[s];
                }
                __syncthreads();
                out.key = (uint32_t)(sh->found[3] >> 32);
                out.idx = (uint32_t)sh->found[3];
            } else {
                const float one = sb_value(lo);
                // one value: its ties in the order of their indices. Number `need` (from 1) is the border.
                const u64 w1 = MODE == SB_COUNT ? 1 : sb_weight(sb_value(lo), r.top, t, sh->table);
                u64 need = left;
                if (w1 > 0) {
                    u64 a = 1, z = left;  // smallest a with before + a * w1 >= target
                    while (a < z) {
                        const u64 mid = (a + z) >> 1;
                        if ((double)(before + mid * w1) >= target) z = mid;
                        else a = mid + 1;
                    }
                    need = a;
                } else if ((double)before >= target) {
                    need = 1;
                }
                const int seg = ((r.n + SB_THREADS - 1) / SB_THREADS) | 1;  // odd: a warp's runs start in different banks
                const int i0 = min(tid * seg, r.n), i1 = min(i0 + seg, r.n);
                uint32_t mine = 0;
                for (int i = i0; i < i1; ++i) mine += r.vals[i] == one && in.keeps(lo, r.base + i);
                u64 all;
                const u64 upto = sb_scan(mine, sh, all);
                if (tid == 0) sh->ties = (uint32_t)all;
                cluster_sync_all();
                u64 ahead = 0;
                for (int q = 0; q < r.rank; ++q) ahead += sb_ld32(&sh->ties, q);
                if (tid == 0) sh->found[3] = ~0ull;
                __syncthreads();
                const u64 mine0 = ahead + upto - mine;
                if (need > mine0 && need <= mine0 + mine) {
                    u64 left_n = need - mine0;
                    for (int i = i0; i < i1; ++i)
                        if (r.vals[i] == one && in.keeps(lo, r.base + i) && --left_n == 0) sh->found[3] = r.base + i;
                }
                cluster_sync_all();
                out.key = lo;
                out.idx = ~0u;
                for (int q = 0; q < r.size; ++q) {
                    const u64 f = sb_ld64(&sh->found[3], q);
                    if (f != ~0ull) out.idx = (uint32_t)f;
                }
            }
            cluster_sync_all();  // the lists may be written again
            return out;
        }
    }
}

template <typename T>
__global__ void __launch_bounds__(SB_THREADS, 2) sample_batch_kernel(const SampleBatch a) {
    extern __shared__ __align__(16) float sb_vals[];
    __shared__ SbShared sh;
    pdl_launch_dependents();
    pdl_wait();
    uint32_t size;
    asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(size));
    const int tid = threadIdx.x, lane = tid & 31;
    const int row = blockIdx.x / size;
    SbRow r;
    r.rank = cluster_rank();
    r.size = size;
    r.base = r.rank * a.slice;
    r.n = max(min(a.slice, a.vocab - r.base), 0);
    r.vals = sb_vals;
    r.sh = &sh;

    // the slice, and the largest with the lowest index
    const T* x = reinterpret_cast<const T*>(a.logits) + row * a.ld + r.base;
    float thread_max = -INFINITY;
    int at = -1;
    constexpr int V = 16 / sizeof(T);
    const bool vec = (reinterpret_cast<uintptr_t>(x) & 15) == 0;
    const int nv = vec ? r.n / V : 0;
    for (int i = tid; i < nv; i += SB_THREADS) {
        const PackV<T, V> v = *reinterpret_cast<const PackV<T, V>*>(x + (long long)i * V);
#pragma unroll
        for (int e = 0; e < V; ++e) {
            const float c = sb_clean(to_f<T>(v.e[e]));
            sb_vals[i * V + e] = c;
            if (c > thread_max || at < 0) {
                thread_max = c;
                at = i * V + e;
            }
        }
    }
    for (int i = nv * V + tid; i < r.n; i += SB_THREADS) {
        const float c = sb_clean(to_f<T>(x[i]));
        sb_vals[i] = c;
        if (c > thread_max || at < 0) {
            thread_max = c;
            at = i;
        }
    }
    u64 best = at < 0 ? 0 : (u64)sb_key(thread_max) << 32 | (uint32_t)~(r.base + at);  // this thread saw its indices in order
    for (int o = 16; o > 0; o >>= 1) best = max(best, __shfl_xor_sync(0xffffffffu, best, o));
    if (tid == 0) sh.best = sh.list_n = 0;
    if (tid < 256) sh.table[tid] = exp2(-tid / 256.0);
    sb_clear(&sh);
    __syncthreads();
    if (lane == 0) atomicMax(&sh.best, best);
    cluster_sync_all();
    u64 bests[SB_MAX_CLUSTER];
    sb_ld_all(&sh.best, r.size, bests);
    best = 0;
#pragma unroll
    for (int q = 0; q < SB_MAX_CLUSTER; ++q) best = max(best, bests[q]);
    cluster_sync_all();
    const uint32_t top_key = (uint32_t)(best >> 32);
    r.top = sb_value(top_key);
    SbBorder pick;
    pick.key = top_key;
    pick.idx = ~(uint32_t)best;

    const float temp = a.temp[row], top_p = a.top_p[row], min_p = a.min_p[row];
    const int top_k = a.top_k[row];
    const bool none = top_key == sb_key(-INFINITY);  // nothing to choose from
    double prob = 1.0, inv_t = 1.0;
    u64 sum = 0;
    if (!none && temp > 0.f) {
        const SbBorder all = {0u, ~0u};
        const bool cut_k = top_k > 0 && top_k < a.vocab, cut_p = top_p < 1.f;
        const double share_p = (double)fmaxf(top_p, 0.f), draw = (double)fminf(fmaxf(a.draws[row], 0.f), 0.99999994f);
        const SbTemp t1 = sb_temp(1.0), t2 = sb_temp((double)temp);
        inv_t = t2.inv_t;
        uint32_t low = 0;  // the smallest key at least min_p as likely as the first: x >= top + log(min_p)
        if (min_p > 0.f) {
            const double thr = min_p < 1.f ? (double)r.top + log((double)min_p) : (double)r.top;
            low = sb_key(__double2float_ru(thr));  // the smallest float that is not below thr
        }
        bool done = false, right;
        SbBorder kept = all;
        if (cut_k) {
            // few, as a rule: the candidates down to a bin that holds the last go through the filters in order
            const int bin = sb_top_bin(r, at >= 0, thread_max, (uint32_t)top_k);
            // (with a value for the bin's end, rounded down: one candidate more does no harm)
            const float end = bin < SB_BINS - 1 ? __fsub_rd(r.top, ((float)bin + 0.51f) / 16.f) : -INFINITY;
            const int n4 = r.n / 4;
            for (int i = tid; i < n4; i += SB_THREADS) {
                const float4 x = *reinterpret_cast<const float4*>(sb_vals + 4 * i);
                if (fmaxf(fmaxf(x.x, x.y), fmaxf(x.z, x.w)) >= end) {
                    if (x.x >= end) sb_note(&sh, sb_key(x.x), r.base + 4 * i);
                    if (x.y >= end) sb_note(&sh, sb_key(x.y), r.base + 4 * i + 1);
                    if (x.z >= end) sb_note(&sh, sb_key(x.z), r.base + 4 * i + 2);
                    if (x.w >= end) sb_note(&sh, sb_key(x.w), r.base + 4 * i + 3);
                }
            }
            for (int i = 4 * n4 + tid; i < r.n; i += SB_THREADS)
                if (sb_vals[i] >= end) sb_note(&sh, sb_key(sb_vals[i]), r.base + i);
            cluster_sync_all();
            uint32_t nq[SB_MAX_CLUSTER];
            const uint32_t n = sb_noted(r, nq);
            u64 v4[SB_E];
            if (r.rank == 0 && n <= SB_FEW) sb_fetch(r, nq, n, v4);
            cluster_sync_all();
            if (n <= SB_FEW) {
                if (r.rank != 0) return;
                u64 part = 0, cut = sb_pick<SB_COUNT>(r, v4, 0, t1, 0, (u64)top_k, -1.0, part, right);
                part = 0;
                if (cut_p) cut = sb_pick<SB_WEIGHT>(r, v4, cut, t1, 0, 0, share_p, part, right);
                if (low) cut = max(cut, (u64)low << 32);
                const u64 got = sb_pick<SB_WEIGHT>(r, v4, cut, t2, 0, 0, draw, sum, right);
                pick.key = (uint32_t)(got >> 32);
                pick.idx = ~(uint32_t)got;
                done = true;
            } else {
                kept = sb_find<SB_COUNT>(r, kept, t1, (u64)top_k, -1.0, sum);
                if (cut_p) kept = sb_find<SB_WEIGHT>(r, kept, t1, 0, share_p, sum);
            }
        } else {
            // Most of the vocabulary may be kept. One pass adds up the exact sum that the first target needs and,
            // coarsely, the bins; then for each border one pass adds up what lies before its bin, exactly, and
            // collects the bin.
            const float c1 = 1.4426950408889634f / 16.f, c2 = (float)(1.4426950408889634 / 16 * t2.inv_t);
            u64 s = 0;
            const float low_x = low ? sb_value(low) : -INFINITY;
            const bool same = temp == 1.f && !low;  // both borders have the same weights: one set of bins
            auto one = [&](float x) {
                const int bin = sb_bin(r.top, x);
                if (cut_p) {
                    s += sb_weight(x, r.top, t1, sh.table);
                    atomicAdd(&sh.part[0][bin], sb_coarse(r.top, x, bin, c1));
                    if (same || !(x >= low_x)) return;
                } else {
                    s += sb_weight(x, r.top, t2, sh.table);
                }
                atomicAdd(&sh.part[1][bin], sb_coarse(r.top, x, bin, c2));
            };
            const float least = cut_p ? -INFINITY : low_x;  // what counts for the sum
            const int n4 = r.n / 4;
            for (int i = tid; i < n4; i += SB_THREADS) {
                const float4 x = *reinterpret_cast<const float4*>(sb_vals + 4 * i);
                if (x.x >= least) one(x.x);
                if (x.y >= least) one(x.y);
                if (x.z >= least) one(x.z);
                if (x.w >= least) one(x.w);
            }
            for (int i = 4 * n4 + tid; i < r.n; i += SB_THREADS)
                if (sb_vals[i] >= least) one(sb_vals[i]);
            u64 block;
            sb_scan(s, &sh, block);
            if (tid == 0) sh.sum[0] = block;
            cluster_sync_all();
            sum = sb_sum_all(&sh.sum[0], r.size);
            u64 w1 = 0, w2 = sb_coarse_bin(r, cut_p && same ? 0 : 1, c2), all1 = 0, all2;
            if (cut_p) {
                w1 = sb_coarse_bin(r, 0, c1);
                w1 = sb_scan(w1, &sh, all1);
            }
            w2 = sb_scan(w2, &sh, all2);
            cluster_sync_all();  // every block has read the bins and the sums
            bool ok = true;
            int last = SB_BINS - 1;  // the bin in which what is kept ends
            if (cut_p) {
                const int bin = sb_first_thread(w1 > 0 && (double)w1 >= share_p * (double)all1, &sh);
                u64 s1 = 0, s2 = 0;
                const bool same_t = temp == 1.f;
                // values above `hi` are certainly in a bin before, those below `lo` in one behind
                const float hi = bin > 0 ? __fsub_ru(r.top, ((float)bin - 0.51f) / 16.f) : INFINITY;
                const float lo = bin < SB_BINS - 1 ? __fsub_rd(r.top, ((float)bin + 0.51f) / 16.f) : -INFINITY;
                auto before = [&](float x) {
                    const u64 w = sb_weight(x, r.top, t1, sh.table);
                    s1 += w;
                    if (x >= low_x) s2 += same_t ? w : sb_weight(x, r.top, t2, sh.table);
                };
                sb_scan_slice(r, lo, hi, [&](float x, int i) {
                    const int b = sb_bin(r.top, x);
                    if (b == bin) sb_note(&sh, sb_key(x), i);
                    else if (b < bin) before(x);
                }, before);
                u64 b1, b2;
                sb_scan(s1, &sh, b1);
                sb_scan(s2, &sh, b2);
                if (tid == 0) {
                    sh.sum[0] = b1;
                    sh.sum[1] = b2;
                }
                cluster_sync_all();
                if (r.rank == 0) {
                    s1 = sb_sum_all(&sh.sum[0], r.size);
                    s2 = sb_sum_all(&sh.sum[1], r.size);
                    uint32_t nq[SB_MAX_CLUSTER];
                    const uint32_t n = sb_noted(r, nq);
                    ok = n > 0 && n <= SB_FEW;
                    if (ok) {
                        u64 v4[SB_E];
                        sb_fetch(r, nq, n, v4);
                        const u64 got = sb_pick<SB_WEIGHT>(r, v4, 0, t1, s1, 0, share_p, sum, right);
                        ok = right;
                        u64 weight = 0;  // of all that is kept
                        if (ok) {        // the draw may fall into this bin
                            const u64 g = sb_pick<SB_WEIGHT>(r, v4, max(got, (u64)low << 32), t2, s2, 0, draw, weight, right);
                            if (weight == 0) weight = s2;  // nothing of the bin is kept
                            sum = weight;
                            if (right) {
                                pick.key = (uint32_t)(g >> 32);
                                pick.idx = ~(uint32_t)g;
                                done = true;
                            }
                        }
                        if (tid == 0) {
                            sh.told[1] = got;
                            sh.told[2] = sum;
                        }
                    }
                    if (tid == 0) sh.told[0] = (ok ? 1u : 0u) | (done ? 2u : 0u);
                }
                cluster_sync_all();
                const u64 told = sb_ld64(&sh.told[0], 0), got = sb_ld64(&sh.told[1], 0);
                if (ok = told & 1; ok) sum = sb_ld64(&sh.told[2], 0);
                done = told & 2;
                cluster_sync_all();
                if (done && r.rank != 0) return;
                if (ok) {
                    kept.key = (uint32_t)(got >> 32);
                    kept.idx = ~(uint32_t)got;
                    last = bin;
                } else {
                    kept = sb_find<SB_WEIGHT>(r, all, t1, 0, share_p, sum);
                }
                if (tid == 0) {
                    sh.first = ~0u;
                    sh.list_n = 0;
                }
                __syncthreads();
            }
            if (!done && ok) {
                const int bin = min(sb_first_thread(w2 > 0 && (double)w2 >= draw * (double)sum, &sh), last);
                u64 s2 = 0;
                const float kept_x = kept.key ? sb_value(kept.key) : -INFINITY;
                // as above; what the filters cut is between (values below low_x or the last kept are never above `hi`)
                const float hi = fmaxf(bin > 0 ? __fsub_ru(r.top, ((float)bin - 0.51f) / 16.f) : INFINITY, fmaxf(kept_x, low_x));
                const float lo = bin < SB_BINS - 1 ? __fsub_rd(r.top, ((float)bin + 0.51f) / 16.f) : -INFINITY;
                auto before = [&](float x) { s2 += sb_weight(x, r.top, t2, sh.table); };
                sb_scan_slice(r, lo, hi, [&](float x, int i) {
                    if (!(x >= low_x) || x < kept_x || (x == kept_x && (uint32_t)i > kept.idx)) return;
                    const int b = sb_bin(r.top, x);
                    if (b == bin) sb_note(&sh, sb_key(x), i);
                    else if (b < bin) before(x);
                }, before);
                u64 b2;
                sb_scan(s2, &sh, b2);
                if (tid == 0) sh.sum[0] = b2;
                cluster_sync_all();
                if (r.rank == 0) {
                    s2 = sb_sum_all(&sh.sum[0], r.size);
                    uint32_t nq[SB_MAX_CLUSTER];
                    const uint32_t n = sb_noted(r, nq);
                    if (n > 0 && n <= SB_FEW) {
                        u64 v4[SB_E];
                        sb_fetch(r, nq, n, v4);
                        const u64 got = sb_pick<SB_WEIGHT>(r, v4, 0, t2, s2, 0, draw, sum, right);
                        if (right) {
                            pick.key = (uint32_t)(got >> 32);
                            pick.idx = ~(uint32_t)got;
                            done = true;
                        }
                    }
                    if (tid == 0) sh.told[0] = done ? 1 : 0;
                }
                cluster_sync_all();
                done = sb_ld64(&sh.told[0], 0) != 0;
                cluster_sync_all();
                if (done && r.rank != 0) return;
            }
        }
        if (!done) {
            // a crowded bin, or coarse sums that named the wrong one: the border of the draw by descent
            const SbBorder likely = {low, ~0u};
            if (low && likely.before(kept)) kept = likely;
            pick = sb_find<SB_WEIGHT>(r, kept, t2, 0, draw, sum);
        }
        const float v = sb_value(pick.key);
        const double e = v == r.top ? 1.0 : exp(((double)v - (double)r.top) * inv_t);
        prob = e * SB_ONE / (double)sum;
    }
    if (r.rank == 0 && tid == 0) {
        a.ids[row] = none ? -1 : (int)pick.idx;
        if (a.probs) a.probs[row] = none ? 0.f : (float)prob;
    }
    // no block leaves while another may still read its shared memory: sb_find and the maximum end with a cluster barrier
}

}  // namespace mf
