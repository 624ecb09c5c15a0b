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
// read from memory once, as order-preserving 32-bit keys, and every later pass
// runs on chip. A border is found by descent: 512 bins of 1/16 below the top,
// the bin that holds the border cut into 512 ranges of keys, and so on, until
// a few candidates are left, which one warp orders, or one value, whose ties
// are counted out by index. Per level the bins of the cluster's blocks are
// added up by every block for itself (one remote read per block and bin).
//
// Sums: weights are exp() in 64 bits, rounded to multiples of 2^-45 and added
// as whole numbers, so a sum does not depend on the order of its terms and is
// off by at most 2^-46 per term. In floats a vocabulary of 10^5 would move the
// border of every hundredth draw.
#pragma once

#include "mf_common.cuh"
#include "paged.cuh"

namespace mf {

constexpr int SB_THREADS = 512;
constexpr int SB_BINS = 512;        // one per thread
constexpr int SB_LIST = 64;         // candidates left to one warp (two per lane)
constexpr int SB_SORT = 2048;       // candidates that one block sorts
constexpr int SB_MAX_CLUSTER = 8;
constexpr int SB_MAX_VOCAB = 1 << 18;  // 2^18 weights of at most 2^45: sums below 2^63
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

MF_DEVICE uint32_t sb_key(float x) {
    if (x != x) x = -INFINITY;
    const uint32_t u = __float_as_uint(x + 0.0f);  // -0 and 0 are equal
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}
MF_DEVICE float sb_value(uint32_t key) { return __uint_as_float(key & 0x80000000u ? key & 0x7fffffffu : ~key); }

// Level-1 bin of a value: never decreases as x falls.
MF_DEVICE int sb_bin(float top, float x) {
    const float d = x == top ? 0.f : top - x;  // top may be infinite
    return d < (float)SB_BINS / 16.f ? (int)(d * 16.f) : SB_BINS - 1;
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

// The last kept candidate of a prefix of the order.
struct SbBorder {
    uint32_t key, idx;
    MF_DEVICE bool keeps(uint32_t k, uint32_t i) const { return k > key || (k == key && i <= idx); }
    MF_DEVICE bool before(const SbBorder& o) const { return key > o.key || (key == o.key && idx < o.idx); }
};

struct SbShared {
    union {
        struct {
            uint32_t cnt[SB_BINS];
            uint32_t part[3][SB_BINS];  // weights in three parts of 16 bits: 32-bit shared atomics, no overflow below 2^16 terms
            u64 wsum[SB_BINS];          // their sum, what the other blocks read
        };
        u64 sorted[SB_SORT];  // candidates of the whole row (its first block)
    };
    u64 cand[SB_SORT];          // (key, ~index) of the block's candidates
    u64 best;                   // (key, ~index) of the block's largest
    u64 scan[34];
    uint32_t scan_c[32];
    u64 found[4];
    uint32_t list_n;
    uint32_t list_key[SB_LIST], list_idx[SB_LIST];
    uint32_t ties;
    uint32_t first;             // smallest position asked for
};

struct SbRow {
    const uint32_t* keys;  // this block's slice
    int n, base;           // its length and first index
    int rank, size;        // of the cluster
    float top;
    SbShared* sh;
};

enum SbMode { SB_COUNT, SB_WEIGHT };

// Where a border falls among the level-1 bins of the whole row.
struct SbLevel {
    int bin;
    u64 before;     // running sum up to the bin
    u64 total;      // over the prefix
    uint32_t in_bin, upto;  // candidates in the bin, and up to its end
    double target;
};

// exp((x - top) / T) in multiples of 2^-45
MF_DEVICE u64 sb_weight(float x, float top, double inv_t) {
    if (x == top) return (u64)SB_ONE;
    const double z = ((double)x - (double)top) * inv_t;
    if (!(z > -32.0)) return 0;  // below half of 2^-45
    return (u64)(exp(z) * SB_ONE + 0.5);
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

// Inclusive scans of a u64 and a count per thread.
MF_DEVICE u64 sb_scan2(u64 v, uint32_t& c, SbShared* sh, u64& total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const u64 u = __shfl_up_sync(0xffffffffu, v, o);
        const uint32_t d = __shfl_up_sync(0xffffffffu, c, o);
        if (lane >= o) {
            v += u;
            c += d;
        }
    }
    __syncthreads();
    if (lane == 31) {
        sh->scan[warp] = v;
        sh->scan_c[warp] = c;
    }
    __syncthreads();
    u64 base = 0;
    uint32_t base_c = 0;
    total = 0;
#pragma unroll
    for (int w = 0; w < SB_THREADS / 32; ++w) {
        const u64 x = sh->scan[w];
        if (w < warp) {
            base += x;
            base_c += sh->scan_c[w];
        }
        total += x;
    }
    c += base_c;
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

// Adds one candidate to a bin.
template <int MODE> MF_DEVICE void sb_add(SbShared* sh, int bin, float x, float top, double inv_t) {
    if (MODE == SB_WEIGHT) {
        const u64 w = sb_weight(x, top, inv_t);
        if (w) {
            atomicAdd(&sh->part[0][bin], (uint32_t)(w & 0xffff));
            atomicAdd(&sh->part[1][bin], (uint32_t)((w >> 16) & 0xffff));
            atomicAdd(&sh->part[2][bin], (uint32_t)(w >> 32));
        }
    }
    atomicAdd(&sh->cnt[bin], 1u);
}

// The bin in which the running sum over the prefix `in` reaches the target:
// `want` ones, or share * (the sum) for weights. The block's bins must be zero
// and in step (sb_clear). The same in every block of the cluster.
MF_DEVICE void sb_clear(SbShared* sh) {
    const int tid = threadIdx.x;
    sh->cnt[tid] = 0;
    sh->part[0][tid] = sh->part[1][tid] = sh->part[2][tid] = 0;
    if (tid == 0) sh->first = ~0u;
}
template <int MODE>
MF_DEVICE SbLevel sb_level(const SbRow& r, const SbBorder& in, double inv_t, u64 want, double share) {
    SbShared* sh = r.sh;
    const int tid = threadIdx.x;
    const uint32_t whole = in.key == 0 ? 1 : 0;  // the prefix is everything
    for (int i = tid; i < r.n; i += SB_THREADS) {
        const uint32_t k = r.keys[i];
        if (!whole && !in.keeps(k, r.base + i)) continue;
        const float x = sb_value(k);
        sb_add<MODE>(sh, sb_bin(r.top, x), x, r.top, inv_t);
    }
    __syncthreads();
    if (MODE == SB_WEIGHT)
        sh->wsum[tid] = (u64)sh->part[0][tid] + ((u64)sh->part[1][tid] << 16) + ((u64)sh->part[2][tid] << 32);
    cluster_sync_all();
    uint32_t c = 0;
    u64 w = 0;
    for (int q = 0; q < r.size; ++q) {
        c += sb_ld32(&sh->cnt[tid], q);
        if (MODE == SB_WEIGHT) w += sb_ld64(&sh->wsum[tid], q);
    }
    if (MODE == SB_COUNT) w = c;
    SbLevel v;
    uint32_t upto = c;
    const u64 inc = sb_scan2(w, upto, sh, v.total);
    v.target = MODE == SB_COUNT ? (double)want : share * (double)v.total;
    const bool hit = c > 0 && (double)inc >= v.target;
    const unsigned hits = __ballot_sync(0xffffffffu, hit);
    if ((tid & 31) == 0 && hits) atomicMin(&sh->first, (uint32_t)tid + __ffs(hits) - 1);
    __syncthreads();
    v.bin = sh->first;
    if (tid == v.bin) {
        sh->found[1] = inc - w;
        sh->found[2] = (u64)upto << 32 | c;
    }
    cluster_sync_all();  // every block has read these bins
    v.before = sh->found[1];
    v.in_bin = (uint32_t)sh->found[2];
    v.upto = (uint32_t)(sh->found[2] >> 32);
    return v;
}

// Brings the candidates with keys in [lo, hi] of the prefix `in` to the row's
// first block and sorts them there (value, then index): n <= SB_SORT of them
// in all. False in the other blocks, which have nothing more to do.
MF_DEVICE bool sb_gather(const SbRow& r, const SbBorder& in, uint32_t lo, uint32_t hi, int n) {
    SbShared* sh = r.sh;
    const int tid = threadIdx.x;
    if (tid == 0) sh->list_n = 0;
    __syncthreads();
    for (int i = tid; i < r.n; i += SB_THREADS) {
        const uint32_t k = r.keys[i];
        if (k < lo || k > hi || !in.keeps(k, r.base + i)) continue;
        sh->cand[atomicAdd(&sh->list_n, 1u)] = (u64)k << 32 | (uint32_t)~(r.base + i);
    }
    cluster_sync_all();
    if (r.rank == 0) {
        int m = 32;
        while (m < n) m *= 2;
        int at = 0;
        for (int q = 0; q < r.size; ++q) {
            const int nq = sb_ld32(&sh->list_n, q);
            for (int i = tid; i < nq; i += SB_THREADS) sh->sorted[at + i] = sb_ld64(&sh->cand[i], q);
            at += nq;
        }
        for (int i = n + tid; i < m; i += SB_THREADS) sh->sorted[i] = 0;
        __syncthreads();
        for (int size = 2; size <= m; size *= 2)
            for (int stride = size / 2; stride > 0; stride /= 2) {
                for (int i = tid; i < m / 2; i += SB_THREADS) {
                    const int x = 2 * i - (i & (stride - 1)), y = x + stride;
                    const u64 u = sh->sorted[x], v = sh->sorted[y];
                    if ((u < v) == ((x & size) == 0)) {
                        sh->sorted[x] = v;
                        sh->sorted[y] = u;
                    }
                }
                __syncthreads();
            }
    }
    cluster_sync_all();  // the lists have been read
    return r.rank == 0;
}

// Position of the first of the n sorted candidates at which before + (running
// sum of weights) reaches share * total, or target if share < 0; n - 1 if none
// does. total 0: the sum over the n. Sets `sum` to that total.
MF_DEVICE int sb_first(const SbRow& r, int n, double inv_t, u64 before, u64 total, double share, u64& sum) {
    SbShared* sh = r.sh;
    const int tid = threadIdx.x;
    constexpr int E = SB_SORT / SB_THREADS;
    u64 w[E], mine = 0;
#pragma unroll
    for (int e = 0; e < E; ++e) {
        const int i = tid * E + e;
        w[e] = i < n ? sb_weight(sb_value((uint32_t)(sh->sorted[i] >> 32)), r.top, inv_t) : 0;
        mine += w[e];
    }
    u64 all;
    u64 run = before + sb_scan(mine, sh, all) - mine;
    sum = total ? total : all;
    const double target = share * (double)sum;
    if (tid == 0) sh->first = n - 1;
    __syncthreads();
#pragma unroll
    for (int e = 0; e < E; ++e) {
        run += w[e];
        if (tid * E + e < n && (double)run >= target) {
            atomicMin(&sh->first, (uint32_t)(tid * E + e));
            break;
        }
    }
    __syncthreads();
    const int at = sh->first;
    __syncthreads();
    return at;
}

// First candidate of the prefix `in` at which the running sum reaches the
// target: target = want (SB_COUNT: want ones; share < 0), or share * (sum over
// the prefix) for weights. Sets `sum` to the whole sum. Every block of the
// cluster calls it and gets the same answer. If rounding leaves the target
// above the sum the last candidate with weight is taken.
template <int MODE>
MF_DEVICE SbBorder sb_find(const SbRow& r, const SbBorder& in, double inv_t, u64 want, double share, u64& sum) {
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
            const uint32_t k = r.keys[i];
            if (k < lo || k > hi || !in.keeps(k, r.base + i)) continue;
            const float x = sb_value(k);
            const int bin = level == 0 ? sb_bin(r.top, x) : (int)((hi - k) >> shift);
            atomicAdd(&sh->cnt[bin], 1u);
            if (MODE == SB_WEIGHT) {
                const u64 w = sb_weight(x, r.top, inv_t);
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
        uint32_t c = 0;
        u64 w = 0;
        for (int q = 0; q < r.size; ++q) {
            c += sb_ld32(&sh->cnt[tid], q);
            if (MODE == SB_WEIGHT) w += sb_ld64(&sh->wsum[tid], q);
        }
        if (MODE == SB_COUNT) w = c;
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
                    const uint32_t k = r.keys[i];
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
                        w2[s] = !has[s] ? 0 : MODE == SB_COUNT ? 1 : sb_weight(sb_value(k[s]), r.top, inv_t);
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
                // one value: its ties in the order of their indices. Number `need` (from 1) is the border.
                const u64 w1 = MODE == SB_COUNT ? 1 : sb_weight(sb_value(lo), r.top, inv_t);
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
                for (int i = i0; i < i1; ++i) mine += r.keys[i] == lo && in.keeps(lo, r.base + i);
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
                        if (r.keys[i] == lo && in.keeps(lo, r.base + i) && --left_n == 0) sh->found[3] = r.base + i;
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
__global__ void __launch_bounds__(SB_THREADS) sample_batch_kernel(const SampleBatch a) {
    extern __shared__ __align__(16) uint32_t sb_keys[];
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
    r.keys = sb_keys;
    r.sh = &sh;

    // the slice as keys, and the largest with the lowest index
    const T* x = reinterpret_cast<const T*>(a.logits) + row * a.ld + r.base;
    u64 best = 0;
    constexpr int V = 16 / sizeof(T);
    const bool vec = (reinterpret_cast<uintptr_t>(x) & 15) == 0;
    const int nv = vec ? r.n / V : 0;
    for (int i = tid; i < nv; i += SB_THREADS) {
        const PackV<T, V> v = *reinterpret_cast<const PackV<T, V>*>(x + (long long)i * V);
#pragma unroll
        for (int e = 0; e < V; ++e) {
            const uint32_t k = sb_key(to_f<T>(v.e[e]));
            sb_keys[i * V + e] = k;
            best = max(best, (u64)k << 32 | (uint32_t)~(r.base + i * V + e));
        }
    }
    for (int i = nv * V + tid; i < r.n; i += SB_THREADS) {
        const uint32_t k = sb_key(to_f<T>(x[i]));
        sb_keys[i] = k;
        best = max(best, (u64)k << 32 | (uint32_t)~(r.base + i));
    }
    for (int o = 16; o > 0; o >>= 1) best = max(best, __shfl_xor_sync(0xffffffffu, best, o));
    if (tid == 0) sh.best = 0;
    sb_clear(&sh);
    __syncthreads();
    if (lane == 0) atomicMax(&sh.best, best);
    cluster_sync_all();
    best = 0;
    for (int q = 0; q < r.size; ++q) best = max(best, sb_ld64(&sh.best, q));
    cluster_sync_all();
    const uint32_t top_key = (uint32_t)(best >> 32);
    r.top = sb_value(top_key);
    SbBorder pick;
    pick.key = top_key;
    pick.idx = ~(uint32_t)best;

    const float temp = a.temp[row], top_p = a.top_p[row], min_p = a.min_p[row];
    const int top_k = a.top_k[row];
    const bool none = top_key == sb_key(-INFINITY);  // nothing to choose from
    double prob = 1.0;
    if (!none && temp > 0.f) {
        const SbBorder all = {0u, ~0u};
        const bool cut_k = top_k > 0 && top_k < a.vocab, cut_p = top_p < 1.f;
        const double share_p = (double)fmaxf(top_p, 0.f), inv_t = 1.0 / (double)temp;
        const double draw = (double)fminf(fmaxf(a.draws[row], 0.f), 0.99999994f);
        SbBorder likely = all;  // the smallest value at least min_p as likely as the first: x >= top + log(min_p)
        if (min_p > 0.f) {
            const double thr = min_p < 1.f ? (double)r.top + log((double)min_p) : (double)r.top;
            uint32_t lo = sb_key(-INFINITY), hi = top_key;
            while (lo < hi) {
                const uint32_t mid = lo + ((hi - lo) >> 1);
                if ((double)sb_value(mid) >= thr) hi = mid;
                else lo = mid + 1;
            }
            likely.key = lo;
        }
        u64 sum = 0;
        bool done = false;
        if (cut_k || cut_p) {
            const SbLevel v = cut_k ? sb_level<SB_COUNT>(r, all, 1.0, (u64)top_k, -1.0) : sb_level<SB_WEIGHT>(r, all, 1.0, 0, share_p);
            if (v.upto <= SB_SORT) {
                // the candidates down to the bin of the first border: what is kept is among the first of them
                if (!sb_gather(r, all, sb_bin_low(r.top, v.bin), top_key, (int)v.upto)) return;
                int n = cut_k ? top_k : (int)v.upto;
                if (cut_p) n = sb_first(r, n, 1.0, 0, cut_k ? 0 : v.total, share_p, sum) + 1;
                if (min_p > 0.f) {
                    if (tid == 0) sh.first = n;
                    __syncthreads();
                    for (int i = tid; i < n; i += SB_THREADS)
                        if ((uint32_t)(sh.sorted[i] >> 32) < likely.key) atomicMin(&sh.first, (uint32_t)i);
                    __syncthreads();
                    n = sh.first;
                    __syncthreads();
                }
                const u64 got = sh.sorted[sb_first(r, n, inv_t, 0, 0, draw, sum)];
                pick.key = (uint32_t)(got >> 32);
                pick.idx = ~(uint32_t)got;
                done = true;
            }
        } else {
            const SbLevel v = sb_level<SB_WEIGHT>(r, likely, inv_t, 0, draw);
            if (v.in_bin <= SB_SORT) {
                // the candidates of the draw's bin
                const uint32_t lo = sb_bin_low(r.top, v.bin), hi = v.bin > 0 ? sb_bin_low(r.top, v.bin - 1) - 1 : top_key;
                if (!sb_gather(r, likely, lo, hi, (int)v.in_bin)) return;
                const u64 got = sh.sorted[sb_first(r, (int)v.in_bin, inv_t, v.before, v.total, draw, sum)];
                pick.key = (uint32_t)(got >> 32);
                pick.idx = ~(uint32_t)got;
                done = true;
            }
        }
        if (!done) {
            // many candidates down to the border: filter by filter, by descent
            SbBorder kept = all;
            if (cut_k) kept = sb_find<SB_COUNT>(r, kept, 1.0, (u64)top_k, -1.0, sum);
            if (cut_p) kept = sb_find<SB_WEIGHT>(r, kept, 1.0, 0, share_p, sum);
            if (likely.before(kept)) kept = likely;
            pick = sb_find<SB_WEIGHT>(r, kept, inv_t, 0, draw, sum);
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
