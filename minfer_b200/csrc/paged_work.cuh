// How the paged attention kernels for few rows share a batch out.
//
// An item is a tile of up to RT query rows (row r of a sequence = token r / G, head
// r % G of the group) of one KV head of one sequence; its work is the number
// of KT-key tiles that its rows see, after one unit for its beginning and end
// (queries, join, output: about a tile's time; without it a CTA of 55 one-tile
// items ran four times as long as one of a few long items). The items of the
// whole batch, laid end to end, are cut into equal ranges, one per CTA,
// wherever the cut falls: lengths from one key to the longest balance by
// themselves, and the grid does not depend on them. An item whose tiles lie
// inside one range is finished by its CTA; of one whose tiles a cut divides
// every CTA leaves (O, m, l) of its part in a slot of its own, and the block
// of the item's first inner cut in a second kernel joins them in order
// (paged_join_kernel). No counters or flags stay behind, and the result does
// not depend on which CTA ran first.
#pragma once

#include "paged.cuh"

namespace mf {

struct PagedAttn {
    void* out;  // [n_tokens][out_stride]
    long long out_stride;
    const void* q;  // [n_tokens][q_stride]
    long long q_stride;
    float scale2;  // softmax scale * log2(e)
    int n_heads, G, window;
    int min_rows, max_rows;  // sequences of other numbers of rows (n_b * G) are another kernel's: min_rows < rows <= max_rows
    int beside;    // launched behind a chunk kernel that it neither reads nor waits for at its start (paged_begin)
    float* part;   // (O, m, l) of divided items: [2 * grid][RT][D], then [2 * grid][RT][2]; l = PAGED_GAVE_UP: none
    int* status;   // bit 2: a wait gave up
    unsigned long long timeout_ns;
};

// The sum that a CTA whose wait gave up leaves in place of its rows': the
// joining kernels write no row with such a part. (Sums are not negative.)
constexpr float PAGED_GAVE_UP = -1.f;

// A kernel for few rows that follows a chunk kernel of the same call works on
// other rows, so it starts on SMs that that kernel's CTAs leave or never had and
// waits for it only at its own end (whoever waits for this one then waits for
// both). Each CTA keeps its place until then: beside a chunk kernel that still
// runs only as many work as fit the free SMs at once, the others follow it.
// What both read was there before: the chunk kernel lets this one start only after
// its own wait.
MF_DEVICE void paged_begin(const PagedAttn& a) {
    if (!a.beside) pdl_wait();
    pdl_launch_dependents();  // after the wait: see paged_join_kernel
}
MF_DEVICE void paged_end(const PagedAttn& a) {
    if (a.beside) pdl_wait();
}

// The keys [lo, hi) that rows [r0, r0 + RT) of a sequence see between them.
struct PagedSpan {
    int lo, hi;
};
MF_HOST_DEVICE PagedSpan paged_span(const PagedSeq& s, const PagedAttn& a, int r0, int rows) {
    const int t0 = r0 / a.G, t1 = (min(r0 + rows, s.n * a.G) - 1) / a.G;
    PagedSpan k;
    k.hi = max(s.first + t1 + 1, 0);
    k.lo = a.window > 0 ? min(max(s.first + t0 - a.window + 1, 0), k.hi) : 0;
    return k;
}
// Number of KT-key tiles of a span; a span without keys still takes one (its rows' zeros are written).
template <int KT> MF_HOST_DEVICE int paged_tiles(const PagedSpan& k) { return max((k.hi + KT - 1) / KT - k.lo / KT, 1); }

// Rows of an item of a sequence of `rows`: as few items as RT allows, of nearly
// equal size (130 rows are three items of 48, not two of 64 and one of 2: a
// warp works on 8 rows, and an item counts by its keys alone).
template <int RT> MF_HOST_DEVICE int paged_step(int rows) {
    const int n = (rows + RT - 1) / RT;
    return n <= 1 ? RT : min(((rows + n - 1) / n + 7) / 8 * 8, RT);
}

// Tiles of one KV head of sequence b (0: no rows, or another kernel's). In 64
// bits: 2^24 tiles for each of 2^24 items are within what a call may ask for.
template <int RT, int KT> MF_HOST_DEVICE long long paged_head_work(const PagedSeq& s, const PagedAttn& a) {
    const int rows = s.n * a.G;
    if (rows <= a.min_rows || rows > a.max_rows) return 0;
    long long w = 0;
    const int step = paged_step<RT>(rows);
    for (int r = 0; r < rows; r += step) w += 1 + paged_tiles<KT>(paged_span(s, a, r, step));
    return w;
}

// Item (b, h, r0) of the batch: its tiles are the units [start, start + tiles) of all, after the one at start - 1.
struct PagedItem {
    int b, h, r0, step;
    long long start;
    int tiles;
    PagedSeq s;
    PagedSpan k;
};

// a / b for a >= 0, b > 0; nearly always both are small, and a 64-bit division is five times as long
MF_DEVICE long long paged_div(long long a, long long b) {
    return (a | b) >> 32 ? a / b : (long long)((uint32_t)a / (uint32_t)b);
}

// Total work, and the item that holds unit `at` (if at < total); at = n * share
// with share = ceil(total / grid). Called by the whole block (a multiple of 32
// threads, <= 1024); `sh` is shared scratch of 34 long longs. Each thread sums
// a run of sequences; the owner of `at` is found in the prefix sums (each warp's
// own for up to 32 sequences, else the block's) and walked by every thread.
template <int RT, int KT>
MF_DEVICE long long paged_find(const PagedKv& p, const PagedAttn& a, int n, int grid, long long* sh, long long& share,
                               PagedItem& it) {
    const int tid = threadIdx.x, nt = blockDim.x, lane = tid & 31, warp = tid >> 5;
    const bool one = p.n_seqs <= 32;
    const int run = one ? 1 : (p.n_seqs + nt - 1) / nt;
    const int b0 = min((one ? lane : tid) * run, p.n_seqs), b1 = min(b0 + run, p.n_seqs);
    long long mine = 0;
    for (int b = b0; b < b1; ++b) mine += p.n_kv_heads * paged_head_work<RT, KT>(paged_seq(p, b), a);
    long long inc = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const long long v = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += v;
    }
    long long base = 0, total = 0;
    if (one) {
        total = __shfl_sync(0xffffffffu, inc, 31);
    } else {
        if (lane == 31) sh[warp] = inc;
        __syncthreads();
        for (int w = 0; w < (nt >> 5); ++w) {
            const long long v = sh[w];
            if (w < warp) base += v;
            total += v;
        }
    }
    share = paged_div(total + grid - 1, grid);
    const long long at = n * share;
    const long long begin = base + inc - mine;
    const bool here = mine > 0 && at >= begin && at < begin + mine;
    long long w = begin;
    int b = b0;
    it.tiles = 0;
    if (one) {
        const unsigned who = __ballot_sync(0xffffffffu, here);
        if (at >= total) return total;
        const int src = __ffs(who) - 1;
        w = __shfl_sync(0xffffffffu, w, src);
        b = __shfl_sync(0xffffffffu, b, src);
    } else {
        if (here) {
            sh[32] = begin;
            sh[33] = b0;
        }
        __syncthreads();
        if (at >= total) return total;
        w = sh[32];
        b = (int)sh[33];
    }
    for (;; ++b) {
        const PagedSeq s = paged_seq(p, b);
        const long long hw = paged_head_work<RT, KT>(s, a);
        if (hw > 0 && at < w + hw * p.n_kv_heads) {
            it.b = b;
            it.s = s;
            it.h = (int)paged_div(at - w, hw);
            w += it.h * hw;
            break;
        }
        w += hw * p.n_kv_heads;
    }
    it.step = paged_step<RT>(it.s.n * a.G);
    for (it.r0 = 0;; it.r0 += it.step) {
        it.k = paged_span(it.s, a, it.r0, it.step);
        it.tiles = paged_tiles<KT>(it.k);
        if (at < w + 1 + it.tiles) break;
        w += 1 + it.tiles;
    }
    it.start = w + 1;
    return total;
}

// The item after `it` (only called while work is left).
template <int RT, int KT> MF_DEVICE void paged_next(const PagedKv& p, const PagedAttn& a, PagedItem& it) {
    it.start += it.tiles + 1;
    it.r0 += it.step;
    if (it.r0 >= it.s.n * a.G) {
        it.r0 = 0;
        if (++it.h == p.n_kv_heads) {
            it.h = 0;
            do {
                it.s = paged_seq(p, ++it.b);
            } while (it.s.n * a.G <= a.min_rows || it.s.n * a.G > a.max_rows);
            it.step = paged_step<RT>(it.s.n * a.G);
        }
    }
    it.k = paged_span(it.s, a, it.r0, it.step);
    it.tiles = paged_tiles<KT>(it.k);
}

// Joins the parts of every item that a cut divides: block c - 1 takes the item
// whose first inner cut is c (1 .. grid - 1). Row by row, with m the largest
// part maximum, out = sum O_i 2^(m_i - m) / sum l_i 2^(m_i - m). A part that
// saw no key has l = 0 and adds nothing; a row without any key is 0. A part
// whose scores were NaN has l = NaN, whatever its m, and makes the row NaN.
// The search for the item runs before the wait for the kernel that leaves the
// parts: that kernel lets this one start only after its own wait, so the
// batch's lengths are there.
template <typename T, int D, int RT, int KT>
__global__ void __launch_bounds__(256) paged_join_kernel(const PagedKv p, const PagedAttn a, int grid) {
    __shared__ long long sh[34];
    pdl_launch_dependents();
    PagedItem it;
    long long share;
    const int c = (int)blockIdx.x + 1;
    const long long total = paged_find<RT, KT>(p, a, c, grid, sh, share, it);
    const long long at = c * share;
    const bool mine = at < total && at > it.start && paged_div(it.start, share) + 1 == c;
    const int last = mine ? (int)paged_div(it.start + it.tiles - 1, share) : 0;
    pdl_wait();
    if (!mine) return;
    const int rows = min(it.step, it.s.n * a.G - it.r0);
    const float* ml = a.part + (long long)2 * grid * RT * D;
    constexpr int V = D / 32, U = 8;
    const int lane = threadIdx.x & 31;
    // a CTA's slot 0 is for the item that its range begins inside of, slot 1 for the one it ends inside of:
    // the parts are slot 1 of CTA c - 1 and slot 0 of the CTAs c .. last
    const int n = last - c + 2;
    for (int r = threadIdx.x >> 5; r < rows; r += blockDim.x >> 5) {
        float m = -INFINITY;
        for (int i = lane; i < n; i += 32) m = fmaxf(m, __ldcg(ml + ((long long)(2 * (c - 1 + i) + (i == 0)) * RT + r) * 2));
        m = warp_max(m);
        if (m == -INFINITY) m = 0.f;
        float l = 0.f, o[V] = {};
        bool gone = false;
        for (int i0 = 0; i0 < n; i0 += 32) {
            float w = 0.f;  // weight of part i0 + lane
            if (i0 + lane < n) {
                const int i = i0 + lane;
                const float2 v = __ldcg(reinterpret_cast<const float2*>(ml) + (long long)(2 * (c - 1 + i) + (i == 0)) * RT + r);
                gone |= v.y == PAGED_GAVE_UP;
                w = v.y == 0.f ? 0.f : exp2f(v.x - m);
                l = fmaf(v.y, w, l);
            }
            for (int i1 = 0; i1 < min(32, n - i0); i1 += U) {  // U loads in flight
                PackV<float, V> x[U];
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    const int i = min(i0 + i1 + u, n - 1);
                    x[u] = *reinterpret_cast<const PackV<float, V>*>(a.part + ((long long)(2 * (c - 1 + i) + (i == 0)) * RT + r) * D + lane * V);
                }
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    const float wu = __shfl_sync(0xffffffffu, w, i1 + u);  // 0 past the last
#pragma unroll
                    for (int e = 0; e < V; ++e) o[e] = wu != 0.f ? fmaf(x[u].e[e], wu, o[e]) : o[e];
                }
            }
        }
        if (__any_sync(0xffffffffu, gone)) continue;
        l = warp_sum(l);
        const float inv = l == 0.f ? 0.f : 1.0f / l;
        PackV<T, V> y;
#pragma unroll
        for (int e = 0; e < V; ++e) y.e[e] = from_f<T>(o[e] * inv);
        const int row = it.r0 + r;
        *reinterpret_cast<PackV<T, V>*>(reinterpret_cast<T*>(a.out) + (long long)(it.s.row + row / a.G) * a.out_stride +
                                        (long long)(it.h * a.G + row % a.G) * D + lane * V) = y;
    }
}

}  // namespace mf
