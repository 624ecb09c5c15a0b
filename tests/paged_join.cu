// The joining kernels of the paged attention over parts that a test made, 16-bit pages of 64-wide heads (test
// infrastructure, built by test_gpu_paged_gave_up.py).
#include "paged_fa.cuh"

using T = __nv_bfloat16;

static mf::PagedKv batch(const int* q_start, const int* kv_lens, int n_seqs, int n_tokens, int n_kv_heads) {
    mf::PagedKv p = {};
    p.q_start = q_start;
    p.kv_lens = kv_lens;
    p.max_pages = 1 << 16;
    p.n_pages = 1;
    p.page_size = 16;
    p.n_seqs = n_seqs;
    p.n_kv_heads = n_kv_heads;
    p.n_tokens = n_tokens;
    return p;
}

static mf::PagedAttn rows(void* out, int n_kv_heads, int G) {
    mf::PagedAttn a = {};
    a.out = out;
    a.n_heads = n_kv_heads * G;
    a.out_stride = a.n_heads * 64;
    a.G = G;
    a.max_rows = 0x7fffffff;
    return a;
}

// part: [2 * grid][16][64] and [2 * grid][16][2] floats, of ranges of 128-key tiles
extern "C" int join_few(void* out, float* part, const int* q_start, const int* kv_lens, int n_seqs, int n_tokens, int n_kv_heads, int G, int grid) {
    mf::PagedAttn a = rows(out, n_kv_heads, G);
    a.part = part;
    mf::paged_join_kernel<T, 64, 16, 128><<<grid - 1, 256>>>(batch(q_start, kv_lens, n_seqs, n_tokens, n_kv_heads), a, grid);
    return (int)cudaDeviceSynchronize();
}

// part_o: [n_split][n_tokens * n_heads][64], part_ml: [n_split][n_tokens * n_heads][2]
extern "C" int join_chunks(void* out, float* part_o, float* part_ml, const int* q_start, const int* kv_lens, int n_seqs, int n_tokens, int n_kv_heads, int G,
                           int n_split) {
    mf::PagedFa f = {};
    f.n_split = n_split;
    f.part_o = part_o;
    f.part_ml = reinterpret_cast<float2*>(part_ml);
    const int n = n_tokens * n_kv_heads * G;
    mf::paged_fa_join_kernel<T, 64><<<(n + 7) / 8, 256>>>(batch(q_start, kv_lens, n_seqs, n_tokens, n_kv_heads), rows(out, n_kv_heads, G), f);
    return (int)cudaDeviceSynchronize();
}
