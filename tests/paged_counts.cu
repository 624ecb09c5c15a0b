// How the paged attention counts a batch's work, for tests on the CPU (built by test_paged_counts.py).
#include "paged_work.cuh"

template <int RT, int KT> static long long work(int n, int first, int G, int window) {
    mf::PagedAttn a = {};
    a.G = G;
    a.window = window;
    a.max_rows = 0x7fffffff;
    return mf::paged_head_work<RT, KT>(mf::PagedSeq{0, n, first}, a);
}

// Work of one KV head of a sequence: n new tokens, the first at position `first`
extern "C" long long head_work(int RT, int KT, int n, int first, int G, int window) {
    if (RT == 16 && KT == 64) return work<16, 64>(n, first, G, window);
    if (RT == 32 && KT == 64) return work<32, 64>(n, first, G, window);
    if (RT == 64 && KT == 64) return work<64, 64>(n, first, G, window);
    if (RT == 16 && KT == 128) return work<16, 128>(n, first, G, window);
    if (RT == 32 && KT == 128) return work<32, 128>(n, first, G, window);
    return -1;
}
