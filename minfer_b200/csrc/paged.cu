// Entry points of the paged KV cache (include/minfer_cuda.h, "One step of a
// batch of sequences over a paged KV cache"): argument checks and launches.
#include <cuda.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>
#include <cmath>
#include <cstdlib>
#include <map>
#include <mutex>
#include <utility>

#include "minfer_cuda.h"
#include "paged_attn.cuh"
#include "paged_fa.cuh"
#include "paged_few.cuh"
#include "paged_rope.cuh"

namespace mf {
int record_error(int code, const char* msg);  // capi.cu: message for mf_last_error
cudaStream_t resolve_stream(void* stream);    // capi.cu: NULL -> manager stream of the current device
}  // namespace mf

namespace {

__device__ int g_paged_status;  // bit 2: a wait of the attention kernels gave up

int fail(int code, const char* msg) { return mf::record_error(code, msg); }

bool pdl_on() {
    const char* e = std::getenv("MF_PDL");
    return !(e && e[0] == '0');
}

cudaError_t launch(const void* fn, dim3 grid, dim3 block, size_t smem, cudaStream_t st, void** args) {
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute at[1];
    cfg.gridDim = grid;
    cfg.blockDim = block;
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    if (pdl_on()) {
        at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        at[0].val.programmaticStreamSerializationAllowed = 1;
        cfg.attrs = at;
        cfg.numAttrs = 1;
    }
    return cudaLaunchKernelExC(&cfg, fn, args);
}

int num_sms() {
    static std::atomic<int> known[64];
    int dev = 0, v = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) {
        cudaGetLastError();
        return 148;
    }
    if ((v = known[dev].load()) > 0) return v;
    if (cudaDeviceGetAttribute(&v, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || v <= 0) {
        cudaGetLastError();
        return 148;
    }
    known[dev] = v;
    return v;
}

unsigned long long timeout_ns() {
    const char* e = std::getenv("MF_PREFILL_TIMEOUT_MS");
    const long v = (e && *e) ? std::atol(e) : 2000;
    return 1000000ull * (unsigned long long)(v > 0 ? v : 2000);
}

int* status_ptr() {
    static int* p[64] = {nullptr};
    static std::mutex mu;
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return nullptr;
    std::lock_guard<std::mutex> lk(mu);
    if (!p[dev] && cudaGetSymbolAddress((void**)&p[dev], g_paged_status) != cudaSuccess) return nullptr;
    return p[dev];
}

using EncodeFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                              const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                              CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
EncodeFn tmap_encoder() {
    static EncodeFn encode = nullptr;
    static std::once_flag once;
    std::call_once(once, [] {
        void* fn = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &fn, cudaEnableDefault, &q) == cudaSuccess &&
            q == cudaDriverEntryPointSuccess)
            encode = (EncodeFn)fn;
    });
    return encode;
}

// Keys of a page that one TMA box brings in: the largest power of two that divides page_size, at most 64.
int page_run(int page_size) { return std::min(page_size & -page_size, 64); }

// Maps of the 16-bit pages: (d, row of the page, head, page, tensor), boxes of
// 64 elements x `run` rows, 128-byte swizzle. One map serves K and V where their
// distance can be its last stride (encoding a map takes about 3 us of host
// time, a third of a decode call), else there are two. *at: K's index along the
// last extent, and V's in bit 1.
int page_tmaps(CUtensorMap* tk, CUtensorMap* tv, const mf::PagedKv& p, int D, int dtype, int run, int* at) {
    EncodeFn encode = tmap_encoder();
    if (!encode) return fail(MF_E_CUDA, "cuTensorMapEncodeTiled is not available");
    char *k = (char*)p.k, *v = (char*)p.v;
    const cuuint64_t apart = k <= v ? (cuuint64_t)(v - k) : (cuuint64_t)(k - v);
    const bool both = apart > 0 && apart < (1ull << 40);
    *at = !both ? 0 : k < v ? 2 : 1;
    const cuuint64_t dims[5] = {(cuuint64_t)D, (cuuint64_t)p.page_size, (cuuint64_t)p.n_kv_heads, (cuuint64_t)p.n_pages, both ? 2u : 1u};
    const cuuint64_t strides[4] = {(cuuint64_t)p.row_stride * 2, (cuuint64_t)p.head_stride * 2, (cuuint64_t)p.page_stride * 2,
                                   both ? apart : 16};
    const cuuint32_t box[5] = {64, (cuuint32_t)run, 1, 1, 1}, es[5] = {1, 1, 1, 1, 1};
    auto make = [&](CUtensorMap* tm, void* base) {
        return encode(tm, dtype == MF_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 5, base, dims,
                      strides, box, es, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                      CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    };
    CUresult r = make(tk, both ? std::min(k, v) : k);
    if (both) *tv = *tk;
    else if (r == CUDA_SUCCESS) r = make(tv, v);
    return r == CUDA_SUCCESS ? MF_OK : fail(MF_E_INVALID, "the pages' strides do not fit a tensor map");
}

size_t dtype_bytes(int dtype) { return dtype == MF_F32 ? 4 : 2; }
bool known_dtype(int dtype) { return dtype == MF_F32 || dtype == MF_F16 || dtype == MF_BF16; }
bool aligned(const void* p, size_t n) { return ((uintptr_t)p & (n - 1)) == 0; }

// Checks a cache's description and resolves it.
int resolve_kv(const mf_paged_kv* c, int n_tokens, mf::PagedKv* p) {
    if (!c || !c->k_pages || !c->v_pages || !c->page_table || !c->q_start || !c->kv_lens)
        return fail(MF_E_INVALID, "paged cache: null argument");
    if (!known_dtype(c->dtype)) return fail(MF_E_INVALID, "paged cache: bad dtype");
    if (c->n_seqs < 0 || n_tokens < 0 || c->n_pages <= 0 || c->max_pages <= 0 || c->n_kv_heads <= 0)
        return fail(MF_E_INVALID, "paged cache: bad sizes");
    if (c->table_stride != 0 && c->table_stride < c->max_pages)
        return fail(MF_E_INVALID, "paged cache: table_stride below max_pages");
    if (c->d_head != 64 && c->d_head != 128) return fail(MF_E_UNSUPPORTED, "paged cache: d_head must be 64 or 128");
    if (c->page_size <= 0 || c->page_size % 8 != 0 || c->page_size > (1 << 20))
        return fail(MF_E_UNSUPPORTED, "paged cache: page_size must be a multiple of 8, up to 2^20");
    const long long row = c->row_stride ? c->row_stride : c->d_head;
    const long long head = c->head_stride ? c->head_stride : (long long)c->page_size * c->d_head;
    const long long page = c->page_stride ? c->page_stride : head * c->n_kv_heads;
    const long long unit = 16 / (long long)dtype_bytes(c->dtype);
    if (row < c->d_head || head < c->d_head || page < c->d_head || row % unit || head % unit || page % unit ||
        !aligned(c->k_pages, 16) || !aligned(c->v_pages, 16))
        return fail(MF_E_INVALID, "paged cache: pages and strides must be 16-byte aligned, strides at least d_head");
    if (!aligned(c->page_table, 4) || !aligned(c->q_start, 4) || !aligned(c->kv_lens, 4))
        return fail(MF_E_INVALID, "paged cache: tables must be 4-byte aligned");
    p->k = c->k_pages;
    p->v = c->v_pages;
    p->page_stride = page;
    p->head_stride = head;
    p->row_stride = row;
    p->table = c->page_table;
    p->q_start = c->q_start;
    p->kv_lens = c->kv_lens;
    p->table_stride = c->table_stride ? c->table_stride : c->max_pages;
    p->max_pages = c->max_pages;
    p->n_pages = c->n_pages;
    p->page_size = c->page_size;
    p->n_seqs = c->n_seqs;
    p->n_kv_heads = c->n_kv_heads;
    p->n_tokens = n_tokens;
    return MF_OK;
}

template <typename X, typename T> const void* rope_fn2(int d) {
    return d == 64 ? (const void*)&mf::paged_rope_kernel<X, T, 64> : (const void*)&mf::paged_rope_kernel<X, T, 128>;
}
template <typename X> const void* rope_fn1(int t, int d) {
    return t == MF_F32   ? rope_fn2<X, float>(d)
           : t == MF_F16 ? rope_fn2<X, __half>(d)
                         : rope_fn2<X, __nv_bfloat16>(d);
}
const void* rope_fn(int x, int t, int d) {
    return x == MF_F32 ? rope_fn1<float>(t, d) : x == MF_F16 ? rope_fn1<__half>(t, d) : rope_fn1<__nv_bfloat16>(t, d);
}

// ---------------------------------------------------------------- attention plans
// A kernel for few rows and the one that joins its parts.
struct FewPlan {
    const void* kernel;
    const void* join;
    size_t smem;
    int threads, RT;
};
template <int D, int RT> FewPlan simt_plan() {
    return {(const void*)&mf::paged_simt_kernel<D, RT>, (const void*)&mf::paged_join_kernel<float, D, RT, mf::PA_SIMT_KT>,
            (size_t)mf::paged_simt_smem<RT, D>(), mf::PA_SIMT_THREADS, RT};
}
template <typename T, int D, int MT> FewPlan mma_plan() {
    return {(const void*)&mf::paged_few_kernel<T, D, MT>, (const void*)&mf::paged_join_kernel<T, D, 16 * MT, mf::pw_kt<D>()>,
            (size_t)mf::pw_smem<D, MT>(), mf::PW_THREADS, 16 * MT};
}
template <typename T> FewPlan mma_plan2(int d, bool one) {
    return d == 64 ? (one ? mma_plan<T, 64, 1>() : mma_plan<T, 64, 2>()) : (one ? mma_plan<T, 128, 1>() : mma_plan<T, 128, 2>());
}
// `rows`: the most rows of a sequence, as far as known
FewPlan few_plan(int dtype, int d, long long rows) {
    const bool one = rows <= 16;
    if (dtype == MF_F32) return d == 64 ? (one ? simt_plan<64, 16>() : simt_plan<64, 64>()) : (one ? simt_plan<128, 16>() : simt_plan<128, 64>());
    return dtype == MF_F16 ? mma_plan2<__half>(d, one) : mma_plan2<__nv_bfloat16>(d, one);
}

// Blocks of `fn` that are resident at once; also sets its shared-memory size
// (always the same for one kernel). Asked of the driver once per device.
int resident(const void* fn, int threads, size_t smem, int* blocks) {
    static std::mutex mu;
    static std::map<std::pair<int, const void*>, int> known;
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return fail(MF_E_CUDA, cudaGetErrorString(e));
    std::lock_guard<std::mutex> lk(mu);
    int& n = known[{dev, fn}];
    if (n == 0) {
        int per = 0;
        e = cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
        if (e == cudaSuccess) e = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per, fn, threads, smem);
        if (e != cudaSuccess) return fail(MF_E_CUDA, cudaGetErrorString(e));
        n = std::max(per, 1) * num_sms();
    }
    *blocks = n;
    return MF_OK;
}

// Blocks per SM that the workspace of the kernels for few rows is sized for.
int per_sm(int RT) { return RT == 16 ? 4 : 2; }

// Row tiles of the chunk kernel as far as the host knows the batch: every
// sequence begins a tile, so one of max_new tokens after the other while there
// are as many left, then the rest in one. Without the hint all tokens are
// taken for one sequence's, the fewest tiles: a count by equal sequences would
// keep the one chunk among many single tokens in one share.
long long row_tiles(int n_tokens, int G, int max_new) {
    const long long most = max_new > 0 ? std::min(max_new, n_tokens) : n_tokens;
    auto tiles = [&](long long n) { return (n * G + mf::PF_ROWS - 1) / mf::PF_ROWS; };
    return n_tokens / most * tiles(most) + tiles(n_tokens % most);
}
// Shares of the keys in which the chunk kernel works, so that a batch of few
// row tiles fills the SMs: the number with the shortest estimate. A CTA takes
// about 1.9 us per tile of 128 keys and as long as three tiles to begin and
// end; joining n shares reads and writes n fp32 rows of D per query row.
// (100 row tiles after 8192 keys: 3 shares, two rounds of a third each, 0.8 of
// the time of one; 128 row tiles after 29184: one.)
constexpr int MAX_SPLIT = 16;
int chunk_split(int n_tokens, int n_heads, int n_kv_heads, int D, int max_new, long long keys) {
    const long long ctas = row_tiles(n_tokens, n_heads / n_kv_heads, max_new) * n_kv_heads;
    const double tiles = std::max(1.0, (double)keys / mf::PF_KT), row_us = 2.0 * n_tokens * n_heads * D * 4 / 6e6;
    const int sms = num_sms();
    int best = 1;
    double least = 0;
    for (int n = 1; n <= MAX_SPLIT && (n == 1 || (ctas * n <= 4ll * sms && tiles >= 2.0 * n)); ++n) {
        const double us = (double)((ctas * n + sms - 1) / sms) * (tiles / n + 3) * 1.9 + (n > 1 ? 4 + n * row_us : 0);
        if (n == 1 || us < least) {
            best = n;
            least = us;
        }
    }
    return best;
}
// Query rows x shares are bounded by the rule above (at most 4 CTAs of 256 rows per SM, or one share), whatever the
// hint: it only adds tiles.
size_t split_bytes(int n_tokens, int n_heads, int n_kv_heads, int D) {
    const long long ctas = row_tiles(n_tokens, n_heads / n_kv_heads, 0) * n_kv_heads;
    const long long n = std::min<long long>(4ll * num_sms() / ctas, MAX_SPLIT);
    return n <= 1 ? 0 : (size_t)n * n_tokens * n_heads * (D + 2) * sizeof(float);
}

template <typename T, int D> const void* fa_fn2(bool join) {
    return join ? (const void*)&mf::paged_fa_join_kernel<T, D> : (const void*)&mf::paged_fa_kernel<T, D>;
}
const void* fa_fn(int dtype, int d, bool join) {
    return dtype == MF_F16 ? (d == 64 ? fa_fn2<__half, 64>(join) : fa_fn2<__half, 128>(join))
                           : (d == 64 ? fa_fn2<__nv_bfloat16, 64>(join) : fa_fn2<__nv_bfloat16, 128>(join));
}

size_t part_bytes(int blocks, int RT, int d) { return (size_t)2 * blocks * RT * (d + 2) * sizeof(float); }

}  // namespace

extern "C" {

int mf_rope_freqs(double* out, int d_rot, double base, int scaling, double factor, double orig_ctx, double beta_fast,
                  double beta_slow, float* mscale) {
    if (!out || !mscale) return fail(MF_E_INVALID, "null argument");
    if (d_rot < 2 || d_rot % 2 != 0 || !(base > 1.0) || !std::isfinite(base)) return fail(MF_E_INVALID, "bad d_rot or base");
    if (scaling < MF_ROPE_PLAIN || scaling > MF_ROPE_YARN) return fail(MF_E_INVALID, "unknown rope scaling");
    if (scaling != MF_ROPE_PLAIN && !(factor >= 1.0 && std::isfinite(factor))) return fail(MF_E_INVALID, "factor must be at least 1");
    if (scaling == MF_ROPE_NTK && d_rot < 4) return fail(MF_E_INVALID, "d_rot must be at least 4 with a stretched base");
    double lo = 0, hi = 1;
    if (scaling == MF_ROPE_YARN) {
        if (!(orig_ctx > 0 && beta_fast > beta_slow && beta_slow > 0 && std::isfinite(orig_ctx) && std::isfinite(beta_fast)))
            return fail(MF_E_INVALID, "need orig_ctx > 0 and beta_fast > beta_slow > 0");
        // pair index at which a dimension makes `beta` turns over the original context
        const double two_pi = 6.283185307179586;
        lo = std::max(std::floor(d_rot * std::log(orig_ctx / (beta_fast * two_pi)) / (2 * std::log(base))), 0.0);
        hi = std::min(std::ceil(d_rot * std::log(orig_ctx / (beta_slow * two_pi)) / (2 * std::log(base))), d_rot - 1.0);
        hi = std::max(hi, lo + 1e-3);
    }
    if (scaling == MF_ROPE_NTK) base *= std::pow(factor, d_rot / (d_rot - 2.0));
    for (int j = 0; j < d_rot / 2; ++j) {
        double f = std::pow(base, -2.0 * j / d_rot);
        if (scaling == MF_ROPE_LINEAR) f /= factor;
        if (scaling == MF_ROPE_YARN) {
            const double ramp = std::min(std::max((j - lo) / (hi - lo), 0.0), 1.0);
            f = f / factor * ramp + f * (1.0 - ramp);
        }
        out[j] = f / 6.283185307179586;
    }
    *mscale = scaling == MF_ROPE_YARN ? (float)(0.1 * std::log(factor) + 1.0) : 1.0f;
    return MF_OK;
}

static int rope_append(const mf_paged_kv* kv, const mf_paged_rope_desc* d, void* stream) {
    mf::PagedKv p;
    if (!kv || !d) return fail(MF_E_INVALID, "null argument");
    if (d->n_tokens == 0 || kv->n_seqs == 0) return MF_OK;  // nothing to do (empty tensors have no address)
    int rc = resolve_kv(kv, d->n_tokens, &p);
    if (rc) return rc;
    if (!d->q_out || !d->qkv || (!d->freqs && d->d_rot > 0)) return fail(MF_E_INVALID, "null argument");
    if (!known_dtype(d->x_dtype)) return fail(MF_E_INVALID, "bad dtype");
    if (d->n_heads <= 0 || d->n_heads % kv->n_kv_heads != 0)
        return fail(MF_E_INVALID, "n_heads must be a positive multiple of n_kv_heads");
    if (d->d_rot < 0 || d->d_rot > kv->d_head || d->d_rot % 8 != 0)
        return fail(MF_E_INVALID, "d_rot must be a multiple of 8, at most d_head");
    if (!(d->eps >= 0.f)) return fail(MF_E_INVALID, "eps must not be negative");
    const int D = kv->d_head;
    const long long width = (long long)(d->n_heads + 2 * kv->n_kv_heads) * D;
    mf::PagedRope r = {};
    r.q_out = d->q_out;
    r.q_stride = d->q_stride ? d->q_stride : (long long)d->n_heads * D;
    r.qkv = d->qkv;
    r.x_stride = d->x_stride ? d->x_stride : width;
    const long long ux = 16 / (long long)dtype_bytes(d->x_dtype), uq = 16 / (long long)dtype_bytes(kv->dtype);
    if (r.q_stride < (long long)d->n_heads * D || r.x_stride < width || r.q_stride % uq || r.x_stride % ux ||
        !aligned(d->q_out, 16) || !aligned(d->qkv, 16))
        return fail(MF_E_INVALID, "qkv and q_out: rows must be 16-byte aligned and not overlap");
    if (!aligned(d->freqs, 8) || !aligned(d->q_norm_w, 4) || !aligned(d->k_norm_w, 4) || !aligned(d->positions, 4))
        return fail(MF_E_INVALID, "misaligned table");
    r.freqs = d->freqs;
    r.q_norm_w = d->q_norm_w;
    r.k_norm_w = d->k_norm_w;
    r.positions = d->positions;
    r.eps = d->eps;
    r.mscale = d->mscale;
    r.n_heads = d->n_heads;
    r.d_rot = d->d_rot;
    r.interleaved = d->interleaved != 0;
    // Heads per warp, in fours: a warp's angles and lookups take as long as about
    // eight heads, and blocks run in whole rounds (three blocks per SM), so the
    // number with the shortest rounds x (heads + 8) is taken. (2533 tokens of 80
    // heads: 20 heads, 3 rounds, 29 us; 32 heads, 3 rounds of which the last is a
    // seventh full, 33 us. One token: 4 heads.)
    const int H = d->n_heads + 2 * kv->n_kv_heads;
    const long long resident_warps = 3ll * num_sms() * mf::ROPE_WARPS;
    long long least = 0;
    for (int n = 4; n == 4 || (n <= 64 && n < H + 4); n += 4) {
        const long long warps = (long long)d->n_tokens * ((H + n - 1) / n);
        const long long cost = (warps + resident_warps - 1) / resident_warps * (n + 8);
        if (n == 4 || cost < least) {
            least = cost;
            r.hpw = n;
        }
    }
    const long long units = (long long)d->n_tokens * ((H + r.hpw - 1) / r.hpw);
    const long long blocks = (units + mf::ROPE_WARPS - 1) / mf::ROPE_WARPS;
    if (blocks > 0x7fffffffll) return fail(MF_E_UNSUPPORTED, "too many rows");
    void* args[] = {&p, &r};
    cudaError_t e = launch(rope_fn(d->x_dtype, kv->dtype, D), dim3((unsigned)blocks), dim3(mf::ROPE_WARPS * 32), 0,
                           mf::resolve_stream(stream), args);
    return e == cudaSuccess ? MF_OK : fail(MF_E_CUDA, cudaGetErrorString(e));
}

size_t mf_paged_attention_workspace_bytes(int n_tokens, int n_heads, int n_kv_heads, int d_head, int dtype) {
    if (n_tokens <= 0 || n_heads <= 0 || n_kv_heads <= 0 || n_heads < n_kv_heads || (d_head != 64 && d_head != 128) || !known_dtype(dtype)) return 0;
    const size_t few = part_bytes(num_sms(), 64, d_head);  // 4 blocks per SM of 16 rows, 2 of 32
    return few + (dtype == MF_F32 ? part_bytes(2 * num_sms(), 64, d_head) : split_bytes(n_tokens, n_heads, n_kv_heads, d_head));
}

static int attention(const mf_paged_kv* kv, const mf_paged_attn_desc* d, void* stream) {
    mf::PagedKv p;
    if (!kv || !d) return fail(MF_E_INVALID, "null argument");
    if (d->n_tokens == 0 || kv->n_seqs == 0) return MF_OK;  // nothing to do (empty tensors have no address)
    int rc = resolve_kv(kv, d->n_tokens, &p);
    if (rc) return rc;
    if (!d->out || !d->q) return fail(MF_E_INVALID, "null argument");
    if (d->n_heads <= 0 || d->n_heads % kv->n_kv_heads != 0)
        return fail(MF_E_INVALID, "n_heads must be a positive multiple of n_kv_heads");
    if (d->window < 0 || d->max_new < 0 || d->max_len < 0) return fail(MF_E_INVALID, "window and hints must not be negative");
    if (!std::isfinite(d->scale)) return fail(MF_E_INVALID, "scale must be finite");
    const int D = kv->d_head, G = d->n_heads / kv->n_kv_heads;
    if ((long long)d->n_tokens * G > 0x40000000ll) return fail(MF_E_UNSUPPORTED, "too many query rows");
    mf::PagedAttn a = {};
    a.out = d->out;
    a.q = d->q;
    a.out_stride = d->out_stride ? d->out_stride : (long long)d->n_heads * D;
    a.q_stride = d->q_stride ? d->q_stride : (long long)d->n_heads * D;
    const long long u = 16 / (long long)dtype_bytes(kv->dtype);
    if (a.out_stride < (long long)d->n_heads * D || a.q_stride < (long long)d->n_heads * D || a.out_stride % u ||
        a.q_stride % u || !aligned(d->out, 16) || !aligned(d->q, 16))
        return fail(MF_E_INVALID, "q and out: rows must be 16-byte aligned and not overlap");
    if (!d->workspace || !aligned(d->workspace, 256) ||
        d->workspace_bytes < mf_paged_attention_workspace_bytes(d->n_tokens, d->n_heads, kv->n_kv_heads, D, kv->dtype))
        return fail(MF_E_INVALID, "workspace missing, too small or not 256-byte aligned");
    a.scale2 = (d->scale == 0.f ? 1.0f / sqrtf((float)D) : d->scale) * 1.4426950408889634f;
    a.n_heads = d->n_heads;
    a.G = G;
    // a window as long as the table hides nothing; beyond 2^30 its arithmetic would leave 32 bits
    a.window = d->window >= std::min<long long>((long long)p.max_pages * p.page_size, 1 << 30) ? 0 : d->window;
    const int most = std::min(d->max_new > 0 ? d->max_new : d->n_tokens, d->n_tokens);
    cudaStream_t st = mf::resolve_stream(stream);

    a.status = status_ptr();
    if (!a.status) return fail(MF_E_CUDA, "status symbol");
    a.timeout_ns = timeout_ns();

    // Sequences of more than few_rows query rows (new tokens x heads of a group)
    // go to the chunk kernels, which work on 256 (16-bit pages, tensor cores) or
    // 64 rows at a time (fp32), the others to the kernels for few rows. A batch
    // of one sequence is served by one of them alone.
    const bool f32 = kv->dtype == MF_F32;
    const int few_rows = f32 ? 16 : 32;
    const bool chunks = (long long)most * G > few_rows;
    const bool few = !chunks || kv->n_seqs > 1;
    cudaError_t e = cudaSuccess;
    CUtensorMap tk, tv;
    int run = page_run(p.page_size), at = 0;
    if (!f32) {
        rc = page_tmaps(&tk, &tv, p, D, kv->dtype, run, &at);
        if (rc) return rc;
    }
    // parts of the kernels for few rows, of the fp32 chunk kernel, of the split chunk kernel
    float* part_few = (float*)d->workspace;
    float* part_chunk = part_few + part_bytes(num_sms(), 64, D) / sizeof(float);
    // a kernel of paged_work.cuh, and the one that joins its parts
    struct Shared {
        FewPlan s;
        int blocks;
        mf::PagedAttn a;
    };
    auto begin = [&](Shared& k, const FewPlan& s, int min_rows, int max_rows, float* part, bool beside) {
        k.s = s;
        k.a = a;
        k.a.min_rows = min_rows;
        k.a.max_rows = max_rows;
        k.a.part = part;
        k.a.beside = beside;
        const int r = resident(s.kernel, s.threads, s.smem, &k.blocks);
        if (r) return r;
        k.blocks = std::min(k.blocks, per_sm(s.RT) * num_sms());
        void* f32_args[] = {&p, &k.a};
        void* args[] = {&tk, &tv, &p, &k.a, &run, &at};
        e = launch(s.kernel, dim3(k.blocks), dim3(s.threads), s.smem, st, f32 ? f32_args : args);
        return e == cudaSuccess ? MF_OK : fail(MF_E_CUDA, cudaGetErrorString(e));
    };
    auto join = [&](Shared& k) {
        if (k.blocks <= 1) return MF_OK;
        void* args[] = {&p, &k.a, &k.blocks};
        e = launch(k.s.join, dim3(k.blocks - 1), dim3(256), 0, st, args);
        return e == cudaSuccess ? MF_OK : fail(MF_E_CUDA, cudaGetErrorString(e));
    };
    Shared chunk = {}, single = {};
    mf::PagedFa f = {};
    const size_t rows = (size_t)d->n_tokens * d->n_heads;
    if (chunks && f32) {
        rc = begin(chunk, few_plan(kv->dtype, D, 64), few ? few_rows : 0, 0x7fffffff, part_chunk, false);
        if (rc) return rc;
    } else if (chunks) {
        f.run = run;
        f.at = at;
        f.min_rows = few ? few_rows : 0;
        long long keys = (long long)p.max_pages * p.page_size;  // that a row tile sees at most
        if (d->max_len > 0) keys = std::min<long long>(keys, d->max_len);
        if (a.window > 0) keys = std::min<long long>(keys, (long long)a.window + mf::PF_ROWS / G);
        f.n_split = chunk_split(d->n_tokens, d->n_heads, kv->n_kv_heads, D, d->max_new, keys);
        f.part_o = part_chunk;
        f.part_ml = (float2*)(f.part_o + f.n_split * rows * D);
        const void* fn = fa_fn(kv->dtype, D, false);
        const size_t smem = D == 64 ? mf::pf_smem<64>() : mf::pf_smem<128>();
        int unused = 0;
        rc = resident(fn, mf::PF_THREADS, smem, &unused);
        if (rc) return rc;
        // every tile of every such sequence: at most T G / 256 whole ones, and one more for each sequence
        const long long tg = (long long)d->n_tokens * G;
        const long long tiles = tg / mf::PF_ROWS + std::min<long long>(kv->n_seqs, tg / (f.min_rows + 1));
        if (tiles * kv->n_kv_heads > 0x7fffffffll) return fail(MF_E_UNSUPPORTED, "too many query rows");
        void* args[] = {&tk, &tv, &p, &a, &f};
        e = launch(fn, dim3((unsigned)(tiles * kv->n_kv_heads), (unsigned)f.n_split), dim3(mf::PF_THREADS), smem, st, args);
        if (e != cudaSuccess) return fail(MF_E_CUDA, cudaGetErrorString(e));
    }
    if (few) {
        rc = begin(single, few_plan(kv->dtype, D, std::min<long long>((long long)most * G, chunks ? few_rows : 0x7fffffff)), 0,
                   chunks ? few_rows : 0x7fffffff, part_few, chunks);
        if (rc) return rc;
    }
    if (chunks && f32) {
        rc = join(chunk);
        if (rc) return rc;
    } else if (chunks && f.n_split > 1) {
        void* args[] = {&p, &a, &f};
        e = launch(fa_fn(kv->dtype, D, true), dim3((unsigned)((rows + 7) / 8)), dim3(256), 0, st, args);
        if (e != cudaSuccess) return fail(MF_E_CUDA, cudaGetErrorString(e));
    }
    return few ? join(single) : MF_OK;
}

// No C++ exception leaves the library (the caches of launch attributes allocate).
int mf_paged_rope_append(const mf_paged_kv* kv, const mf_paged_rope_desc* desc, void* stream) {
    try {
        return rope_append(kv, desc, stream);
    } catch (...) {
        return fail(MF_E_OOM, "out of host memory");
    }
}

int mf_paged_attention(const mf_paged_kv* kv, const mf_paged_attn_desc* desc, void* stream) {
    try {
        return attention(kv, desc, stream);
    } catch (...) {
        return fail(MF_E_OOM, "out of host memory");
    }
}

int mf_paged_status(int* status, int clear) {
    if (!status) return fail(MF_E_INVALID, "null argument");
    int* p = status_ptr();
    if (!p) return fail(MF_E_CUDA, "status symbol");
    cudaError_t e = cudaDeviceSynchronize();
    if (e == cudaSuccess) e = cudaMemcpy(status, p, sizeof(int), cudaMemcpyDeviceToHost);
    if (e == cudaSuccess && clear) e = cudaMemset(p, 0, sizeof(int));
    return e == cudaSuccess ? MF_OK : fail(MF_E_CUDA, cudaGetErrorString(e));
}

}  // extern "C"
