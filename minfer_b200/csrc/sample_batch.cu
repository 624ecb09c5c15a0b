// mf_sample_batch (include/minfer_cuda.h, "Sampling on the device").
#include <cuda_runtime.h>

#include <algorithm>
#include <cstdlib>
#include <mutex>
#include <set>
#include <utility>

#include "minfer_cuda.h"
#include "sample_batch.cuh"

namespace mf {
int record_error(int code, const char* msg);
cudaStream_t resolve_stream(void* stream);
}  // namespace mf

namespace {
int sample_batch(int* ids, float* probs, const void* logits, int dtype, long long ld, int n_rows, int vocab,
                               const float* draws, const float* temp, const int* top_k, const float* top_p,
                               const float* min_p, void* stream) {
    auto fail = [](int code, const char* msg) { return mf::record_error(code, msg); };
    if (n_rows == 0) return MF_OK;  // nothing to do (empty tensors have no address)
    if (!ids || !logits || !draws || !temp || !top_k || !top_p || !min_p) return fail(MF_E_INVALID, "null argument");
    if (n_rows < 0 || vocab <= 0 || ld < vocab) return fail(MF_E_INVALID, "need n_rows > 0, vocab > 0 and ld >= vocab");
    if (vocab > mf::SB_MAX_VOCAB) return fail(MF_E_UNSUPPORTED, "vocabulary above 2^18");
    const void* fn = dtype == MF_F32    ? (const void*)&mf::sample_batch_kernel<float>
                     : dtype == MF_F16  ? (const void*)&mf::sample_batch_kernel<__half>
                     : dtype == MF_BF16 ? (const void*)&mf::sample_batch_kernel<__nv_bfloat16>
                                        : nullptr;
    if (!fn) return fail(MF_E_INVALID, "bad dtype");
    const size_t size = dtype == MF_F32 ? 4 : 2;
    if (((uintptr_t)logits & (size - 1)) != 0 ||
        (((uintptr_t)ids | (uintptr_t)probs | (uintptr_t)draws | (uintptr_t)temp | (uintptr_t)top_k | (uintptr_t)top_p |
          (uintptr_t)min_p) & 3) != 0)
        return fail(MF_E_INVALID, "misaligned argument");
    // Blocks per row: as few as keep a block's slice at 4096 logits or fewer, at most 8.
    int cluster = 1;
    while (cluster < mf::SB_MAX_CLUSTER && (vocab + cluster - 1) / cluster > 4096) cluster *= 2;
    if ((long long)n_rows * cluster > 0x7fffffffll) return fail(MF_E_UNSUPPORTED, "too many rows");
    mf::SampleBatch a;
    a.logits = logits;
    a.ld = ld;
    a.draws = draws;
    a.temp = temp;
    a.top_k = top_k;
    a.top_p = top_p;
    a.min_p = min_p;
    a.ids = ids;
    a.probs = probs;
    a.vocab = vocab;
    a.slice = ((vocab + cluster - 1) / cluster + 7) / 8 * 8;  // 16-byte pieces of aligned rows
    const size_t smem = (size_t)a.slice * sizeof(float);
    {
        static std::mutex mu;
        static std::set<std::pair<int, const void*>> set;  // per device and kernel, once
        int dev = 0;
        cudaError_t e = cudaGetDevice(&dev);
        std::lock_guard<std::mutex> lk(mu);
        if (e == cudaSuccess && !set.count({dev, fn})) {
            e = cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                     (mf::SB_MAX_VOCAB / mf::SB_MAX_CLUSTER) * (int)sizeof(float));
            if (e == cudaSuccess) set.insert({dev, fn});
        }
        if (e != cudaSuccess) return fail(MF_E_CUDA, cudaGetErrorString(e));
    }
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute at[2];
    cfg.gridDim = dim3((unsigned)(n_rows * cluster));
    cfg.blockDim = dim3(mf::SB_THREADS);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = mf::resolve_stream(stream);
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = (unsigned)cluster;
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    at[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    const char* pdl = std::getenv("MF_PDL");
    at[1].val.programmaticStreamSerializationAllowed = !(pdl && pdl[0] == '0');
    cfg.attrs = at;
    cfg.numAttrs = 2;
    void* args[] = {&a};
    cudaError_t e = cudaLaunchKernelExC(&cfg, fn, args);
    return e == cudaSuccess ? MF_OK : fail(MF_E_CUDA, cudaGetErrorString(e));
}
}  // namespace

extern "C" int mf_sample_batch(int* ids, float* probs, const void* logits, int dtype, long long ld, int n_rows, int vocab,
                               const float* draws, const float* temp, const int* top_k, const float* top_p,
                               const float* min_p, void* stream) {
    try {
        return sample_batch(ids, probs, logits, dtype, ld, n_rows, vocab, draws, temp, top_k, top_p, min_p, stream);
    } catch (...) {
        return mf::record_error(MF_E_OOM, "out of host memory");
    }
}
