// qms_rows.cuh - what the kernels over rows of logits share (qms_verify.cu, qms_logprobs.cu): a row's split over a cluster of
// CTAs and its launch. Not part of the C ABI.
#pragma once

#include <string.h>

#include "qms_kv.cuh"

namespace qms {

// A row is cut over a cluster of up to 8 CTAs, which exchange their partial results through distributed
// shared memory once.
constexpr int kRowCtas = 8;

__device__ __forceinline__ float ex2f(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// Values of a row that a CTA keeps in shared memory (76 KB: three CTAs per SM, and a row of 155,648 values
// in a cluster of 8); what a longer slice has beyond them is read from memory in each pass.
constexpr int kProbsKeep = 19456, kProbsThreads = 512, kProbsWarps = kProbsThreads / 32;

// Cluster and PDL launch of a row kernel.
template <typename... P, typename... Q>
static int launch_rows(void (*kern)(P...), int threads, int rows, int nc, size_t smem, cudaStream_t s, Q... args) {
    QMS_REQUIRE((int64_t)rows * nc < (1ll << 31), QMS_CUDA_EINVAL, "too many rows (%d)", rows);
    cudaLaunchConfig_t cfg;
    memset(&cfg, 0, sizeof cfg);
    cfg.gridDim = dim3((unsigned)(rows * nc));
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute at[2];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    at[1].id = cudaLaunchAttributeClusterDimension;
    at[1].val.clusterDim.x = nc;
    at[1].val.clusterDim.y = at[1].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = 2;
    QMS_CK(cudaLaunchKernelEx(&cfg, kern, ((P)args)...));
    return QMS_CUDA_OK;
}

// CTAs per row: as many as hold it in shared memory (k_probs), then, while all of them are at most `sms`, twice as many (of
// 4096 values or more). A row of 32,000 in us, by two CTAs and by four: k_probs (up to 74) 1 row 5.6, 4.5; 16 rows 5.7, 4.8; 37
// rows 5.8, 6.7; k_verify (up to 148) 32 sequences
// 8.3, 6.4.
inline int row_ctas(int rows, int V, int sms) {
    int nc = 1;
    while (nc < kRowCtas && (V > nc * kProbsKeep || ((int64_t)rows * nc * 2 <= sms && V > nc * 8192))) nc *= 2;
    return nc;
}

}  // namespace qms
