// qms_kv.cuh - device helpers shared by the attention kernels over the contiguous caches (qms_trunk.cu)
// and the paged ones (qms_paged*.cu): cache elements, asynchronous copies, QK-norm + rotation of a row.
#pragma once

#include <atomic>

#include "qms_async.cuh"
#include "qms_common.cuh"

namespace qms {

constexpr unsigned kFull = 0xffffffffu;

__device__ __forceinline__ double warp_sum_d(double v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(kFull, v, o);
    return v;
}
__device__ __forceinline__ double warp_max_d(double v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v = fmax(v, __shfl_xor_sync(kFull, v, o));
    return v;
}

// That much dynamic shared memory for a kernel, once per device (a bit of `done` each). Any number of threads may call.
template <typename K>
inline int allow_smem(std::atomic<unsigned long long> &done, K *kern, int bytes) {
    int dev = 0;
    QMS_CK(cudaGetDevice(&dev));
    if (!(done.load() >> (dev & 63) & 1)) {
        QMS_CK(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
        done.fetch_or(1ull << (dev & 63));
    }
    return QMS_CUDA_OK;
}

// KV cache elements: fp32 (the reference's cache, src/model.c:459-460) or fp16 (compacted: each K / V
// value rounded once when appended, read back as fp32).
__device__ __forceinline__ void kv_st(float *p, float v) { *p = v; }
__device__ __forceinline__ void kv_st(__half *p, float v) { *p = __float2half_rn(v); }
__device__ __forceinline__ float kv_ld(const float *p) { return __ldcg(p); }
__device__ __forceinline__ float kv_ld(const __half *p) { return __half2float(__ldcg(p)); }
__device__ __forceinline__ float4 kv_ld4(const float *p) { return *reinterpret_cast<const float4 *>(p); }
__device__ __forceinline__ float4 kv_ld4(const __half *p) {
    const uint2 u = *reinterpret_cast<const uint2 *>(p);
    const float2 lo = __half22float2(*reinterpret_cast<const __half2 *>(&u.x));
    const float2 hi = __half22float2(*reinterpret_cast<const __half2 *>(&u.y));
    return make_float4(lo.x, lo.y, hi.x, hi.y);
}
__device__ __forceinline__ float2 kv_ld2(const float *p) { return *reinterpret_cast<const float2 *>(p); }
__device__ __forceinline__ float2 kv_ld2(const __half *p) { return __half22float2(*reinterpret_cast<const __half2 *>(p)); }
// the same from global memory through L2 only
__device__ __forceinline__ float4 kv_ldg4(const float *p) { return __ldcg(reinterpret_cast<const float4 *>(p)); }
__device__ __forceinline__ float4 kv_ldg4(const __half *p) {
    const uint2 u = __ldcg(reinterpret_cast<const uint2 *>(p));
    const float2 lo = __half22float2(*reinterpret_cast<const __half2 *>(&u.x));
    const float2 hi = __half22float2(*reinterpret_cast<const __half2 *>(&u.y));
    return make_float4(lo.x, lo.y, hi.x, hi.y);
}
__device__ __forceinline__ float2 kv_ldg2(const float *p) { return __ldcg(reinterpret_cast<const float2 *>(p)); }
__device__ __forceinline__ float2 kv_ldg2(const __half *p) {
    const uint32_t u = __ldcg(reinterpret_cast<const unsigned int *>(p));
    return __half22float2(*reinterpret_cast<const __half2 *>(&u));
}

// 16-byte asynchronous copy global -> shared (L2 only; no register staging).
__device__ __forceinline__ void cp_async16(void *dst, const void *src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(dst)), "l"(src) : "memory");
}
// 8-byte asynchronous copy (through L1: the 16-byte form is the only L2-only one).
__device__ __forceinline__ void cp_async8(void *dst, const void *src) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(smem_u32(dst)), "l"(src) : "memory");
}
// Four cache elements: 16 bytes of fp32 or 8 bytes of fp16.
__device__ __forceinline__ void cp_async_kv4(float *dst, const float *src) { cp_async16(dst, src); }
__device__ __forceinline__ void cp_async_kv4(__half *dst, const __half *src) { cp_async8(dst, src); }
__device__ __forceinline__ void cp_async4(void *dst, const void *src) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(smem_u32(dst)), "l"(src) : "memory");
}

// x w inv, rotated: the second half of norm_rope_pre.
template <int D>
__device__ __forceinline__ void rope_scaled(float (&x)[D / 32], const float (&w)[D / 32], const float (&c)[D / 64], const float (&sn)[D / 64],
                                            double inv) {
    constexpr int J = D / 32, JH = J / 2;
#pragma unroll
    for (int j = 0; j < J; j++) x[j] = __fmul_rn((float)((double)x[j] * inv), w[j]);
#pragma unroll
    for (int j = 0; j < JH; j++) {
        const float x1 = x[j], x2 = x[j + JH];
        x[j] = __fsub_rn(__fmul_rn(x1, c[j]), __fmul_rn(x2, sn[j]));
        x[j + JH] = __fadd_rn(__fmul_rn(x2, c[j]), __fmul_rn(x1, sn[j]));
    }
}

// RMSNorm + NEOX rotation of one head row from preloaded values: x (the row), w (norm weights) and
// c / s (cos / sin of the position) as lane + 32 j (src/model.c:403-422, 441-447).
template <int D>
__device__ __forceinline__ void norm_rope_pre(float (&x)[D / 32], const float (&w)[D / 32], const float (&c)[D / 64],
                                              const float (&sn)[D / 64], float eps) {
    constexpr int J = D / 32;
    double ss = 0.0;
#pragma unroll
    for (int j = 0; j < J; j++) ss = fma((double)x[j], (double)x[j], ss);
    ss = warp_sum_d(ss);
    rope_scaled<D>(x, w, c, sn, 1.0 / sqrt(ss / D + (double)eps));
}

}  // namespace qms
