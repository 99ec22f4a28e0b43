// paged_types.cuh -- what the serving-step attention kernels share: the two 16-bit types, copies, launches.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "paged.cuh"

namespace kvx {

constexpr float kPagedLn2 = 0.6931471805599453f;

// Softmax weights enter the tensor cores in the cache's type, rounded to nearest: 8 significant
// bits in BF16, 11 in FP16, the same relative size as the output's own rounding (the normaliser l
// sums them unrounded, in FP32, so the log-sum-exp does not see it).  Against 64 bits the outputs are off by
// 0.0018 to 0.0024 of their size in BF16 (FP16: 0.00028), of which the outputs' own rounding is 0.0017
// (0.00021).  A second term (the weight less its rounding) in a second product would leave the latter
// alone: measured, it takes 64 sequences behind 32768 tokens from 68.4 to 77.8 us, 7 behind 131072 from 96.0
// to 104.0 and the other calls 2 to 6 % longer, and since it is 0 for a weight that the type holds, an
// infinite V would give inf + 0 inf = NaN where the formula has inf.  kBias: weights are formed as
// 2^(x - m + kBias); FP16's normal numbers end at 2^-14, so a bias of 10 keeps weights down to
// 2^-24 of the largest at full precision (and its largest, 2^10 times the growth a kernel allows
// before it rescales, below 65504).  The bias is part of the stored m, so it cancels.
template <int DT> struct Elem;
template <> struct Elem<KVX_DTYPE_BF16> {
    static constexpr float kBias = 0.f;
    static __device__ __forceinline__ uint32_t pack(float lo, float hi) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
        return *reinterpret_cast<const uint32_t *>(&h);
    }
    static __device__ __forceinline__ uint16_t one(float x) { return __bfloat16_as_ushort(__float2bfloat16_rn(x)); }
};
template <> struct Elem<KVX_DTYPE_FP16> {
    static constexpr float kBias = 10.f;
    static __device__ __forceinline__ uint32_t pack(float lo, float hi) {
        const __half2 h = __floats2half2_rn(lo, hi);
        return *reinterpret_cast<const uint32_t *>(&h);
    }
    static __device__ __forceinline__ uint16_t one(float x) { return __half_as_ushort(__float2half_rn(x)); }
};

// 2^x by the SFU; results below 2^-126 flush to zero.
__device__ __forceinline__ float exp2_sfu(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// lens[b] clamped to [0, max_len] (reported when it was outside).
__device__ __forceinline__ int tail_len(const PagedArgs &a, int b) {
    const int n = __ldg(a.lens + b);
    if (n >= 0 && n <= a.max_len) return n;
    report(a.status, KVX_ERR_RUNTIME, DERR_LENGTH);
    return n < 0 ? 0 : a.max_len;
}

// 16 bytes global -> shared, zeros when there is no such row.
__device__ __forceinline__ void copy16(uint32_t dst, const void *src, bool live) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(live ? 16 : 0) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void copy_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// Lets a kernel take up to `bytes` of dynamic shared memory a CTA and all of the SM's (the default split
// with L1 may leave room for one CTA where two fit), on the current device.
template <class K> cudaError_t allow_smem(K k, int bytes) {
    cudaError_t e = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e == cudaSuccess) e = cudaFuncSetAttribute(k, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared);
    return e;
}

// A launch that may be set up while the grid before it in the stream drains (programmatic dependent
// launch; every kernel launched so waits for that grid itself).
template <class K, class... More>
cudaError_t launch_paged(K k, dim3 grid, int threads, int smem, cudaStream_t s, const PagedArgs &a, const More &...more) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(unsigned(threads));
    cfg.dynamicSmemBytes = size_t(smem);
    cfg.stream = s;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, k, a, more...);
}

}  // namespace kvx

// The instantiation of fn<D, type> for a head dim and type given at run time, called with the other arguments.
#define KVX_PAGED_TYPE(fn, D, ...) \
    return dtype == KVX_DTYPE_BF16 ? fn<D, KVX_DTYPE_BF16>(__VA_ARGS__) : fn<D, KVX_DTYPE_FP16>(__VA_ARGS__)
#define KVX_PAGED_DIM(fn, ...)                           \
    switch (dim) {                                       \
    case 32: KVX_PAGED_TYPE(fn, 32, __VA_ARGS__);        \
    case 64: KVX_PAGED_TYPE(fn, 64, __VA_ARGS__);        \
    case 128: KVX_PAGED_TYPE(fn, 128, __VA_ARGS__);      \
    case 256: KVX_PAGED_TYPE(fn, 256, __VA_ARGS__);      \
    default: return cudaErrorInvalidValue;               \
    }
