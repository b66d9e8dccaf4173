// Helpers shared by the decoder-layer kernels (rmsnorm.cu, kv_cache.cu,
// kv_attention.cu, kv_attention_tc.cu).
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "../../include/lcml_decoder.h"
#include "lcml_device.cuh"
#include "lcml_internal.h"

namespace lcml {

// Join the codes of DeviceError. A page number outside the cache or a position
// past the block table (the access is skipped), and a sequence longer than
// the call's bounds (its surplus is not computed) or of negative length.
constexpr int kDevBadPage = 6;
constexpr int kDevBadBatch = 7;

template <typename T>
struct Elem;
template <>
struct Elem<float> {
    static __device__ __forceinline__ float load(const float *p) { return *p; }
    static __device__ __forceinline__ float from(float v) { return v; }
};
template <>
struct Elem<__half> {
    static __device__ __forceinline__ float load(const __half *p) { return __half2float(*p); }
    static __device__ __forceinline__ __half from(float v) { return __float2half_rn(v); }
};
template <>
struct Elem<__nv_bfloat16> {
    static __device__ __forceinline__ float load(const __nv_bfloat16 *p) { return __bfloat162float(*p); }
    static __device__ __forceinline__ __nv_bfloat16 from(float v) { return __float2bfloat16_rn(v); }
};

// E consecutive elements of T as one aligned access of E * sizeof(T) bytes
// (two for 32 bytes), widened to or rounded from fp32. kReadOnly: nothing writes
// the memory while the kernel runs.
template <typename T, int E, bool kReadOnly = true>
__device__ __forceinline__ void load_vec(const T *p, float *v) {
    constexpr int B = E * static_cast<int>(sizeof(T));
    alignas(16) T t[E];
    auto get = [&](auto *dst, int i) {
        const auto *src = reinterpret_cast<decltype(dst)>(const_cast<T *>(p)) + i;
        if constexpr (kReadOnly) dst[i] = __ldg(src);
        else dst[i] = *src;
    };
    if constexpr (B == 32) {
        get(reinterpret_cast<uint4 *>(t), 0);
        get(reinterpret_cast<uint4 *>(t), 1);
    } else if constexpr (B == 16) {
        get(reinterpret_cast<uint4 *>(t), 0);
    } else if constexpr (B == 8) {
        get(reinterpret_cast<uint2 *>(t), 0);
    } else {
#pragma unroll
        for (int i = 0; i < E; ++i) t[i] = p[i];
    }
#pragma unroll
    for (int i = 0; i < E; ++i) v[i] = Elem<T>::load(t + i);
}

template <typename T, int E>
__device__ __forceinline__ void store_vec(T *p, const float *v) {
    constexpr int B = E * static_cast<int>(sizeof(T));
    alignas(16) T t[E];
#pragma unroll
    for (int i = 0; i < E; ++i) t[i] = Elem<T>::from(v[i]);
    if constexpr (B % 16 == 0) {
#pragma unroll
        for (int i = 0; i < B / 16; ++i) reinterpret_cast<uint4 *>(p)[i] = reinterpret_cast<uint4 *>(t)[i];
    } else if constexpr (B == 8) {
        *reinterpret_cast<uint2 *>(p) = *reinterpret_cast<uint2 *>(t);
    } else {
#pragma unroll
        for (int i = 0; i < E; ++i) p[i] = t[i];
    }
}

// The sequence that owns work unit `u` of a ragged batch whose sequence b owns
// the units from first(b) = cu[b] * mul / div + add * b on (strictly
// increasing in b for add >= 1): the largest b with first(b) <= u. One warp
// searches together, 32 probes a step, so B <= 32 costs one load latency and
// B <= 1024 two. All 32 lanes must call it; all get the answer.
__device__ __forceinline__ int find_sequence(const int32_t *__restrict__ cu, int batch, int64_t u, int mul, int div,
                                             int add) {
    int lo = 0, n = batch;  // the answer is in [lo, lo + n)
    const int lane = threadIdx.x & 31;
    while (n > 1) {
        const int step = (n + 31) / 32;
        const int b = lo + lane * step;
        const bool le = lane * step < n && static_cast<int64_t>(__ldg(cu + b)) * mul / div + static_cast<int64_t>(add) * b <= u;
        const int k = __popc(__ballot_sync(0xffffffffu, le));  // monotone: lanes 0 .. k - 1
        const int at = k > 0 ? (k - 1) * step : 0;
        lo += at;
        n = min(step, n - at);
    }
    return lo;
}

// Launch with programmatic stream serialization (see griddep_wait()): every
// decoder kernel waits for the previous kernel before it reads anything.
template <typename... Params, typename... Args>
int launch_dependent(void (*kern)(Params...), dim3 grid, unsigned threads, size_t smem, cudaStream_t st,
                     const char *name, Args &&...args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads, 1, 1);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kern, static_cast<Params>(args)...);
    g_launches.fetch_add(1, std::memory_order_relaxed);
    if (e != cudaSuccess) {
        cudaGetLastError();
        return set_error(LCML_ERR_CUDA, "%s launch failed: %s", name, cudaGetErrorString(e));
    }
    return LCML_OK;
}

// Argument checks shared by the cache's entry points.
int check_cache(const lcml_kv_cache *c, const char *what);
int check_batch(const lcml_kv_batch *b, const char *what);

}// namespace lcml
