// Element types of the model operators (fp32, bf16, fp16) and the loads and stores they share.
// Arithmetic is in fp32 whatever the storage type; a 16-bit result is rounded once, to nearest even.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

enum { SA_FP32 = 0, SA_BF16 = 1, SA_FP16 = 2 };

inline int sa_element_size(int dtype) { return dtype == SA_FP32 ? 4 : 2; }

#if defined(__CUDACC__)
namespace { // internal linkage: included by several translation units

__device__ __forceinline__ float sa_to_float(float v) { return v; }
__device__ __forceinline__ float sa_to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float sa_to_float(__half v) { return __half2float(v); }
template <class T>
__device__ __forceinline__ T sa_from_float(float v);
template <>
__device__ __forceinline__ float sa_from_float<float>(float v) { return v; }
template <>
__device__ __forceinline__ __nv_bfloat16 sa_from_float<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <>
__device__ __forceinline__ __half sa_from_float<__half>(float v) { return __float2half_rn(v); }

// V elements that are loaded and stored as one word of V * sizeof(T) bytes (2 to 16)
template <class T, int V>
struct alignas(sizeof(T) * V) SaVec {
    T e[V];
};

// data that is used once: evict-first
template <class T, int V>
__device__ __forceinline__ SaVec<T, V> sa_load_stream(const T* p) {
    SaVec<T, V> r;
    if constexpr (sizeof(r) == 16) {
        const uint4 w = __ldcs(reinterpret_cast<const uint4*>(p));
        r = *reinterpret_cast<const SaVec<T, V>*>(&w);
    } else if constexpr (sizeof(r) == 8) {
        const uint2 w = __ldcs(reinterpret_cast<const uint2*>(p));
        r = *reinterpret_cast<const SaVec<T, V>*>(&w);
    } else if constexpr (sizeof(r) == 4) {
        const uint32_t w = __ldcs(reinterpret_cast<const uint32_t*>(p));
        r = *reinterpret_cast<const SaVec<T, V>*>(&w);
    } else {
        const uint16_t w = __ldcs(reinterpret_cast<const uint16_t*>(p));
        r = *reinterpret_cast<const SaVec<T, V>*>(&w);
    }
    return r;
}

template <class T, int V>
__device__ __forceinline__ SaVec<T, V> sa_load(const T* p) {
    return *reinterpret_cast<const SaVec<T, V>*>(p);
}

template <class T, int V>
__device__ __forceinline__ void sa_store(T* p, const SaVec<T, V>& v) {
    *reinterpret_cast<SaVec<T, V>*>(p) = v;
}

// one entry of a parameter vector (weight, bias) whose type is known at run time only
__device__ __forceinline__ float sa_param(const void* p, long long i, int dtype) {
    if (dtype == SA_FP32) return static_cast<const float*>(p)[i];
    if (dtype == SA_BF16) return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
    return __half2float(static_cast<const __half*>(p)[i]);
}

__device__ __forceinline__ void sa_set_param(void* p, long long i, int dtype, float v) {
    if (dtype == SA_FP32) static_cast<float*>(p)[i] = v;
    else if (dtype == SA_BF16) static_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(v);
    else static_cast<__half*>(p)[i] = __float2half_rn(v);
}

} // namespace
#endif
