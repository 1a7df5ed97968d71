// Element types of the model operators (fp32, bf16, fp16) and the loads and stores they share.
// Arithmetic is in fp32 whatever the storage type; a 16-bit result is rounded once, to nearest even.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <type_traits>

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

// Two fp32 numbers that one instruction works on (sm_100a: add, mul and fma .f32x2, each half rounded as usual).
struct F2 {
    unsigned long long v;
};
__device__ __forceinline__ F2 f2(float x, float y) {
    F2 r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r.v) : "f"(x), "f"(y));
    return r;
}
__device__ __forceinline__ void split(F2 a, float& x, float& y) { asm("mov.b64 {%0, %1}, %2;" : "=f"(x), "=f"(y) : "l"(a.v)); }
__device__ __forceinline__ F2 operator+(F2 a, F2 b) {
    F2 r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
    return r;
}
__device__ __forceinline__ F2 operator*(F2 a, F2 b) {
    F2 r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
    return r;
}
__device__ __forceinline__ F2 fma2(F2 a, F2 b, F2 c) {
    F2 r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
    return r;
}
__device__ __forceinline__ F2 negative(F2 a) { return F2{a.v ^ 0x8000000080000000ull}; }

// elements 2k and 2k + 1 of a word (a word of one element: the second half is 0)
template <class T, int V>
__device__ __forceinline__ F2 pair_of(const SaVec<T, V>& v, int k) {
    if constexpr (V == 1) {
        return f2(sa_to_float(v.e[0]), 0.0f);
    } else if constexpr (sizeof(T) == 2 && std::is_same<T, __nv_bfloat16>::value) {
        const uint32_t w = reinterpret_cast<const uint32_t*>(&v)[k];
        return f2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
    } else if constexpr (sizeof(T) == 2) {
        const float2 f = __half22float2(reinterpret_cast<const __half2*>(&v)[k]);
        return f2(f.x, f.y);
    } else {
        return f2(v.e[2 * k], v.e[2 * k + 1]);
    }
}
template <class T, int V>
__device__ __forceinline__ void set_pair(SaVec<T, V>& v, int k, F2 a) {
    float x, y;
    split(a, x, y);
    if constexpr (V == 1) {
        v.e[0] = sa_from_float<T>(x);
    } else if constexpr (sizeof(T) == 2 && std::is_same<T, __nv_bfloat16>::value) {
        reinterpret_cast<__nv_bfloat162*>(&v)[k] = __floats2bfloat162_rn(x, y);
    } else if constexpr (sizeof(T) == 2) {
        reinterpret_cast<__half2*>(&v)[k] = __floats2half2_rn(x, y);
    } else {
        v.e[2 * k] = x;
        v.e[2 * k + 1] = y;
    }
}
// Division by a launch constant: exact for n * d < 2^32 (n * (2^32 / d + 1) overshoots n / d * 2^32 by at most n).
struct Divisor {
    uint32_t d, m;
    __device__ __forceinline__ uint32_t div(uint32_t n) const { return d == 1u ? n : __umulhi(n, m); }
};
inline Divisor divisor(uint32_t d) { return Divisor{d, d > 1 ? (uint32_t)(0x100000000ull / d + 1) : 0u}; }

// a result that is not read again soon: evict-first
template <class T, int V>
__device__ __forceinline__ void sa_store_stream(T* p, const SaVec<T, V>& v) {
    if constexpr (sizeof(v) == 16) __stcs(reinterpret_cast<uint4*>(p), *reinterpret_cast<const uint4*>(&v));
    else if constexpr (sizeof(v) == 8) __stcs(reinterpret_cast<uint2*>(p), *reinterpret_cast<const uint2*>(&v));
    else if constexpr (sizeof(v) == 4) __stcs(reinterpret_cast<uint32_t*>(p), *reinterpret_cast<const uint32_t*>(&v));
    else __stcs(reinterpret_cast<uint16_t*>(p), *reinterpret_cast<const uint16_t*>(&v));
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
