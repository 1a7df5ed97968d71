// Dropout whose mask is drawn again instead of stored: out = residual + (keep ? x / (1 - p) : 0).
//
// Element i belongs to group g = i / 8.  Philox4x32-10 (Salmon, Moraes, Dror, Shaw: "Parallel random numbers: as easy
// as 1, 2, 3", 2011) with the counter (g, call) and the key `seed` gives 128 bits, 16 for each element of the group:
// the upper half of the element's 32-bit number u.  An element is dropped when u < round(p 2^32).  The lower half of u
// comes from a second block (the same counter with its 64th bit set) and is only looked at where the upper half equals
// the threshold's, once in 65,536 elements: the decision has 32 bits for the price of 16.
// (seed, call) are read from device memory, so a recorded graph draws new masks when its replays advance them.
//
// Bound: HBM.  One block is 20 multiplications 32 x 32 -> 64 and about as many logic operations for eight elements.
#include <cmath>

#include "sa_elem.cuh"
#include "sa_ops.hpp"

namespace {

constexpr int kThreads = 256;

struct Draw {
    uint32_t upper, lower; // halves of round(p 2^32); upper = 65536 for p = 1
    float scale;           // 1 / (1 - p)
};

__device__ __forceinline__ uint4 philox(uint32_t c0, uint32_t c1, uint32_t c2, uint32_t c3, uint32_t k0, uint32_t k1) {
#pragma unroll
    for (int r = 0; r < 10; ++r) {
        const uint64_t a = (uint64_t)c0 * 0xD2511F53u, b = (uint64_t)c2 * 0xCD9E8D57u;
        c0 = (uint32_t)(b >> 32) ^ c1 ^ k0;
        c1 = (uint32_t)b;
        c2 = (uint32_t)(a >> 32) ^ c3 ^ k1;
        c3 = (uint32_t)a;
        k0 += 0x9E3779B9u;
        k1 += 0xBB67AE85u;
    }
    return make_uint4(c0, c1, c2, c3);
}

__device__ __forceinline__ uint32_t half_of(const uint4& b, int i) {
    const uint32_t w = i < 2 ? b.x : i < 4 ? b.y : i < 6 ? b.z : b.w;
    return i & 1 ? w >> 16 : w & 0xffffu;
}

// bit i: element i of group g is kept
__device__ __forceinline__ uint32_t keep_mask(uint64_t g, ulonglong2 rng, const Draw& d) {
    const uint32_t s0 = (uint32_t)rng.x, s1 = (uint32_t)(rng.x >> 32), n0 = (uint32_t)rng.y, n1 = (uint32_t)(rng.y >> 32);
    const uint4 b = philox((uint32_t)g, (uint32_t)(g >> 32), n0, n1, s0, s1);
    uint32_t keep = 0, tie = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const uint32_t u = half_of(b, i);
        keep |= (u >= d.upper ? 1u : 0u) << i;
        tie |= (u == d.upper ? 1u : 0u) << i;
    }
    if (tie != 0u && d.lower != 0u) {
        const uint4 c = philox((uint32_t)g, (uint32_t)(g >> 32) | 0x80000000u, n0, n1, s0, s1);
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (((tie >> i) & 1u) && half_of(c, i) < d.lower) keep &= ~(1u << i);
    }
    return keep;
}

// elements of group g in two halves of four (fp32) or one word of eight (16 bits)
template <class T>
struct Eight {
    static constexpr int kWords = sizeof(T) / 2, kPer = 8 / kWords;
    SaVec<T, kPer> w[kWords];
};

template <class T, bool RESIDUAL, bool ALIGNED>
__global__ void __launch_bounds__(kThreads)
sa_dropout_kernel(T* out, const T* x, const T* residual, const ulonglong2* rng_state, const __grid_constant__ Draw d, uint64_t n) {
    const uint64_t g = (uint64_t)blockIdx.x * kThreads + threadIdx.x;
    const uint64_t i0 = g * 8;
    if (i0 >= n) return;
    const ulonglong2 rng = __ldg(rng_state);
    if (ALIGNED && i0 + 8 <= n) {
        Eight<T> a, r;
#pragma unroll
        for (int k = 0; k < a.kWords; ++k) {
            a.w[k] = sa_load_stream<T, a.kPer>(x + i0 + k * a.kPer);
            if (RESIDUAL) r.w[k] = sa_load_stream<T, a.kPer>(residual + i0 + k * a.kPer);
        }
        const uint32_t keep = keep_mask(g, rng, d);
#pragma unroll
        for (int k = 0; k < a.kWords; ++k) {
#pragma unroll
            for (int j = 0; j < a.kPer; ++j) {
                float v = (keep >> (k * a.kPer + j)) & 1u ? sa_to_float(a.w[k].e[j]) * d.scale : 0.0f;
                if (RESIDUAL) v += sa_to_float(r.w[k].e[j]);
                a.w[k].e[j] = sa_from_float<T>(v);
            }
            sa_store<T, a.kPer>(out + i0 + k * a.kPer, a.w[k]);
        }
    } else {
        const uint32_t keep = keep_mask(g, rng, d);
        for (int j = 0; j < 8 && i0 + j < n; ++j) {
            float v = (keep >> j) & 1u ? sa_to_float(x[i0 + j]) * d.scale : 0.0f;
            if (RESIDUAL) v += sa_to_float(residual[i0 + j]);
            out[i0 + j] = sa_from_float<T>(v);
        }
    }
}

template <class T>
cudaError_t launch(void* out, const void* x, const void* residual, const void* rng, const Draw& d, size_t n, cudaStream_t stream) {
    const bool aligned = sa_common_alignment((uint64_t)out | (uint64_t)x | (uint64_t)residual) == 16;
    const uint64_t blocks = ((n + 7) / 8 + kThreads - 1) / kThreads;
    if (blocks > 0x7fffffffull) return cudaErrorInvalidValue;
    auto k = residual ? (aligned ? sa_dropout_kernel<T, true, true> : sa_dropout_kernel<T, true, false>)
                      : (aligned ? sa_dropout_kernel<T, false, true> : sa_dropout_kernel<T, false, false>);
    k<<<(unsigned)blocks, kThreads, 0, stream>>>((T*)out, (const T*)x, (const T*)residual, (const ulonglong2*)rng, d, n);
    return cudaGetLastError();
}

} // namespace

cudaError_t sa_launch_dropout(void* out, const void* x, const void* residual, const void* rng, double p, size_t n, int dtype,
                              cudaStream_t stream) {
    const uint64_t threshold = (uint64_t)std::llrint(p * 4294967296.0);
    Draw d;
    d.upper = (uint32_t)(threshold >> 16);
    d.lower = (uint32_t)(threshold & 0xffffu);
    d.scale = p < 1.0 ? (float)(1.0 / (1.0 - p)) : 0.0f;
    if (dtype == SA_FP32) return launch<float>(out, x, residual, rng, d, n, stream);
    if (dtype == SA_BF16) return launch<__nv_bfloat16>(out, x, residual, rng, d, n, stream);
    return launch<__half>(out, x, residual, rng, d, n, stream);
}
