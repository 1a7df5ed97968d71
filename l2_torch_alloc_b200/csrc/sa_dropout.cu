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

// U blocks at once: the key's schedule is shared, and so is whatever depends on the call alone.
template <int U>
__device__ __forceinline__ void philox(uint4 (&c)[U], uint32_t k0, uint32_t k1) {
#pragma unroll
    for (int r = 0; r < 10; ++r) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const uint64_t a = (uint64_t)c[u].x * 0xD2511F53u, b = (uint64_t)c[u].z * 0xCD9E8D57u;
            c[u] = make_uint4((uint32_t)(b >> 32) ^ c[u].y ^ k0, (uint32_t)b, (uint32_t)(a >> 32) ^ c[u].w ^ k1, (uint32_t)a);
        }
        k0 += 0x9E3779B9u;
        k1 += 0xBB67AE85u;
    }
}

// Which 16-bit halves of w equal h (given twice): the classic zero-byte test on halves, non-zero if any is.
__device__ __forceinline__ uint32_t equal_halves(uint32_t w, uint32_t hh) {
    const uint32_t x = w ^ hh;
    return (x - 0x00010001u) & ~x & 0x80008000u;
}

// Bit i: element i of group g is kept, once its upper half has tied: the lower half decides.
__device__ __noinline__ uint32_t settle_ties(uint32_t keep, uint4 b, uint64_t g, ulonglong2 rng, uint32_t upper, uint32_t lower) {
    uint4 c[1] = {make_uint4((uint32_t)g, (uint32_t)(g >> 32) | 0x80000000u, (uint32_t)rng.y, (uint32_t)(rng.y >> 32))};
    philox<1>(c, (uint32_t)rng.x, (uint32_t)(rng.x >> 32));
    const uint32_t first[4] = {b.x, b.y, b.z, b.w}, second[4] = {c[0].x, c[0].y, c[0].z, c[0].w};
    for (int i = 0; i < 8; ++i) {
        const int shift = 16 * (i & 1);
        if (((first[i / 2] >> shift) & 0xffffu) == upper && ((second[i / 2] >> shift) & 0xffffu) < lower) keep &= ~(1u << i);
    }
    return keep;
}

// bit i: element i of the group is kept
__device__ __forceinline__ uint32_t keep_mask(const uint4& b, uint64_t g, ulonglong2 rng, const Draw& d) {
    const uint32_t w[4] = {b.x, b.y, b.z, b.w};
    uint32_t keep = 0, tie = 0;
    if (d.upper < 65536u) {
        const uint32_t top = d.upper << 16, twice = top | d.upper;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            keep |= (w[k] << 16) >= top ? 1u << (2 * k) : 0u; // the halves as the upper 16 bits of a word
            keep |= w[k] >= top ? 2u << (2 * k) : 0u;
            tie |= equal_halves(w[k], twice);
        }
        if (tie != 0u && d.lower != 0u) keep = settle_ties(keep, b, g, rng, d.upper, d.lower);
    }
    return keep;
}

// elements of a group in two words of four (fp32) or one word of eight (16 bits)
template <class T>
struct Eight {
    static constexpr int kWords = sizeof(T) / 2, kPer = 8 / kWords;
    SaVec<T, kPer> w[kWords];
    __device__ __forceinline__ void load(const T* p) {
#pragma unroll
        for (int k = 0; k < kWords; ++k) w[k] = sa_load_stream<T, kPer>(p + k * kPer);
    }
};

// U groups of each thread, kThreads groups apart.
template <class T, bool RESIDUAL, int U>
__global__ void __launch_bounds__(kThreads)
sa_dropout_kernel(T* out, const T* x, const T* residual, const ulonglong2* rng_state, const __grid_constant__ Draw d, uint64_t n) {
    const uint64_t g0 = (uint64_t)blockIdx.x * (U * kThreads) + threadIdx.x;
    const ulonglong2 rng = __ldg(rng_state);
    Eight<T> a[U], r[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const uint64_t i0 = (g0 + u * kThreads) * 8;
        if (i0 + 8 <= n) {
            a[u].load(x + i0);
            if (RESIDUAL) r[u].load(residual + i0);
        }
    }
    uint4 c[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const uint64_t g = g0 + u * kThreads;
        c[u] = make_uint4((uint32_t)g, (uint32_t)(g >> 32), (uint32_t)rng.y, (uint32_t)(rng.y >> 32));
    }
    philox<U>(c, (uint32_t)rng.x, (uint32_t)(rng.x >> 32));
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const uint64_t g = g0 + u * kThreads, i0 = g * 8;
        if (i0 >= n) continue;
        const uint32_t keep = keep_mask(c[u], g, rng, d);
        if (i0 + 8 <= n) {
            const F2 scale = f2(d.scale, d.scale);
#pragma unroll
            for (int k = 0; k < Eight<T>::kWords; ++k) {
#pragma unroll
                for (int j = 0; j < Eight<T>::kPer / 2; ++j) {
                    const int e = k * Eight<T>::kPer + 2 * j;
                    float p, q;
                    split(pair_of(a[u].w[k], j) * scale, p, q);
                    F2 v = f2((keep >> e) & 1u ? p : 0.0f, (keep >> e) & 2u ? q : 0.0f);
                    if (RESIDUAL) v = v + pair_of(r[u].w[k], j);
                    set_pair(a[u].w[k], j, v);
                }
                sa_store<T, Eight<T>::kPer>(out + i0 + k * Eight<T>::kPer, a[u].w[k]);
            }
        } else { // the last, partial group
            for (int j = 0; j < 8 && i0 + j < n; ++j) {
                float v = (keep >> j) & 1u ? sa_to_float(x[i0 + j]) * d.scale : 0.0f;
                if (RESIDUAL) v += sa_to_float(residual[i0 + j]);
                out[i0 + j] = sa_from_float<T>(v);
            }
        }
    }
}

// Arrays off a 16-byte boundary, element by element.
template <class T, bool RESIDUAL>
__global__ void __launch_bounds__(kThreads)
sa_dropout_unaligned_kernel(T* out, const T* x, const T* residual, const ulonglong2* rng_state, const __grid_constant__ Draw d, uint64_t n) {
    const uint64_t g = (uint64_t)blockIdx.x * kThreads + threadIdx.x, i0 = g * 8;
    if (i0 >= n) return;
    const ulonglong2 rng = __ldg(rng_state);
    uint4 c[1] = {make_uint4((uint32_t)g, (uint32_t)(g >> 32), (uint32_t)rng.y, (uint32_t)(rng.y >> 32))};
    philox<1>(c, (uint32_t)rng.x, (uint32_t)(rng.x >> 32));
    const uint32_t keep = keep_mask(c[0], g, rng, d);
    for (int j = 0; j < 8 && i0 + j < n; ++j) {
        float v = (keep >> j) & 1u ? sa_to_float(x[i0 + j]) * d.scale : 0.0f;
        if (RESIDUAL) v += sa_to_float(residual[i0 + j]);
        out[i0 + j] = sa_from_float<T>(v);
    }
}

template <class T>
cudaError_t launch(void* out, const void* x, const void* residual, const void* rng, const Draw& d, size_t n, cudaStream_t stream) {
    const bool aligned = sa_common_alignment((uint64_t)out | (uint64_t)x | (uint64_t)residual) == 16;
    const uint64_t groups = (n + 7) / 8;
    // four groups of a thread (two of fp32: 64 bytes of x in flight either way) once that leaves every SM its threads
    constexpr int U = sizeof(T) == 2 ? 4 : 2;
    const int each = !aligned || groups < 148ull * 2048 * U ? 1 : U;
    const uint64_t blocks = (groups + (uint64_t)kThreads * each - 1) / ((uint64_t)kThreads * each);
    if (blocks > 0x7fffffffull) return cudaErrorInvalidValue;
    auto k = !aligned  ? (residual ? sa_dropout_unaligned_kernel<T, true> : sa_dropout_unaligned_kernel<T, false>)
             : each == 1 ? (residual ? sa_dropout_kernel<T, true, 1> : sa_dropout_kernel<T, false, 1>)
                         : (residual ? sa_dropout_kernel<T, true, U> : sa_dropout_kernel<T, false, U>);
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
