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

// Whether one of the eight 16-bit halves of b equals `upper` (and there is a lower half to look at): the halves' differences
// by exclusive or, their minimum two at a time, then the classic test for a zero half.
__device__ __forceinline__ bool has_tie(const uint4& b, const Draw& d) {
    const uint32_t twice = d.upper << 16 | d.upper;
    uint32_t m = b.x ^ twice;
    asm("min.u16x2 %0, %0, %1;" : "+r"(m) : "r"(b.y ^ twice));
    asm("min.u16x2 %0, %0, %1;" : "+r"(m) : "r"(b.z ^ twice));
    asm("min.u16x2 %0, %0, %1;" : "+r"(m) : "r"(b.w ^ twice));
    return ((m - 0x00010001u) & ~m & 0x80008000u) != 0u && d.upper < 65536u && d.lower != 0u;
}

// bit i: element i of group g is kept, with both halves of its number
__device__ __noinline__ uint32_t exact_mask(uint4 b, uint64_t g, ulonglong2 rng, uint32_t upper, uint32_t lower) {
    uint4 c[1] = {make_uint4((uint32_t)g, (uint32_t)(g >> 32) | 0x80000000u, (uint32_t)rng.y, (uint32_t)(rng.y >> 32))};
    philox<1>(c, (uint32_t)rng.x, (uint32_t)(rng.x >> 32));
    const uint32_t first[4] = {b.x, b.y, b.z, b.w}, second[4] = {c[0].x, c[0].y, c[0].z, c[0].w};
    uint32_t keep = 0;
    for (int i = 0; i < 8; ++i) {
        const int shift = 16 * (i & 1);
        const uint32_t u = (first[i / 2] >> shift) & 0xffffu, v = (second[i / 2] >> shift) & 0xffffu;
        if (u > upper || (u == upper && v >= lower)) keep |= 1u << i;
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

// A group's results; kept(i): element i is kept.
template <class T, bool RESIDUAL, class F>
__device__ __forceinline__ void finish(T* out, Eight<T>& a, const Eight<T>& r, float scale, F&& kept) {
    const F2 both = f2(scale, scale);
#pragma unroll
    for (int k = 0; k < Eight<T>::kWords; ++k) {
#pragma unroll
        for (int j = 0; j < Eight<T>::kPer / 2; ++j) {
            const int e = k * Eight<T>::kPer + 2 * j;
            float p, q;
            split(pair_of(a.w[k], j) * both, p, q);
            F2 v = f2(kept(e) ? p : 0.0f, kept(e + 1) ? q : 0.0f);
            if (RESIDUAL) v = v + pair_of(r.w[k], j);
            set_pair(a.w[k], j, v);
        }
        sa_store_stream<T, Eight<T>::kPer>(out + k * Eight<T>::kPer, a.w[k]);
    }
}

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
    const uint32_t top = d.upper << 16; // a half against `upper`, both as the upper half of a word
    const bool none = d.upper >= 65536u;
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const uint64_t g = g0 + u * kThreads, i0 = g * 8;
        if (i0 + 8 <= n) {
            if (none || has_tie(c[u], d)) {
                const uint32_t keep = none ? 0u : exact_mask(c[u], g, rng, d.upper, d.lower);
                finish<T, RESIDUAL>(out + i0, a[u], r[u], d.scale, [&](int i) { return (keep >> i) & 1u; });
            } else {
                const uint32_t w[4] = {c[u].x, c[u].y, c[u].z, c[u].w};
                finish<T, RESIDUAL>(out + i0, a[u], r[u], d.scale, [&](int i) { return (i & 1 ? w[i / 2] : w[i / 2] << 16) >= top; });
            }
        } else if (i0 < n) { // the last, partial group
            const uint32_t keep = none ? 0u : exact_mask(c[u], g, rng, d.upper, d.lower);
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
    const uint32_t keep = d.upper >= 65536u ? 0u : exact_mask(c[0], g, rng, d.upper, d.lower);
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
    // two groups of a thread share the key schedule once that leaves every SM its threads (four: 5 % slower, the registers cost
    // warps); fp32 moves twice the bytes for the same numbers and is 3 % faster with one
    constexpr int U = sizeof(T) == 2 ? 2 : 1;
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
