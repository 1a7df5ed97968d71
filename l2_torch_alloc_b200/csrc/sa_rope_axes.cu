// Rotary positions with several axes (time, height, width, ...), in place on packed [B, T, Nq + 2 Nkv, HS].
//
// Pair i of a head turns by the angle pos[axis(i)][b][t] * f(i): (x, y) -> (x cos - y sin, x sin + y cos).  Q and K heads
// are turned, V heads and whatever a head holds behind its 2 * pairs turned elements are neither read nor written.
//
// Angles: the spectrum holds f(i) / 2 pi as a 61-bit binary fraction of a turn (the low three bits name the axis), so the
// integer product with the position, modulo 2^64, is the fraction of a turn without a rounding of its own: no table, and an
// error of |position| 2^-62 turns (theta >= 1), so that position 10^6 is as accurate as position 1.  Its upper 32 bits are kept.
// The nearest quarter turn is split off in integers and what is left, at most an eighth of a turn, becomes an fp32 angle (off by
// 2^-26.3 turns, from the conversion, the constant and the product) for Taylor polynomials (truncation below 2e-9).
//
// Bound: HBM, each turned element is read once and written once.  A thread has one place in the head (its cos and sin
// are computed once) and several heads of one token in flight.
#include "sa_elem.cuh"
#include "sa_ops.hpp"

namespace {

constexpr uint32_t kMostThreads = 512;

struct Shape {
    uint32_t tokens, T;               // B * T tokens
    uint32_t heads, head_groups;      // Nq + Nkv; threads of a token and a place = ceil(heads / heads per thread)
    Divisor by_slots;                 // places: words (interleaved) or pairs of words (halves) of a head
    Divisor by_token;                 // threads of a token
    uint32_t tokens_per_block;
    uint32_t axes;
    int HS, pairs;
    int inverse, wide_positions;
    long long stride_b, stride_t, pos_stride_axis, pos_stride_b, pos_stride_t;
};

// cos and sin of `turn` / 2^32 turns
__device__ __forceinline__ void cos_sin_of_turn(uint32_t turn, float& c, float& s) {
    const uint32_t q = (turn + 0x20000000u) >> 30;
    const float x = (float)(int32_t)(turn - (q << 30)) * 1.46291807926715968e-9f; // 2 pi / 2^32
    const float z = x * x;
    float p = fmaf(z, 2.75573192e-6f, -1.98412698e-4f); // 1/9!, -1/7!, 1/5!, -1/3!
    p = fmaf(z, p, 8.33333333e-3f);
    p = fmaf(z, p, -1.66666667e-1f);
    const float sn = fmaf(x * z, p, x);
    float r = fmaf(z, -2.75573192e-7f, 2.48015873e-5f); // -1/10!, 1/8!, -1/6!, 1/4!, -1/2!
    r = fmaf(z, r, -1.38888889e-3f);
    r = fmaf(z, r, 4.16666667e-2f);
    r = fmaf(z, r, -0.5f);
    const float cs = fmaf(z, r, 1.0f);
    c = q & 1u ? sn : cs;
    s = q & 1u ? cs : sn;
    if (((q + 1u) & 2u) != 0u) c = -c; // quarters 1 and 2
    if ((q & 2u) != 0u) s = -s;        // quarters 2 and 3
}

// V elements in words of W
template <class T, int V, int W>
struct Words {
    SaVec<T, W> w[V / W];
    __device__ __forceinline__ void load(const T* p) {
#pragma unroll
        for (int k = 0; k < V / W; ++k) w[k] = sa_load_stream<T, W>(p + k * W);
    }
    __device__ __forceinline__ void store(T* p) const {
#pragma unroll
        for (int k = 0; k < V / W; ++k) sa_store<T, W>(p + k * W, w[k]);
    }
    __device__ __forceinline__ T& operator[](int i) { return w[i / W].e[i % W]; }
};

// (x, y) -> (x cos - y sin, x sin + y cos) for two pairs at once
__device__ __forceinline__ void turn(F2& x, F2& y, F2 c, F2 s) {
    const F2 a = fma2(x, c, negative(y * s));
    y = fma2(x, s, y * c);
    x = a;
}
template <class T>
__device__ __forceinline__ void turn(T& xa, T& ya, T& xb, T& yb, F2 c, F2 s) {
    F2 x = f2(sa_to_float(xa), sa_to_float(xb)), y = f2(sa_to_float(ya), sa_to_float(yb));
    turn(x, y, c, s);
    float p, q;
    split(x, p, q);
    xa = sa_from_float<T>(p);
    xb = sa_from_float<T>(q);
    split(y, p, q);
    ya = sa_from_float<T>(p);
    yb = sa_from_float<T>(q);
}

// HALVES: pair i = elements (i, i + pairs), a thread has two words of V elements (V pairs) of each of U heads;
// else pair i = elements (2 i, 2 i + 1), one word of V elements (V / 2 pairs) of each of U heads.
template <class T, int V, int W, bool HALVES, int U>
__global__ void __launch_bounds__(kMostThreads, 2)
sa_rope_axes_kernel(T* __restrict__ x, const void* __restrict__ positions, const unsigned long long* __restrict__ spectrum,
                    const __grid_constant__ Shape sh) {
    constexpr int kPairs = HALVES ? V : V / 2;
    constexpr int kParts = HALVES ? 2 : 1;
    const uint32_t local = blockIdx.y * blockDim.x + threadIdx.x;
    const uint32_t in_block = sh.tokens_per_block > 1 ? sh.by_token.div(local) : local >= sh.by_token.d ? 1u : 0u;
    const uint32_t unit = local - in_block * sh.by_token.d;
    const uint32_t token = blockIdx.x * sh.tokens_per_block + in_block;
    if (in_block >= sh.tokens_per_block || token >= sh.tokens) return;
    const uint32_t hg = sh.by_slots.div(unit), slot = unit - hg * sh.by_slots.d;
    const uint32_t b = token < sh.T ? 0u : token / sh.T, t = token - b * sh.T;
    T* const row = x + b * sh.stride_b + t * sh.stride_t + slot * V + hg * (uint32_t)sh.HS;
    const uint32_t step = sh.head_groups * (uint32_t)sh.HS; // from one of this thread's heads to the next

    Words<T, V, W> v[U][kParts];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        if (hg + u * sh.head_groups < sh.heads) {
#pragma unroll
            for (int k = 0; k < kParts; ++k) v[u][k].load(row + u * step + k * sh.pairs);
        }
    }
    float c[kPairs], s[kPairs];
    const long long place = b * sh.pos_stride_b + t * sh.pos_stride_t;
    uint32_t have = 0xffffffffu; // neighbouring pairs mostly share their axis
    bool lacking = false;
    long long pos = 0;
#pragma unroll
    for (int i = 0; i < kPairs; ++i) {
        const unsigned long long f = __ldg(spectrum + slot * kPairs + i);
        const uint32_t axis = (uint32_t)f & 7u;
        if (axis != have) {
            lacking |= axis >= sh.axes;
            const long long at = place + (axis < sh.axes ? axis : 0u) * sh.pos_stride_axis;
            pos = sh.wide_positions ? __ldg(static_cast<const long long*>(positions) + at)
                                    : (long long)__ldg(static_cast<const int*>(positions) + at);
            have = axis;
        }
        const unsigned long long product = (unsigned long long)pos * (f & ~7ull);
        cos_sin_of_turn((uint32_t)(product >> 32), c[i], s[i]);
    }
    // a spectrum of other positions: no number rather than a wrong one
    const float direction = lacking ? __int_as_float(0x7fffffff) : sh.inverse ? -1.0f : 1.0f;
#pragma unroll
    for (int i = 0; i < kPairs; ++i) s[i] *= direction;
    if constexpr (HALVES && V > 1) { // two neighbouring pairs of a head at a time
#pragma unroll
        for (int u = 0; u < U; ++u) {
#pragma unroll
            for (int i = 0; i < V; i += 2)
                turn(v[u][0][i], v[u][1][i], v[u][0][i + 1], v[u][1][i + 1], f2(c[i], c[i + 1]), f2(s[i], s[i + 1]));
        }
    } else { // the same pair of two heads at a time
#pragma unroll
        for (int u = 0; u < U; u += 2) {
#pragma unroll
            for (int i = 0; i < kPairs; ++i) {
                constexpr int y = HALVES ? kParts - 1 : 0;
                const int xi = HALVES ? i : 2 * i, yi = HALVES ? i : 2 * i + 1;
                turn(v[u][0][xi], v[u][y][yi], v[u + 1][0][xi], v[u + 1][y][yi], f2(c[i], c[i]), f2(s[i], s[i]));
            }
        }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
        if (hg + u * sh.head_groups < sh.heads) {
#pragma unroll
            for (int k = 0; k < kParts; ++k) v[u][k].store(row + u * step + k * sh.pairs);
        }
    }
}

template <class T, int V, int W, bool HALVES>
cudaError_t launch(void* qkv, const void* positions, const void* spectrum, Shape s, cudaStream_t stream) {
    constexpr int U = V * (int)sizeof(T) == 16 && HALVES ? 2 : 4; // 64 bytes of each thread are in flight, 32 of narrow words
    const uint32_t slots = (uint32_t)(HALVES ? s.pairs / V : 2 * s.pairs / V);
    s.head_groups = (s.heads + U - 1) / U;
    // at most 256 places and 65,536 heads: 2^22 threads of a token, so 2^14 blocks of it and divisions of up to 2^30
    const uint32_t per_token = slots * s.head_groups;
    s.by_slots = divisor(slots);
    s.by_token = divisor(per_token);
    uint32_t threads, rows = 1; // blocks of 160 threads or a little more (256: 7 % slower on 65,536 tokens): whole tokens, or a part of one
    if (per_token <= kMostThreads) {
        s.tokens_per_block = (160 + per_token - 1) / per_token;
        if (s.tokens_per_block * per_token > kMostThreads) s.tokens_per_block = 1;
        threads = (s.tokens_per_block * per_token + 31) / 32 * 32;
    } else {
        s.tokens_per_block = 1;
        rows = (per_token + 255) / 256;
        threads = ((per_token + rows - 1) / rows + 31) / 32 * 32;
    }
    const uint32_t blocks = (s.tokens + s.tokens_per_block - 1) / s.tokens_per_block;
    sa_rope_axes_kernel<T, V, W, HALVES, U><<<dim3(blocks, rows), threads, 0, stream>>>(
        (T*)qkv, positions, (const unsigned long long*)spectrum, s);
    return cudaGetLastError();
}

// Words as wide as the addresses, strides, heads and runs of pairs allow.
template <class T>
cudaError_t launch_type(void* qkv, const void* positions, const void* spectrum, const Shape& s, bool halves, cudaStream_t stream) {
    const uint64_t e = sizeof(T);
    const int a = sa_common_alignment((uint64_t)qkv | (uint64_t)s.stride_b * e | (uint64_t)s.stride_t * e | (uint64_t)s.HS * e |
                                      (uint64_t)s.pairs * e * (halves ? 1 : 2));
    constexpr int V16 = 16 / (int)sizeof(T), V8 = 8 / (int)sizeof(T);
    if (halves) {
        if (a == 16) return launch<T, V16, V16, true>(qkv, positions, spectrum, s, stream);
        if (a == 8) return launch<T, V8, V8, true>(qkv, positions, spectrum, s, stream);
        return launch<T, 1, 1, true>(qkv, positions, spectrum, s, stream);
    }
    if (a == 16) return launch<T, V16, V16, false>(qkv, positions, spectrum, s, stream);
    if (a == 8) return launch<T, V8, V8, false>(qkv, positions, spectrum, s, stream);
    return launch<T, 2, 1, false>(qkv, positions, spectrum, s, stream);
}

struct Turns {
    unsigned long long v[256];
};

__global__ void sa_rope_axes_spectrum_kernel(unsigned long long* spectrum, const __grid_constant__ Turns turns, int pairs) {
    for (int i = threadIdx.x; i < pairs; i += blockDim.x) spectrum[i] = turns.v[i];
}

} // namespace

cudaError_t sa_launch_rope_axes(void* qkv, const void* positions, const void* spectrum, const sideaware_rope_axes_t& sh,
                                bool inverse, cudaStream_t stream) {
    Shape s{};
    s.tokens = (uint32_t)((uint64_t)sh.B * (uint64_t)sh.T);
    s.T = (uint32_t)sh.T;
    s.heads = (uint32_t)(sh.Nq + sh.Nkv);
    s.axes = (uint32_t)sh.axes;
    s.HS = sh.HS;
    s.pairs = sh.pairs;
    s.inverse = inverse ? 1 : 0;
    s.wide_positions = sh.position_dtype;
    s.stride_b = sh.B > 1 ? sh.stride_b : 0;
    s.stride_t = sh.T > 1 ? sh.stride_t : 0;
    s.pos_stride_axis = sh.pos_stride_axis;
    s.pos_stride_b = sh.pos_stride_b;
    s.pos_stride_t = sh.pos_stride_t;
    const bool halves = sh.layout == 1;
    if (sh.dtype == SA_FP32) return launch_type<float>(qkv, positions, spectrum, s, halves, stream);
    if (sh.dtype == SA_BF16) return launch_type<__nv_bfloat16>(qkv, positions, spectrum, s, halves, stream);
    return launch_type<__half>(qkv, positions, spectrum, s, halves, stream);
}

cudaError_t sa_launch_rope_axes_spectrum(void* spectrum, const uint64_t* turns, int pairs, cudaStream_t stream) {
    Turns t{};
    for (int i = 0; i < pairs; ++i) t.v[i] = turns[i];
    sa_rope_axes_spectrum_kernel<<<1, 256, 0, stream>>>((unsigned long long*)spectrum, t, pairs);
    return cudaGetLastError();
}
