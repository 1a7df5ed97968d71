// Group norm with an optional SiLU, channels last: x [N, S, C], groups of D = C / G neighbouring channels.
//
//   mean, rstd = 1 / sqrt(var + eps) over the S * D elements of (n, g);  z = (x - mean) rstd w + b;  y = z or z sigmoid(z)
//
// Backward, with u = (x - mean) rstd, dz = dy act'(z), A[n][c] = sum_s dz, B[n][c] = sum_s dz u:
//   dbias = sum_n A, dweight = sum_n B,
//   dx = rstd (w dz - m1 - u m2), m1 = sum_{c in g} w A / (S D), m2 = sum_{c in g} w B / (S D)
//
// Statistics: a thread takes the exact two-step mean and squared deviation of a few rows at a time and joins them with
// the pairwise update of Chan, Golub and LeVeque (1983), all in fp32: no cancellation however far the mean is from zero.
// All sums go through fixed trees (no atomics): the same inputs give the same bits.
//
// Two ways, chosen by plan_resident below:
//  * resident: a thread-block cluster owns some neighbouring groups of one sample, all rows of them lie in the shared
//    memory of its blocks, which exchange their statistics through distributed shared memory.  One launch, each element
//    is read once and written once.
//  * for samples too long for that, three launches: partial statistics of runs of rows, joining them, applying them.
#include <cooperative_groups.h>

#include <type_traits>

#include "sa_elem.cuh"
#include "sa_ops.hpp"

namespace cg = cooperative_groups;

namespace {

constexpr int kThreads = 256;
constexpr int kResidentThreads = 512, kResidentBackwardThreads = 256; // threads of a resident block, at most
constexpr int kBatch = 8; // rows whose statistics a thread takes in one go

struct Norm {
    long long S, C;         // rows of a sample, channels
    int G, D;               // groups, channels of a group
    int splits;             // runs of rows a sample is cut into
    long long rows;         // rows of a run (the last one may be shorter)
    int columns, row_lanes; // words across a block's tile, rows it takes at a time
    int N;
    int silu, param_dtype;
    float eps;
    const void* weight;
    const void* bias;
};

// V neighbouring entries of a parameter vector, `missing` where there is none.  One branch on the type, then V loads
// that are in flight together.
template <int V>
__device__ __forceinline__ void load_params(float (&out)[V], const void* p, long long c0, int dtype, float missing) {
    if (!p) {
#pragma unroll
        for (int i = 0; i < V; ++i) out[i] = missing;
    } else if (dtype == SA_FP32) {
#pragma unroll
        for (int i = 0; i < V; ++i) out[i] = static_cast<const float*>(p)[c0 + i];
    } else if (dtype == SA_BF16) {
#pragma unroll
        for (int i = 0; i < V; ++i) out[i] = __bfloat162float(static_cast<const __nv_bfloat16*>(p)[c0 + i]);
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i) out[i] = __half2float(static_cast<const __half*>(p)[c0 + i]);
    }
}

// mean and sum of squared deviations of `n` values
struct Moments {
    float n, mean, m2;
};

__device__ __forceinline__ void join(Moments& a, const Moments& b) {
    const float n = a.n + b.n;
    if (n == 0.0f) return;
    const float d = b.mean - a.mean, f = __fdividef(b.n, n); // a weight: two roundings more do no harm
    a.mean = fmaf(d, f, a.mean);
    a.m2 += b.m2 + d * d * a.n * f;
    a.n = n;
}

// sigmoid: fp32 storage wants all of fp32, for 16-bit storage the fast forms' 2^-21 is far below a rounding
template <class T>
__device__ __forceinline__ float sigmoid(float z) {
    if constexpr (sizeof(T) == 4) return 1.0f / (1.0f + expf(-z));
    return __fdividef(1.0f, 1.0f + __expf(-z));
}

template <class T>
__device__ __forceinline__ float activate(float z, int silu) {
    return silu ? z * sigmoid<T>(z) : z;
}

// dy act'(z)
template <class T>
__device__ __forceinline__ float through_activation(float dy, float z, int silu) {
    if (!silu) return dy;
    const float s = sigmoid<T>(z);
    return dy * (s * fmaf(z, 1.0f - s, 1.0f));
}

// ---------------------------------------------------------------------------
// forward
// ---------------------------------------------------------------------------
// partial[n][split][c] = (mean, m2) of channel c over the run's rows
template <class T, int V>
__global__ void __launch_bounds__(kThreads)
sa_norm_partial_kernel(const T* __restrict__ x, float2* __restrict__ partial, const __grid_constant__ Norm p) {
    __shared__ float2 tile[kThreads * V];
    __shared__ float count[kThreads];
    const int lane_column = threadIdx.x % p.columns, row_lane = threadIdx.x / p.columns;
    const long long c0 = ((long long)blockIdx.y * p.columns + lane_column) * V;
    const int split = blockIdx.x % p.splits, n = blockIdx.x / p.splits;
    const long long first = split * p.rows, end = min(first + p.rows, p.S);
    const bool mine = row_lane < p.row_lanes && c0 < p.C;
    Moments a[V];
#pragma unroll
    for (int i = 0; i < V; ++i) a[i] = Moments{0.0f, 0.0f, 0.0f};
    if (mine) {
        const T* base = x + ((long long)n * p.S) * p.C + c0;
        for (long long s = first + row_lane; s < end; s += (long long)kBatch * p.row_lanes) {
            SaVec<T, V> v[kBatch];
            int have = 0;
#pragma unroll
            for (int k = 0; k < kBatch; ++k)
                if (s + (long long)k * p.row_lanes < end) {
                    v[k] = sa_load<T, V>(base + (s + (long long)k * p.row_lanes) * p.C);
                    have = k + 1;
                }
            const float inv = 1.0f / (float)have;
#pragma unroll
            for (int i = 0; i < V; ++i) {
                float sum = 0.0f, m2 = 0.0f;
#pragma unroll
                for (int k = 0; k < kBatch; ++k) sum += k < have ? sa_to_float(v[k].e[i]) : 0.0f;
                const float mean = sum * inv;
#pragma unroll
                for (int k = 0; k < kBatch; ++k) {
                    const float d = k < have ? sa_to_float(v[k].e[i]) - mean : 0.0f;
                    m2 = fmaf(d, d, m2);
                }
                join(a[i], Moments{(float)have, mean, m2});
            }
        }
    }
    count[threadIdx.x] = mine ? a[0].n : 0.0f;
#pragma unroll
    for (int i = 0; i < V; ++i) tile[threadIdx.x * V + i] = make_float2(a[i].mean, a[i].m2);
    __syncthreads();
    // the tile's channels, each over its row lanes
    for (int j = threadIdx.x; j < p.columns * V; j += kThreads) {
        const long long c = (long long)blockIdx.y * p.columns * V + j;
        if (c >= p.C) continue;
        Moments m{0.0f, 0.0f, 0.0f};
        for (int r = 0; r < p.row_lanes; ++r) {
            const int t = r * p.columns + j / V;
            const float2 e = tile[t * V + j % V];
            join(m, Moments{count[t], e.x, e.y});
        }
        partial[((long long)n * p.splits + split) * p.C + c] = make_float2(m.mean, m.m2);
    }
}

__device__ __forceinline__ Moments warp_join(Moments m) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const Moments b{__shfl_down_sync(0xffffffffu, m.n, o), __shfl_down_sync(0xffffffffu, m.mean, o), __shfl_down_sync(0xffffffffu, m.m2, o)};
        join(m, b);
    }
    return m;
}

// mean and rstd of (n, g): one block each
__global__ void __launch_bounds__(kThreads)
sa_norm_join_kernel(const float2* __restrict__ partial, float* __restrict__ mean, float* __restrict__ rstd, const __grid_constant__ Norm p) {
    __shared__ Moments warps[kThreads / 32];
    const int n = blockIdx.x / p.G, g = blockIdx.x % p.G;
    Moments m{0.0f, 0.0f, 0.0f};
    const long long entries = (long long)p.splits * p.D;
    for (long long i = threadIdx.x; i < entries; i += kThreads) {
        const long long split = i / p.D;
        const long long rows = min(p.rows, p.S - split * p.rows);
        const float2 e = partial[((long long)n * p.splits + split) * p.C + (long long)g * p.D + i % p.D];
        join(m, Moments{(float)rows, e.x, e.y});
    }
    m = warp_join(m);
    if (threadIdx.x % 32 == 0) warps[threadIdx.x / 32] = m;
    __syncthreads();
    if (threadIdx.x < 32) {
        m = threadIdx.x < kThreads / 32 ? warps[threadIdx.x] : Moments{0.0f, 0.0f, 0.0f};
        m = warp_join(m);
        if (threadIdx.x == 0) {
            mean[blockIdx.x] = m.mean;
            rstd[blockIdx.x] = 1.0f / sqrtf(m.m2 / m.n + p.eps);
        }
    }
}

template <class T, int V>
__global__ void __launch_bounds__(kThreads)
sa_norm_apply_kernel(T* out, const T* x, const float* __restrict__ mean, const float* __restrict__ rstd, const __grid_constant__ Norm p) {
    const int lane_column = threadIdx.x % p.columns, row_lane = threadIdx.x / p.columns;
    const long long c0 = ((long long)blockIdx.y * p.columns + lane_column) * V;
    if (row_lane >= p.row_lanes || c0 >= p.C) return;
    const int split = blockIdx.x % p.splits, n = blockIdx.x / p.splits;
    float m[V], a[V], b[V];
    load_params<V>(a, p.weight, c0, p.param_dtype, 1.0f);
    load_params<V>(b, p.bias, c0, p.param_dtype, 0.0f);
#pragma unroll
    for (int i = 0; i < V; ++i) {
        const long long at = (long long)n * p.G + (uint32_t)(c0 + i) / (uint32_t)p.D;
        m[i] = mean[at];
        a[i] *= rstd[at];
    }
    const long long first = split * p.rows, end = min(first + p.rows, p.S);
    const long long base = (long long)n * p.S * p.C + c0;
#pragma unroll 4
    for (long long s = first + row_lane; s < end; s += p.row_lanes) {
        SaVec<T, V> v = sa_load_stream<T, V>(x + base + s * p.C);
#pragma unroll
        for (int i = 0; i < V; ++i)
            v.e[i] = sa_from_float<T>(activate<T>(fmaf(sa_to_float(v.e[i]) - m[i], a[i], b[i]), p.silu));
        sa_store<T, V>(out + base + s * p.C, v);
    }
}

// ---------------------------------------------------------------------------
// backward
// ---------------------------------------------------------------------------
// partial[n][split][c] = (sum dz, sum dz u) over the run's rows
template <class T, int V>
__global__ void __launch_bounds__(kThreads)
sa_norm_backward_partial_kernel(const T* __restrict__ dout, const T* __restrict__ x, const float* __restrict__ mean,
                                const float* __restrict__ rstd, float2* __restrict__ partial, const __grid_constant__ Norm p) {
    __shared__ float2 tile[kThreads * V];
    const int lane_column = threadIdx.x % p.columns, row_lane = threadIdx.x / p.columns;
    const long long c0 = ((long long)blockIdx.y * p.columns + lane_column) * V;
    const int split = blockIdx.x % p.splits, n = blockIdx.x / p.splits;
    const long long first = split * p.rows, end = min(first + p.rows, p.S);
    const bool mine = row_lane < p.row_lanes && c0 < p.C;
    float sa[V], sb[V];
#pragma unroll
    for (int i = 0; i < V; ++i) sa[i] = sb[i] = 0.0f;
    if (mine) {
        float m[V], r[V], w[V], b[V];
        load_params<V>(w, p.weight, c0, p.param_dtype, 1.0f);
        load_params<V>(b, p.bias, c0, p.param_dtype, 0.0f);
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const long long at = (long long)n * p.G + (uint32_t)(c0 + i) / (uint32_t)p.D;
            m[i] = mean[at];
            r[i] = rstd[at];
        }
        const long long base = (long long)n * p.S * p.C + c0;
#pragma unroll 4
        for (long long s = first + row_lane; s < end; s += p.row_lanes) {
            const SaVec<T, V> vx = sa_load<T, V>(x + base + s * p.C), vd = sa_load<T, V>(dout + base + s * p.C);
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const float u = (sa_to_float(vx.e[i]) - m[i]) * r[i];
                const float dz = through_activation<T>(sa_to_float(vd.e[i]), fmaf(u, w[i], b[i]), p.silu);
                sa[i] += dz;
                sb[i] = fmaf(dz, u, sb[i]);
            }
        }
    }
#pragma unroll
    for (int i = 0; i < V; ++i) tile[threadIdx.x * V + i] = make_float2(sa[i], sb[i]);
    __syncthreads();
    for (int j = threadIdx.x; j < p.columns * V; j += kThreads) {
        const long long c = (long long)blockIdx.y * p.columns * V + j;
        if (c >= p.C) continue;
        float2 sum = make_float2(0.0f, 0.0f);
        for (int q = 0; q < p.row_lanes; ++q) {
            const float2 e = tile[(q * p.columns + j / V) * V + j % V];
            sum.x += e.x;
            sum.y += e.y;
        }
        partial[((long long)n * p.splits + split) * p.C + c] = sum;
    }
}

// sums[n][c] over the runs, and of every (n, g) m1 and m2: one block each
__global__ void __launch_bounds__(kThreads)
sa_norm_backward_join_kernel(const float2* __restrict__ partial, float2* __restrict__ sums, float2* __restrict__ means,
                             const __grid_constant__ Norm p) {
    __shared__ float2 warps[kThreads / 32];
    const int n = blockIdx.x / p.G, g = blockIdx.x % p.G;
    float2 m = make_float2(0.0f, 0.0f);
    for (int d = threadIdx.x; d < p.D; d += kThreads) {
        const long long c = (long long)g * p.D + d;
        float2 s = make_float2(0.0f, 0.0f);
        for (int k = 0; k < p.splits; ++k) {
            const float2 e = partial[((long long)n * p.splits + k) * p.C + c];
            s.x += e.x;
            s.y += e.y;
        }
        sums[(long long)n * p.C + c] = s;
        const float w = p.weight ? sa_param(p.weight, c, p.param_dtype) : 1.0f;
        m.x = fmaf(w, s.x, m.x);
        m.y = fmaf(w, s.y, m.y);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        m.x += __shfl_down_sync(0xffffffffu, m.x, o);
        m.y += __shfl_down_sync(0xffffffffu, m.y, o);
    }
    if (threadIdx.x % 32 == 0) warps[threadIdx.x / 32] = m;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int k = 1; k < kThreads / 32; ++k) {
            m.x += warps[k].x;
            m.y += warps[k].y;
        }
        const float inv = 1.0f / ((float)p.S * (float)p.D);
        means[blockIdx.x] = make_float2(m.x * inv, m.y * inv);
    }
}

__global__ void __launch_bounds__(kThreads)
sa_norm_backward_params_kernel(const float2* __restrict__ sums, void* __restrict__ dweight, void* __restrict__ dbias, const __grid_constant__ Norm p) {
    const long long c = (long long)blockIdx.x * kThreads + threadIdx.x;
    if (c >= p.C) return;
    float2 s = make_float2(0.0f, 0.0f);
    for (int n = 0; n < p.N; ++n) {
        const float2 e = sums[(long long)n * p.C + c];
        s.x += e.x;
        s.y += e.y;
    }
    if (dbias) sa_set_param(dbias, c, p.param_dtype, s.x);
    if (dweight) sa_set_param(dweight, c, p.param_dtype, s.y);
}

template <class T, int V>
__global__ void __launch_bounds__(kThreads)
sa_norm_backward_apply_kernel(T* dx, const T* dout, const T* x, const float* __restrict__ mean, const float* __restrict__ rstd,
                              const float2* __restrict__ means, const __grid_constant__ Norm p) {
    const int lane_column = threadIdx.x % p.columns, row_lane = threadIdx.x / p.columns;
    const long long c0 = ((long long)blockIdx.y * p.columns + lane_column) * V;
    if (row_lane >= p.row_lanes || c0 >= p.C) return;
    const int split = blockIdx.x % p.splits, n = blockIdx.x / p.splits;
    float m[V], r[V], w[V], b[V], m1[V], m2[V];
    load_params<V>(w, p.weight, c0, p.param_dtype, 1.0f);
    load_params<V>(b, p.bias, c0, p.param_dtype, 0.0f);
#pragma unroll
    for (int i = 0; i < V; ++i) {
        const long long at = (long long)n * p.G + (uint32_t)(c0 + i) / (uint32_t)p.D;
        m[i] = mean[at];
        r[i] = rstd[at];
        m1[i] = means[at].x;
        m2[i] = means[at].y;
    }
    const long long first = split * p.rows, end = min(first + p.rows, p.S);
    const long long base = (long long)n * p.S * p.C + c0;
#pragma unroll 2
    for (long long s = first + row_lane; s < end; s += p.row_lanes) {
        const SaVec<T, V> vx = sa_load_stream<T, V>(x + base + s * p.C), vd = sa_load_stream<T, V>(dout + base + s * p.C);
        SaVec<T, V> o;
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const float u = (sa_to_float(vx.e[i]) - m[i]) * r[i];
            const float dz = through_activation<T>(sa_to_float(vd.e[i]), fmaf(u, w[i], b[i]), p.silu);
            o.e[i] = sa_from_float<T>(r[i] * (fmaf(w[i], dz, -m1[i]) - u * m2[i]));
        }
        sa_store<T, V>(dx + base + s * p.C, o);
    }
}

// ---------------------------------------------------------------------------
// resident: a cluster for a slab of groups of one sample
// ---------------------------------------------------------------------------
struct Slab {
    Norm p;
    int groups, width;     // groups of a slab, its channels = groups * D, a whole number of words
    int words;             // words of a row
    int row_lanes;         // rows a block takes at a time: a thread has one word of every row_lanes-th row
    int slabs;             // of a sample
    int blocks;            // of a cluster
    int rows;              // of a block
    int parts;             // threads that share a channel's column when the block's threads are joined
    int threads;
    Divisor by_words, by_width, by_D;
    size_t shared;         // bytes of shared memory of a block
};

// What this block and thread work on.
struct Place {
    int n, rank;
    int word, row_lane;
    int channels, groups; // of this slab (the last one of a sample may be narrower)
    long long first;      // first channel of the slab
    int group0;           // first group of the slab
    int block_rows;       // of this block
    int rows;             // of this thread: row_lane, row_lane + row_lanes, ...
};

template <int V>
__device__ __forceinline__ Place place_of(const Slab& s) {
    Place w;
    const uint32_t cluster = s.blocks > 1 ? blockIdx.x / (uint32_t)s.blocks : blockIdx.x;
    w.rank = (int)(blockIdx.x - cluster * s.blocks);
    w.n = (int)(cluster / (uint32_t)s.slabs);
    const int slab = (int)cluster - w.n * s.slabs;
    w.row_lane = (int)s.by_words.div(threadIdx.x);
    w.word = (int)threadIdx.x - w.row_lane * s.words;
    w.group0 = slab * s.groups;
    w.first = (long long)slab * s.width;
    w.groups = min(s.groups, s.p.G - w.group0);
    w.channels = w.groups * s.p.D;
    w.block_rows = max(0, min(s.rows, (int)s.p.S - w.rank * s.rows)); // a sample that fits is short
    const int left = w.block_rows - w.row_lane;
    w.rows = w.row_lane < s.row_lanes && w.word * V < w.channels && left > 0 ? (left + s.row_lanes - 1) / s.row_lanes : 0;
    return w;
}

// This thread's words of its block's rows from global into shared memory, without passing through registers (words of 4
// bytes or more); complete for this thread after wait_for_rows.  The rows come in kStages groups, so that the first ones can
// be worked on while the others travel.
constexpr int kStages = 4;
__device__ __forceinline__ int stage_end(int rows, int stage) { return stage == kStages - 1 ? rows : rows * (stage + 1) / kStages; }

template <class T, int V>
__device__ __forceinline__ void fetch_rows(SaVec<T, V>* to, const T* from, int rows, int stride, long long step) {
#pragma unroll 4
    for (int u = 0; u < rows; ++u, to += stride, from += step) {
        if constexpr (sizeof(SaVec<T, V>) == 16)
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"((uint32_t)__cvta_generic_to_shared(to)), "l"(from) : "memory");
        else if constexpr (sizeof(SaVec<T, V>) >= 4)
            asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"((uint32_t)__cvta_generic_to_shared(to)), "l"(from), "n"(sizeof(SaVec<T, V>)) : "memory");
        else
            *to = sa_load<T, V>(from);
    }
}
__device__ __forceinline__ void end_of_stage() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int STAGE>
__device__ __forceinline__ void wait_for_stage() {
    asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 1 - STAGE) : "memory");
}
// f(first row, end) for every stage's rows as they arrive
template <class F>
__device__ __forceinline__ void as_rows_arrive(int rows, F&& f) {
    wait_for_stage<0>();
    f(0, stage_end(rows, 0));
    wait_for_stage<1>();
    f(stage_end(rows, 0), stage_end(rows, 1));
    wait_for_stage<2>();
    f(stage_end(rows, 1), stage_end(rows, 2));
    wait_for_stage<3>();
    f(stage_end(rows, 2), rows);
}

// V floats of shared memory as pairs
template <int V>
__device__ __forceinline__ void shared_pairs(F2 (&out)[(V + 1) / 2], const float* p) {
#pragma unroll
    for (int k = 0; k < (V + 1) / 2; ++k) out[k] = f2(p[2 * k], 2 * k + 1 < V ? p[2 * k + 1] : 0.0f);
}

// 16-bit storage: one reciprocal for both, 1 / a = b / (a b).  The special-function unit is what an activation waits for (8
// cycles a warp and operation), so 1.5 of them for each element instead of 2.  The exponent is held below 60 so that a b stays
// finite: sigmoid is off by less than 1e-18 beyond that.
template <class T>
__device__ __forceinline__ F2 sigmoid2(F2 z) {
    float x, y;
    if constexpr (sizeof(T) == 4) {
        split(z, x, y);
        return f2(sigmoid<T>(x), sigmoid<T>(y));
    }
    split(z * f2(-1.44269504f, -1.44269504f), x, y); // -log2 e
    x = fminf(x, 60.0f);
    y = fminf(y, 60.0f);
    asm("ex2.approx.ftz.f32 %0, %0;" : "+f"(x));
    asm("ex2.approx.ftz.f32 %0, %0;" : "+f"(y));
    split(f2(x, y) + f2(1.0f, 1.0f), x, y);
    float r = x * y;
    asm("rcp.approx.ftz.f32 %0, %0;" : "+f"(r));
    return f2(r, r) * f2(y, x);
}

// dy act'(z)
template <class T>
__device__ __forceinline__ F2 through_activation2(F2 dy, F2 z, int silu) {
    if (!silu) return dy;
    const F2 sg = sigmoid2<T>(z), one = f2(1.0f, 1.0f);
    return dy * (sg * fma2(z, one + negative(sg), one));
}

// A channel's row lanes, `parts` threads for each channel; the sum stands in the first row of each share.
__device__ __forceinline__ void column_sums(const Slab& s, int lanes, float2* tile) {
    for (int j = threadIdx.x; j < s.parts * s.width; j += blockDim.x) {
        const int part = s.parts > 1 ? (int)s.by_width.div(j) : 0; // j = part * width + channel
        float2 t = tile[j];
        const float2* e = tile + j;
        for (int r = part + s.parts; r < lanes; r += s.parts) {
            e += s.parts * s.width;
            t.x += e->x;
            t.y += e->y;
        }
        tile[j] = t;
    }
}

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// weight and bias of the slab's channels (1 and 0 where there are none) into shared memory, without a barrier
__device__ __forceinline__ void stage_params(const Slab& s, const Place& w, float* weight, float* bias) {
    for (int j = threadIdx.x; j < s.width; j += blockDim.x) {
        const bool is = j < w.channels;
        weight[j] = is && s.p.weight ? sa_param(s.p.weight, w.first + j, s.p.param_dtype) : 1.0f;
        bias[j] = is && s.p.bias ? sa_param(s.p.bias, w.first + j, s.p.param_dtype) : 0.0f;
    }
}

// Place of channel c in a row of the tile: pairs of channels, the words' first pairs side by side, then their second pairs and
// so on, so that neighbouring threads write neighbouring 16 bytes.
template <int V>
__device__ __forceinline__ int tile_place(const Slab& s, int c) {
    return V == 1 ? c : (((c & (V - 1)) >> 1) * s.words + c / V) * 2 + (c & 1);
}

// The pairs (a, b) of every thread's channels, summed over the block: tile[part][tile_place(channel)], `parts` values for each
// channel (all zero where a thread has no rows).  The upper half of the row lanes hands its values to the lower half first, so that
// the tile has (row_lanes + 1) / 2 rows.  Ends with a barrier.
template <int V>
__device__ __forceinline__ void block_sums(const Slab& s, const Place& w, float2* tile, const F2 (&a)[(V + 1) / 2], const F2 (&b)[(V + 1) / 2]) {
    const int half = (s.row_lanes + 1) / 2;
    float2* const at = tile + (w.row_lane < half ? w.row_lane : w.row_lane - half) * s.width + w.word * (V == 1 ? 1 : 2);
    const bool upper = w.row_lane >= half && w.row_lane < s.row_lanes, taken = w.row_lane + half < s.row_lanes;
#pragma unroll
    for (int turn = 0; turn < 2; ++turn) {
        if (turn == 0 ? upper : w.row_lane < half) {
#pragma unroll
            for (int k = 0; k < (V + 1) / 2; ++k) {
                float4 e;
                split(a[k], e.x, e.z);
                split(b[k], e.y, e.w);
                if constexpr (V == 1) {
                    if (turn == 1 && taken) {
                        e.x += at->x;
                        e.y += at->y;
                    }
                    *at = make_float2(e.x, e.y);
                } else {
                    float4* const to = reinterpret_cast<float4*>(at + 2 * k * s.words);
                    if (turn == 1 && taken) {
                        const float4 o = *to;
                        e = make_float4(e.x + o.x, e.y + o.y, e.z + o.z, e.w + o.w);
                    }
                    *to = e;
                }
            }
        }
        __syncthreads();
    }
    column_sums(s, half, tile);
    __syncthreads();
}

// Statistics of a thread: sums of x - K and of its square, K being the thread's first row.  What cancels when they are put
// together is of the size of K's own square, and K is one of a few values: nothing is lost.  The block's threads then refer
// their sums to the mean of row lane 0 (the same argument, with its rows among the block's), which makes them plain sums;
// the channels of a group have equally many values, and the blocks of a cluster are joined by Chan's rule.
template <class T, int V>
__global__ void __launch_bounds__(kResidentThreads, 2)
sa_norm_resident_kernel(T* out, const T* x, float* __restrict__ mean, float* __restrict__ rstd, const __grid_constant__ Slab s) {
    constexpr int P = (V + 1) / 2;
    extern __shared__ __align__(16) unsigned char memory[];
    SaVec<T, V>* const data = (SaVec<T, V>*)memory;                                           // [rows][words]
    float2* const tile = (float2*)(memory + ((size_t)s.rows * s.words * sizeof(*data) + 15) / 16 * 16); // [lanes][width] sums
    float2* const joined = tile + (s.row_lanes + 1) / 2 * s.width;                             // [groups] (mean, m2) of this block
    float* const weight = (float*)(joined + s.groups); // [width] each: weight, then weight * rstd; bias; the means of row lane 0, then the groups'
    float* const bias = weight + s.width;
    float* const centre = bias + s.width;
    const Place w = place_of<V>(s);
    const Norm& p = s.p;

    const long long base = ((long long)w.n * p.S + (long long)w.rank * s.rows + w.row_lane) * p.C + w.first + w.word * V;
    const long long step = (long long)s.row_lanes * p.C;
    const int stride = s.row_lanes * s.words;
    SaVec<T, V>* const mine = data + threadIdx.x;
    for (int stage = 0, u = 0; stage < kStages; ++stage) {
        const int end = stage_end(w.rows, stage);
        fetch_rows<T, V>(mine + u * stride, x + base + u * step, end - u, stride, step);
        end_of_stage();
        u = end;
    }
    stage_params(s, w, weight, bias); // travels beside the data
    const float n = (float)w.rows;
    F2 m[P], q[P]; // mean and sum of squared deviations of this thread's rows
#pragma unroll
    for (int k = 0; k < P; ++k) m[k] = q[k] = f2(0.0f, 0.0f);
    F2 k0[P];
    as_rows_arrive(w.rows, [&](int u, int end) {
        if (u == 0 && end > 0) {
            const SaVec<T, V> v = *mine;
#pragma unroll
            for (int k = 0; k < P; ++k) k0[k] = negative(pair_of(v, k));
            u = 1;
        }
#pragma unroll 4
        for (; u < end; ++u) {
            const SaVec<T, V> v = mine[u * stride];
#pragma unroll
            for (int k = 0; k < P; ++k) {
                const F2 d = pair_of(v, k) + k0[k];
                m[k] = m[k] + d;
                q[k] = fma2(d, d, q[k]);
            }
        }
    });
    if (w.rows > 0) {
        const F2 inv = f2(1.0f / n, 1.0f / n);
#pragma unroll
        for (int k = 0; k < P; ++k) {
            const F2 part = m[k] * inv;
            q[k] = fma2(negative(m[k]), part, q[k]);
            m[k] = part + negative(k0[k]);
        }
    }
    if (w.row_lane == 0) {
#pragma unroll
        for (int k = 0; k < P; ++k) {
            float mx, my;
            split(m[k], mx, my);
            centre[w.word * V + 2 * k] = mx;
            if (2 * k + 1 < V) centre[w.word * V + 2 * k + 1] = my;
        }
    }
    __syncthreads();
    if (w.rows > 0) { // without rows both stay 0
        F2 c[P];
        shared_pairs<V>(c, centre + w.word * V);
#pragma unroll
        for (int k = 0; k < P; ++k) {
            const F2 d = m[k] + negative(c[k]);
            m[k] = f2(n, n) * d;
            q[k] = fma2(m[k], d, q[k]);
        }
    }
    block_sums<V>(s, w, tile, m, q);
    // a warp for each group
    const float rows_inv = w.block_rows > 0 ? 1.0f / (float)w.block_rows : 0.0f, D_inv = 1.0f / (float)p.D;
    for (int g = threadIdx.x / 32; g < w.groups; g += blockDim.x / 32) {
        float sum = 0.0f, m2 = 0.0f;
        for (int d = threadIdx.x % 32; d < p.D; d += 32) { // a channel's mean and squared deviations
            const int c = g * p.D + d;
            float2* const at = tile + tile_place<V>(s, c);
            float2 t = *at;
            for (int part = 1; part < s.parts; ++part) {
                const float2 e = at[part * s.width];
                t.x += e.x;
                t.y += e.y;
            }
            const float off = t.x * rows_inv, mc = centre[c] + off;
            at->x = mc;
            m2 += fmaf(-t.x, off, t.y);
            sum += mc;
        }
        const float mg = warp_sum(sum) * D_inv;
        for (int d = threadIdx.x % 32; d < p.D; d += 32) {
            const float off = tile[tile_place<V>(s, g * p.D + d)].x - mg; // written by this lane
            m2 = fmaf(off * off, (float)w.block_rows, m2);
        }
        m2 = warp_sum(m2);
        if (threadIdx.x % 32 == 0) joined[g] = make_float2(mg, m2);
    }

    cg::cluster_group cluster = cg::this_cluster();
    if (s.blocks > 1) cluster.sync();
    else __syncthreads();
    for (int j = threadIdx.x; j < w.channels; j += blockDim.x) { // every channel joins its group's blocks
        const int g = (int)s.by_D.div(j);
        Moments t{0.0f, 0.0f, 0.0f};
        if (s.blocks == 1) {
            t = Moments{(float)w.block_rows * (float)p.D, joined[g].x, joined[g].y};
        } else {
            int left = (int)p.S;
#pragma unroll 4
            for (int r = 0; r < s.blocks; ++r, left -= s.rows) {
                const float2 e = *cluster.map_shared_rank(joined + g, r);
                join(t, Moments{(float)max(0, min(left, s.rows)) * (float)p.D, e.x, e.y});
            }
        }
        const float rs = 1.0f / sqrtf(t.m2 / t.n + p.eps);
        centre[j] = t.mean;
        weight[j] *= rs;
        if (w.rank == 0 && j == g * p.D) {
            const long long at = (long long)w.n * p.G + w.group0 + g;
            mean[at] = t.mean;
            rstd[at] = rs;
        }
    }
    __syncthreads();
    if (s.blocks > 1) cluster.barrier_arrive(); // this block has read its neighbours
    if (w.rows > 0) {
        F2 a[P], b[P];
        shared_pairs<V>(m, centre + w.word * V);
        shared_pairs<V>(a, weight + w.word * V);
        shared_pairs<V>(b, bias + w.word * V);
#pragma unroll
        for (int k = 0; k < P; ++k) m[k] = negative(m[k]);
        T* to = out + base;
#pragma unroll 2
        for (int u = 0; u < w.rows; ++u, to += step) {
            SaVec<T, V> v = mine[u * stride];
#pragma unroll
            for (int k = 0; k < P; ++k) {
                const F2 z = fma2(pair_of(v, k) + m[k], a[k], b[k]);
                set_pair(v, k, p.silu ? z * sigmoid2<T>(z) : z);
            }
            sa_store<T, V>(to, v);
        }
    }
    if (s.blocks > 1) cluster.barrier_wait(); // no block leaves while a neighbour may still read its shared memory
}

// The deviations x - mean stand for u = (x - mean) rstd throughout, rstd goes into the constants:
//   z = (x - mean) (w rstd) + b,  dx = (w rstd) dz - rstd m1 - (x - mean) rstd^2 m2
// `sums`: (sum dz, sum dz u) of every (n, c); NULL: there is one sample, dweight and dbias are written here
template <class T, int V>
__global__ void __launch_bounds__(kResidentBackwardThreads, 3)
sa_norm_resident_backward_kernel(T* dx, const T* dout, const T* x, const float* __restrict__ mean, const float* __restrict__ rstd,
                                 float2* __restrict__ sums, void* __restrict__ dweight, void* __restrict__ dbias,
                                 const __grid_constant__ Slab s) {
    constexpr int P = (V + 1) / 2;
    extern __shared__ __align__(16) unsigned char memory[];
    const size_t bytes = ((size_t)s.rows * s.words * sizeof(SaVec<T, V>) + 15) / 16 * 16;
    SaVec<T, V>* const data = (SaVec<T, V>*)memory;              // [rows][words] of x
    SaVec<T, V>* const grad = (SaVec<T, V>*)(memory + bytes);    // [rows][words] of dout
    float2* const tile = (float2*)(memory + 2 * bytes);          // [lanes][width] sums
    float2* const channel = tile + (s.row_lanes + 1) / 2 * s.width; // [width] sums of dz and dz (x - mean) of this block
    float2* const total = channel + s.width;                     // [width] sums of the cluster, times weight and slope
    float2* const means = total + s.width;                       // [groups] rstd, later (rstd m1, rstd^2 m2), negative
    float* const weight = (float*)(means + s.groups);            // [width] each
    float* const bias = weight + s.width;
    float* const centre = bias + s.width;
    float* const slope = centre + s.width; // weight * rstd
    const Place w = place_of<V>(s);
    const Norm& p = s.p;

    const long long base = ((long long)w.n * p.S + (long long)w.rank * s.rows + w.row_lane) * p.C + w.first + w.word * V;
    const long long step = (long long)s.row_lanes * p.C;
    const int stride = s.row_lanes * s.words;
    SaVec<T, V>* const mine = data + threadIdx.x;
    SaVec<T, V>* const theirs = grad + threadIdx.x;
    for (int stage = 0, u = 0; stage < kStages; ++stage) {
        const int end = stage_end(w.rows, stage);
        fetch_rows<T, V>(mine + u * stride, x + base + u * step, end - u, stride, step);
        fetch_rows<T, V>(theirs + u * stride, dout + base + u * step, end - u, stride, step);
        end_of_stage();
        u = end;
    }
    stage_params(s, w, weight, bias); // these and the statistics travel beside the data
    for (int j = threadIdx.x; j < w.channels; j += blockDim.x) {
        const int g = (int)s.by_D.div(j);
        const long long at = (long long)w.n * p.G + w.group0 + g;
        const float rs = rstd[at];
        centre[j] = mean[at];
        slope[j] = weight[j] * rs; // staged by this thread
        if (j == g * p.D) means[g].x = rs;
    }
    __syncthreads();
    F2 m[P], sl[P], b[P];
    {
        F2 a0[P], a1[P];
#pragma unroll
        for (int k = 0; k < P; ++k) a0[k] = a1[k] = f2(0.0f, 0.0f);
        if (w.row_lane < s.row_lanes) {
            shared_pairs<V>(m, centre + w.word * V);
            shared_pairs<V>(sl, slope + w.word * V);
            shared_pairs<V>(b, bias + w.word * V);
#pragma unroll
            for (int k = 0; k < P; ++k) m[k] = negative(m[k]);
        }
        as_rows_arrive(w.rows, [&](int u, int end) {
            for (; u < end; ++u) {
                const SaVec<T, V> v = mine[u * stride], d = theirs[u * stride];
#pragma unroll
                for (int k = 0; k < P; ++k) {
                    const F2 dev = pair_of(v, k) + m[k];
                    const F2 dz = through_activation2<T>(pair_of(d, k), fma2(dev, sl[k], b[k]), p.silu);
                    a0[k] = a0[k] + dz;
                    a1[k] = fma2(dz, dev, a1[k]);
                }
            }
        });
        block_sums<V>(s, w, tile, a0, a1);
    }
    for (int j = threadIdx.x; j < s.width; j += blockDim.x) {
        const float2* const at = tile + tile_place<V>(s, j);
        float2 t = *at;
        for (int part = 1; part < s.parts; ++part) {
            const float2 e = at[part * s.width];
            t.x += e.x;
            t.y += e.y;
        }
        channel[j] = t;
    }
    cg::cluster_group cluster = cg::this_cluster();
    if (s.blocks > 1) cluster.sync();
    else __syncthreads();
    for (int j = threadIdx.x; j < w.channels; j += blockDim.x) {
        float2 t = make_float2(0.0f, 0.0f);
#pragma unroll 4
        for (int r = 0; r < s.blocks; ++r) {
            const float2 e = s.blocks > 1 ? *cluster.map_shared_rank(channel + j, r) : channel[j];
            t.x += e.x;
            t.y += e.y;
        }
        total[j] = make_float2(weight[j] * t.x, slope[j] * t.y);
        t.y *= means[s.by_D.div(j)].x; // sum of dz u
        if (w.rank == 0) {
            if (sums) sums[(long long)w.n * p.C + w.first + j] = t;
            else {
                if (dbias) sa_set_param(dbias, w.first + j, p.param_dtype, t.x);
                if (dweight) sa_set_param(dweight, w.first + j, p.param_dtype, t.y);
            }
        }
    }
    __syncthreads();
    if (s.blocks > 1) cluster.barrier_arrive(); // this block has read its neighbours
    const float inv = 1.0f / ((float)p.S * (float)p.D);
    for (int g = threadIdx.x / 32; g < w.groups; g += blockDim.x / 32) {
        float2 t = make_float2(0.0f, 0.0f);
        for (int c = threadIdx.x % 32; c < p.D; c += 32) {
            const float2 e = total[g * p.D + c];
            t.x += e.x;
            t.y += e.y;
        }
        t = make_float2(warp_sum(t.x), warp_sum(t.y));
        if (threadIdx.x % 32 == 0) {
            const float rs = means[g].x;
            means[g] = make_float2(-rs * (t.x * inv), -rs * rs * (t.y * inv));
        }
    }
    __syncthreads();
    if (w.rows > 0) {
        F2 m1[P], m2[P];
        {
            float x1[2 * P] = {}, x2[2 * P] = {};
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const float2 e = means[s.by_D.div(w.word * V + i)];
                x1[i] = e.x;
                x2[i] = e.y;
            }
#pragma unroll
            for (int k = 0; k < P; ++k) {
                m1[k] = f2(x1[2 * k], x1[2 * k + 1]);
                m2[k] = f2(x2[2 * k], x2[2 * k + 1]);
            }
        }
        T* to = dx + base;
        for (int u = 0; u < w.rows; ++u, to += step) {
            SaVec<T, V> v = mine[u * stride];
            const SaVec<T, V> d = theirs[u * stride];
#pragma unroll
            for (int k = 0; k < P; ++k) {
                const F2 dev = pair_of(v, k) + m[k];
                const F2 dz = through_activation2<T>(pair_of(d, k), fma2(dev, sl[k], b[k]), p.silu);
                set_pair(v, k, fma2(dev, m2[k], fma2(sl[k], dz, m1[k])));
            }
            sa_store<T, V>(to, v);
        }
    }
    if (s.blocks > 1) cluster.barrier_wait(); // no block leaves while a neighbour may still read its shared memory
}

// ---------------------------------------------------------------------------
// launches
// ---------------------------------------------------------------------------
// How a sample is cut: words across a block, rows at a time, runs of rows.  About four blocks for each SM, but runs of
// at least `kBatch` rows for each row lane, so that partial results stay a small part of the traffic.
void cut(Norm& p, int V, int* column_tiles) {
    const long long words = p.C / V;
    p.columns = (int)(words < kThreads ? words : kThreads);
    p.row_lanes = kThreads / p.columns;
    *column_tiles = (int)((words + p.columns - 1) / p.columns);
    long long splits = 148 * 4 / ((long long)p.N * *column_tiles);
    const long long most = (p.S + (long long)kBatch * p.row_lanes - 1) / ((long long)kBatch * p.row_lanes);
    if (splits > most) splits = most;
    if (splits < 1) splits = 1;
    p.rows = (p.S + splits - 1) / splits;
    p.splits = (int)((p.S + p.rows - 1) / p.rows);
}

Norm describe(const sideaware_group_norm_t& sh, const void* weight, const void* bias) {
    Norm p{};
    p.N = sh.N;
    p.S = sh.S;
    p.C = sh.C;
    p.G = sh.G;
    p.D = sh.C / sh.G;
    p.silu = sh.silu;
    p.param_dtype = sh.param_dtype;
    p.eps = sh.eps;
    p.weight = weight;
    p.bias = bias;
    return p;
}

// elements of a word: 16 bytes where addresses and rows allow them, else 4, else one element
int word_elements(const sideaware_group_norm_t& sh, uint64_t addresses) {
    const int e = sa_element_size(sh.dtype);
    const int a = sa_common_alignment(addresses | (uint64_t)sh.C * (uint64_t)e);
    return a == 16 ? 16 / e : a >= 4 ? 4 / e : 1;
}

constexpr int kMaxCluster = 8; // blocks of a cluster that every GPU schedules

// Whether the groups of a sample fit into the shared memory of clusters, and how.  `tensors`: 1 (forward) or 2.  Of every slab
// width (multiples of the narrowest one that is whole words, up to 512 bytes of a row) and cluster size the one with the least
// estimated time: rounds of blocks, each with a fixed part (latency, barriers) and its bytes at the SM's share of the HBM.
bool plan_resident(const Norm& p, int V, int esize, int tensors, Slab* best) {
    const int most_threads = tensors == 1 ? kResidentThreads : kResidentBackwardThreads, most_blocks = tensors == 1 ? 2 : 3;
    if (p.S > 1 << 20) return false;
    int unit = 1; // groups of the narrowest slab
    while ((unit * (long long)p.D) % V) ++unit;
    double least = 1e300;
    for (int m = 1; m == 1 || unit * m <= p.G; ++m) {
        const int groups = unit * m < p.G ? unit * m : p.G;
        const long long width = (long long)groups * p.D;
        if (width % V || width / V > most_threads / 2 || (m > 1 && width * esize > 512)) break;
        Slab s{};
        s.p = p;
        s.groups = groups;
        s.width = (int)width;
        s.words = (int)(width / V);
        s.slabs = (p.G + groups - 1) / groups;
        s.by_words = divisor((uint32_t)s.words);
        s.by_width = divisor((uint32_t)width);
        s.by_D = divisor((uint32_t)p.D);
        for (int blocks = 1; blocks <= kMaxCluster; ++blocks) {
            const int rows = (int)((p.S + blocks - 1) / blocks);
            if (blocks > 1 && rows < 8) break;
            s.blocks = blocks;
            s.rows = rows;
            // about four rows for each thread
            long long threads = ((long long)rows * s.words / 4 + 31) / 32 * 32;
            if (threads < 2 * s.words) threads = (2 * s.words + 31) / 32 * 32;
            if (threads < 128) threads = 128;
            s.threads = threads > most_threads ? most_threads : (int)threads;
            s.row_lanes = s.threads / s.words;
            const int half = (s.row_lanes + 1) / 2;
            s.parts = s.width >= s.threads ? 1 : s.threads / s.width < half ? s.threads / s.width : half;
            const size_t data = ((size_t)rows * s.words * V * esize + 15) / 16 * 16;
            s.shared = tensors * data + sizeof(float2) * ((size_t)half * s.width + s.groups + (tensors == 1 ? 0 : 2 * s.width)) +
                       sizeof(float) * (size_t)(tensors == 1 ? 3 : 4) * s.width;
            if (s.shared > 226 * 1024) continue;
            const double grid = (double)p.N * s.slabs * blocks;
            if (grid > 1e9) continue;
            int resident = (int)(228 * 1024 / (s.shared + 1024));
            if (resident > most_blocks) resident = most_blocks;
            const double segment = (double)width * esize, ragged = (width * esize) % 32 ? (segment + 16.0) / segment : 1.0;
            const double fixed = 2.5 + (blocks > 1 ? 0.7 : 0.0) + 0.1 * blocks;
            const double bytes = (tensors + 1) * (double)data * ragged / 44e3; // us for one block's traffic at an SM's share
            const double rounds = grid / (148.0 * resident);
            const double cost = rounds <= 1.0 ? fixed + bytes * (grid > 148.0 ? resident : 1.0)
                                              : fixed + (double)(long long)(rounds + 0.999) * (bytes * resident + fixed / resident);
            if (cost < least) {
                least = cost;
                *best = s;
            }
        }
    }
    return least < 1e300;
}

template <class K, class... Args>
cudaError_t launch_clusters(K kernel, const Slab& s, cudaStream_t stream, Args... args) {
    if (s.shared > 48 * 1024) {
        const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)s.shared);
        if (e != cudaSuccess) return e;
    }
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)(s.p.N * s.slabs * s.blocks));
    cfg.blockDim = dim3((unsigned)s.threads);
    cfg.dynamicSmemBytes = s.shared;
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = (unsigned)s.blocks;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = s.blocks > 1 ? 1 : 0;
    return cudaLaunchKernelEx(&cfg, kernel, args...);
}

template <class T, int V>
cudaError_t forward(void* out, float* mean, float* rstd, const void* x, Norm p, void* workspace, cudaStream_t stream) {
    Slab s;
    if (plan_resident(p, V, sizeof(T), 1, &s))
        return launch_clusters(sa_norm_resident_kernel<T, V>, s, stream, (T*)out, (const T*)x, mean, rstd, s);
    int tiles = 0;
    cut(p, V, &tiles);
    const dim3 grid((unsigned)p.N * p.splits, tiles);
    float2* partial = (float2*)workspace;
    sa_norm_partial_kernel<T, V><<<grid, kThreads, 0, stream>>>((const T*)x, partial, p);
    sa_norm_join_kernel<<<p.N * p.G, kThreads, 0, stream>>>(partial, mean, rstd, p);
    sa_norm_apply_kernel<T, V><<<grid, kThreads, 0, stream>>>((T*)out, (const T*)x, mean, rstd, p);
    return cudaGetLastError();
}

template <class T, int V>
cudaError_t backward(void* dx, void* dweight, void* dbias, const void* dout, const void* x, const float* mean, const float* rstd,
                     Norm p, void* workspace, cudaStream_t stream) {
    Slab s;
    if (plan_resident(p, V, sizeof(T), 2, &s)) {
        float2* const sums = p.N > 1 && (dweight || dbias) ? (float2*)workspace : nullptr;
        const cudaError_t e = launch_clusters(sa_norm_resident_backward_kernel<T, V>, s, stream, (T*)dx, (const T*)dout, (const T*)x,
                                              mean, rstd, sums, p.N > 1 ? nullptr : dweight, p.N > 1 ? nullptr : dbias, s);
        if (e != cudaSuccess || !sums) return e;
        sa_norm_backward_params_kernel<<<(unsigned)((p.C + kThreads - 1) / kThreads), kThreads, 0, stream>>>(sums, dweight, dbias, p);
        return cudaGetLastError();
    }
    int tiles = 0;
    cut(p, V, &tiles);
    const dim3 grid((unsigned)p.N * p.splits, tiles);
    float2* partial = (float2*)workspace;
    float2* sums = partial + (long long)p.N * p.splits * p.C;
    float2* means = sums + (long long)p.N * p.C;
    sa_norm_backward_partial_kernel<T, V><<<grid, kThreads, 0, stream>>>((const T*)dout, (const T*)x, mean, rstd, partial, p);
    sa_norm_backward_join_kernel<<<p.N * p.G, kThreads, 0, stream>>>(partial, sums, means, p);
    if (dweight || dbias)
        sa_norm_backward_params_kernel<<<(unsigned)((p.C + kThreads - 1) / kThreads), kThreads, 0, stream>>>(sums, dweight, dbias, p);
    sa_norm_backward_apply_kernel<T, V><<<grid, kThreads, 0, stream>>>((T*)dx, (const T*)dout, (const T*)x, mean, rstd, means, p);
    return cudaGetLastError();
}

template <class F>
cudaError_t by_type(const sideaware_group_norm_t& sh, int V, F&& f) {
    if (sh.dtype == SA_FP32) {
        if (V == 4) return f(float(), std::integral_constant<int, 4>());
        return f(float(), std::integral_constant<int, 1>());
    }
    if (sh.dtype == SA_BF16) {
        if (V == 8) return f(__nv_bfloat16(), std::integral_constant<int, 8>());
        if (V == 2) return f(__nv_bfloat16(), std::integral_constant<int, 2>());
        return f(__nv_bfloat16(), std::integral_constant<int, 1>());
    }
    if (V == 8) return f(__half(), std::integral_constant<int, 8>());
    if (V == 2) return f(__half(), std::integral_constant<int, 2>());
    return f(__half(), std::integral_constant<int, 1>());
}

} // namespace

// Enough for words of any width, so that it follows from the shape alone.  Long samples: the partial results of all runs,
// backward also the sums of every (n, c) and the means of every (n, g).  Resident ones: those sums, if there is more than one sample.
size_t sa_group_norm_workspace(const sideaware_group_norm_t& sh, bool backward) {
    const int e = sa_element_size(sh.dtype);
    long long most = 0;
    for (int V : {16 / e, 4 / e, 1}) {
        if (sh.C % V) continue;
        Norm p = describe(sh, nullptr, nullptr);
        Slab s;
        int tiles = 0;
        long long entries = backward && sh.N > 1 ? (long long)sh.N * sh.C : 0;
        if (!plan_resident(p, V, e, backward ? 2 : 1, &s)) {
            cut(p, V, &tiles);
            entries = (long long)sh.N * p.splits * sh.C + (backward ? (long long)sh.N * (sh.C + sh.G) : 0);
        }
        if (entries > most) most = entries;
    }
    return (size_t)most * sizeof(float2);
}

cudaError_t sa_launch_group_norm(void* out, float* mean, float* rstd, const void* x, const void* weight, const void* bias,
                                 const sideaware_group_norm_t& sh, void* workspace, cudaStream_t stream) {
    const Norm p = describe(sh, weight, bias);
    return by_type(sh, word_elements(sh, (uint64_t)out | (uint64_t)x), [&](auto type, auto v) {
        return forward<decltype(type), v.value>(out, mean, rstd, x, p, workspace, stream);
    });
}

cudaError_t sa_launch_group_norm_backward(void* dx, void* dweight, void* dbias, const void* dout, const void* x, const float* mean,
                                          const float* rstd, const void* weight, const void* bias,
                                          const sideaware_group_norm_t& sh, void* workspace, cudaStream_t stream) {
    const Norm p = describe(sh, weight, bias);
    return by_type(sh, word_elements(sh, (uint64_t)dx | (uint64_t)dout | (uint64_t)x), [&](auto type, auto v) {
        return backward<decltype(type), v.value>(dx, dweight, dbias, dout, x, mean, rstd, p, workspace, stream);
    });
}
