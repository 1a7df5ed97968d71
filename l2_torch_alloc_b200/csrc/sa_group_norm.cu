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
// Three launches: partial statistics of runs of rows, joining them, applying them.
#include <climits>

#include "sa_elem.cuh"
#include "sa_ops.hpp"

namespace {

constexpr int kThreads = 256;
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

// mean and sum of squared deviations of `n` values
struct Moments {
    float n, mean, m2;
};

__device__ __forceinline__ void join(Moments& a, const Moments& b) {
    const float n = a.n + b.n;
    if (n == 0.0f) return;
    const float d = b.mean - a.mean, f = b.n / n;
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
#pragma unroll
    for (int i = 0; i < V; ++i) {
        const long long c = c0 + i, at = (long long)n * p.G + c / p.D;
        m[i] = mean[at];
        a[i] = rstd[at] * (p.weight ? sa_param(p.weight, c, p.param_dtype) : 1.0f);
        b[i] = p.bias ? sa_param(p.bias, c, p.param_dtype) : 0.0f;
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
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const long long c = c0 + i, at = (long long)n * p.G + c / p.D;
            m[i] = mean[at];
            r[i] = rstd[at];
            w[i] = p.weight ? sa_param(p.weight, c, p.param_dtype) : 1.0f;
            b[i] = p.bias ? sa_param(p.bias, c, p.param_dtype) : 0.0f;
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
#pragma unroll
    for (int i = 0; i < V; ++i) {
        const long long c = c0 + i, at = (long long)n * p.G + c / p.D;
        m[i] = mean[at];
        r[i] = rstd[at];
        w[i] = p.weight ? sa_param(p.weight, c, p.param_dtype) : 1.0f;
        b[i] = p.bias ? sa_param(p.bias, c, p.param_dtype) : 0.0f;
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

template <class T, int V>
cudaError_t forward(void* out, float* mean, float* rstd, const void* x, Norm p, void* workspace, cudaStream_t stream) {
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

// partial results of all runs; backward: also the sums of every (n, c) and the means of every (n, g).  Enough for words
// of any width, so that it follows from the shape alone.
size_t sa_group_norm_workspace(const sideaware_group_norm_t& sh, bool backward) {
    long long most = 0;
    for (int V : {16 / sa_element_size(sh.dtype), 4 / sa_element_size(sh.dtype), 1}) {
        if (sh.C % V) continue;
        Norm p = describe(sh, nullptr, nullptr);
        int tiles = 0;
        cut(p, V, &tiles);
        if (p.splits > most) most = p.splits;
    }
    const long long entries = (long long)sh.N * most * sh.C + (backward ? (long long)sh.N * (sh.C + sh.G) : 0);
    return (size_t)entries * sizeof(float2);
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
