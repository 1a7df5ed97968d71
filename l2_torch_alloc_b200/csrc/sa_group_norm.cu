// Group norm with an optional SiLU, channels last: x [N, S, C], groups of D = C / G neighbouring channels.
//
//   mean, rstd = 1 / sqrt(var + eps) over the S * D elements of (n, g);  z = (x - mean) rstd w + b;  y = z or z sigmoid(z)
//
// Backward, with u = (x - mean) rstd, dz = dy act'(z), A[n][c] = sum_s dz, B[n][c] = sum_s dz u:
//   dbias = sum_n A, dweight = sum_n B,
//   dx = rstd (w dz - m1 - u m2), m1 = sum_{c in g} w A / (S D), m2 = sum_{c in g} w B / (S D)
//
// Statistics: sums about a value that is one of the data, kept for a few rows, then joined with the pairwise update of Chan,
// Golub and LeVeque (1983), all in fp32: no cancellation however far the mean is from zero.  All sums go through fixed trees
// (no atomics): the same inputs give the same bits.
//
// Three ways, chosen by estimated times in search_plan below:
//  * resident: a thread-block cluster owns some neighbouring groups of one sample, all rows of them lie in the shared
//    memory of its blocks, which exchange their statistics through distributed shared memory.  One launch, each element
//    is read once and written once.
//  * streamed, for samples too long for that: partial statistics of runs of rows, joining them, applying them; three
//    launches that overlap, x is read twice (a part of it from L2).
//  * packed, for many short samples (a token's channels, a small image) and for little work: a block has several whole samples
//    in its shared memory at a time and goes on to the next ones, which are already on their way.
//
// Bound and measured on a B200 (device time of a call, three sets of inputs in turn):
//  * resident: the phases of a block follow one another, and each moves about 4 TB/s alone.  8 x 4096 x 320 bf16: 17.1 us (6.4
//    at the copy's rate), of 31,000 cycles 12,000 are for the rows to arrive, 5,000 for the statistics to go around and
//    11,500 for SiLU and the stores (without SiLU: 1.6 us less).  Backward the activation's derivative is worked out twice, 32
//    operations of the special-function unit for 8 elements: 8 x 1024 x 640 fp16 17.5 us.
//  * streamed: HBM.  2 x 262144 x 128 bf16: 75.6 us, 29 us for reading x (a plain sum of as many bytes takes as long) and 41
//    us for the copy-like second pass.
//  * packed: instructions, 190 of a warp for a word of each lane forward and 550 backward.  16384 x 1 x 2048 bf16: 45 us
//    and 117 us (resident: 580 and 1080); 1 x 64 x 1280 bf16: 4.1 us, which is latency (resident 5.1).
#include <cooperative_groups.h>

#include <algorithm>
#include <cmath>
#include <mutex>
#include <type_traits>

#include "sa_elem.cuh"
#include "sa_kernels.hpp"
#include "sa_ops.hpp"

namespace cg = cooperative_groups;

namespace {

constexpr int kThreads = 256;
constexpr int kMaxCluster = 8; // blocks of a cluster that every GPU schedules
constexpr int kResidentThreads = 1024; // threads of a resident block, at most
constexpr int kResidentRegisters = 64, kResidentBackwardRegisters = 80; // 32 and 25 warps on an SM

struct Norm {
    long long S, C; // rows of a sample, channels
    int G, D;       // groups, channels of a group
    int fold;       // so many pixels lie side by side in a row: S and C are those of such rows, the operator has C / fold channels
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
    if (a.n == 0.0f) { // b as it is: a weight of nearly 1 would move a mean far from zero by more than the deviations
        a = b;
        return;
    }
    const float n = a.n + b.n;
    const float d = b.mean - a.mean, f = __fdividef(b.n, n); // a weight: two roundings more do no harm
    a.mean = fmaf(d, f, a.mean);
    a.m2 += b.m2 + d * (d * (a.n * f));
    a.n = n;
}

// ---------------------------------------------------------------------------
// what the kernels share: a block has some rows of a slab (neighbouring channels) of one sample
// ---------------------------------------------------------------------------
struct Slab {
    Norm p;
    int groups, width;     // groups of a slab (streamed: that it touches, at most), its channels: a whole number of words
    int words;             // words of a row
    int row_lanes;         // rows a block takes at a time: a thread has one word of every row_lanes-th row
    int slabs;             // of a sample
    int blocks;            // of a slab of a sample; resident: a cluster
    int rows;              // of a block
    int parts;             // threads that share a channel's column when the block's threads are joined
    int threads;
    int samples;           // packed: whole samples of a tile, else 0
    int tiles, lanes;      // packed: tiles of a slab; threads that work on a group of a sample
    int pitch;             // packed: words from a row to the next in shared memory (odd: rows meet different banks)
    Divisor by_words, by_width, by_D, by_S, by_groups;
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
__device__ __forceinline__ Place place_of(const Slab& s, uint32_t block) {
    Place w;
    const uint32_t cluster = s.blocks > 1 ? block / (uint32_t)s.blocks : block;
    w.rank = (int)(block - cluster * s.blocks);
    w.n = (int)(cluster / (uint32_t)s.slabs);
    const int slab = (int)cluster - w.n * s.slabs;
    w.row_lane = (int)s.by_words.div(threadIdx.x);
    w.word = (int)threadIdx.x - w.row_lane * s.words;
    w.group0 = slab * s.groups;
    w.first = (long long)slab * s.width;
    w.groups = min(s.groups, s.p.G - w.group0);
    w.channels = (int)min((long long)s.width, s.p.C - w.first);
    w.block_rows = (int)max(0ll, min((long long)s.rows, s.p.S - (long long)w.rank * s.rows));
    const int left = w.block_rows - w.row_lane;
    w.rows = w.row_lane < s.row_lanes && w.word * V < w.channels && left > 0 ? (left + s.row_lanes - 1) / s.row_lanes : 0;
    return w;
}

// This thread's words of its block's rows from global into shared memory, without passing through registers (words of 4
// bytes or more).  The rows come in kStages groups, so that the first ones can be worked on while the others travel; a thread
// waits for its own words only.  (Through registers instead: 8 to 40 % slower; hints to fetch whole lines: no difference.)
constexpr int kStages = 4;
__device__ __forceinline__ int stage_end(int rows, int stage) { return stage == kStages - 1 ? rows : rows * (stage + 1) / kStages; }

template <class T, int V>
__device__ __forceinline__ void fetch_row(SaVec<T, V>* to, const T* from) {
    if constexpr (sizeof(SaVec<T, V>) == 16)
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"((uint32_t)__cvta_generic_to_shared(to)), "l"(from) : "memory");
    else if constexpr (sizeof(SaVec<T, V>) >= 4)
        asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"((uint32_t)__cvta_generic_to_shared(to)), "l"(from), "n"(sizeof(SaVec<T, V>)) : "memory");
    else
        *to = sa_load<T, V>(from);
}
template <class T, int V>
__device__ __forceinline__ void fetch_rows(SaVec<T, V>* to, const T* from, int rows, int stride, long long step) {
#pragma unroll 4
    for (int u = 0; u < rows; ++u, to += stride, from += step) fetch_row<T, V>(to, from);
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

// The activation of a word's pairs.  fp32 storage wants all of fp32.  16-bit storage takes the fast exponential and reciprocal, whose
// 2^-22 (and a rounding of the exponent) are far below a rounding of the result; below z = -87 sigmoid is 0, and z sigmoid(z)
// and the derivative with it, which are under 2^-119 there.
__device__ __forceinline__ float exp2_fast(float v) {
    asm("ex2.approx.ftz.f32 %0, %0;" : "+f"(v));
    return v;
}
__device__ __forceinline__ float reciprocal_fast(float v) {
    asm("rcp.approx.ftz.f32 %0, %0;" : "+f"(v));
    return v;
}
// 1 + exp(-z)
__device__ __forceinline__ void denominators(F2 z, float& a, float& b) {
    split(z * f2(-1.44269504f, -1.44269504f), a, b); // -log2 e
    split(f2(exp2_fast(a), exp2_fast(b)) + f2(1.0f, 1.0f), a, b);
}
template <class T>
__device__ __forceinline__ F2 sigmoid2(F2 z) {
    float a, b;
    if constexpr (sizeof(T) == 4) {
        split(z, a, b);
        return f2(1.0f / (1.0f + expf(-a)), 1.0f / (1.0f + expf(-b)));
    }
    denominators(z, a, b);
    return f2(reciprocal_fast(a), reciprocal_fast(b));
}

// The inner loops exist with and without the activation, which is one branch around them: with_activation(silu, f) calls
// f(std::true_type) or f(std::false_type).
template <class F>
__device__ __forceinline__ void with_activation(int silu, F&& f) {
    if (silu) f(std::true_type{});
    else f(std::false_type{});
}

// use(k, activation of z(k)) for the P pairs of a word, possibly a second time.  16-bit storage: the special-function unit is what
// an activation waits for (8 cycles a warp and operation), so a pair has one reciprocal, 1 / a = b / (a b), 1.5 operations for each
// element instead of 2.  Where a b is no number any more (from z = -43 on) or a NaN, which its neighbour must not see, the word is
// done again with one for each element.  (The smallest of the reciprocals tells; a test of z before them took 1 to 5 % of a call,
// limits on z 1 to 4 %, a reciprocal for each element always 3 to 12 %.)
template <class T, bool SILU, int P, class Z, class Use>
__device__ __forceinline__ void activation(Z&& z, Use&& use) {
    if constexpr (!SILU) {
#pragma unroll
        for (int k = 0; k < P; ++k) use(k, z(k));
    } else if constexpr (sizeof(T) == 4 || P == 1) {
#pragma unroll
        for (int k = 0; k < P; ++k) {
            const F2 v = z(k);
            use(k, v * sigmoid2<T>(v));
        }
    } else {
        float least = 1.0f;
#pragma unroll
        for (int k = 0; k < P; ++k) {
            float a, b;
            const F2 v = z(k);
            denominators(v, a, b);
            const float r = reciprocal_fast(a * b);
            asm("min.NaN.f32 %0, %0, %1;" : "+f"(least) : "f"(r));
            use(k, v * (f2(r, r) * f2(b, a)));
        }
        if (__builtin_expect(!(least > 0.0f), 0)) {
#pragma unroll
            for (int k = 0; k < P; ++k) {
                const F2 v = z(k);
                use(k, v * sigmoid2<T>(v));
            }
        }
    }
}

// dy act'(z) = dy s (1 + z (1 - s)).  A reciprocal for each element: 1 - s is exactly 0 for large z then.  (One for a pair, and
// 1 - s = exp(-z) s: no faster.)
template <class T, bool SILU>
__device__ __forceinline__ F2 through_activation2(F2 dy, F2 z) {
    if constexpr (!SILU) return dy;
    const F2 sg = sigmoid2<T>(z), one = f2(1.0f, 1.0f);
    return dy * (sg * fma2(z, fma2(sg, f2(-1.0f, -1.0f), one), one));
}

// A channel's row lanes, `parts` threads for each channel; the sum stands in the first row of each share.
__device__ __forceinline__ void column_sums(const Slab& s, int lanes, float2* tile) {
    for (int j = threadIdx.x; j < s.parts * s.width; j += blockDim.x) {
        const int part = s.parts > 1 ? (int)s.by_width.div(j) : 0; // j = part * width + channel
        float2 t = tile[j];
        const float2* at = tile + j;
#pragma unroll 4
        for (int r = part + s.parts; r < lanes; r += s.parts) {
            at += s.parts * s.width;
            const float2 e = *at;
            t.x += e.x;
            t.y += e.y;
        }
        tile[j] = t;
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

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// the operator's channel at place c of a row
__device__ __forceinline__ long long channel_of(const Norm& p, long long c) {
    return p.fold > 1 ? (long long)((uint32_t)c % ((uint32_t)p.C / (uint32_t)p.fold)) : c;
}

// weight and bias of the slab's channels (1 and 0 where there are none) into shared memory, without a barrier
__device__ __forceinline__ void stage_params(const Slab& s, const Place& w, float* weight, float* bias) {
    for (int j = threadIdx.x; j < s.width; j += blockDim.x) {
        const bool is = j < w.channels;
        const long long c = channel_of(s.p, w.first + j);
        weight[j] = is && s.p.weight ? sa_param(s.p.weight, c, s.p.param_dtype) : 1.0f;
        bias[j] = is && s.p.bias ? sa_param(s.p.bias, c, s.p.param_dtype) : 0.0f;
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

// Row lane 0's means for everybody; a barrier has to follow.
template <int V>
__device__ __forceinline__ void share_centre(const Place& w, const F2 (&m)[(V + 1) / 2], float* centre) {
    if (w.row_lane == 0) {
#pragma unroll
        for (int k = 0; k < (V + 1) / 2; ++k) {
            float mx, my;
            split(m[k], mx, my);
            centre[w.word * V + 2 * k] = mx;
            if (2 * k + 1 < V) centre[w.word * V + 2 * k + 1] = my;
        }
    }
}

// (mean, m2) of this thread's n rows become the sums of x - centre and of its square.
template <int V>
__device__ __forceinline__ void refer_to_centre(const Place& w, F2 (&m)[(V + 1) / 2], F2 (&q)[(V + 1) / 2], float n, const float* centre) {
    if (w.rows <= 0) return; // without rows both are 0
    F2 c[(V + 1) / 2];
    shared_pairs<V>(c, centre + w.word * V);
#pragma unroll
    for (int k = 0; k < (V + 1) / 2; ++k) {
        const F2 d = m[k] + negative(c[k]);
        m[k] = f2(n, n) * d;
        q[k] = fma2(m[k], d, q[k]);
    }
}

// channel c's sums once block_sums is through
template <int V>
__device__ __forceinline__ float2 channel_sum(const Slab& s, const float2* tile, int c) {
    const float2* const at = tile + tile_place<V>(s, c);
    float2 t = *at;
#pragma unroll 4
    for (int part = 1; part < s.parts; ++part) {
        const float2 e = at[part * s.width];
        t.x += e.x;
        t.y += e.y;
    }
    return t;
}

// ---------------------------------------------------------------------------
// streamed: partial results of runs of rows, joined, then applied
// ---------------------------------------------------------------------------
// A thread's rows (one word of each) on their way through a ring in shared memory that only this thread uses: four stages of
// ROWS rows are in flight.  16 words of each thread in all (64 KiB of a block, three blocks of an SM): 4 rows of one tensor or
// 2 of two.
constexpr int kStreamStages = 4, kRingWords = 16;

template <class T, int V>
struct Stream {
    SaVec<T, V>* ring; // [rows][kThreads], this thread's column
    const T* from;
    long long step;
    __device__ __forceinline__ Stream(void* memory, const T* first, long long rows_apart)
        : ring((SaVec<T, V>*)memory + threadIdx.x), from(first), step(rows_apart) {}
    __device__ __forceinline__ void fetch(int slot) {
        fetch_row<T, V>(ring + slot * kThreads, from);
        from += step;
    }
    __device__ __forceinline__ SaVec<T, V> row(int slot) const { return ring[slot * kThreads]; }
};

// fetch(slot) sets the next row under way, f(slot) works on the row in a slot; stage(slot, rows) comes before a stage's rows.
// Slots are constants once the loops are unrolled, and a whole stage takes one test.
template <int ROWS, class Fetch, class Stage, class F>
__device__ __forceinline__ void stream_rows(int rows, Fetch&& fetch, Stage&& stage, F&& f) {
    auto fetch_stage = [&](int slot, int left) {
        if (left >= ROWS) {
#pragma unroll
            for (int r = 0; r < ROWS; ++r) fetch(slot + r);
        } else {
#pragma unroll
            for (int r = 0; r < ROWS; ++r)
                if (r < left) fetch(slot + r);
        }
        end_of_stage();
    };
    int left = rows, ahead = rows; // rows to work on, rows to fetch
#pragma unroll
    for (int k = 0; k < kStreamStages; ++k, ahead -= ROWS) fetch_stage(k * ROWS, ahead);
    while (left > 0) {
#pragma unroll
        for (int k = 0; k < kStreamStages; ++k) {
            asm volatile("cp.async.wait_group %0;" ::"n"(kStreamStages - 1) : "memory");
            if (left >= ROWS) {
                stage(k * ROWS, ROWS);
#pragma unroll
                for (int r = 0; r < ROWS; ++r) f(k * ROWS + r);
            } else if (left > 0) {
                stage(k * ROWS, left);
#pragma unroll
                for (int r = 0; r < ROWS; ++r)
                    if (r < left) f(k * ROWS + r);
            }
            fetch_stage(k * ROWS, ahead);
            left -= ROWS;
            ahead -= ROWS;
        }
    }
}

// Kernels of one call overlap their launches (programmatic dependent launch): a later one waits here before it reads
// what an earlier one wrote.
__device__ __forceinline__ void may_follow() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void await_previous() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

// The groups that a slab touches: with folded rows (one slab) all of them.
__device__ __forceinline__ int first_group(const Norm& p, long long first) { return p.fold > 1 ? 0 : (int)((uint32_t)first / (uint32_t)p.D); }
__device__ __forceinline__ int last_group(const Norm& p, long long first, int channels) {
    return p.fold > 1 ? p.G - 1 : (int)((uint32_t)(first + channels - 1) / (uint32_t)p.D);
}
// Lanes that work on a group together: the power of two that its places of a slab keep busy.
__device__ __forceinline__ int group_lanes(const Norm& p) {
    const int places = p.D * p.fold;
    return places > 16 ? 32 : places > 8 ? 16 : places > 4 ? 8 : 4;
}
__device__ __forceinline__ float lanes_sum(float v, int lanes) {
    for (int o = lanes / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}
// f(g, whether there is such a group) for the groups g0 to g1, `lanes` threads for each; all threads of a warp call f together
template <class F>
__device__ __forceinline__ void for_groups(int g0, int g1, int lanes, F&& f) {
    const int at_once = kThreads / lanes;
    for (int g = g0; g <= g1; g += at_once) {
        const int mine = g + (int)threadIdx.x / lanes;
        f(min(mine, g1), mine <= g1);
    }
}
// Place of the first channel of group g in a slab.
__device__ __forceinline__ int first_place(const Norm& p, long long first, int g) { return (int)max((long long)g * p.D - first, 0ll); }
// f(j) for this lane's share of the places j of group g in a slab
template <class F>
__device__ __forceinline__ void for_group(const Norm& p, long long first, int channels, int g, int lanes, F&& f) {
    const long long each = p.C / p.fold;
    for (int copy = 0; copy < p.fold; ++copy) {
        const long long base = copy * each - first;
        const long long from = max((long long)g * p.D, -base), end = min((long long)(g + 1) * p.D, channels - base);
        for (long long c = from + (threadIdx.x & (lanes - 1)); c < end; c += lanes) f((int)(base + c));
    }
}

// partial[n][run][slab][group of the slab] = (mean, m2) of the group's channels in the slab over the run's rows
template <class T, int V>
__global__ void __launch_bounds__(kThreads, 3)
sa_norm_partial_kernel(const T* __restrict__ x, float2* __restrict__ partial, const __grid_constant__ Slab s) {
    constexpr int P = (V + 1) / 2;
    extern __shared__ __align__(16) unsigned char memory[];
    float2* const tile = (float2*)memory;              // [lanes][width], after the stream has passed
    float* const centre = (float*)(memory + s.shared); // [width] each: the means of row lane 0, then the channels'; m2
    may_follow();
    const Place w = place_of<V>(s, blockIdx.x);
    const Norm& p = s.p;
    // sums about the first of every kFold rows (what cancels is of the size of a value's own square), joined by Chan's rule
    constexpr int kFold = 32, kRows = kRingWords / kStreamStages;
    F2 k0[P], sum[P], square[P], m[P], q[P];
    float n = 0.0f;
    int have = 0;
#pragma unroll
    for (int k = 0; k < P; ++k) k0[k] = sum[k] = square[k] = m[k] = q[k] = f2(0.0f, 0.0f);
    auto fold = [&] {
        const float c = (float)have, inv = 1.0f / c, share = n > 0.0f ? __fdividef(c, n + c) : 1.0f, weight = n * share;
#pragma unroll
        for (int k = 0; k < P; ++k) {
            const F2 part = sum[k] * f2(inv, inv), d = part + negative(k0[k] + m[k]);
            q[k] = q[k] + fma2(negative(sum[k]), part, square[k]);
            q[k] = fma2(d * f2(weight, weight), d, q[k]); // weight first: 0 for the first rows, however far they are from zero
            m[k] = fma2(d, f2(share, share), m[k]);
            sum[k] = square[k] = f2(0.0f, 0.0f);
        }
        n += c;
        have = 0;
    };
    Stream<T, V> in(memory, x + ((long long)w.n * p.S + (long long)w.rank * s.rows + w.row_lane) * p.C + w.first + w.word * V,
                    (long long)s.row_lanes * p.C);
    stream_rows<kRows>(
        w.rows, [&](int slot) { in.fetch(slot); },
        [&](int slot, int rows) {
            if (have == kFold) fold();
            if (have == 0) {
                const SaVec<T, V> v = in.row(slot);
#pragma unroll
                for (int k = 0; k < P; ++k) k0[k] = negative(pair_of(v, k));
            }
            have += rows;
        },
        [&](int slot) {
            const SaVec<T, V> v = in.row(slot);
#pragma unroll
            for (int k = 0; k < P; ++k) {
                const F2 e = pair_of(v, k) + k0[k];
                sum[k] = sum[k] + e;
                square[k] = fma2(e, e, square[k]);
            }
        });
    if (have > 0) fold();
    __syncthreads(); // the ring becomes the tile
    share_centre<V>(w, m, centre);
    __syncthreads();
    refer_to_centre<V>(w, m, q, n, centre);
    block_sums<V>(s, w, tile, m, q);
    // the channels' means and squared deviations, then some lanes for each group: equally many values in each channel
    float* const deviation = centre + s.width;
    const float rows_inv = w.block_rows > 0 ? 1.0f / (float)w.block_rows : 0.0f;
    for (int j = threadIdx.x; j < w.channels; j += blockDim.x) {
        const float2 t = channel_sum<V>(s, tile, j);
        const float off = t.x * rows_inv;
        centre[j] += off;
        deviation[j] = fmaf(-t.x, off, t.y);
    }
    __syncthreads();
    const int g0 = first_group(p, w.first), g1 = last_group(p, w.first, w.channels);
    float2* const to = partial + (((long long)w.n * s.blocks + w.rank) * s.slabs + w.first / s.width) * s.groups;
    const int lanes = group_lanes(p);
    for_groups(g0, g1, lanes, [&](int g, bool is) {
        float n_channels = 0.0f, sum = 0.0f, m2 = 0.0f;
        const float about = centre[first_place(p, w.first, g)]; // the mean of the group's first channel here: what is summed is small
        for_group(p, w.first, w.channels, g, lanes, [&](int j) {
            n_channels += 1.0f;
            sum += centre[j] - about;
            m2 += deviation[j];
        });
        const float mg = about + __fdividef(lanes_sum(sum, lanes), lanes_sum(n_channels, lanes));
        for_group(p, w.first, w.channels, g, lanes, [&](int j) {
            const float off = centre[j] - mg;
            m2 = fmaf(off * off, (float)w.block_rows, m2);
        });
        m2 = lanes_sum(m2, lanes);
        if (is && (threadIdx.x & (lanes - 1)) == 0) to[g - g0] = make_float2(mg, m2);
    });
}

// mean and rstd of (n, g): one block each
__global__ void __launch_bounds__(kThreads)
sa_norm_join_kernel(const float2* __restrict__ partial, float* __restrict__ mean, float* __restrict__ rstd, const __grid_constant__ Slab s) {
    __shared__ Moments warps[kThreads / 32];
    may_follow();
    const Norm& p = s.p;
    const uint32_t n = blockIdx.x / (uint32_t)p.G, g = blockIdx.x - n * (uint32_t)p.G;
    const float last = (float)(p.S - (long long)(s.blocks - 1) * s.rows);
    const uint32_t c0 = g * (uint32_t)p.D, c1 = c0 + (uint32_t)p.D; // the group's channels lie in slabs t0 to t1
    const uint32_t t0 = p.fold > 1 ? 0 : c0 / (uint32_t)s.width, t1 = p.fold > 1 ? 0 : (c1 - 1) / (uint32_t)s.width;
    Moments m{0.0f, 0.0f, 0.0f};
    await_previous();
    for (uint32_t t = t0; t <= t1; ++t) {
        const uint32_t first = t * (uint32_t)s.width;
        const float channels = p.fold > 1 ? (float)p.D * (float)p.fold : (float)(min(c1, first + (uint32_t)s.width) - max(c0, first));
        const float2* const from = partial + ((long long)n * s.blocks * s.slabs + t) * s.groups + (g - first_group(p, first));
#pragma unroll 4
        for (int r = threadIdx.x; r < s.blocks; r += kThreads) {
            const float2 e = from[(long long)r * s.slabs * s.groups];
            join(m, Moments{(r + 1 == s.blocks ? last : (float)s.rows) * channels, e.x, e.y});
        }
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

// The rows are taken from the end: what the statistics read last is still in L2.
template <class T, int V>
__global__ void __launch_bounds__(kThreads, 3)
sa_norm_apply_kernel(T* out, const T* x, const float* __restrict__ mean, const float* __restrict__ rstd, const __grid_constant__ Slab s) {
    constexpr int P = (V + 1) / 2;
    extern __shared__ __align__(16) unsigned char memory[];
    float* const weight = (float*)(memory + s.shared); // [width] each: weight * rstd, bias, mean
    float* const bias = weight + s.width;
    float* const centre = bias + s.width;
    const Place w = place_of<V>(s, gridDim.x - 1 - blockIdx.x);
    const Norm& p = s.p;
    stage_params(s, w, weight, bias);
    await_previous();
    for (int j = threadIdx.x; j < w.channels; j += blockDim.x) {
        const long long at = (long long)w.n * p.G + (uint32_t)channel_of(p, w.first + j) / (uint32_t)p.D;
        centre[j] = mean[at];
        weight[j] *= rstd[at];
    }
    __syncthreads();
    if (w.rows <= 0) return;
    F2 m[P], a[P], b[P];
    shared_pairs<V>(m, centre + w.word * V);
    shared_pairs<V>(a, weight + w.word * V);
    shared_pairs<V>(b, bias + w.word * V);
#pragma unroll
    for (int k = 0; k < P; ++k) m[k] = negative(m[k]);
    const long long step = (long long)s.row_lanes * p.C;
    const long long base = ((long long)w.n * p.S + (long long)w.rank * s.rows + w.row_lane) * p.C + w.first + w.word * V + (w.rows - 1) * step;
    Stream<T, V> in(memory, x + base, -step);
    T* to = out + base;
    with_activation(p.silu, [&](auto silu) {
        stream_rows<kRingWords / kStreamStages>(
            w.rows, [&](int slot) { in.fetch(slot); }, [](int, int) {},
            [&](int slot) {
                const SaVec<T, V> v = in.row(slot);
                SaVec<T, V> y;
                activation<T, silu.value, P>([&](int k) { return fma2(pair_of(v, k) + m[k], a[k], b[k]); }, [&](int k, F2 e) { set_pair(y, k, e); });
                sa_store_stream<T, V>(to, y);
                to -= step;
            });
    });
}

// partial[n][run][c] = (sum dz, sum dz (x - mean)) over the run's rows
template <class T, int V>
__global__ void __launch_bounds__(kThreads, 3)
sa_norm_backward_partial_kernel(const T* __restrict__ dout, const T* __restrict__ x, const float* __restrict__ mean,
                                const float* __restrict__ rstd, float2* __restrict__ partial, const __grid_constant__ Slab s) {
    constexpr int P = (V + 1) / 2;
    extern __shared__ __align__(16) unsigned char memory[];
    constexpr int kRows = kRingWords / 2 / kStreamStages;
    constexpr size_t kRing = kRingWords / 2 * kThreads * sizeof(SaVec<T, V>);
    float2* const tile = (float2*)memory;             // [lanes][width], after the streams have passed
    float* const slope = (float*)(memory + s.shared); // [width] each: weight * rstd, bias, mean
    float* const bias = slope + s.width;
    float* const centre = bias + s.width;
    may_follow();
    const Place w = place_of<V>(s, blockIdx.x);
    const Norm& p = s.p;
    stage_params(s, w, slope, bias);
    for (int j = threadIdx.x; j < w.channels; j += blockDim.x) {
        const long long at = (long long)w.n * p.G + (uint32_t)channel_of(p, w.first + j) / (uint32_t)p.D;
        centre[j] = mean[at];
        slope[j] *= rstd[at];
    }
    __syncthreads();
    F2 m[P], sl[P], b[P], a0[P], a1[P];
    if (w.row_lane < s.row_lanes) {
        shared_pairs<V>(m, centre + w.word * V);
        shared_pairs<V>(sl, slope + w.word * V);
        shared_pairs<V>(b, bias + w.word * V);
    }
#pragma unroll
    for (int k = 0; k < P; ++k) {
        m[k] = negative(m[k]);
        a0[k] = a1[k] = f2(0.0f, 0.0f);
    }
    const long long step = (long long)s.row_lanes * p.C;
    const long long base = ((long long)w.n * p.S + (long long)w.rank * s.rows + w.row_lane) * p.C + w.first + w.word * V;
    Stream<T, V> in(memory, x + base, step), grad(memory + kRing, dout + base, step);
    with_activation(p.silu, [&](auto silu) {
        stream_rows<kRows>(
            w.rows,
            [&](int slot) {
                in.fetch(slot);
                grad.fetch(slot);
            },
            [](int, int) {},
            [&](int slot) {
                const SaVec<T, V> v = in.row(slot), d = grad.row(slot);
#pragma unroll
                for (int k = 0; k < P; ++k) {
                    const F2 dev = pair_of(v, k) + m[k];
                    const F2 dz = through_activation2<T, silu.value>(pair_of(d, k), fma2(dev, sl[k], b[k]));
                    a0[k] = a0[k] + dz;
                    a1[k] = fma2(dz, dev, a1[k]);
                }
            });
    });
    __syncthreads(); // the rings become the tile
    block_sums<V>(s, w, tile, a0, a1);
    for (int j = threadIdx.x; j < w.channels; j += blockDim.x)
        partial[((long long)w.n * s.blocks + w.rank) * p.C + w.first + j] = channel_sum<V>(s, tile, j);
}

// 32 channels of a block of 1024 threads, which have added up a 32nd of something each (lane = channel, warp = share): the
// sums of channel w in warp w.
__device__ __forceinline__ float2 joined_shares(float2 t) {
    __shared__ float2 tile[32][33];
    tile[threadIdx.x / 32][threadIdx.x % 32] = t;
    __syncthreads();
    t = tile[threadIdx.x % 32][threadIdx.x / 32];
    return make_float2(warp_sum(t.x), warp_sum(t.y));
}

// sums[n][c] = (sum dz, sum dz u): a block for 32 channels of a sample, 32 shares of the runs
__global__ void __launch_bounds__(1024)
sa_norm_backward_sums_kernel(const float2* __restrict__ partial, const float* __restrict__ rstd, float2* __restrict__ sums, const __grid_constant__ Slab s) {
    may_follow();
    const Norm& p = s.p;
    const long long channels = p.C / p.fold;
    const uint32_t tiles = (uint32_t)((channels + 31) / 32), n = blockIdx.x / tiles;
    const long long first = (long long)(blockIdx.x - n * tiles) * 32, c = first + threadIdx.x % 32;
    const int share = threadIdx.x / 32;
    float2 t = make_float2(0.0f, 0.0f);
    await_previous();
    if (c < channels) {
        for (int copy = 0; copy < p.fold; ++copy) { // the pixels side by side
            const float2* const from = partial + (long long)n * s.blocks * p.C + copy * channels + c;
#pragma unroll 4
            for (int r = share; r < s.blocks; r += 32) {
                const float2 e = from[(long long)r * p.C];
                t.x += e.x;
                t.y += e.y;
            }
        }
    }
    t = joined_shares(t);
    const long long mine = first + share;
    if (threadIdx.x % 32 == 0 && mine < channels)
        sums[(long long)n * channels + mine] = make_float2(t.x, t.y * rstd[(long long)n * p.G + (uint32_t)mine / (uint32_t)p.D]);
}

// dbias, dweight = the sums of the `count` rows of sums[count][C]: a block for 32 channels, 32 shares of the rows
__global__ void __launch_bounds__(1024)
sa_norm_backward_params_kernel(const float2* __restrict__ sums, void* __restrict__ dweight, void* __restrict__ dbias, int count, int C, int dtype) {
    await_previous();
    const int first = (int)blockIdx.x * 32, c = first + (int)threadIdx.x % 32, share = threadIdx.x / 32;
    float2 t = make_float2(0.0f, 0.0f);
    if (c < C) {
#pragma unroll 8
        for (int r = share; r < count; r += 32) {
            const float2 e = sums[(long long)r * C + c];
            t.x += e.x;
            t.y += e.y;
        }
    }
    t = joined_shares(t);
    const int mine = first + share;
    if (threadIdx.x % 32 != 0 || mine >= C) return;
    if (dbias) sa_set_param(dbias, mine, dtype, t.x);
    if (dweight) sa_set_param(dweight, mine, dtype, t.y);
}

// The rows are taken from the end, as above.
template <class T, int V>
__global__ void __launch_bounds__(kThreads, 3)
sa_norm_backward_apply_kernel(T* dx, const T* dout, const T* x, const float* __restrict__ mean, const float* __restrict__ rstd,
                              const float2* __restrict__ sums, const __grid_constant__ Slab s) {
    constexpr int P = (V + 1) / 2;
    extern __shared__ __align__(16) unsigned char memory[];
    constexpr int kRows = kRingWords / 2 / kStreamStages;
    constexpr size_t kRing = kRingWords / 2 * kThreads * sizeof(SaVec<T, V>);
    float* const slope = (float*)(memory + s.shared); // [width] each: weight * rstd, bias, mean, the two means of the gradient
    float* const bias = slope + s.width;
    float* const centre = bias + s.width;
    float* const first = centre + s.width;
    float* const second = first + s.width;
    const Place w = place_of<V>(s, gridDim.x - 1 - blockIdx.x);
    const Norm& p = s.p;
    may_follow();
    stage_params(s, w, slope, bias);
    await_previous();
    for (int j = threadIdx.x; j < w.channels; j += blockDim.x) {
        const long long at = (long long)w.n * p.G + (uint32_t)channel_of(p, w.first + j) / (uint32_t)p.D;
        centre[j] = mean[at];
        slope[j] *= rstd[at];
    }
    // -rstd m1 and -rstd^2 m2 of the groups, from the sums of all their channels: these are in this slab (and come through
    // shared memory), unless there are several slabs
    const long long each = p.C / p.fold;
    const float2* const of_sample = sums + (long long)w.n * each;
    auto weighted = [&](long long c) {
        const float wc = p.weight ? sa_param(p.weight, c, p.param_dtype) : 1.0f;
        const float2 e = of_sample[c];
        return make_float2(wc * e.x, wc * e.y);
    };
    if (s.slabs == 1) {
        for (int j = threadIdx.x; j < (int)each; j += kThreads) {
            const float2 e = weighted(j);
            first[j] = e.x;
            second[j] = e.y;
        }
        __syncthreads();
    }
    const float inv = 1.0f / ((float)p.S * (float)p.fold * (float)p.D);
    const int lanes = s.slabs == 1 ? group_lanes(p) : 32;
    for_groups(first_group(p, w.first), last_group(p, w.first, w.channels), lanes, [&](int g, bool is) {
        float2 t = make_float2(0.0f, 0.0f);
        // (lanes without a group of their own leave the last one's channels alone: its own lanes overwrite them below)
        for (int d = threadIdx.x & (lanes - 1); is && d < p.D; d += lanes) {
            const int c = g * p.D + d;
            const float2 e = s.slabs == 1 ? make_float2(first[c], second[c]) : weighted(c);
            t.x += e.x;
            t.y += e.y;
        }
        const float rs = rstd[(long long)w.n * p.G + g];
        const float m1 = -rs * (lanes_sum(t.x, lanes) * inv), m2 = -rs * (lanes_sum(t.y, lanes) * inv) * rs;
        __syncwarp(); // every lane of the group has read its channels
        if (is)
            for_group(p, w.first, w.channels, g, lanes, [&](int j) {
                first[j] = m1;
                second[j] = m2;
            });
        __syncwarp();
    });
    __syncthreads();
    if (w.rows <= 0) return;
    F2 m[P], sl[P], b[P], m1[P], m2[P];
    shared_pairs<V>(m, centre + w.word * V);
    shared_pairs<V>(sl, slope + w.word * V);
    shared_pairs<V>(b, bias + w.word * V);
    shared_pairs<V>(m1, first + w.word * V);
    shared_pairs<V>(m2, second + w.word * V);
#pragma unroll
    for (int k = 0; k < P; ++k) m[k] = negative(m[k]);
    const long long step = (long long)s.row_lanes * p.C;
    const long long base = ((long long)w.n * p.S + (long long)w.rank * s.rows + w.row_lane) * p.C + w.first + w.word * V + (w.rows - 1) * step;
    Stream<T, V> in(memory, x + base, -step), grad(memory + kRing, dout + base, -step);
    T* to = dx + base;
    with_activation(p.silu, [&](auto silu) {
        stream_rows<kRows>(
            w.rows,
            [&](int slot) {
                in.fetch(slot);
                grad.fetch(slot);
            },
            [](int, int) {},
            [&](int slot) {
                SaVec<T, V> v = in.row(slot);
                const SaVec<T, V> d = grad.row(slot);
#pragma unroll
                for (int k = 0; k < P; ++k) {
                    const F2 dev = pair_of(v, k) + m[k];
                    const F2 dz = through_activation2<T, silu.value>(pair_of(d, k), fma2(dev, sl[k], b[k]));
                    set_pair(v, k, fma2(dev, m2[k], fma2(sl[k], dz, m1[k])));
                }
                sa_store_stream<T, V>(to, v);
                to -= step;
            });
    });
}

// ---------------------------------------------------------------------------
// resident: a cluster for a slab of groups of one sample
// ---------------------------------------------------------------------------
// Statistics of a thread: sums of x - K and of its square, K being the thread's first row.  What cancels when they are put
// together is of the size of K's own square, and K is one of a few values: nothing is lost.  The block's threads then refer
// their sums to the mean of row lane 0 (the same argument, with its rows among the block's), which makes them plain sums;
// the channels of a group have equally many values, and the blocks of a cluster are joined by Chan's rule.
template <class T, int V>
__global__ void __maxnreg__(kResidentRegisters)
sa_norm_resident_kernel(T* out, const T* x, float* __restrict__ mean, float* __restrict__ rstd, const __grid_constant__ Slab s) {
    constexpr int P = (V + 1) / 2;
    extern __shared__ __align__(16) unsigned char memory[];
    SaVec<T, V>* const data = (SaVec<T, V>*)memory;                                           // [rows][words]
    float2* const tile = (float2*)(memory + ((size_t)s.rows * s.words * sizeof(*data) + 15) / 16 * 16); // [lanes][width] sums
    float2* const joined = tile + (s.row_lanes + 1) / 2 * s.width;                             // [groups] (mean, m2) of this block
    float* const weight = (float*)(joined + s.groups); // [width] each: weight, then weight * rstd; bias; the means of row lane 0, then the groups'
    float* const bias = weight + s.width;
    float* const centre = bias + s.width;
    const Place w = place_of<V>(s, blockIdx.x);
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
        const float share = __fdividef(1.0f, n);
        const F2 inv = f2(share, share);
#pragma unroll
        for (int k = 0; k < P; ++k) {
            const F2 part = m[k] * inv;
            q[k] = fma2(negative(m[k]), part, q[k]);
            m[k] = part + negative(k0[k]);
        }
    }
    share_centre<V>(w, m, centre);
    __syncthreads();
    refer_to_centre<V>(w, m, q, n, centre);
    block_sums<V>(s, w, tile, m, q);
    // a warp for each group: its channels, then the blocks of the cluster (lane r has block r), then the channels' constants
    const int lane = threadIdx.x % 32, warp = threadIdx.x / 32, warps = blockDim.x / 32;
    const float rows_inv = w.block_rows > 0 ? __fdividef(1.0f, (float)w.block_rows) : 0.0f, D_inv = __fdividef(1.0f, (float)p.D);
    auto finish = [&](int g, float mg, float m2, float count) { // all lanes have the group's moments
        const float rs = 1.0f / sqrtf(m2 / count + p.eps);
        for (int d = lane; d < p.D; d += 32) {
            centre[g * p.D + d] = mg;
            weight[g * p.D + d] *= rs;
        }
        if (w.rank == 0 && lane == 0) {
            const long long at = (long long)w.n * p.G + w.group0 + g;
            mean[at] = mg;
            rstd[at] = rs;
        }
    };
    for (int g = warp; g < w.groups; g += warps) {
        float sum = 0.0f, m2 = 0.0f;
        const float about = centre[g * p.D]; // a mean of the group's first channel: what is summed is small
        __syncwarp();                        // before it becomes that of all rows
        for (int d = lane; d < p.D; d += 32) { // a channel's mean and squared deviations
            const int c = g * p.D + d;
            const float2 t = channel_sum<V>(s, tile, c);
            const float off = t.x * rows_inv, mc = centre[c] + off;
            centre[c] = mc;
            m2 += fmaf(-t.x, off, t.y);
            sum += mc - about;
        }
        const float mg = about + warp_sum(sum) * D_inv;
        for (int d = lane; d < p.D; d += 32) {
            const float off = centre[g * p.D + d] - mg; // written by this lane
            m2 = fmaf(off * off, (float)w.block_rows, m2);
        }
        m2 = warp_sum(m2);
        if (s.blocks == 1) finish(g, mg, m2, (float)w.block_rows * (float)p.D);
        else if (lane == 0) joined[g] = make_float2(mg, m2);
    }

    cg::cluster_group cluster = cg::this_cluster();
    if (s.blocks > 1) {
        cluster.sync();
        for (int g = warp; g < w.groups; g += warps) {
            Moments t{0.0f, 0.0f, 0.0f};
            if (lane < s.blocks) {
                const float2 e = *cluster.map_shared_rank(joined + g, lane);
                t = Moments{(float)max(0, min((int)p.S - lane * s.rows, s.rows)) * (float)p.D, e.x, e.y};
            }
#pragma unroll
            for (int o = kMaxCluster / 2; o > 0; o >>= 1)
                join(t, Moments{__shfl_down_sync(0xffffffffu, t.n, o), __shfl_down_sync(0xffffffffu, t.mean, o), __shfl_down_sync(0xffffffffu, t.m2, o)});
            finish(g, __shfl_sync(0xffffffffu, t.mean, 0), __shfl_sync(0xffffffffu, t.m2, 0), __shfl_sync(0xffffffffu, t.n, 0));
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
        with_activation(p.silu, [&](auto silu) {
            T* to = out + base;
            const SaVec<T, V>* row = mine;
#pragma unroll 2
            for (int u = 0; u < w.rows; ++u, to += step, row += stride) {
                const SaVec<T, V> v = *row;
                SaVec<T, V> y;
                activation<T, silu.value, P>([&](int k) { return fma2(pair_of(v, k) + m[k], a[k], b[k]); }, [&](int k, F2 e) { set_pair(y, k, e); });
                sa_store<T, V>(to, y);
            }
        });
    }
    if (s.blocks > 1) cluster.barrier_wait(); // no block leaves while a neighbour may still read its shared memory
}

// The deviations x - mean stand for u = (x - mean) rstd throughout, rstd goes into the constants:
//   z = (x - mean) (w rstd) + b,  dx = (w rstd) dz - rstd m1 - (x - mean) rstd^2 m2
// `sums`: (sum dz, sum dz u) of every (n, c); NULL: there is one sample, dweight and dbias are written here
template <class T, int V>
__global__ void __maxnreg__(kResidentBackwardRegisters)
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
    may_follow();
    const Place w = place_of<V>(s, blockIdx.x);
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
        with_activation(p.silu, [&](auto silu) {
            as_rows_arrive(w.rows, [&](int u, int end) {
                const SaVec<T, V>*row = mine + u * stride, *other = theirs + u * stride;
#pragma unroll 2
                for (; u < end; ++u, row += stride, other += stride) {
                    const SaVec<T, V> v = *row, d = *other;
#pragma unroll
                    for (int k = 0; k < P; ++k) {
                        const F2 dev = pair_of(v, k) + m[k];
                        const F2 dz = through_activation2<T, silu.value>(pair_of(d, k), fma2(dev, sl[k], b[k]));
                        a0[k] = a0[k] + dz;
                        a1[k] = fma2(dz, dev, a1[k]);
                    }
                }
            });
        });
        block_sums<V>(s, w, tile, a0, a1);
    }
    for (int j = threadIdx.x; j < s.width; j += blockDim.x) channel[j] = channel_sum<V>(s, tile, j);
    cg::cluster_group cluster = cg::this_cluster();
    if (s.blocks > 1) cluster.sync();
    else __syncthreads();
    for (int j = threadIdx.x; j < w.channels; j += blockDim.x) {
        float2 t = channel[j];
        if (s.blocks > 1) {
            t = make_float2(0.0f, 0.0f);
#pragma unroll
            for (int r = 0; r < kMaxCluster; ++r) { // all in flight together
                if (r < s.blocks) {
                    const float2 e = *cluster.map_shared_rank(channel + j, r);
                    t.x += e.x;
                    t.y += e.y;
                }
            }
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
            int g = (int)s.by_D.div(w.word * V), r = w.word * V - g * p.D;
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const float2 e = means[g];
                x1[i] = e.x;
                x2[i] = e.y;
                if (++r == p.D) {
                    r = 0;
                    ++g;
                }
            }
#pragma unroll
            for (int k = 0; k < P; ++k) {
                m1[k] = f2(x1[2 * k], x1[2 * k + 1]);
                m2[k] = f2(x2[2 * k], x2[2 * k + 1]);
            }
        }
        with_activation(p.silu, [&](auto silu) {
            T* to = dx + base;
            const SaVec<T, V>*row = mine, *other = theirs;
#pragma unroll 2
            for (int u = 0; u < w.rows; ++u, to += step, row += stride, other += stride) {
                SaVec<T, V> v = *row;
                const SaVec<T, V> d = *other;
#pragma unroll
                for (int k = 0; k < P; ++k) {
                    const F2 dev = pair_of(v, k) + m[k];
                    const F2 dz = through_activation2<T, silu.value>(pair_of(d, k), fma2(dev, sl[k], b[k]));
                    set_pair(v, k, fma2(dev, m2[k], fma2(sl[k], dz, m1[k])));
                }
                sa_store<T, V>(to, v);
            }
        });
    }
    if (s.blocks > 1) cluster.barrier_wait(); // no block leaves while a neighbour may still read its shared memory
}

// ---------------------------------------------------------------------------
// packed: short samples, several of them in a block's shared memory at a time
// ---------------------------------------------------------------------------
// A block goes through tiles of `samples` whole samples of its slab; the next tile travels while one is worked on.  A thread
// has one word of the row, so parameters and their gradients stay in its registers; `lanes` neighbouring threads take the
// statistics of a group of a sample: its mean about one of its elements, then the squared deviations from that.
// Blocks of an SM: what the registers allow without spills; forward four of whole words were slower than three with larger tiles
// (65536 x 4 x 64 bf16: 30.9 against 24.2 us).
constexpr int packed_on_sm(int tensors, bool whole) { return tensors == 1 || whole ? 3 : 2; }

struct Pack {
    int slab, first_tile;
    int word, row_lane;
    int channels, groups; // of this slab (the last one of a sample may be narrower)
    long long first;      // first channel of the slab
    int group0;           // first group of the slab
    int g, rem;           // group of the thread's first channel in the slab, place in that group
    int next, edge;       // the group after it, if the word reaches that far; first channel of the word that belongs to it
    bool busy;            // has a word
};

template <int V>
__device__ __forceinline__ Pack pack_of(const Slab& s) {
    Pack w;
    w.slab = (int)(blockIdx.x / (uint32_t)s.blocks);
    w.first_tile = (int)(blockIdx.x - (uint32_t)w.slab * s.blocks);
    w.row_lane = (int)s.by_words.div(threadIdx.x);
    w.word = (int)threadIdx.x - w.row_lane * s.words;
    w.group0 = w.slab * s.groups;
    w.first = (long long)w.slab * s.width;
    w.groups = min(s.groups, s.p.G - w.group0);
    w.channels = (int)min((long long)s.width, s.p.C - w.first);
    w.g = (int)s.by_D.div((uint32_t)(w.word * V));
    w.rem = w.word * V - w.g * s.p.D;
    w.edge = s.p.D - w.rem;
    w.next = w.g + (w.edge < V ? 1 : 0);
    w.busy = w.row_lane < s.row_lanes && w.word * V < w.channels;
    return w;
}
// Rows of a tile (they follow one another in memory, whole samples).
__device__ __forceinline__ int tile_samples(const Slab& s, int tile) { return min(s.samples, s.p.N - tile * s.samples); }

// WHOLE in these kernels: groups are whole words, which takes a register instead of a word of them for every group's value
// (16384 x 1 x 2048 bf16 backward: 137 us without it).
// The values of this thread's channels out of one for each group, as pairs.  Otherwise words have at most one border between
// pairs, or any, the same for all threads.
template <int V, bool WHOLE>
__device__ __forceinline__ void of_groups(const Pack& w, int D, const float* at, F2 (&out)[(V + 1) / 2]) {
    if (WHOLE) {
        const float v = at[w.g];
#pragma unroll
        for (int k = 0; k < (V + 1) / 2; ++k) out[k] = f2(v, v);
    } else if (D >= V && D % 2 == 0) {
        const float v0 = at[w.g], v1 = at[w.next];
#pragma unroll
        for (int k = 0; k < (V + 1) / 2; ++k) {
            const float v = 2 * k < w.edge ? v0 : v1;
            out[k] = f2(v, v);
        }
    } else {
        float v[(V + 1) / 2 * 2] = {};
        int g = w.g, r = w.rem;
#pragma unroll
        for (int i = 0; i < V; ++i) {
            v[i] = at[g];
            if (++r == D) {
                r = 0;
                ++g;
            }
        }
#pragma unroll
        for (int k = 0; k < (V + 1) / 2; ++k) out[k] = f2(v[2 * k], v[2 * k + 1]);
    }
}

// Elements of an item, what a thread takes of a group at a time: as many as divide the group, up to a word.
// f(std::integral_constant) for that number, the same for all threads.
template <int V, bool WHOLE, class F>
__device__ __forceinline__ void with_items(int D, F&& f) {
    if constexpr (WHOLE) f(std::integral_constant<int, V>());
    else if (V > 4 && D % 4 == 0) f(std::integral_constant<int, (V > 4 ? 4 : V)>());
    else if (V > 2 && D % 2 == 0) f(std::integral_constant<int, (V > 2 ? 2 : V)>());
    else f(std::integral_constant<int, 1>());
}

// weight and bias of this thread's channels
template <int V>
__device__ __forceinline__ void params_of(const Norm& p, const Pack& w, F2 (&weight)[(V + 1) / 2], F2 (&bias)[(V + 1) / 2]) {
    float a[(V + 1) / 2 * 2] = {}, b[(V + 1) / 2 * 2] = {};
    if (w.busy) {
#pragma unroll
        for (int i = 0; i < V; ++i) {
            a[i] = p.weight ? sa_param(p.weight, w.first + w.word * V + i, p.param_dtype) : 1.0f;
            b[i] = p.bias ? sa_param(p.bias, w.first + w.word * V + i, p.param_dtype) : 0.0f;
        }
    }
#pragma unroll
    for (int k = 0; k < (V + 1) / 2; ++k) {
        weight[k] = f2(a[2 * k], a[2 * k + 1]);
        bias[k] = f2(b[2 * k], b[2 * k + 1]);
    }
}

// f(sample, group, first element or word, last + 1, whether there is such a group) for the groups of a tile, `lanes` threads each;
// all threads of a warp call f together.
template <class F>
__device__ __forceinline__ void for_teams(const Slab& s, int samples, F&& f) {
    const int teams = samples * s.groups, at_once = kThreads / s.lanes;
    for (int t0 = 0; t0 < teams; t0 += at_once) {
        const int t = min(t0 + (int)threadIdx.x / s.lanes, teams - 1);
        const int sample = (int)s.by_groups.div((uint32_t)t);
        f(sample, t - sample * s.groups, t, t0 + (int)threadIdx.x / s.lanes < teams);
    }
}

template <class T, int V, bool WHOLE>
__global__ void __launch_bounds__(kThreads, packed_on_sm(1, WHOLE))
sa_norm_packed_kernel(T* out, const T* x, float* __restrict__ mean, float* __restrict__ rstd, const __grid_constant__ Slab s) {
    constexpr int P = (V + 1) / 2;
    using Word = SaVec<T, V>;
    extern __shared__ __align__(16) unsigned char memory[];
    const size_t bytes = ((size_t)s.rows * s.pitch * sizeof(Word) + 15) / 16 * 16;
    float* const centre = (float*)(memory + 2 * bytes); // [samples][groups] each: mean, rstd
    float* const scale = centre + s.samples * s.groups;
    const Pack w = pack_of<V>(s);
    const Norm& p = s.p;
    const int S = (int)p.S, D = p.D, width = s.pitch * V;
    const long long step = (long long)s.row_lanes * p.C, base = (long long)w.row_lane * p.C + w.first + w.word * V;
    const int own = w.row_lane * s.pitch + w.word, stride = s.row_lanes * s.pitch;
    auto fetch = [&](int tile, int buffer) {
        if (tile < s.tiles && w.busy) {
            const T* from = x + (long long)tile * s.samples * S * p.C + base;
            Word* to = (Word*)(memory + buffer * bytes) + own;
            const int rows = tile_samples(s, tile) * S;
#pragma unroll 4
            for (int r = w.row_lane; r < rows; r += s.row_lanes, from += step, to += stride) fetch_row<T, V>(to, from);
        }
        end_of_stage();
    };
    fetch(w.first_tile, 0);
    F2 weight[P], bias[P];
    params_of<V>(p, w, weight, bias);
    const float inv = 1.0f / ((float)S * (float)D);
    int buffer = 0;
    for (int tile = w.first_tile; tile < s.tiles; tile += s.blocks, buffer ^= 1) {
        asm volatile("cp.async.wait_group 0;" ::: "memory");
        __syncthreads();
        fetch(tile + s.blocks, buffer ^ 1);
        const Word* const data = (const Word*)(memory + buffer * bytes);
        const int samples = tile_samples(s, tile);
        for_teams(s, samples, [&](int sample, int g, int t, bool is) {
            const T* const at = (const T*)data + sample * S * width + g * D;
            const bool real = g < w.groups;
            const int sub = threadIdx.x & (s.lanes - 1), count = real ? S * D : 0;
            const float k0 = real ? sa_to_float(*at) : 0.0f;
            float m = 0.0f, m2 = 0.0f;
            with_items<V, WHOLE>(D, [&](auto size) {
                constexpr int W = size.value;
                auto each = [&](float about, auto&& f) {
                    const F2 c = f2(-about, -about);
#pragma unroll 2
                    for (int e = sub * W; e < count; e += s.lanes * W) {
                        const SaVec<T, W> v = sa_load<T, W>(at + e + (int)s.by_D.div((uint32_t)e) * (width - D));
                        if constexpr (W == 1) f(f2(sa_to_float(v.e[0]) - about, 0.0f));
                        else {
#pragma unroll
                            for (int k = 0; k < W / 2; ++k) f(pair_of(v, k) + c);
                        }
                    }
                };
                auto all = [&](F2 v) {
                    float a, b;
                    split(v, a, b);
                    return lanes_sum(a + b, s.lanes);
                };
                F2 total = f2(0.0f, 0.0f), square = total;
                each(k0, [&](F2 d) {
                    total = total + d;
                    square = fma2(d, d, square);
                });
                const float sum = all(total), squares = all(square), off = sum * inv;
                m = k0 + off;
                m2 = fmaf(-sum, off, squares);
                // the first element is far out: what cancels would be 16 times what is left, so once more about the mean
                const bool again = !(squares <= 16.0f * m2);
                if (__any_sync(0xffffffffu, again)) {
                    square = f2(0.0f, 0.0f);
                    each(m, [&](F2 d) { square = fma2(d, d, square); });
                    const float exact = all(square);
                    if (again) m2 = exact;
                }
            });
            if (is && real && sub == 0) {
                const float rs = 1.0f / sqrtf(m2 * inv + p.eps);
                centre[t] = m;
                scale[t] = rs;
                const long long to = ((long long)tile * s.samples + sample) * p.G + w.group0 + g;
                mean[to] = m;
                rstd[to] = rs;
            }
        });
        __syncthreads();
        if (!w.busy) continue;
        T* to = out + (long long)tile * s.samples * S * p.C + base;
        const Word* row = data + own;
        const int rows = samples * S;
        F2 m[P], a[P];
        int have = -1;
        with_activation(p.silu, [&](auto silu) {
            for (int r = w.row_lane; r < rows; r += s.row_lanes, to += step, row += stride) {
                const Word v = *row;
                if (const int of = (int)s.by_S.div((uint32_t)r) * s.groups; of != have) { // the next sample
                    have = of;
                    of_groups<V, WHOLE>(w, D, centre + of, m);
                    of_groups<V, WHOLE>(w, D, scale + of, a);
#pragma unroll
                    for (int k = 0; k < P; ++k) {
                        m[k] = negative(m[k]);
                        a[k] = a[k] * weight[k];
                    }
                }
                Word y;
                activation<T, silu.value, P>([&](int k) { return fma2(pair_of(v, k) + m[k], a[k], bias[k]); }, [&](int k, F2 e) { set_pair(y, k, e); });
                sa_store_stream<T, V>(to, y);
            }
        });
    }
}

// `partial`: [blocks of a slab][C], each block's sums of (dz, dz u) over its samples; NULL: there is one block, dweight and
// dbias are written here.  dz is kept in fp32 in
// shared memory, so that the activation's derivative is worked out once.
template <class T, int V, bool WHOLE>
__global__ void __launch_bounds__(kThreads, packed_on_sm(2, WHOLE))
sa_norm_packed_backward_kernel(T* dx, const T* dout, const T* x, const float* __restrict__ mean, const float* __restrict__ rstd,
                               float2* __restrict__ partial, void* __restrict__ dweight, void* __restrict__ dbias,
                               const __grid_constant__ Slab s) {
    constexpr int P = (V + 1) / 2;
    using Word = SaVec<T, V>;
    using Floats = SaVec<float, (V >= 4 ? 4 : V)>;
    constexpr int kPer = V >= 4 ? 4 : V;
    extern __shared__ __align__(16) unsigned char memory[];
    const size_t bytes = ((size_t)s.rows * s.pitch * sizeof(Word) + 15) / 16 * 16;
    const int teams = s.samples * s.groups, width = s.pitch * V;
    float* const flow = (float*)(memory + 4 * bytes); // dz, as x lies; in the end the sums of the block
    const size_t tile_floats = (size_t)s.rows * width, sum_floats = (size_t)(s.row_lanes + 1) / 2 * s.width * 2;
    float* const weights = flow + ((tile_floats > sum_floats ? tile_floats : sum_floats) + 3) / 4 * 4; // [width]
    float* const biases = weights + (s.width + 3) / 4 * 4;
    float* const first = biases + (s.width + 3) / 4 * 4;  // [teams] each: -rstd m1, -rstd^2 m2
    float* const second = first + teams;
    float* const stats = second + teams;                  // [2][teams] means, [2][teams] rstd
    may_follow();
    const Pack w = pack_of<V>(s);
    const Norm& p = s.p;
    const int S = (int)p.S, D = p.D;
    const long long step = (long long)s.row_lanes * p.C, base = (long long)w.row_lane * p.C + w.first + w.word * V;
    const int own = w.row_lane * s.pitch + w.word, stride = s.row_lanes * s.pitch;
    auto fetch = [&](int tile, int buffer) {
        if (tile < s.tiles) {
            const int samples = tile_samples(s, tile), rows = samples * S;
            if (w.busy) {
                const long long at = (long long)tile * s.samples * S * p.C + base;
                const T *from = x + at, *other = dout + at;
                Word* to = (Word*)(memory + buffer * bytes) + own;
                Word* beside = (Word*)(memory + (2 + buffer) * bytes) + own;
#pragma unroll 2
                for (int r = w.row_lane; r < rows; r += s.row_lanes, from += step, other += step, to += stride, beside += stride) {
                    fetch_row<T, V>(to, from);
                    fetch_row<T, V>(beside, other);
                }
            }
            for (int t = threadIdx.x; t < samples * s.groups; t += kThreads) {
                const int sample = (int)s.by_groups.div((uint32_t)t), g = t - sample * s.groups;
                if (g >= w.groups) continue;
                const long long at = ((long long)tile * s.samples + sample) * p.G + w.group0 + g;
                fetch_row<float, 1>((SaVec<float, 1>*)(stats + buffer * teams + t), mean + at);
                fetch_row<float, 1>((SaVec<float, 1>*)(stats + (2 + buffer) * teams + t), rstd + at);
            }
        }
        end_of_stage();
    };
    fetch(w.first_tile, 0);
    for (int j = threadIdx.x; j < s.width; j += kThreads) {
        weights[j] = p.weight && j < w.channels ? sa_param(p.weight, w.first + j, p.param_dtype) : 1.0f;
        biases[j] = p.bias && j < w.channels ? sa_param(p.bias, w.first + j, p.param_dtype) : 0.0f;
    }
    F2 a0[P], a1[P];
#pragma unroll
    for (int k = 0; k < P; ++k) a0[k] = a1[k] = f2(0.0f, 0.0f);
    const float inv = 1.0f / ((float)S * (float)D);
    int buffer = 0;
    for (int tile = w.first_tile; tile < s.tiles; tile += s.blocks, buffer ^= 1) {
        asm volatile("cp.async.wait_group 0;" ::: "memory");
        __syncthreads();
        fetch(tile + s.blocks, buffer ^ 1);
        const Word* const data = (const Word*)(memory + buffer * bytes);
        const Word* const grad = (const Word*)(memory + (2 + buffer) * bytes);
        const float *const centre = stats + buffer * teams, *const scale = stats + (2 + buffer) * teams;
        const int samples = tile_samples(s, tile), rows = samples * S;
        if (w.busy) {
            with_activation(p.silu, [&](auto silu) {
                int at = own, have = -1;
                F2 m[P], rs[P];
                for (int r = w.row_lane; r < rows; r += s.row_lanes, at += stride) {
                    const Word v = data[at], d = grad[at];
                    if (const int of = (int)s.by_S.div((uint32_t)r) * s.groups; of != have) { // the next sample
                        have = of;
                        of_groups<V, WHOLE>(w, D, centre + of, m);
                        of_groups<V, WHOLE>(w, D, scale + of, rs);
                    }
                    F2 weight[P], bias[P];
                    shared_pairs<V>(weight, weights + w.word * V);
                    shared_pairs<V>(bias, biases + w.word * V);
                    float dzs[2 * P];
#pragma unroll
                    for (int k = 0; k < P; ++k) {
                        const F2 u = (pair_of(v, k) + negative(m[k])) * rs[k];
                        const F2 dz = through_activation2<T, silu.value>(pair_of(d, k), fma2(u, weight[k], bias[k]));
                        a0[k] = a0[k] + dz;
                        a1[k] = fma2(dz, u, a1[k]);
                        split(dz, dzs[2 * k], dzs[2 * k + 1]);
                    }
#pragma unroll
                    for (int k = 0; k < V / kPer; ++k) {
                        Floats f;
#pragma unroll
                        for (int i = 0; i < kPer; ++i) f.e[i] = dzs[k * kPer + i];
                        *(Floats*)(flow + (size_t)at * V + k * kPer) = f;
                    }
                }
            });
        }
        __syncthreads();
        for_teams(s, samples, [&](int sample, int g, int t, bool is) {
            const bool real = g < w.groups;
            const int sub = threadIdx.x & (s.lanes - 1), count = real ? S * D : 0, from = sample * S * width + g * D;
            const T* const at = (const T*)data + from;
            const float *const dz = flow + from, *const wg = weights + g * D;
            const float m = real ? centre[t] : 0.0f, rs = real ? scale[t] : 0.0f;
            float t1 = 0.0f, t2 = 0.0f;
            with_items<V, WHOLE>(D, [&](auto size) {
                constexpr int W = size.value;
                constexpr int kPiece = W >= 4 ? 4 : W;
                F2 s1 = f2(0.0f, 0.0f), s2 = s1;
#pragma unroll 2
                for (int e = sub * W; e < count; e += s.lanes * W) {
                    const int row = (int)s.by_D.div((uint32_t)e), place = e + row * (width - D);
                    const SaVec<T, W> v = sa_load<T, W>(at + place);
#pragma unroll
                    for (int k = 0; k < W; k += kPiece) {
                        const auto z = sa_load<float, kPiece>(dz + place + k), we = sa_load<float, kPiece>(wg + e - row * D + k);
                        if constexpr (W == 1) {
                            const float q = z.e[0] * we.e[0];
                            s1 = s1 + f2(q, 0.0f);
                            s2 = s2 + f2(q * (sa_to_float(v.e[0]) - m), 0.0f);
                        } else {
#pragma unroll
                            for (int i = 0; i < kPiece / 2; ++i) {
                                const F2 q = f2(z.e[2 * i], z.e[2 * i + 1]) * f2(we.e[2 * i], we.e[2 * i + 1]);
                                s1 = s1 + q;
                                s2 = fma2(q, pair_of(v, k / 2 + i) + f2(-m, -m), s2);
                            }
                        }
                    }
                }
                float a, b;
                split(s1, a, b);
                t1 = a + b;
                split(s2, a, b);
                t2 = a + b;
            });
            t1 = lanes_sum(t1, s.lanes) * inv;
            t2 = lanes_sum(t2, s.lanes) * inv;
            if (is && real && sub == 0) { // dx = (w rstd) dz - rstd m1 - (x - mean) rstd^2 m2, m2 = rstd t2
                first[t] = -rs * t1;
                second[t] = -rs * (rs * (rs * t2));
            }
        });
        __syncthreads();
        if (!w.busy) continue;
        T* to = dx + (long long)tile * s.samples * S * p.C + base;
        int at = own, have = -1;
        F2 m[P], a[P], m1[P], m2[P];
        for (int r = w.row_lane; r < rows; r += s.row_lanes, at += stride, to += step) {
            Word v = data[at];
            if (const int of = (int)s.by_S.div((uint32_t)r) * s.groups; of != have) {
                have = of;
                F2 weight[P];
                shared_pairs<V>(weight, weights + w.word * V);
                of_groups<V, WHOLE>(w, D, centre + of, m);
                of_groups<V, WHOLE>(w, D, scale + of, a);
                of_groups<V, WHOLE>(w, D, first + of, m1);
                of_groups<V, WHOLE>(w, D, second + of, m2);
#pragma unroll
                for (int k = 0; k < P; ++k) a[k] = a[k] * weight[k];
            }
            F2 dz[P];
            shared_pairs<V>(dz, flow + (size_t)at * V);
#pragma unroll
            for (int k = 0; k < P; ++k) set_pair(v, k, fma2(pair_of(v, k) + negative(m[k]), m2[k], fma2(a[k], dz[k], m1[k])));
            sa_store_stream<T, V>(to, v);
        }
    }
    if (!partial && !dweight && !dbias) return;
    __syncthreads(); // dz becomes the sums
    Place place{};
    place.word = w.word;
    place.row_lane = w.row_lane;
    block_sums<V>(s, place, (float2*)flow, a0, a1);
    for (int j = threadIdx.x; j < w.channels; j += kThreads) {
        const float2 t = channel_sum<V>(s, (const float2*)flow, j);
        if (partial) partial[(long long)w.first_tile * p.C + w.first + j] = t;
        else {
            if (dbias) sa_set_param(dbias, w.first + j, p.param_dtype, t.x);
            if (dweight) sa_set_param(dweight, w.first + j, p.param_dtype, t.y);
        }
    }
}

// ---------------------------------------------------------------------------
// launches
// ---------------------------------------------------------------------------
// Threads that share a channel's column of `lanes` values: the column is added up in lanes / shares steps, the shares in
// `shares` steps, so the square root is best.
int shares(int lanes, int most) {
    int n = 1;
    while (n < most && n * n < lanes) ++n;
    return n;
}

// Samples too long to be resident: words across a block, rows at a time, runs of rows.  Three blocks for each SM, but runs
// of at least 8 rows for each row lane (4 x 100000 x 6 bf16: 12.3 us, with 32 rows 16.3).
Slab cut(const Norm& p, int V) {
    Slab s{};
    s.p = p;
    const long long words = p.C / V;
    const long long tiles = (words + kThreads - 1) / kThreads;
    s.words = (int)((words + tiles - 1) / tiles);
    s.width = s.words * V;
    s.slabs = (int)tiles;
    s.threads = kThreads;
    s.row_lanes = kThreads / s.words;
    const int half = (s.row_lanes + 1) / 2;
    s.parts = shares(half, kThreads / s.width);
    s.by_words = divisor((uint32_t)s.words);
    s.by_width = divisor((uint32_t)s.width);
    long long runs = 148 * 3 / ((long long)p.N * tiles);
    const long long most = (p.S + 8ll * s.row_lanes - 1) / (8ll * s.row_lanes);
    if (runs > most) runs = most;
    if (runs < p.S >> 30) runs = (p.S >> 30) + 1; // a run's rows are counted in 32 bits
    if (runs < 1) runs = 1;
    s.rows = (int)((p.S + runs - 1) / runs);
    s.blocks = (int)((p.S + s.rows - 1) / s.rows);
    s.shared = sizeof(float2) * (size_t)half * s.width;
    s.groups = p.fold > 1 || s.width / p.D + 2 > p.G ? p.G : s.width / p.D + 2; // that a slab touches, at most
    return s;
}

Norm describe(const sideaware_group_norm_t& sh, const void* weight, const void* bias) {
    Norm p{};
    p.N = sh.N;
    p.S = sh.S;
    p.C = sh.C;
    p.G = sh.G;
    p.D = sh.C / sh.G;
    p.fold = 1;
    p.silu = sh.silu;
    p.param_dtype = sh.param_dtype;
    p.eps = sh.eps;
    p.weight = weight;
    p.bias = bias;
    return p;
}


constexpr int kMostShared = 226 * 1024; // dynamic shared memory of a block

// How a resident launch would run, in microseconds.  The form is a sum of what an SM has to do in each round of blocks; the
// constants were fitted to 3,000 measured launches (13 shapes, forward and backward, all slab widths, cluster sizes and block
// sizes) with a mean error of 13 %: the choice that follows from it took 5 % longer than each shape's best one.
double resident_time(const Norm& p, const Slab& s, int V, int esize, int tensors) {
    // blocks that run at once when each has an SM (or a share of one) to itself: a cluster stays inside a GPC, so sizes that
    // do not divide a GPC's SMs leave some idle (cudaOccupancyMaxActiveClusters)
    static const int kAlone[kMaxCluster + 1] = {0, 148, 148, 135, 132, 130, 132, 105, 120};
    const int registers = tensors == 1 ? kResidentRegisters : kResidentBackwardRegisters;
    int on_sm = (int)(228 * 1024 / (s.shared + 1024));
    if (on_sm > 65536 / (registers * s.threads)) on_sm = 65536 / (registers * s.threads);
    const double grid = (double)p.N * s.slabs * s.blocks;
    const double at_once = on_sm == 1 ? kAlone[s.blocks] : 148.0 * on_sm * (s.blocks <= 2 ? 1.0 : 0.92);
    const double rounds = grid <= at_once ? 1.0 : std::ceil(grid / at_once);
    const double of_sm = std::min((double)on_sm, std::ceil(grid / 148.0)); // blocks of the busiest SM
    // memory: segments that do not start and end on sectors, or are shorter than two of them, cost more than their bytes
    const double segment = (double)s.width * esize, bytes = (double)s.rows * s.words * V * esize;
    double ragged = (s.width * esize) % 32 ? (segment + 16.0) / segment : 1.0;
    if (segment < 64.0) ragged *= 2.0 - segment / 64.0;
    const double memory = of_sm * bytes * (tensors + 1) * ragged / 59e3;
    // arithmetic: cycles of a warp for a row of its words (V = 8), on four schedulers, fewer than 20 warps do not fill them
    const double warps = of_sm * s.threads / 32, row = (tensors == 1 ? 54.0 : 237.0) * std::max(V / 8.0, 0.3) * (esize == 4 ? 1.3 : 1.0);
    const double lanes = std::ceil((double)s.rows / s.row_lanes);
    const double arithmetic = of_sm * lanes * (s.threads / 32) * row / 4 / 1900 / std::min(1.0, warps / 20.0);
    const double fixed = 3.8 + (s.blocks > 1 ? 1.4 : 0.0) + 0.26 * s.blocks + (tensors == 1 ? 0.0 : 0.7); // latencies and barriers
    return fixed + rounds * (memory + arithmetic) + (rounds - 1.0) * 6.0;
}

// The same for tiles of short samples: instructions, of the SM with the most tiles or of a block alone (fitted to 20 shapes, with
// 1,000 to 34 million elements; the choice took at most 9 % longer than the better way).
double packed_time(const Norm& p, const Slab& s, int V, int tensors) {
    const double each = std::ceil((double)s.tiles / s.blocks), on_sm = std::ceil((double)s.slabs * s.blocks / 148);
    const double thousands = s.rows * s.width * 1e-3 * (V == 8 ? 1.0 : V == 4 ? 1.7 : 2.4) * (p.D % V ? 1.3 : 1.0);
    const double most = std::min(on_sm, (double)packed_on_sm(tensors, p.D % V == 0)), rounds = std::ceil(on_sm / most);
    if (tensors == 1) return 3.0 + rounds * each * (0.4 + thousands * std::max(0.3, 0.18 * most));
    return 5.6 + rounds * each * (0.7 + thousands * std::max(0.5, 0.38 * most));
}

// The same for the way of long samples: three or four launches (fitted to 0.2-134 MB of x; within 20 %).
double streamed_time(const Norm& p, int V, int esize, int tensors) {
    const double mb = (double)p.N * (double)p.S * (double)p.C * esize * 1e-6 * (V * esize == 16 ? 1.0 : V * esize == 4 ? 4.0 : 8.0);
    // many samples are many blocks, of the kernel that joins as well
    const double blocks = (double)p.N * std::ceil((double)p.C / V / kThreads);
    const double joins = (double)p.N * (tensors == 1 ? p.G / 8.0 : std::ceil((double)p.C / 32) / 2);
    return (tensors == 1 ? 17.0 + 0.45 * mb : 31.0 + 0.75 * mb) + blocks / (148 * 3) * 8.0 + joins / 148 * 3.0;
}

// Short samples: tiles of whole samples with up to `cap` bytes of x, fewer where that leaves SMs without any.
bool pack(const Norm& p, int V, int esize, int tensors, int unit, int cap, Slab* best) {
    const long long column = p.S * p.D * esize; // bytes of a group of a sample
    long long groups = std::min(std::min(cap / column, 256ll * V / p.D) / unit * unit, (long long)p.G);
    if (groups < 1) return false;
    Slab s{};
    s.p = p;
    s.slabs = (int)((p.G + groups - 1) / groups);
    groups = ((p.G + s.slabs - 1) / s.slabs + unit - 1) / unit * unit;
    s.slabs = (int)((p.G + groups - 1) / groups);
    s.groups = (int)groups;
    s.width = s.groups * p.D;
    s.words = s.width / V;
    s.pitch = s.words | 1;
    s.threads = kThreads;
    s.row_lanes = kThreads / s.words;
    s.parts = shares((s.row_lanes + 1) / 2, kThreads / s.width);
    const int on_sm = packed_on_sm(tensors, p.D % V == 0);
    const size_t most = (228 / on_sm - 1) * 1024;
    s.samples = (int)std::max(1ll, std::min({cap / (column * groups), (long long)p.N, (long long)p.N * s.slabs / (148 * on_sm)}));
    for (;; --s.samples) {
        const size_t words = (size_t)s.samples * p.S * s.pitch, bytes = (words * V * esize + 15) / 16 * 16, teams = (size_t)s.samples * s.groups;
        if (tensors == 1) s.shared = 2 * bytes + sizeof(float) * 2 * teams;
        else
            s.shared = 4 * bytes + sizeof(float) * ((std::max(words * V, (size_t)(s.row_lanes + 1) / 2 * s.width * 2) + 3) / 4 * 4 +
                                                    (s.width + 3) / 4 * 4 * 2 + 6 * teams);
        if (s.shared <= most || s.samples == 1) break;
    }
    if (s.shared > kMostShared) return false;
    s.rows = s.samples * (int)p.S;
    s.tiles = (p.N + s.samples - 1) / s.samples;
    const int at_once = std::min(s.tiles, std::max(1, 148 * on_sm / s.slabs)), each = (s.tiles + at_once - 1) / at_once;
    s.blocks = (s.tiles + each - 1) / each;
    const int items = (int)p.S * p.D / (p.D % V == 0 ? V : p.D % 4 == 0 && V > 4 ? 4 : p.D % 2 == 0 && V > 2 ? 2 : 1);
    for (s.lanes = 1; s.lanes < 32 && s.lanes * 2 <= items && s.lanes * s.samples * s.groups < kThreads;) s.lanes *= 2;
    s.by_words = divisor((uint32_t)s.words);
    s.by_width = divisor((uint32_t)s.width);
    s.by_D = divisor((uint32_t)p.D);
    s.by_S = divisor((uint32_t)p.S);
    s.by_groups = divisor((uint32_t)s.groups);
    *best = s;
    return true;
}

// Whether the groups of a sample are to be resident or packed, and how: every slab width (multiples of the narrowest one that is
// whole words, up to 512 bytes of a row), cluster size and block size that fits, against each other and against streaming.
bool search_plan(const Norm& p, int V, int esize, int tensors, Slab* best) {
    if (p.S > 1 << 20) return false;
    const int registers = tensors == 1 ? kResidentRegisters : kResidentBackwardRegisters;
    int unit = 1; // groups of the narrowest slab
    while ((unit * (long long)p.D) % V) ++unit;
    double least = streamed_time(p, V, esize, tensors);
    bool found = false;
    for (int cap = 32 * 1024 / tensors; cap >= 4 * 1024 / tensors; cap /= 2) {
        Slab packed{};
        if (!pack(p, V, esize, tensors, unit, cap, &packed)) continue;
        if (const double time = packed_time(p, packed, V, tensors); time < least) {
            least = time;
            *best = packed;
            found = true;
        }
    }
    for (int m = 1; m == 1 || unit * (m - 1) < p.G; ++m) {
        const int groups = unit * m < p.G ? unit * m : p.G;
        const long long width = (long long)groups * p.D;
        if (width % V || width / V > 256 || (m > 1 && width * esize > 512)) break;
        Slab s{};
        s.p = p;
        s.groups = groups;
        s.width = (int)width;
        s.words = (int)(width / V);
        s.slabs = (p.G + groups - 1) / groups;
        s.by_words = divisor((uint32_t)s.words);
        s.by_width = divisor((uint32_t)width);
        s.by_D = divisor((uint32_t)p.D);
        for (s.blocks = 1; s.blocks <= kMaxCluster; ++s.blocks) {
            s.rows = (int)((p.S + s.blocks - 1) / s.blocks);
            if ((s.blocks > 1 && s.rows < 8) || (double)p.N * s.slabs * s.blocks > 1e9) break;
            const size_t data = ((size_t)s.rows * s.words * V * esize + 15) / 16 * 16;
            for (s.threads = 128; s.threads <= kResidentThreads; s.threads += 128) {
                if (s.threads < 2 * s.words || s.threads * registers > 65536) continue;
                s.row_lanes = s.threads / s.words;
                const int half = (s.row_lanes + 1) / 2;
                s.parts = shares(half, s.threads / s.width);
                s.shared = tensors * data + sizeof(float2) * ((size_t)half * s.width + s.groups + (tensors == 1 ? 0 : 2 * s.width)) +
                           sizeof(float) * (size_t)(tensors == 1 ? 3 : 4) * s.width;
                if (s.shared > kMostShared) continue;
                const double time = resident_time(p, s, V, esize, tensors);
                if (time < least) {
                    least = time;
                    *best = s;
                    found = true;
                }
            }
        }
    }
    return found;
}

// The search takes some ten microseconds; the last shapes of a thread are looked up instead.
bool plan_of(const Norm& p, int V, int esize, int tensors, Slab* best) {
    struct Entry {
        long long S, C;
        int N, G, V, esize, tensors;
        bool fits;
        Slab slab;
    };
    constexpr unsigned kEntries = 16;
    thread_local Entry entries[kEntries] = {};
    thread_local unsigned next = 0;
    for (const Entry& e : entries) {
        if (e.S == p.S && e.C == p.C && e.N == p.N && e.G == p.G && e.V == V && e.esize == esize && e.tensors == tensors) {
            *best = e.slab;
            best->p = p;
            return e.fits;
        }
    }
    Entry& e = entries[next++ % kEntries];
    e = Entry{p.S, p.C, p.N, p.G, V, esize, tensors, false, Slab{}};
    e.fits = search_plan(p, V, esize, tensors, &e.slab);
    *best = e.slab;
    return e.fits;
}

// Elements of a word: 16 bytes where addresses and rows allow them.  Rows of another length are folded, 2, 4 or 8 pixels to a
// row, where that makes them whole words and divides the sample; otherwise words have 4 bytes or one element.
int word_elements(Norm& p, int dtype, uint64_t addresses) {
    const int e = sa_element_size(dtype);
    const int a = sa_common_alignment(addresses | (uint64_t)p.C * (uint64_t)e);
    if (a == 16) return 16 / e;
    if (sa_common_alignment(addresses) == 16) {
        for (int k = 2; k <= 8; k *= 2) {
            if ((uint64_t)p.C * k * e % 16 || p.S % k || (uint64_t)p.C * k * e > 16ull * kThreads) continue;
            Slab s;
            const int V = a >= 4 ? 4 / e : 1;
            if (plan_of(p, V, e, 1, &s)) break; // short: better off in shared memory
            p.fold = k;
            p.S /= k;
            p.C *= k;
            return 16 / e;
        }
    }
    return a >= 4 ? 4 / e : 1;
}

// Lets a kernel have more than 48 KiB of dynamic shared memory, once for each kernel and device (a full table only means that
// the attribute is set again).
cudaError_t allow_shared(const void* kernel, size_t bytes) {
    if (bytes <= 48 * 1024) return cudaSuccess;
    struct Allowed {
        const void* kernel;
        int device;
    };
    static std::mutex mu;
    static Allowed allowed[256];
    static int count = 0;
    int device = 0;
    cudaGetDevice(&device);
    std::lock_guard<std::mutex> lock(mu);
    for (int i = 0; i < count; ++i)
        if (allowed[i].kernel == kernel && allowed[i].device == device) return cudaSuccess;
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kMostShared);
    if (e == cudaSuccess && count < 256) allowed[count++] = Allowed{kernel, device};
    return e;
}

// `follows`: the launch may begin while the previous kernel of the same call ends
template <class... P, class... Args>
cudaError_t launch(void (*kernel)(P...), long long grid, int threads, size_t shared, bool follows, cudaStream_t stream, int& launched, Args... args) {
    if (const cudaError_t e = allow_shared((const void*)kernel, shared); e != cudaSuccess) return e;
    cudaLaunchConfig_t cfg{};
    if (grid > 0x7fffffffll) return cudaErrorInvalidValue;
    cfg.gridDim = dim3((unsigned)grid);
    cfg.blockDim = dim3((unsigned)threads);
    cfg.dynamicSmemBytes = shared;
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = follows && sa_pdl_enabled() ? 1 : 0;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, static_cast<P>(args)...);
    if (e == cudaSuccess) ++launched;
    return e;
}

template <class K, class... Args>
cudaError_t launch_clusters(K kernel, const Slab& s, cudaStream_t stream, int& launched, Args... args) {
    if (const cudaError_t e = allow_shared((const void*)kernel, s.shared); e != cudaSuccess) return e;
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
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, args...);
    if (e == cudaSuccess) ++launched;
    return e;
}

template <class T, int V>
size_t ring_bytes(size_t tile) {
    const size_t rings = (size_t)kRingWords * kThreads * sizeof(SaVec<T, V>);
    return rings > tile ? rings : (tile + 15) / 16 * 16;
}

template <class T, int V>
cudaError_t forward(void* out, float* mean, float* rstd, const void* x, Norm p, void* workspace, cudaStream_t stream, int& launched) {
    Slab s;
    const bool planned = p.fold == 1 && plan_of(p, V, sizeof(T), 1, &s);
    if (planned && s.samples)
        return launch(p.D % V == 0 ? sa_norm_packed_kernel<T, V, true> : sa_norm_packed_kernel<T, V, V == 1>, (long long)s.slabs * s.blocks, kThreads, s.shared, false, stream, launched, (T*)out,
                      (const T*)x, mean, rstd, s);
    if (planned)
        return launch_clusters(sa_norm_resident_kernel<T, V>, s, stream, launched, (T*)out, (const T*)x, mean, rstd, s);
    s = cut(p, V);
    const size_t params = sizeof(float) * 3 * (size_t)s.width;
    s.shared = ring_bytes<T, V>(s.shared); // stream, then tile; the parameters behind
    float2* const partial = (float2*)workspace;
    const long long grid = (long long)p.N * s.slabs * s.blocks;
    cudaError_t e = launch(sa_norm_partial_kernel<T, V>, grid, kThreads, s.shared + params, false, stream, launched, (const T*)x, partial, s);
    if (e == cudaSuccess) e = launch(sa_norm_join_kernel, (long long)p.N * p.G, kThreads, 0, true, stream, launched, partial, mean, rstd, s);
    if (e == cudaSuccess)
        e = launch(sa_norm_apply_kernel<T, V>, grid, kThreads, s.shared + params, true, stream, launched, (T*)out, (const T*)x, mean, rstd, s);
    return e;
}

template <class T, int V>
cudaError_t backward(void* dx, void* dweight, void* dbias, const void* dout, const void* x, const float* mean, const float* rstd,
                     const Norm& p, void* workspace, cudaStream_t stream, int& launched) {
    Slab s;
    auto join_params = [&](const float2* sums, int count, int C) {
        return launch(sa_norm_backward_params_kernel, (C + 31) / 32, 1024, 0, true, stream, launched, sums, dweight, dbias, count, C, p.param_dtype);
    };
    const bool planned = p.fold == 1 && plan_of(p, V, sizeof(T), 2, &s);
    if (planned && s.samples) {
        float2* const sums = s.blocks > 1 && (dweight || dbias) ? (float2*)workspace : nullptr; // [blocks of a slab][C]
        const cudaError_t e = launch(p.D % V == 0 ? sa_norm_packed_backward_kernel<T, V, true> : sa_norm_packed_backward_kernel<T, V, V == 1>, (long long)s.slabs * s.blocks, kThreads, s.shared, false, stream,
                                     launched, (T*)dx, (const T*)dout, (const T*)x, mean, rstd, sums, s.blocks > 1 ? nullptr : dweight,
                                     s.blocks > 1 ? nullptr : dbias, s);
        return e != cudaSuccess || !sums ? e : join_params(sums, s.blocks, (int)p.C);
    }
    if (planned) {
        float2* const sums = p.N > 1 && (dweight || dbias) ? (float2*)workspace : nullptr;
        const cudaError_t e = launch_clusters(sa_norm_resident_backward_kernel<T, V>, s, stream, launched, (T*)dx, (const T*)dout, (const T*)x,
                                              mean, rstd, sums, p.N > 1 ? nullptr : dweight, p.N > 1 ? nullptr : dbias, s);
        if (e != cudaSuccess || !sums) return e;
        return join_params(sums, p.N, (int)p.C);
    }
    s = cut(p, V);
    const long long grid = (long long)p.N * s.slabs * s.blocks;
    const size_t params = sizeof(float) * 5 * (size_t)s.width;
    s.shared = ring_bytes<T, V>(s.shared); // streams, then tile; the parameters behind
    float2* const partial = (float2*)workspace; // [N][runs][C]
    float2* const sums = partial + (long long)p.N * s.blocks * p.C;
    const long long channels = p.C / p.fold;
    cudaError_t e = launch(sa_norm_backward_partial_kernel<T, V>, grid, kThreads, s.shared + params, false, stream, launched, (const T*)dout,
                           (const T*)x, mean, rstd, partial, s);
    if (e == cudaSuccess)
        e = launch(sa_norm_backward_sums_kernel, p.N * ((channels + 31) / 32), 1024, 0, true, stream, launched, partial, rstd, sums, s);
    if (e == cudaSuccess)
        e = launch(sa_norm_backward_apply_kernel<T, V>, grid, kThreads, s.shared + params, true, stream, launched, (T*)dx, (const T*)dout, (const T*)x,
                   mean, rstd, sums, s);
    if (e == cudaSuccess && (dweight || dbias)) e = join_params(sums, p.N, (int)channels);
    return e;
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

// Enough for words of any width, so that it follows from the shape alone.  Streamed samples: the partial results of all runs,
// backward also the sums of every (n, c).  Resident ones: those sums, if there is more than one sample.
size_t sa_group_norm_workspace(const sideaware_group_norm_t& sh, bool backward) {
    const int e = sa_element_size(sh.dtype);
    long long most = 0;
    auto streamed = [&](const Norm& p, int V) {
        const Slab s = cut(p, V);
        return backward ? (long long)p.N * s.blocks * p.C + (long long)sh.N * sh.C : (long long)p.N * s.blocks * s.slabs * s.groups;
    };
    for (int V : {16 / e, 4 / e, 1}) {
        if (sh.C % V) continue;
        const Norm p = describe(sh, nullptr, nullptr);
        Slab s;
        long long entries;
        if (!plan_of(p, V, e, backward ? 2 : 1, &s)) entries = streamed(p, V);
        else if (!backward) entries = 0;
        else if (s.samples) entries = s.blocks > 1 ? (long long)s.blocks * sh.C : 0;
        else entries = sh.N > 1 ? (long long)sh.N * sh.C : 0;
        if (entries > most) most = entries;
    }
    Norm p = describe(sh, nullptr, nullptr);
    const int V = word_elements(p, sh.dtype, 0);
    if (p.fold > 1 && streamed(p, V) > most) most = streamed(p, V);
    return (size_t)most * sizeof(float2);
}

cudaError_t sa_launch_group_norm(void* out, float* mean, float* rstd, const void* x, const void* weight, const void* bias,
                                 const sideaware_group_norm_t& sh, void* workspace, cudaStream_t stream, int& launched) {
    Norm p = describe(sh, weight, bias);
    const int V = word_elements(p, sh.dtype, (uint64_t)out | (uint64_t)x);
    return by_type(sh, V, [&](auto type, auto v) {
        return forward<decltype(type), v.value>(out, mean, rstd, x, p, workspace, stream, launched);
    });
}

cudaError_t sa_launch_group_norm_backward(void* dx, void* dweight, void* dbias, const void* dout, const void* x, const float* mean,
                                          const float* rstd, const void* weight, const void* bias,
                                          const sideaware_group_norm_t& sh, void* workspace, cudaStream_t stream, int& launched) {
    Norm p = describe(sh, weight, bias);
    const int V = word_elements(p, sh.dtype, (uint64_t)dx | (uint64_t)dout | (uint64_t)x);
    return by_type(sh, V, [&](auto type, auto v) {
        return backward<decltype(type), v.value>(dx, dweight, dbias, dout, x, mean, rstd, p, workspace, stream, launched);
    });
}
