// extern "C" entry points of the operators of image and video models: argument checks, then the launch.
#include <cuda_runtime.h>

#include <cmath>

#include "../../include/sideaware.h"
#include "sa_context.hpp"
#include "sa_elem.cuh"
#include "sa_ops.hpp"

#define SA_API extern "C" __attribute__((visibility("default")))

namespace {

bool aligned_to(const void* p, uintptr_t a) { return ((uintptr_t)p & (a - 1)) == 0; }

// two arrays of `bytes` bytes that overlap without being the same
bool overlaps(const void* a, const void* b, size_t bytes) {
    if (!a || !b || a == b) return false;
    const uintptr_t x = (uintptr_t)a, y = (uintptr_t)b;
    return (x < y ? y - x : x - y) < bytes;
}

cudaError_t refuse(const char* what, const char* why) {
    sa_set_error("%s: %s", what, why);
    return cudaErrorInvalidValue;
}

// Runs launch(count) on the device and records what went wrong; it adds the kernels it has launched to `count`.  These kernels
// need nothing of the library's per-device set-up (topology, counters), so a first call may be part of a stream capture;
// launches are counted once that set-up exists.
template <class F>
cudaError_t on_device(const char* what, int device, F&& launch) {
    int count = 0;
    if (cudaGetDeviceCount(&count) != cudaSuccess || count <= 0 || (device < 0 && cudaGetDevice(&device) != cudaSuccess)) {
        cudaGetLastError();
        sa_set_error("%s: no CUDA device available (this library has no CPU path)", what);
        return cudaErrorInitializationError;
    }
    if (device >= count) {
        sa_set_error("%s: device %d out of range (%d devices)", what, device, count);
        return cudaErrorInvalidDevice;
    }
    SaScopedDevice guard(device);
    int launched = 0;
    const cudaError_t e = launch(launched);
    if (SaDevice* dev = sa_device_if_ready(device)) dev->launches.fetch_add((unsigned long long)launched);
    if (e != cudaSuccess) sa_set_error("%s launch: %s", what, cudaGetErrorString(e));
    return e;
}

// an operator of one kernel
cudaError_t one(cudaError_t e, int& launched) {
    if (e == cudaSuccess) ++launched;
    return e;
}

// ---------------------------------------------------------------------------
// rotary positions with several axes
// ---------------------------------------------------------------------------
cudaError_t rope_axes(const char* what, void* qkv, const void* positions, const void* spectrum, const sideaware_rope_axes_t* sh,
                      int device, cudaStream_t stream, bool inverse) {
    if (!sh) return refuse(what, "no shape given");
    if (sh->B < 0 || sh->T < 0 || sh->Nq < 0 || sh->Nkv < 0 || sh->HS <= 0) return refuse(what, "negative size");
    if (sh->axes < 1 || sh->axes > SIDEAWARE_ROPE_MAX_AXES) return refuse(what, "1 to 8 axes");
    if (sh->pairs < 1 || sh->pairs > SIDEAWARE_ROPE_MAX_PAIRS || 2 * sh->pairs > sh->HS)
        return refuse(what, "pairs must be at least 1, at most 256 and at most half the head size");
    if (sh->layout < 0 || sh->layout > 1) return refuse(what, "layout is 0 (neighbouring elements) or 1 (halves)");
    if (sh->dtype < 0 || sh->dtype > 2) return refuse(what, "dtype is 0 (fp32), 1 (bf16) or 2 (fp16)");
    if (sh->position_dtype < 0 || sh->position_dtype > 1) return refuse(what, "position_dtype is 0 (int32) or 1 (int64)");
    const long long tokens = (long long)sh->B * sh->T;
    const long long heads = (long long)sh->Nq + 2ll * sh->Nkv;
    if (tokens > 0x7fffffffll || heads > 65536 || sh->HS > 65536) return refuse(what, "more than 2^31 - 1 tokens, 65536 heads or 65536 elements of a head");
    if (tokens == 0 || sh->Nq + sh->Nkv == 0) return cudaSuccess;
    if (!qkv || !positions || !spectrum) return refuse(what, "null pointer");
    const int e = sa_element_size(sh->dtype);
    if (!aligned_to(qkv, e) || !aligned_to(positions, sh->position_dtype ? 8 : 4) || !aligned_to(spectrum, 8))
        return refuse(what, "a pointer is not aligned to its elements");
    // tokens must not share memory: a row is `row` elements, rows of one index lie inside a step of the other
    const long long row = heads * sh->HS;
    if (row > (1ll << 30)) return refuse(what, "more than 2^30 elements of a row");
    const long long sb = sh->stride_b, st = sh->stride_t;
    if ((sh->T > 1 && (st < row || st > (1ll << 40))) || (sh->B > 1 && (sb < row || sb > (1ll << 46)))) return refuse(what, "a stride of qkv is shorter than a row (or absurdly long)");
    if (sh->T > 1 && sh->B > 1 && sb < (__int128)(sh->T - 1) * st + row && st < (__int128)(sh->B - 1) * sb + row)
        return refuse(what, "rows of qkv overlap");
    return on_device(what, device, [&](int& launched) { return one(sa_launch_rope_axes(qkv, positions, spectrum, *sh, inverse, stream), launched); });
}

// ---------------------------------------------------------------------------
// group norm
// ---------------------------------------------------------------------------
const char* bad_norm_shape(const sideaware_group_norm_t* sh) {
    if (!sh) return "no shape given";
    if (sh->N < 0 || sh->S < 0 || sh->C <= 0 || sh->G <= 0) return "sizes must not be negative, C and G positive";
    if (sh->C % sh->G) return "the channels must divide evenly into the groups";
    if (sh->C > (1 << 20) || (long long)sh->N * sh->G > (1 << 24) || (double)sh->N * (double)sh->S * sh->C > 1e13) return "more than 2^20 channels, 2^24 groups over all samples or 10^13 elements";
    if (sh->dtype < 0 || sh->dtype > 2 || sh->param_dtype < 0 || sh->param_dtype > 2) return "dtypes are 0 (fp32), 1 (bf16) or 2 (fp16)";
    if (!(sh->eps >= 0.0f) || std::isinf(sh->eps)) return "eps must be finite and not negative";
    if (sh->silu < 0 || sh->silu > 1) return "silu is 0 or 1";
    return nullptr;
}

cudaError_t dropout(const char* what, void* out, const void* x, const void* residual, const void* rng, double p, size_t n, int dtype,
                    int device, cudaStream_t stream) {
    if (!(p >= 0.0 && p <= 1.0)) return refuse(what, "p must lie in [0, 1]");
    if (dtype < 0 || dtype > 2) return refuse(what, "dtype is 0 (fp32), 1 (bf16) or 2 (fp16)");
    if (n > (1ull << 43)) return refuse(what, "more than 2^43 elements");
    if (n == 0) return cudaSuccess;
    if (!out || !x || !rng) return refuse(what, "null pointer");
    const int e = sa_element_size(dtype);
    if (!aligned_to(out, e) || !aligned_to(x, e) || !aligned_to(residual, e) || !aligned_to(rng, 16))
        return refuse(what, "a pointer is not aligned to its elements (rng: 16 bytes)");
    if (overlaps(out, x, n * e) || overlaps(out, residual, n * e)) return refuse(what, "out overlaps an input without being that input");
    return on_device(what, device, [&](int& launched) { return one(sa_launch_dropout(out, x, residual, rng, p, n, dtype, stream), launched); });
}

} // namespace

SA_API sideaware_status_t sideaware_rope_axes_spectrum(void* spectrum, const int* pairs_per_axis, int axes, double theta,
                                                       int arrangement, int device, sideaware_stream_t stream) {
    const char* what = "sideaware_rope_axes_spectrum";
    if (!spectrum || !pairs_per_axis) return refuse(what, "null pointer");
    if (!aligned_to(spectrum, 8)) return refuse(what, "the spectrum must be 8-byte aligned");
    if (axes < 1 || axes > SIDEAWARE_ROPE_MAX_AXES) return refuse(what, "1 to 8 axes");
    if (!(theta > 0.0) || std::isinf(theta)) return refuse(what, "theta must be positive and finite");
    if (arrangement < 0 || arrangement > 2) return refuse(what, "arrangement is 0 (own), 1 (shared) or 2 (interleaved)");
    long long total = 0;
    for (int a = 0; a < axes; ++a) {
        if (pairs_per_axis[a] < 0) return refuse(what, "negative number of pairs");
        total += pairs_per_axis[a];
    }
    if (total < 1 || total > SIDEAWARE_ROPE_MAX_PAIRS) return refuse(what, "1 to 256 pairs over all axes");
    uint64_t turns[SIDEAWARE_ROPE_MAX_PAIRS];
    int used[SIDEAWARE_ROPE_MAX_AXES] = {0};
    int axis = 0;
    for (int i = 0; i < (int)total; ++i) {
        while (used[axis] == pairs_per_axis[axis]) axis = (axis + 1) % axes; // the next axis that has pairs left
        const long double power = arrangement == 0 ? (long double)used[axis] / pairs_per_axis[axis] : (long double)i / total;
        const long double turn = powl((long double)theta, -power) / (2.0L * 3.14159265358979323846264338327950288L);
        const long double part = turn - floorl(turn);
        turns[i] = ((uint64_t)llroundl(ldexpl(part, 61)) << 3) | (uint64_t)axis;
        ++used[axis];
        if (arrangement == 2) axis = (axis + 1) % axes;
    }
    return on_device(what, device, [&](int& launched) { return one(sa_launch_rope_axes_spectrum(spectrum, turns, (int)total, (cudaStream_t)stream), launched); });
}

SA_API sideaware_status_t sideaware_rope_axes_forward(void* qkv, const void* positions, const void* spectrum,
                                                      const sideaware_rope_axes_t* shape, int device, sideaware_stream_t stream) {
    return rope_axes("sideaware_rope_axes_forward", qkv, positions, spectrum, shape, device, (cudaStream_t)stream, false);
}

SA_API sideaware_status_t sideaware_rope_axes_backward(void* dqkv, const void* positions, const void* spectrum,
                                                       const sideaware_rope_axes_t* shape, int device, sideaware_stream_t stream) {
    return rope_axes("sideaware_rope_axes_backward", dqkv, positions, spectrum, shape, device, (cudaStream_t)stream, true);
}

SA_API size_t sideaware_group_norm_workspace(const sideaware_group_norm_t* shape, int backward) {
    if (const char* why = bad_norm_shape(shape)) {
        sa_set_error("sideaware_group_norm_workspace: %s", why);
        return 0;
    }
    return shape->N == 0 || shape->S == 0 ? 0 : sa_group_norm_workspace(*shape, backward != 0);
}

SA_API sideaware_status_t sideaware_group_norm_forward(void* out, float* mean, float* rstd, const void* x, const void* weight,
                                                       const void* bias, const sideaware_group_norm_t* shape, void* workspace,
                                                       size_t workspace_bytes, int device, sideaware_stream_t stream) {
    const char* what = "sideaware_group_norm_forward";
    if (const char* why = bad_norm_shape(shape)) return refuse(what, why);
    if (shape->N == 0) return cudaSuccess;
    if (shape->S == 0) return refuse(what, "a sample without elements has no mean");
    if (!out || !mean || !rstd || !x) return refuse(what, "null pointer");
    const int e = sa_element_size(shape->dtype), pe = sa_element_size(shape->param_dtype);
    if (!aligned_to(out, e) || !aligned_to(x, e) || !aligned_to(mean, 4) || !aligned_to(rstd, 4) || !aligned_to(weight, pe) || !aligned_to(bias, pe))
        return refuse(what, "a pointer is not aligned to its elements");
    if (overlaps(out, x, (size_t)shape->N * shape->S * shape->C * e)) return refuse(what, "out overlaps x without being x");
    const size_t need = sa_group_norm_workspace(*shape, false);
    if (need && (!workspace || workspace_bytes < need || !aligned_to(workspace, 16)))
        return refuse(what, "the workspace is missing, smaller than sideaware_group_norm_workspace says or not 16-byte aligned");
    return on_device(what, device, [&](int& launched) {
        return sa_launch_group_norm(out, mean, rstd, x, weight, bias, *shape, workspace, (cudaStream_t)stream, launched);
    });
}

SA_API sideaware_status_t sideaware_group_norm_backward(void* dx, void* dweight, void* dbias, const void* dout, const void* x,
                                                        const float* mean, const float* rstd, const void* weight, const void* bias,
                                                        const sideaware_group_norm_t* shape, void* workspace, size_t workspace_bytes,
                                                        int device, sideaware_stream_t stream) {
    const char* what = "sideaware_group_norm_backward";
    if (const char* why = bad_norm_shape(shape)) return refuse(what, why);
    if (shape->N == 0 || shape->S == 0) return refuse(what, "no elements: the gradients of weight and bias would be left as they are");
    if (!dx || !dout || !x || !mean || !rstd) return refuse(what, "null pointer");
    const int e = sa_element_size(shape->dtype), pe = sa_element_size(shape->param_dtype);
    if (!aligned_to(dx, e) || !aligned_to(dout, e) || !aligned_to(x, e) || !aligned_to(mean, 4) || !aligned_to(rstd, 4) ||
        !aligned_to(weight, pe) || !aligned_to(bias, pe) || !aligned_to(dweight, pe) || !aligned_to(dbias, pe))
        return refuse(what, "a pointer is not aligned to its elements");
    const size_t bytes = (size_t)shape->N * shape->S * shape->C * e;
    if (overlaps(dx, x, bytes) || overlaps(dx, dout, bytes)) return refuse(what, "dx overlaps an input without being that input");
    const size_t need = sa_group_norm_workspace(*shape, true);
    if (need && (!workspace || workspace_bytes < need || !aligned_to(workspace, 16)))
        return refuse(what, "the workspace is missing, smaller than sideaware_group_norm_workspace says or not 16-byte aligned");
    return on_device(what, device, [&](int& launched) {
        return sa_launch_group_norm_backward(dx, dweight, dbias, dout, x, mean, rstd, weight, bias, *shape, workspace, (cudaStream_t)stream, launched);
    });
}

SA_API sideaware_status_t sideaware_dropout_forward(void* out, const void* x, const void* residual, const void* rng, double p,
                                                    size_t n, int dtype, int device, sideaware_stream_t stream) {
    return dropout("sideaware_dropout_forward", out, x, residual, rng, p, n, dtype, device, (cudaStream_t)stream);
}

SA_API sideaware_status_t sideaware_dropout_backward(void* dx, const void* dout, const void* rng, double p, size_t n, int dtype,
                                                     int device, sideaware_stream_t stream) {
    return dropout("sideaware_dropout_backward", dx, dout, nullptr, rng, p, n, dtype, device, (cudaStream_t)stream);
}
