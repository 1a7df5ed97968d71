// Launch interface of the operators of image and video models (sa_rope_axes.cu, sa_group_norm.cu, sa_dropout.cu).
// Arguments are checked by the C entry points (sa_ops_api.cpp).  One kernel each, but for group norm, which adds the number of
// kernels it has launched to `launched`.
#pragma once
#include <cuda_runtime.h>
#include <stddef.h>
#include <stdint.h>

#include "../../include/sideaware.h"

// largest power of two that divides the address and every byte count or stride or-ed into `bits`, at most 16
inline int sa_common_alignment(uint64_t bits) {
    int a = 16;
    while (a > 1 && (bits & (uint64_t)(a - 1))) a >>= 1;
    return a;
}

cudaError_t sa_launch_rope_axes(void* qkv, const void* positions, const void* spectrum, const sideaware_rope_axes_t& sh,
                                bool inverse, cudaStream_t stream);
// spectrum[i] = turns[i], `pairs` (<= 256) entries of host memory
cudaError_t sa_launch_rope_axes_spectrum(void* spectrum, const uint64_t* turns, int pairs, cudaStream_t stream);

size_t sa_group_norm_workspace(const sideaware_group_norm_t& sh, bool backward);
cudaError_t sa_launch_group_norm(void* out, float* mean, float* rstd, const void* x, const void* weight, const void* bias,
                                 const sideaware_group_norm_t& sh, void* workspace, cudaStream_t stream, int& launched);
cudaError_t sa_launch_group_norm_backward(void* dx, void* dweight, void* dbias, const void* dout, const void* x, const float* mean,
                                          const float* rstd, const void* weight, const void* bias,
                                          const sideaware_group_norm_t& sh, void* workspace, cudaStream_t stream, int& launched);

cudaError_t sa_launch_dropout(void* out, const void* x, const void* residual, const void* rng, double p, size_t n, int dtype,
                              cudaStream_t stream);
