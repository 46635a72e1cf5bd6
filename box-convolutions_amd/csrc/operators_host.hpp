// Host-side declarations of the operators around a box convolution: group norm (group_norm.hip) and the pointwise
// product (linear*.hip).
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace boxconv {

// element type codes, BOXCONV_F32 / F16 / BF16 of include/boxconv.h
constexpr int kF32 = 0, kF16 = 1, kBF16 = 2;

constexpr int64_t kMostThreads = (int64_t(1) << 32) - 1;     // of a grid along x

// Arguments as in boxconv_group_norm_forward / _backward (include/boxconv.h), checked by the caller.
struct NormCall {
    const void *x, *weight, *bias, *residual;
    void* y;
    float *mean, *rstd;          // both null where the caller does not keep them
    int dtype;
    bool float_params;
    int64_t batch, pixels;
    int channels, groups;
    float eps;
    int activation;
};
struct NormGradCall {
    const void *x, *weight, *bias, *residual, *dy;
    const float *mean, *rstd;
    void *dx, *dweight, *dbias, *dresidual;
    int dtype;
    bool float_params;
    int64_t batch, pixels;
    int channels, groups;
    int activation;
};
size_t norm_workspace_bytes(int64_t batch, int64_t pixels, int channels, int groups, int dtype, bool backward);
hipError_t norm_forward_launch(const NormCall& n, void* workspace, hipStream_t stream);
hipError_t norm_backward_launch(const NormGradCall& n, void* workspace, hipStream_t stream);

// Arguments as in boxconv_linear_forward / _backward (include/boxconv.h), checked by the caller. T: float, _Float16, __bf16.
struct LinearCall {
    const void *x, *weight, *bias, *residual;
    int64_t ld_x, ld_residual;
    void *y, *slope;
    int64_t rows, K, N;
    int activation;
};
struct LinearGradCall {
    const void *x, *weight, *dy, *kept;
    int64_t ld_x;
    void *dx, *dweight, *dbias, *dresidual;
    int64_t rows, K, N;
    int activation;
};
template <class T> size_t linear_forward_workspace(int64_t rows, int64_t K, int64_t N);
template <class T> size_t linear_backward_workspace(int64_t rows, int64_t K, int64_t N);
template <class T> hipError_t linear_forward(const LinearCall& c, void* workspace, hipStream_t stream);
template <class T> hipError_t linear_backward(const LinearGradCall& c, void* workspace, hipStream_t stream);

}  // namespace boxconv
