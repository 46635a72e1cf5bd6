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

// Arguments as in boxconv_quantize_blocks and boxconv_linear_float8_forward (include/boxconv.h), checked by the caller.
constexpr int kE4M3 = 8;           // BOXCONV_E4M3
struct QuantizeCall {
    const void* x;
    int64_t ld;
    int dtype;
    int64_t rows, columns;
    uint8_t *codes, *exponents;
};
hipError_t quantize_launch(const QuantizeCall& q, hipStream_t stream);
struct LinearFloat8Call {
    const void* x;
    int64_t ld_x;
    int input_dtype;
    const uint8_t *x_exponents, *weight, *weight_exponents;
    const void *bias, *residual;
    int64_t ld_residual;
    void* y;
    int64_t rows, K, N;
    int activation;
};
template <class T> size_t linear_float8_workspace(int64_t rows, int64_t K, int64_t N, bool values);
template <class T> hipError_t linear_float8_forward(const LinearFloat8Call& c, void* workspace, hipStream_t stream);

// Arguments as in boxconv_residual_norm_forward / _backward (include/boxconv.h), checked by the caller.
constexpr int kGateNone = 0, kGateChannel = 1, kGateItem = 2, kGateFull = 3;
struct ResidualNormCall {
    const void *x, *residual, *gate, *after_weight, *after_bias, *before_weight, *before_bias;
    int gate_kind;
    bool after, before, centre, float_params, float_gate;
    int64_t batch, pixels;
    int channels;
    float scale, eps;
};
struct ResidualNormOut {
    void *stream, *normed;
    uint8_t* exponents;          // not null: `normed` is codes
    float* statistics;           // [row][mean and rstd of x, of the stream], or null
};
struct ResidualNormGrads {
    const float* statistics;     // null: formed again
    const void *dstream, *dnormed;
    void *dx, *dresidual, *dgate, *dafter_weight, *dafter_bias, *dbefore_weight, *dbefore_bias;
};
template <class T> hipError_t residual_norm_forward(const ResidualNormCall& c, const ResidualNormOut& out, hipStream_t stream);
template <class T> size_t residual_norm_workspace(const ResidualNormCall& c);
// Rows of more channels keep their statistics for the backward: a workgroup works on them, and forming them again takes it two of four
// barriers a row (8192 rows of 4096 bfloat16 128 us, kept 96). Within a wave they cost next to nothing (131072 rows of 128 48 and 45 us), and
// short rows would have as much to read instead.
constexpr int kMostChannelsWithoutStatistics = 512;
template <class T> hipError_t residual_norm_backward(const ResidualNormCall& c, const ResidualNormGrads& g, void* workspace, hipStream_t stream);

}  // namespace boxconv
