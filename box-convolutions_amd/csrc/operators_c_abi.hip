// extern "C" entry points of group norm, the norms between residual blocks and the pointwise product (declared in include/boxconv.h): argument checks on the
// host, then the launches. No torch types, no allocation, no synchronisation.
#include "../../include/boxconv.h"
#include "boxconv_host.hpp"
#include "operators_host.hpp"

namespace {

using namespace boxconv;

constexpr int64_t kMaxExtent = (int64_t(1) << 31) - 1;

bool known_dtype(int dtype) { return dtype == BOXCONV_F32 || dtype == BOXCONV_F16 || dtype == BOXCONV_BF16; }

int check_norm(int dtype, int param_dtype, int64_t batch, int64_t pixels, int channels, int groups, int activation, bool backward) {
    if (!known_dtype(dtype)) return fail(BOXCONV_E_INVALID_ARGUMENT, "group norm: dtype must be BOXCONV_F32, BOXCONV_F16 or BOXCONV_BF16, got %d", dtype);
    if (param_dtype != BOXCONV_F32 && param_dtype != dtype)
        return fail(BOXCONV_E_INVALID_ARGUMENT, "group norm: param_dtype must be BOXCONV_F32 or that of the input, got %d", param_dtype);
    if (batch < 0 || pixels < 0 || channels < 1 || groups < 1 || channels % groups != 0)
        return fail(BOXCONV_E_INVALID_ARGUMENT, "group norm: invalid sizes: batch=%lld pixels=%lld channels=%d groups=%d", static_cast<long long>(batch),
                    static_cast<long long>(pixels), channels, groups);
    if (activation < BOXCONV_ACT_NONE || activation > BOXCONV_ACT_GELU)
        return fail(BOXCONV_E_INVALID_ARGUMENT, "group norm: unknown activation %d", activation);
    // batch items are split over launches where a grid would have 2^32 threads or more; one item has at most a workgroup of 256 per group, in the
    // backward per channel
    if ((backward ? channels : groups) > kMostThreads / 256 || batch > kMaxExtent / channels || pixels > (int64_t(1) << 46) / channels)
        return fail(BOXCONV_E_TOO_LARGE, "group norm: batch=%lld items of pixels=%lld x channels=%d are too many", static_cast<long long>(batch),
                    static_cast<long long>(pixels), channels);
    return 0;
}

int check_linear(int dtype, int64_t rows, int64_t in_features, int64_t out_features, int64_t ld_input, int activation) {
    if (!known_dtype(dtype)) return fail(BOXCONV_E_INVALID_ARGUMENT, "linear: dtype must be BOXCONV_F32, BOXCONV_F16 or BOXCONV_BF16, got %d", dtype);
    if (rows < 0 || in_features < 0 || out_features < 0 || ld_input < 0)
        return fail(BOXCONV_E_INVALID_ARGUMENT, "linear: invalid sizes: rows=%lld in_features=%lld out_features=%lld ld_input=%lld", static_cast<long long>(rows),
                    static_cast<long long>(in_features), static_cast<long long>(out_features), static_cast<long long>(ld_input));
    if (activation < BOXCONV_ACT_NONE || activation > BOXCONV_ACT_GELU) return fail(BOXCONV_E_INVALID_ARGUMENT, "linear: unknown activation %d", activation);
    // tiles of 64 x 64 of every product are counted in 31 bits, and no tensor's bytes overflow 63
    const int64_t tm = (rows + 63) / 64, tk = (in_features + 63) / 64, tn = (out_features + 63) / 64;
    if (rows > (int64_t(1) << 40) || in_features > kMaxExtent || out_features > kMaxExtent || tm > kMaxExtent / std::max<int64_t>({tk, tn, 1}) ||
        tk * tn > kMaxExtent || out_features > int64_t(256) * 65535)
        return fail(BOXCONV_E_TOO_LARGE, "linear: rows=%lld in_features=%lld out_features=%lld are too large", static_cast<long long>(rows),
                    static_cast<long long>(in_features), static_cast<long long>(out_features));
    return 0;
}

// Sizes as the 16-bit product's; in_features of 0 (no blocks) are refused.
int check_linear_float8(int dtype, int input_dtype, int64_t rows, int64_t in_features, int64_t out_features, int64_t ld_input, int activation) {
    if (const int rc = check_linear(dtype, rows, in_features, out_features, ld_input, activation)) return rc;
    if (input_dtype != BOXCONV_E4M3 && input_dtype != dtype)
        return fail(BOXCONV_E_INVALID_ARGUMENT, "linear float8: input_dtype must be BOXCONV_E4M3 or that of the output, got %d", input_dtype);
    if (in_features == 0) return fail(BOXCONV_E_INVALID_ARGUMENT, "linear float8: invalid sizes: in_features=0");
    // a workgroup's tile is addressed in 31 bits: 256 rows of codes
    if (in_features > (int64_t(1) << 22)) return fail(BOXCONV_E_TOO_LARGE, "linear float8: in_features=%lld are too large", static_cast<long long>(in_features));
    return 0;
}

int check_residual_norm(int dtype, int param_dtype, int gate_dtype, int gate_kind, bool gate, int norms, int64_t batch, int64_t pixels, int channels) {
    if (!known_dtype(dtype)) return fail(BOXCONV_E_INVALID_ARGUMENT, "residual norm: dtype must be BOXCONV_F32, BOXCONV_F16 or BOXCONV_BF16, got %d", dtype);
    if (param_dtype != BOXCONV_F32 && param_dtype != dtype)
        return fail(BOXCONV_E_INVALID_ARGUMENT, "residual norm: param_dtype must be BOXCONV_F32 or that of the input, got %d", param_dtype);
    if (gate_kind < BOXCONV_GATE_NONE || gate_kind > BOXCONV_GATE_FULL) return fail(BOXCONV_E_INVALID_ARGUMENT, "residual norm: unknown gate_kind %d", gate_kind);
    if (gate != (gate_kind != BOXCONV_GATE_NONE)) return fail(BOXCONV_E_INVALID_ARGUMENT, "residual norm: gate and gate_kind do not agree");
    if (gate && gate_dtype != dtype && (gate_dtype != BOXCONV_F32 || gate_kind == BOXCONV_GATE_FULL))
        return fail(BOXCONV_E_INVALID_ARGUMENT, "residual norm: gate_dtype must be that of the input, or BOXCONV_F32 where the gate is no whole tensor, got %d", gate_dtype);
    if (norms < 0 || norms > (BOXCONV_NORM_AFTER | BOXCONV_NORM_BEFORE | BOXCONV_NORM_CENTRE))
        return fail(BOXCONV_E_INVALID_ARGUMENT, "residual norm: unknown norms %d", norms);
    if (batch < 0 || pixels < 0 || channels < 1)
        return fail(BOXCONV_E_INVALID_ARGUMENT, "residual norm: invalid sizes: batch=%lld pixels=%lld channels=%d", static_cast<long long>(batch),
                    static_cast<long long>(pixels), channels);
    // (no tensor's bytes overflow 63 bits; the joining launch has a workgroup of 1024 threads for every 32 channels)
    if (batch > kMaxExtent || pixels > (int64_t(1) << 46) / channels / std::max<int64_t>(batch, 1) || channels / 32 >= kMostThreads / 1024)
        return fail(BOXCONV_E_TOO_LARGE, "residual norm: batch=%lld items of pixels=%lld x channels=%d are too many", static_cast<long long>(batch),
                    static_cast<long long>(pixels), channels);
    return 0;
}

int check_statistics(const void* statistics, int64_t batch, int64_t pixels, int channels) {
    if (statistics == nullptr) return 0;
    if (boxconv_residual_norm_statistics_bytes(batch, pixels, channels) == 0)
        return fail(BOXCONV_E_INVALID_ARGUMENT, "residual norm: statistics of rows that do without");
    if (reinterpret_cast<uintptr_t>(statistics) % 16 != 0) return fail(BOXCONV_E_INVALID_ARGUMENT, "residual norm: statistics must be 16-byte aligned");
    return 0;
}

int check_workspace(const char* what, const void* workspace, size_t have, size_t need) {
    if (need == 0) return 0;
    if (workspace == nullptr || have < need)
        return fail(BOXCONV_E_WORKSPACE, "%s: workspace of %zu bytes is missing or too small (%zu bytes needed)", what, have, need);
    return 0;
}

__global__ void __launch_bounds__(256) zero_kernel(uint16_t* __restrict__ p, int64_t n) {
    for (int64_t i = blockIdx.x * 256ll + threadIdx.x; i < n; i += gridDim.x * 256ll) p[i] = 0;
}

// Sums of nothing: zeros in a gradient of `elements` of type `dtype`, unless it is not wanted.
int write_zeros(void* p, int64_t elements, int dtype, const char* what, hipStream_t stream) {
    if (p == nullptr || elements == 0) return 0;
    const int64_t n = elements * (dtype == BOXCONV_F32 ? 2 : 1), groups = std::min<int64_t>((n + 255) / 256, 4096);
    BOXCONV_LAUNCH("fill_zero", zero_kernel, dim3(static_cast<unsigned>(groups)), dim3(256), 0, stream, static_cast<uint16_t*>(p), n);
    return hip_result(hipGetLastError(), what);
}

template <class F>
auto with_type(int dtype, F f) {
    if (dtype == BOXCONV_F32) return f(float());
    if (dtype == BOXCONV_F16) return f(_Float16());
    return f(__bf16());
}

}  // namespace

extern "C" {

size_t boxconv_group_norm_workspace_bytes(int64_t batch, int64_t pixels, int channels, int groups, int dtype, int backward) {
    if (check_norm(dtype, BOXCONV_F32, batch, pixels, channels, groups, 0, backward != 0) != 0 || batch == 0 || pixels == 0) return 0;
    return norm_workspace_bytes(batch, pixels, channels, groups, dtype, backward != 0);
}

int boxconv_group_norm_forward(const void* input, const void* weight, const void* bias, int param_dtype, const void* residual, void* output,
                               float* mean, float* rstd, int dtype, int64_t batch, int64_t pixels, int channels, int groups, float eps,
                               int activation, void* workspace, size_t workspace_bytes, void* stream) {
    if (const int rc = check_norm(dtype, param_dtype, batch, pixels, channels, groups, activation, false)) return rc;
    if ((mean == nullptr) != (rstd == nullptr)) return fail(BOXCONV_E_INVALID_ARGUMENT, "group norm: mean and rstd go together");
    if (batch == 0 || pixels == 0) return 0;
    if (input == nullptr || output == nullptr) return fail(BOXCONV_E_INVALID_ARGUMENT, "group norm: null input or output pointer");
    if (const int rc = check_workspace("group norm", workspace, workspace_bytes, norm_workspace_bytes(batch, pixels, channels, groups, dtype, false))) return rc;
    const NormCall call = {input, weight, bias, residual, output, mean, rstd, dtype, param_dtype == BOXCONV_F32, batch, pixels, channels, groups, eps, activation};
    return hip_result(norm_forward_launch(call, workspace, static_cast<hipStream_t>(stream)), "group norm");
}

int boxconv_group_norm_backward(const void* input, const void* weight, const void* bias, int param_dtype, const void* residual,
                                const void* grad_output, const float* mean, const float* rstd, void* grad_input, void* grad_weight, void* grad_bias,
                                void* grad_residual, int dtype, int64_t batch, int64_t pixels, int channels, int groups, int activation, void* workspace,
                                size_t workspace_bytes, void* stream) {
    if (const int rc = check_norm(dtype, param_dtype, batch, pixels, channels, groups, activation, true)) return rc;
    if (batch == 0 || pixels == 0) {
        if (const int rc = write_zeros(grad_weight, channels, param_dtype, "group norm", static_cast<hipStream_t>(stream))) return rc;
        return write_zeros(grad_bias, channels, param_dtype, "group norm", static_cast<hipStream_t>(stream));
    }
    if (grad_input == nullptr && grad_weight == nullptr && grad_bias == nullptr && grad_residual == nullptr) return 0;
    if (input == nullptr || grad_output == nullptr || mean == nullptr || rstd == nullptr)
        return fail(BOXCONV_E_INVALID_ARGUMENT, "group norm: null input, grad_output, mean or rstd pointer");
    if (const int rc = check_workspace("group norm", workspace, workspace_bytes, norm_workspace_bytes(batch, pixels, channels, groups, dtype, true))) return rc;
    const NormGradCall call = {input, weight, bias, residual, grad_output, mean, rstd, grad_input, grad_weight, grad_bias, grad_residual, dtype,
                               param_dtype == BOXCONV_F32, batch, pixels, channels, groups, activation};
    return hip_result(norm_backward_launch(call, workspace, static_cast<hipStream_t>(stream)), "group norm");
}

int boxconv_residual_norm_forward(const void* input, const void* residual, const void* gate, int gate_kind, int gate_dtype, float scale, int norms,
                                  const void* after_weight, const void* after_bias, const void* before_weight, const void* before_bias, int param_dtype,
                                  float eps, void* stream_output, void* normed, void* normed_exponents, void* statistics, int dtype, int64_t batch,
                                  int64_t pixels, int channels, void* stream) {
    if (const int rc = check_residual_norm(dtype, param_dtype, gate_dtype, gate_kind, gate != nullptr, norms, batch, pixels, channels)) return rc;
    if (normed != nullptr && !(norms & BOXCONV_NORM_BEFORE)) return fail(BOXCONV_E_INVALID_ARGUMENT, "residual norm: normed without BOXCONV_NORM_BEFORE");
    if (normed == nullptr && normed_exponents != nullptr) return fail(BOXCONV_E_INVALID_ARGUMENT, "residual norm: normed_exponents without normed");
    if (normed_exponents != nullptr && (reinterpret_cast<uintptr_t>(normed) % 16 != 0 || reinterpret_cast<uintptr_t>(normed_exponents) % 4 != 0))
        return fail(BOXCONV_E_INVALID_ARGUMENT, "residual norm: codes must be 16-byte aligned, exponents 4-byte aligned");
    if (const int rc = check_statistics(statistics, batch, pixels, channels)) return rc;
    if (batch == 0 || pixels == 0 || (stream_output == nullptr && normed == nullptr && statistics == nullptr)) return 0;
    if (input == nullptr) return fail(BOXCONV_E_INVALID_ARGUMENT, "residual norm: null input pointer");
    const ResidualNormCall call = {input, residual, gate, after_weight, after_bias, before_weight, before_bias, gate_kind, (norms & BOXCONV_NORM_AFTER) != 0,
                                   normed != nullptr || (statistics != nullptr && (norms & BOXCONV_NORM_BEFORE)), (norms & BOXCONV_NORM_CENTRE) != 0, param_dtype == BOXCONV_F32, gate_dtype == BOXCONV_F32, batch,
                                   pixels, channels, scale, eps};
    const ResidualNormOut out = {stream_output, normed, static_cast<uint8_t*>(normed_exponents), static_cast<float*>(statistics)};
    return hip_result(with_type(dtype, [&](auto t) { return residual_norm_forward<decltype(t)>(call, out, static_cast<hipStream_t>(stream)); }), "residual norm");
}

size_t boxconv_residual_norm_statistics_bytes(int64_t batch, int64_t pixels, int channels) {
    if (check_residual_norm(BOXCONV_F32, BOXCONV_F32, BOXCONV_F32, BOXCONV_GATE_NONE, false, 0, batch, pixels, channels) != 0) return 0;
    return channels > kMostChannelsWithoutStatistics ? static_cast<size_t>(batch) * pixels * 4 * sizeof(float) : 0;
}

size_t boxconv_residual_norm_workspace_bytes(int64_t batch, int64_t pixels, int channels, int gate_kind, int dtype) {
    if (check_residual_norm(dtype, BOXCONV_F32, dtype, gate_kind, gate_kind != BOXCONV_GATE_NONE, 0, batch, pixels, channels) != 0 || batch == 0 || pixels == 0) return 0;
    ResidualNormCall call = {};
    call.gate_kind = gate_kind;
    call.batch = batch;
    call.pixels = pixels;
    call.channels = channels;
    return with_type(dtype, [&](auto t) { return residual_norm_workspace<decltype(t)>(call); });
}

int boxconv_residual_norm_backward(const void* input, const void* residual, const void* gate, int gate_kind, int gate_dtype, float scale, int norms,
                                   const void* after_weight, const void* after_bias, const void* before_weight, const void* before_bias, int param_dtype,
                                   float eps, const void* statistics, const void* grad_stream, const void* grad_normed, void* grad_input, void* grad_residual, void* grad_gate,
                                   void* grad_after_weight, void* grad_after_bias, void* grad_before_weight, void* grad_before_bias, int dtype,
                                   int64_t batch, int64_t pixels, int channels, void* workspace, size_t workspace_bytes, void* stream) {
    if (const int rc = check_residual_norm(dtype, param_dtype, gate_dtype, gate_kind, gate != nullptr, norms, batch, pixels, channels)) return rc;
    if (gate == nullptr && grad_gate != nullptr) return fail(BOXCONV_E_INVALID_ARGUMENT, "residual norm: grad_gate without a gate");
    if ((!(norms & BOXCONV_NORM_AFTER) && (grad_after_weight != nullptr || grad_after_bias != nullptr)) ||
        (!(norms & BOXCONV_NORM_BEFORE) && (grad_normed != nullptr || grad_before_weight != nullptr || grad_before_bias != nullptr)))
        return fail(BOXCONV_E_INVALID_ARGUMENT, "residual norm: gradients of a norm that norms does not have");
    if ((grad_after_bias != nullptr && after_bias == nullptr) || (grad_before_bias != nullptr && before_bias == nullptr))
        return fail(BOXCONV_E_INVALID_ARGUMENT, "residual norm: a bias' gradient without the bias");
    if (batch == 0 || pixels == 0) {
        for (void* p : {grad_after_weight, grad_after_bias, grad_before_weight, grad_before_bias})
            if (const int rc = write_zeros(p, channels, param_dtype, "residual norm", static_cast<hipStream_t>(stream))) return rc;
        const int64_t gates = gate_kind == BOXCONV_GATE_CHANNEL ? channels : gate_kind == BOXCONV_GATE_ITEM ? batch * channels : 0;
        return write_zeros(grad_gate, gates, gate_dtype, "residual norm", static_cast<hipStream_t>(stream));
    }
    if (const int rc = check_statistics(statistics, batch, pixels, channels)) return rc;
    const bool sums = grad_after_weight != nullptr || grad_after_bias != nullptr || grad_before_weight != nullptr || grad_before_bias != nullptr ||
                      (grad_gate != nullptr && gate_kind != BOXCONV_GATE_FULL);
    if (!sums && grad_input == nullptr && grad_residual == nullptr && grad_gate == nullptr) return 0;
    if (input == nullptr) return fail(BOXCONV_E_INVALID_ARGUMENT, "residual norm: null input pointer");
    if (sums)
        if (const int rc = check_workspace("residual norm", workspace, workspace_bytes, boxconv_residual_norm_workspace_bytes(batch, pixels, channels, gate_kind, dtype)))
            return rc;
    const ResidualNormCall call = {input, residual, gate, after_weight, after_bias, before_weight, before_bias, gate_kind, (norms & BOXCONV_NORM_AFTER) != 0,
                                   (norms & BOXCONV_NORM_BEFORE) != 0, (norms & BOXCONV_NORM_CENTRE) != 0, param_dtype == BOXCONV_F32,
                                   gate_dtype == BOXCONV_F32, batch, pixels, channels, scale, eps};
    const ResidualNormGrads grads = {static_cast<const float*>(statistics), grad_stream, grad_normed, grad_input, grad_residual, grad_gate, grad_after_weight, grad_after_bias, grad_before_weight, grad_before_bias};
    return hip_result(with_type(dtype, [&](auto t) { return residual_norm_backward<decltype(t)>(call, grads, workspace, static_cast<hipStream_t>(stream)); }),
                      "residual norm");
}

size_t boxconv_linear_workspace_bytes(int64_t rows, int64_t in_features, int64_t out_features, int dtype, int backward) {
    if (check_linear(dtype, rows, in_features, out_features, 0, 0) != 0 || rows == 0 || out_features == 0) return 0;
    return with_type(dtype, [&](auto t) {
        return backward ? linear_backward_workspace<decltype(t)>(rows, in_features, out_features)
                        : linear_forward_workspace<decltype(t)>(rows, in_features, out_features);
    });
}

int boxconv_linear_forward(const void* input, int64_t ld_input, const void* weight, const void* bias, const void* residual, int64_t ld_residual,
                           void* output, void* slope, int dtype, int64_t rows, int64_t in_features, int64_t out_features, int activation,
                           void* workspace, size_t workspace_bytes, void* stream) {
    if (const int rc = check_linear(dtype, rows, in_features, out_features, ld_input, activation)) return rc;
    if (ld_residual < 0) return fail(BOXCONV_E_INVALID_ARGUMENT, "linear: negative ld_residual");
    if (rows == 0 || out_features == 0) return 0;
    if (output == nullptr || (in_features > 0 && (input == nullptr || weight == nullptr)))
        return fail(BOXCONV_E_INVALID_ARGUMENT, "linear: null input, weight or output pointer");
    const size_t need = boxconv_linear_workspace_bytes(rows, in_features, out_features, dtype, 0);
    if (const int rc = check_workspace("linear", workspace, workspace_bytes, need)) return rc;
    const bool keeps = activation == BOXCONV_ACT_SILU || activation == BOXCONV_ACT_GELU;
    const LinearCall call = {input, weight, bias, residual, ld_input, ld_residual, output, keeps ? slope : nullptr, rows, in_features, out_features, activation};
    return hip_result(with_type(dtype, [&](auto t) { return linear_forward<decltype(t)>(call, workspace, static_cast<hipStream_t>(stream)); }), "linear");
}

int boxconv_linear_backward(const void* input, int64_t ld_input, const void* weight, const void* grad_output, const void* kept, void* grad_input,
                            void* grad_weight, void* grad_bias, void* grad_residual, int dtype, int64_t rows, int64_t in_features,
                            int64_t out_features, int activation, void* workspace, size_t workspace_bytes, void* stream) {
    if (const int rc = check_linear(dtype, rows, in_features, out_features, ld_input, activation)) return rc;
    if (rows == 0 || out_features == 0) {
        const auto zeros = [&](void* p, int64_t elements) { return write_zeros(p, elements, dtype, "linear", static_cast<hipStream_t>(stream)); };
        if (const int rc = zeros(grad_input, rows * in_features)) return rc;
        if (const int rc = zeros(grad_weight, out_features * in_features)) return rc;
        return zeros(grad_bias, out_features);
    }
    if (in_features == 0) grad_input = grad_weight = nullptr;
    if (grad_input == nullptr && grad_weight == nullptr && grad_bias == nullptr && grad_residual == nullptr) return 0;
    if (grad_output == nullptr || (activation != BOXCONV_ACT_NONE && kept == nullptr) || (grad_input != nullptr && weight == nullptr) ||
        (grad_weight != nullptr && input == nullptr))
        return fail(BOXCONV_E_INVALID_ARGUMENT, "linear: null input, weight, grad_output or kept pointer");
    // (rows of tiles are split over launches where a grid would have 2^32 threads or more; one row of them has to fit)
    if ((grad_input != nullptr || grad_weight != nullptr) && (in_features + 63) / 64 > kMostThreads / 256)
        return fail(BOXCONV_E_TOO_LARGE, "linear: gradients of in_features=%lld are too large", static_cast<long long>(in_features));
    const size_t need = boxconv_linear_workspace_bytes(rows, in_features, out_features, dtype, 1);
    if (const int rc = check_workspace("linear", workspace, workspace_bytes, need)) return rc;
    const LinearGradCall call = {input, weight, grad_output, kept, ld_input, grad_input, grad_weight, grad_bias, grad_residual, rows, in_features, out_features,
                                 activation};
    return hip_result(with_type(dtype, [&](auto t) { return linear_backward<decltype(t)>(call, workspace, static_cast<hipStream_t>(stream)); }), "linear");
}

int boxconv_quantize_blocks(const void* input, int64_t ld_input, int dtype, int64_t rows, int64_t columns, void* codes, void* exponents, void* stream) {
    if (!known_dtype(dtype)) return fail(BOXCONV_E_INVALID_ARGUMENT, "quantize: dtype must be BOXCONV_F32, BOXCONV_F16 or BOXCONV_BF16, got %d", dtype);
    if (rows < 0 || columns < 0 || ld_input < 0)
        return fail(BOXCONV_E_INVALID_ARGUMENT, "quantize: invalid sizes: rows=%lld columns=%lld ld_input=%lld", static_cast<long long>(rows),
                    static_cast<long long>(columns), static_cast<long long>(ld_input));
    if (rows > (int64_t(1) << 40) || columns > kMaxExtent - 512 || rows > (int64_t(1) << 46) / std::max<int64_t>({columns, ld_input, 1}))
        return fail(BOXCONV_E_TOO_LARGE, "quantize: rows=%lld columns=%lld are too large", static_cast<long long>(rows), static_cast<long long>(columns));
    if (rows == 0 || columns == 0) return 0;
    if (input == nullptr || codes == nullptr || exponents == nullptr) return fail(BOXCONV_E_INVALID_ARGUMENT, "quantize: null input, codes or exponents pointer");
    if (reinterpret_cast<uintptr_t>(codes) % 16 != 0 || reinterpret_cast<uintptr_t>(exponents) % 4 != 0)
        return fail(BOXCONV_E_INVALID_ARGUMENT, "quantize: codes must be 16-byte aligned, exponents 4-byte aligned");
    const QuantizeCall call = {input, ld_input, dtype, rows, columns, static_cast<uint8_t*>(codes), static_cast<uint8_t*>(exponents)};
    return hip_result(quantize_launch(call, static_cast<hipStream_t>(stream)), "quantize");
}

size_t boxconv_linear_float8_workspace_bytes(int64_t rows, int64_t in_features, int64_t out_features, int input_dtype, int dtype) {
    if (check_linear_float8(dtype, input_dtype, rows, in_features, out_features, 0, 0) != 0 || rows == 0 || in_features == 0 || out_features == 0) return 0;
    return with_type(dtype, [&](auto t) { return linear_float8_workspace<decltype(t)>(rows, in_features, out_features, input_dtype != BOXCONV_E4M3); });
}

int boxconv_linear_float8_forward(const void* input, int64_t ld_input, int input_dtype, const void* input_exponents, const void* weight,
                                  const void* weight_exponents, const void* bias, const void* residual, int64_t ld_residual, void* output, int dtype,
                                  int64_t rows, int64_t in_features, int64_t out_features, int activation, void* workspace, size_t workspace_bytes,
                                  void* stream) {
    if (const int rc = check_linear_float8(dtype, input_dtype, rows, in_features, out_features, ld_input, activation)) return rc;
    if (ld_residual < 0) return fail(BOXCONV_E_INVALID_ARGUMENT, "linear float8: negative ld_residual");
    if (rows == 0 || out_features == 0) return 0;
    const bool coded = input_dtype == BOXCONV_E4M3;
    if (output == nullptr || input == nullptr || weight == nullptr || weight_exponents == nullptr || coded != (input_exponents != nullptr))
        return fail(BOXCONV_E_INVALID_ARGUMENT, "linear float8: null input, weight, exponents or output pointer, or exponents of values");
    for (const void* p : {coded ? input : nullptr, weight})
        if (reinterpret_cast<uintptr_t>(p) % 16 != 0) return fail(BOXCONV_E_INVALID_ARGUMENT, "linear float8: codes must be 16-byte aligned");
    for (const void* p : {input_exponents, weight_exponents})
        if (reinterpret_cast<uintptr_t>(p) % 4 != 0) return fail(BOXCONV_E_INVALID_ARGUMENT, "linear float8: exponents must be 4-byte aligned");
    const size_t need = boxconv_linear_float8_workspace_bytes(rows, in_features, out_features, input_dtype, dtype);
    if (const int rc = check_workspace("linear float8", workspace, workspace_bytes, need)) return rc;
    const LinearFloat8Call call = {input, ld_input, input_dtype, static_cast<const uint8_t*>(input_exponents), static_cast<const uint8_t*>(weight),
                                   static_cast<const uint8_t*>(weight_exponents), bias, residual, ld_residual, output, rows, in_features, out_features, activation};
    return hip_result(with_type(dtype, [&](auto t) { return linear_float8_forward<decltype(t)>(call, workspace, static_cast<hipStream_t>(stream)); }), "linear float8");
}

}  // extern "C"
