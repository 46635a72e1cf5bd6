// Host side of group_norm_act and linear_act in C++ (part of torch_glue.cpp): checks, allocations and autograd nodes around
// the C ABI's calls, as box_convolution/operators.py has them in Python. A training step of a small layer costs the Python
// version 130 to 200 us of host time.
#pragma once

#include <torch/extension.h>

#include <algorithm>
#include <cstdint>
#include <optional>

namespace {

using Optional = std::optional<at::Tensor>;

struct OperatorAbi {
    size_t (*norm_bytes)(int64_t, int64_t, int, int, int, int) = nullptr;
    int (*norm_forward)(const void*, const void*, const void*, int, const void*, void*, float*, float*, int, int64_t, int64_t, int, int, float, int,
                        void*, size_t, void*) = nullptr;
    int (*norm_backward)(const void*, const void*, const void*, int, const void*, const void*, const float*, const float*, void*, void*, void*, void*,
                         int, int64_t, int64_t, int, int, int, void*, size_t, void*) = nullptr;
    size_t (*linear_bytes)(int64_t, int64_t, int64_t, int, int) = nullptr;
    int (*linear_forward)(const void*, int64_t, const void*, const void*, const void*, int64_t, void*, void*, int, int64_t, int64_t, int64_t, int,
                          void*, size_t, void*) = nullptr;
    int (*linear_backward)(const void*, int64_t, const void*, const void*, const void*, void*, void*, void*, void*, int, int64_t, int64_t, int64_t, int,
                           void*, size_t, void*) = nullptr;
} g_operators;

void init_operators(uint64_t norm_bytes, uint64_t norm_forward, uint64_t norm_backward, uint64_t linear_bytes, uint64_t linear_forward,
                    uint64_t linear_backward) {
    g_operators.norm_bytes = reinterpret_cast<decltype(g_operators.norm_bytes)>(norm_bytes);
    g_operators.norm_forward = reinterpret_cast<decltype(g_operators.norm_forward)>(norm_forward);
    g_operators.norm_backward = reinterpret_cast<decltype(g_operators.norm_backward)>(norm_backward);
    g_operators.linear_bytes = reinterpret_cast<decltype(g_operators.linear_bytes)>(linear_bytes);
    g_operators.linear_forward = reinterpret_cast<decltype(g_operators.linear_forward)>(linear_forward);
    g_operators.linear_backward = reinterpret_cast<decltype(g_operators.linear_backward)>(linear_backward);
}

int type_code(at::ScalarType t) { return t == at::kFloat ? 0 : t == at::kHalf ? 1 : 2; }        // BOXCONV_F32, F16, BF16

const void* address(const Optional& t) { return t ? t->data_ptr() : nullptr; }
void* address(const at::Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }

// Scratch from the allocator (by the stream, and aware of a capture), given back when the call returns.
at::Tensor scratch(size_t nbytes, const at::Tensor& like) {
    return nbytes ? at::empty({static_cast<int64_t>(nbytes)}, like.options().dtype(at::kByte)) : at::Tensor();
}

Optional contiguous(const Optional& t) { return t ? Optional(t->contiguous()) : t; }

bool wants_grad(const at::Tensor& a, std::initializer_list<const Optional*> more) {
    if (!at::GradMode::is_enabled()) return false;
    if (a.requires_grad()) return true;
    for (const Optional* t : more)
        if (*t && (*t)->requires_grad()) return true;
    return false;
}

// Neither the kernels nor the nodes know forward-mode derivatives: a tangent is refused, since dropping it would make it zero.
void refuse_tangents(std::initializer_list<const at::Tensor*> tensors) {
    for (const at::Tensor* t : tensors)
        TORCH_CHECK(!t->defined() || !t->_fw_grad(/*level=*/0).defined(), "box_convolution: group_norm_act and linear_act have no forward-mode derivative");
}
const at::Tensor& or_undefined(const Optional& t) {
    static const at::Tensor none;
    return t ? *t : none;
}

// Which of the arguments of a node, in their order, have a gradient to form (absent ones have no edge).
std::vector<bool> needed(torch::autograd::AutogradContext* ctx, const std::vector<bool>& present) {
    std::vector<bool> out;
    size_t edge = 0;
    for (bool p : present) out.push_back(p && ctx->needs_input_grad(edge++));
    return out;
}

// The gradients are formed by kernels that leave no graph. Where a graph of the backward is asked for, every gradient gets a
// node that refuses to be differentiated, in place of none, which would count as a constant.
struct Once : public torch::autograd::Function<Once> {
    static at::Tensor forward(torch::autograd::AutogradContext*, const at::Tensor& grad, const at::Tensor& /*x*/, const at::Tensor& /*grad_output*/,
                              const at::Tensor& /*needs_grad: that there always is a node*/) {
        return grad.detach();
    }
    static torch::autograd::variable_list backward(torch::autograd::AutogradContext*, torch::autograd::variable_list) {
        TORCH_CHECK(false, "box_convolution: group_norm_act and linear_act can be differentiated once, not twice");
    }
};

torch::autograd::variable_list once(torch::autograd::variable_list grads, const at::Tensor& x, const at::Tensor& grad_output) {
    if (!at::GradMode::is_enabled()) return grads;
    const at::Tensor needs_grad = at::empty({0}, x.options()).requires_grad_();
    for (at::Tensor& g : grads)
        if (g.defined()) g = Once::apply(g, x, grad_output, needs_grad);
    return grads;
}

// What was saved, as the kernels take it: hooks on saved tensors may hand the values back in any memory order.
Optional saved_or_none(const at::Tensor& t) { return t.defined() ? Optional(t.contiguous()) : std::nullopt; }

// ---- group norm ------------------------------------------------------------------------------------------
// A new tensor of x's shape [B, C, ...] in channels-last memory.
at::Tensor empty_channels_last(const at::Tensor& x) {
    std::vector<int64_t> strides(x.dim());
    int64_t step = x.size(1);
    for (int64_t d = x.dim() - 1; d >= 2; --d) {
        strides[d] = step;
        step *= x.size(d);
    }
    strides[0] = step;
    strides[1] = 1;
    return at::empty_strided(x.sizes(), strides, x.options());
}
// x itself where it has that memory, else a copy that does ([B, C, ...] both).
at::Tensor channels_last(const at::Tensor& x) {
    const at::Tensor t = x.dim() == 2 ? x : x.movedim(1, -1);
    if (t.is_contiguous()) return x;
    return x.dim() == 2 ? x.contiguous() : t.contiguous().movedim(-1, 1);
}

struct GroupNormAct : public torch::autograd::Function<GroupNormAct> {
    struct Sizes { int64_t batch, pixels; int channels; };
    static Sizes sizes(const at::Tensor& x) {
        const int64_t b = x.size(0), c = x.size(1);
        return {b, b * c ? x.numel() / (b * c) : 0, static_cast<int>(c)};
    }
    static int param_code(const Optional& weight, const Optional& bias) {
        return weight ? type_code(weight->scalar_type()) : bias ? type_code(bias->scalar_type()) : 0;
    }
    // x and residual in channels-last memory
    static at::Tensor call(const at::Tensor& x, int groups, const Optional& weight, const Optional& bias, const Optional& residual, int act, double eps,
                           int64_t stream, at::Tensor* statistics) {
        const Sizes n = sizes(x);
        at::Tensor y = empty_channels_last(x);
        if (statistics) *statistics = at::empty({2, n.batch, groups}, x.options().dtype(at::kFloat));
        if (x.numel() == 0) return y;
        const int code = type_code(x.scalar_type());
        const size_t nbytes = g_operators.norm_bytes(n.batch, n.pixels, n.channels, groups, code, 0);
        const at::Tensor ws = scratch(nbytes, x);
        float* mean = statistics ? statistics->data_ptr<float>() : nullptr;
        check_rc(g_operators.norm_forward(x.data_ptr(), address(weight), address(bias), param_code(weight, bias), address(residual), y.data_ptr(), mean,
                                          mean ? mean + n.batch * groups : nullptr, code, n.batch, n.pixels, n.channels, groups, static_cast<float>(eps), act,
                                          address(ws), nbytes, reinterpret_cast<void*>(stream)),
                 "group_norm");
        return y;
    }
    static at::Tensor forward(torch::autograd::AutogradContext* ctx, const at::Tensor& input, const Optional& weight, const Optional& bias,
                              const Optional& residual, int64_t groups, int64_t act, double eps, int64_t stream) {
        const at::Tensor x = channels_last(input);
        const Optional w = contiguous(weight), b = contiguous(bias), r = residual ? Optional(channels_last(*residual)) : std::nullopt;
        at::Tensor statistics;
        at::Tensor y = call(x, static_cast<int>(groups), w, b, r, static_cast<int>(act), eps, stream, &statistics);
        // (the residual moves the point at which the activation's derivative is taken, and nothing else)
        ctx->save_for_backward({x, w.value_or(at::Tensor()), b.value_or(at::Tensor()), act && r ? *r : at::Tensor(), statistics});
        ctx->saved_data["present"] = c10::List<bool>({true, weight.has_value(), bias.has_value(), residual.has_value()});
        ctx->saved_data["groups"] = groups;
        ctx->saved_data["act"] = act;
        ctx->saved_data["stream"] = stream;
        return y;
    }
    static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list grad_outputs) {
        refuse_tangents({&grad_outputs[0]});
        const auto saved = ctx->get_saved_variables();
        const at::Tensor x = channels_last(saved[0]), residual = saved[3].defined() ? channels_last(saved[3]) : at::Tensor();
        const at::Tensor statistics = saved[4].contiguous();
        const Optional w = saved_or_none(saved[1]), b = saved_or_none(saved[2]);
        const int groups = static_cast<int>(ctx->saved_data["groups"].toInt()), act = static_cast<int>(ctx->saved_data["act"].toInt());
        const std::vector<bool> need = needed(ctx, ctx->saved_data["present"].toBoolList().vec());
        const at::Tensor g = channels_last(grad_outputs[0]);
        const Sizes n = sizes(x);
        torch::autograd::variable_list grads(8);               // one per argument of forward
        const auto param_options = x.options().dtype(w ? w->scalar_type() : b ? b->scalar_type() : at::kFloat);
        if (need[0]) grads[0] = empty_channels_last(x);
        for (int k = 1; k <= 2; ++k)
            if (need[k]) grads[k] = x.numel() ? at::empty({n.channels}, param_options) : at::zeros({n.channels}, param_options);
        if (need[3]) grads[3] = empty_channels_last(x);
        if (x.numel() == 0) return once(grads, x, g);
        const int code = type_code(x.scalar_type());
        const size_t nbytes = g_operators.norm_bytes(n.batch, n.pixels, n.channels, groups, code, 1);
        const at::Tensor ws = scratch(nbytes, x);
        const float* mean = statistics.data_ptr<float>();
        check_rc(g_operators.norm_backward(x.data_ptr(), address(w), address(b), param_code(w, b), address(residual), g.data_ptr(), mean,
                                           mean + n.batch * groups, address(grads[0]), address(grads[1]), address(grads[2]), address(grads[3]), code,
                                           n.batch, n.pixels, n.channels, groups, act, address(ws), nbytes,
                                           reinterpret_cast<void*>(ctx->saved_data["stream"].toInt())),
                 "group_norm backward");
        return once(grads, x, g);
    }
};

void check_operator_input(const at::Tensor& t, const char* what) {
    TORCH_CHECK(g_operators.norm_bytes != nullptr, "box_convolution: the native glue was not initialised");
    TORCH_CHECK(t.is_cuda(), "box_convolution: ", what, " is on '", t.device(), "'; this build runs on AMD GPUs only (no CPU path)");
    TORCH_CHECK(t.scalar_type() == at::kFloat || t.scalar_type() == at::kHalf || t.scalar_type() == at::kBFloat16, "box_convolution: ", what,
                " must be float32, float16 or bfloat16, got ", t.scalar_type());
}

void check_same(const Optional& t, at::IntArrayRef shape, const at::Tensor& like, const char* name) {
    TORCH_CHECK(!t || (t->sizes() == shape && t->scalar_type() == like.scalar_type() && t->device() == like.device()), "box_convolution: ", name,
                " must have the shape ", shape, ", type ", like.scalar_type(), " and device ", like.device(), ", got ", t ? t->sizes() : shape, ", ",
                t ? t->scalar_type() : like.scalar_type(), ", ", t ? t->device() : like.device());
}

at::Tensor group_norm_act(const at::Tensor& input, int64_t groups, const Optional& weight, const Optional& bias, const Optional& residual, int64_t act,
                          double eps, int64_t stream) {
    check_operator_input(input, "group norm input");
    refuse_tangents({&input, &or_undefined(weight), &or_undefined(bias), &or_undefined(residual)});
    TORCH_CHECK(input.dim() >= 2, "box_convolution: group norm input must have >=2 dimensions");
    const int64_t channels = input.size(1);
    TORCH_CHECK(groups >= 1 && channels >= 1 && channels % groups == 0 && channels <= INT32_MAX, "box_convolution: ", channels,
                " channels cannot be split into ", groups, " groups");
    const at::ScalarType kind = weight ? weight->scalar_type() : bias ? bias->scalar_type() : at::kFloat;
    for (const auto& [name, p] : {std::pair<const char*, const Optional*>{"weight", &weight}, {"bias", &bias}}) {
        if (!*p) continue;
        TORCH_CHECK((*p)->device() == input.device() && (*p)->dim() == 1 && (*p)->size(0) == channels, "box_convolution: ", name, " must hold ", channels,
                    " values on ", input.device());
        TORCH_CHECK((*p)->scalar_type() == kind && (kind == at::kFloat || kind == input.scalar_type()),
                    "box_convolution: weight and bias must both be float32 or both of the input's type");
    }
    check_same(residual, input.sizes(), input, "residual");
    if (wants_grad(input, {&weight, &bias, &residual})) return GroupNormAct::apply(input, weight, bias, residual, groups, act, eps, stream);
    return GroupNormAct::call(channels_last(input), static_cast<int>(groups), contiguous(weight), contiguous(bias),
                              residual ? Optional(channels_last(*residual)) : std::nullopt, static_cast<int>(act), eps, stream, nullptr);
}

// ---- the pointwise product -----------------------------------------------------------------------------------
// [..., width] as rows: where they start and how far apart; `hold` keeps a copy, where one was needed, alive.
struct Rows {
    at::Tensor hold;
    int64_t ld;
    Rows(const at::Tensor& t, int64_t rows, int64_t width) {
        hold = t.dim() == 2 ? t : t.reshape({rows, width});
        if (hold.stride(1) != 1 && width != 1) hold = hold.contiguous();
        ld = hold.stride(0);
    }
};

struct LinearAct : public torch::autograd::Function<LinearAct> {
    static at::Tensor call(const at::Tensor& input, const at::Tensor& weight, const Optional& bias, const Optional& residual, int act, int64_t stream,
                           at::Tensor* kept, at::Tensor* rows_of_input) {
        const int64_t N = weight.size(0), K = weight.size(1);
        std::vector<int64_t> shape(input.sizes().begin(), input.sizes().end());
        shape.back() = N;
        int64_t rows = 1;
        for (size_t d = 0; d + 1 < shape.size(); ++d) rows *= shape[d];
        at::Tensor y = at::empty(shape, input.options());
        const Rows x(input, rows, K);
        if (rows_of_input) *rows_of_input = x.hold;
        const int code = type_code(input.scalar_type());
        at::Tensor slope;
        if (kept && act >= 2) slope = at::empty({rows, N}, input.options().dtype(code == 0 ? at::kFloat : at::kShort));
        if (kept) *kept = act >= 2 ? slope : act == 1 ? y : at::Tensor();
        if (y.numel() == 0) return y;
        const std::optional<Rows> r = residual ? std::optional<Rows>(Rows(*residual, rows, N)) : std::nullopt;
        const size_t nbytes = g_operators.linear_bytes(rows, K, N, code, 0);
        const at::Tensor ws = scratch(nbytes, input);
        check_rc(g_operators.linear_forward(x.hold.data_ptr(), x.ld, weight.data_ptr(), address(bias), r ? r->hold.data_ptr() : nullptr, r ? r->ld : 0,
                                            y.data_ptr(), address(slope), code, rows, K, N, act, address(ws), nbytes, reinterpret_cast<void*>(stream)),
                 "linear");
        return y;
    }
    static at::Tensor forward(torch::autograd::AutogradContext* ctx, const at::Tensor& input, const at::Tensor& weight, const Optional& bias,
                              const Optional& residual, int64_t act, int64_t stream) {
        const at::Tensor w = weight.contiguous();
        at::Tensor kept, x;
        at::Tensor y = call(input, w, contiguous(bias), residual, static_cast<int>(act), stream, &kept, &x);
        ctx->save_for_backward({x, w, kept});
        ctx->saved_data["present"] = c10::List<bool>({true, true, bias.has_value(), residual.has_value()});
        ctx->saved_data["shape"] = input.sizes().vec();
        ctx->saved_data["act"] = act;
        ctx->saved_data["stream"] = stream;
        return y;
    }
    static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list grad_outputs) {
        refuse_tangents({&grad_outputs[0]});
        const auto saved = ctx->get_saved_variables();
        const at::Tensor w = saved[1].contiguous(), kept = saved[2].defined() ? saved[2].contiguous() : at::Tensor();
        const int act = static_cast<int>(ctx->saved_data["act"].toInt());
        const std::vector<bool> need = needed(ctx, ctx->saved_data["present"].toBoolList().vec());
        const at::Tensor g = grad_outputs[0].contiguous();
        const int64_t rows = saved[0].size(0), N = w.size(0), K = w.size(1);
        const Rows held(saved[0], rows, K);
        const at::Tensor& x = held.hold;
        const bool none = rows == 0 || N == 0;
        const auto fresh = [&](at::IntArrayRef shape) { return none || K == 0 ? at::zeros(shape, x.options()) : at::empty(shape, x.options()); };
        torch::autograd::variable_list grads(6);               // one per argument of forward
        if (need[0]) grads[0] = fresh(ctx->saved_data["shape"].toIntVector());
        if (need[1]) grads[1] = fresh({N, K});
        if (need[2]) grads[2] = fresh({N});
        if (need[3]) grads[3] = act ? at::empty_like(g) : g;   // without an activation the residual's gradient is grad_output itself
        if (none) return once(grads, x, g);
        const int code = type_code(x.scalar_type());
        const size_t nbytes = g_operators.linear_bytes(rows, K, N, code, 1);
        const at::Tensor ws = scratch(nbytes, x);
        check_rc(g_operators.linear_backward(x.data_ptr(), held.ld, w.data_ptr(), g.data_ptr(), address(kept), address(grads[0]), address(grads[1]),
                                             address(grads[2]), act ? address(grads[3]) : nullptr, code, rows, K, N, act, address(ws), nbytes,
                                             reinterpret_cast<void*>(ctx->saved_data["stream"].toInt())),
                 "linear backward");
        return once(grads, x, g);
    }
};

at::Tensor linear_act(const at::Tensor& input, const at::Tensor& weight, const Optional& bias, const Optional& residual, int64_t act, int64_t stream) {
    check_operator_input(input, "linear input");
    refuse_tangents({&input, &weight, &or_undefined(bias), &or_undefined(residual)});
    TORCH_CHECK(input.dim() >= 1 && weight.dim() == 2 && weight.size(1) == input.size(-1),
                "box_convolution: linear needs an input [..., K] and a weight [N, K], got ", input.sizes(), " and ", weight.sizes());
    std::vector<int64_t> shape(input.sizes().begin(), input.sizes().end());
    shape.back() = weight.size(0);
    check_same(weight, weight.sizes(), input, "weight");
    check_same(bias, {weight.size(0)}, input, "bias");
    check_same(residual, shape, input, "residual");
    if (wants_grad(input, {&bias, &residual}) || (at::GradMode::is_enabled() && weight.requires_grad()))
        return LinearAct::apply(input, weight, bias, residual, act, stream);
    return LinearAct::call(input, weight.contiguous(), contiguous(bias), residual, static_cast<int>(act), stream, nullptr, nullptr);
}

}  // namespace
