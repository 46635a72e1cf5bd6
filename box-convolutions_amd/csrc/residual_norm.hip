// What lies between two blocks of a residual network, on rows of C channels, forward and backward, for one element type
// (BOXCONV_INST_T: float, _Float16 or __bf16; compiled once for each).
//
//   n(v; w, b) = (v - mean) * rstd * w + b, mean and rstd = 1/sqrt(variance + eps) over the row's channels; without centring the mean
//   counts as 0 (root mean square)
//   u = n(x; after) or x;  stream s = residual + scale * gate * u;  normed h = n(s; before)
//
//   With p, q the normalised x and s, and the means taken over a row (those of e and f only with centring):
//   ds = dstream + rstd_s * (e - mean(e) - q * mean(e q)), e = dh * w_before;  dresidual = ds
//   dgate = sum of scale * u * ds;  du = scale * gate * ds;  dx = rstd_x * (f - mean(f) - p * mean(f p)), f = du * w_after
//   dw_before = sum dh q, db_before = sum dh, dw_after = sum du p, db_after = sum du
//
// s is formed in float32 and h and the backward take it unrounded: the backward forms it again from x, the residual and the gate.
#include "float8_blocks.hpp"
#include "residual_norm.hpp"

namespace boxconv {

namespace {

// What the kernels take. Null pointers leave their piece out; `fused` holds the flags.
template <class T>
struct Rows {
    const T *x, *residual;
    const void *gate, *after_weight, *after_bias, *before_weight, *before_bias;
    T *stream, *normed;
    uint8_t *codes, *exponents;        // the normed rows in 8 bits, in place of `normed`
    int channels, gate_kind;
    bool after, before, centre, float_params, float_gate;
    float scale, eps;
    int64_t pixels;                    // rows of an item; an item is what shares a gate
    RowPlan plan;
    // backward
    const T *dstream, *dnormed;
    T *dx, *dresidual, *dgate_full;
    void* dgate;                       // of an item, where a workgroup has all its rows
    float* sums;                       // [workgroup][kSums][channels]
};

// The rows [first, last) of item i of the workgroup's, counted over the whole tensor; none from `items` on.
struct Span { int64_t item, first, last; };
__device__ __forceinline__ Span span_of(const RowPlan& p, int64_t pixels, int64_t i) {
    const int64_t item = p.parts > 1 ? blockIdx.x / p.parts : blockIdx.x * p.items + i;
    if (i >= p.items || item >= p.batch) return {item, 0, 0};
    const int64_t part = p.parts > 1 ? blockIdx.x % p.parts : 0, begin = part * p.rows;
    return {item, item * pixels + begin, item * pixels + min(pixels, begin + p.rows)};
}

// ---- any number of channels -------------------------------------------------------------------------------------
// A workgroup takes a row at a time and reads it again for every mean; the rows it does so with come from the caches.
constexpr int kAnyThreads = 1024;

template <int N>
__device__ __forceinline__ void sum_of_workgroup(float (&v)[N], float* lds) {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = sum_of_lanes(v[i], 64);
    __syncthreads();                                           // (what was there has been read)
    if (threadIdx.x % 64 == 0) {
#pragma unroll
        for (int i = 0; i < N; ++i) lds[threadIdx.x / 64 * N + i] = v[i];
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; ++i) {
        v[i] = 0.0f;
        for (int w = 0; w < kAnyThreads / 64; ++w) v[i] += lds[w * N + i];
    }
}

struct Moments { float mean, rstd; };

template <class F>
__device__ __forceinline__ Moments moments_any(F value, int channels, bool centre, float eps, float* lds) {
    float v[1] = {};
    Moments m = {0.0f, 0.0f};
    if (centre) {
        for (int c = threadIdx.x; c < channels; c += kAnyThreads) v[0] += value(c);
        sum_of_workgroup(v, lds);
        m.mean = v[0] / static_cast<float>(channels);
        v[0] = 0.0f;
    }
    for (int c = threadIdx.x; c < channels; c += kAnyThreads) {
        const float d = value(c) - m.mean;
        v[0] += d * d;
    }
    sum_of_workgroup(v, lds);
    m.rstd = rsqrtf(v[0] / static_cast<float>(channels) + eps);
    return m;
}

// The pieces of one row, element by element.
template <class T>
struct AnyRow {
    const Rows<T>& a;
    int64_t at;            // its first element
    int64_t item;
    Moments x = {}, s = {};
    __device__ __forceinline__ float param(const void* p, int c, float none) const { return p == nullptr ? none : load_param<T>(p, a.float_params, c); }
    __device__ __forceinline__ float input(int c) const { return static_cast<float>(a.x[at + c]); }
    __device__ __forceinline__ float unit(int c) const { return (input(c) - x.mean) * x.rstd; }
    __device__ __forceinline__ float u(int c) const {
        return a.after ? unit(c) * param(a.after_weight, c, 1.0f) + param(a.after_bias, c, 0.0f) : input(c);
    }
    __device__ __forceinline__ float gate(int c) const {
        switch (a.gate_kind) {
            case kGateChannel: return load_param<T>(a.gate, a.float_gate, c);
            case kGateItem: return a.float_gate ? static_cast<const float*>(a.gate)[item * a.channels + c] : static_cast<float>(static_cast<const T*>(a.gate)[item * a.channels + c]);
            case kGateFull: return static_cast<float>(static_cast<const T*>(a.gate)[at + c]);
            default: return 1.0f;
        }
    }
    __device__ __forceinline__ float stream(int c) const {
        const float t = u(c) * gate(c) * a.scale;
        return a.residual != nullptr ? static_cast<float>(a.residual[at + c]) + t : t;
    }
    __device__ __forceinline__ void measure(float* lds) {
        if (a.after) x = moments_any([&](int c) { return input(c); }, a.channels, a.centre, a.eps, lds);
        if (a.before) s = moments_any([&](int c) { return stream(c); }, a.channels, a.centre, a.eps, lds);
    }
    __device__ __forceinline__ float normed(int c) const { return (stream(c) - s.mean) * s.rstd * param(a.before_weight, c, 1.0f) + param(a.before_bias, c, 0.0f); }
};

template <class T>
__global__ void __launch_bounds__(kAnyThreads) norm_rows_any_kernel(Rows<T> a) {
    __shared__ float lds[kAnyThreads / 64];
    for (int64_t i = 0; i < a.plan.items; ++i) {
        const Span span = span_of(a.plan, a.pixels, i);
        for (int64_t row = span.first; row < span.last; ++row) {
            AnyRow<T> r = {a, row * a.channels, span.item};
            r.measure(lds);
            if (a.stream != nullptr)
                for (int c = threadIdx.x; c < a.channels; c += kAnyThreads) a.stream[r.at + c] = static_cast<T>(r.stream(c));
            if (a.normed != nullptr)
                for (int c = threadIdx.x; c < a.channels; c += kAnyThreads) a.normed[r.at + c] = static_cast<T>(r.normed(c));
            if (a.codes != nullptr) {
                // a wave takes a block of 128, a lane two of its values
                const int blocks = blocks_of(a.channels), padded = exponents_of(a.channels), l = threadIdx.x % 64;
                for (int b = threadIdx.x / 64; b < blocks; b += kAnyThreads / 64) {
                    const int c = b * kBlock + 2 * l;
                    float v[2] = {c < a.channels ? r.normed(c) : 0.0f, c + 1 < a.channels ? r.normed(c + 1) : 0.0f};
                    const int e = block_exponent(most_of_lanes(largest(v), 64));
                    *reinterpret_cast<uint16_t*>(a.codes + row * blocks * kBlock + c) = static_cast<uint16_t>(to_codes(v, e)[0]);
                    if (l == 0) a.exponents[row * padded + b] = static_cast<uint8_t>(e);
                }
                for (int b = blocks + threadIdx.x; b < padded; b += kAnyThreads) a.exponents[row * padded + b] = 127;
            }
        }
    }
}

template <class T>
__global__ void __launch_bounds__(kAnyThreads) norm_rows_any_grad_kernel(Rows<T> a) {
    __shared__ float lds[kAnyThreads / 64 * 2];
    const float inverse = 1.0f / static_cast<float>(a.channels);
    float* const sums = a.sums == nullptr ? nullptr : a.sums + static_cast<int64_t>(blockIdx.x) * kSums * a.channels;
    // (each thread adds to sums of its own channels only; the first row's are stored)
    bool first = true;
    for (int64_t i = 0; i < a.plan.items; ++i) {
        const Span span = span_of(a.plan, a.pixels, i);
        for (int64_t row = span.first; row < span.last; ++row) {
            AnyRow<T> r = {a, row * a.channels, span.item};
            r.measure(lds);
            const auto dh = [&](int c) { return a.before && a.dnormed != nullptr ? static_cast<float>(a.dnormed[r.at + c]) : 0.0f; };
            const auto q = [&](int c) { return (r.stream(c) - r.s.mean) * r.s.rstd; };
            const auto e = [&](int c) { return dh(c) * r.param(a.before_weight, c, 1.0f); };
            float m[2] = {};
            if (a.before && a.dnormed != nullptr) {
                for (int c = threadIdx.x; c < a.channels; c += kAnyThreads) {
                    m[0] += e(c);
                    m[1] += e(c) * q(c);
                }
                sum_of_workgroup(m, lds);
            }
            const float e_mean = a.centre ? m[0] * inverse : 0.0f, eq_mean = m[1] * inverse;
            const auto ds = [&](int c) {
                const float d = a.dstream != nullptr ? static_cast<float>(a.dstream[r.at + c]) : 0.0f;
                return a.before && a.dnormed != nullptr ? d + r.s.rstd * (e(c) - e_mean - q(c) * eq_mean) : d;
            };
            const auto du = [&](int c) { return ds(c) * a.scale * r.gate(c); };
            const auto f = [&](int c) { return du(c) * r.param(a.after_weight, c, 1.0f); };
            float n[2] = {};
            if (a.after) {
                for (int c = threadIdx.x; c < a.channels; c += kAnyThreads) {
                    n[0] += f(c);
                    n[1] += f(c) * r.unit(c);
                }
                sum_of_workgroup(n, lds);
            }
            const float f_mean = a.centre ? n[0] * inverse : 0.0f, fp_mean = n[1] * inverse;
            for (int c = threadIdx.x; c < a.channels; c += kAnyThreads) {
                if (a.dresidual != nullptr) a.dresidual[r.at + c] = static_cast<T>(ds(c));
                if (a.dx != nullptr) a.dx[r.at + c] = static_cast<T>(a.after ? r.x.rstd * (f(c) - f_mean - r.unit(c) * fp_mean) : du(c));
                if (a.dgate_full != nullptr) a.dgate_full[r.at + c] = static_cast<T>(ds(c) * a.scale * r.u(c));
                if (sums != nullptr) {
                    const float part[kSums] = {a.after ? du(c) * r.unit(c) : 0.0f, du(c), a.before ? dh(c) * q(c) : 0.0f, dh(c), ds(c) * a.scale * r.u(c)};
#pragma unroll
                    for (int k = 0; k < kSums; ++k) {
                        const bool fresh = k == kSumGate && a.gate_kind == kGateItem ? row == span.first : first;
                        sums[k * a.channels + c] = fresh ? part[k] : sums[k * a.channels + c] + part[k];
                    }
                }
            }
            first = false;
        }
        if (a.dgate != nullptr && span.last > span.first) {        // the item's rows are all this workgroup's
            for (int c = threadIdx.x; c < a.channels; c += kAnyThreads) {
                const float v = sums[kSumGate * a.channels + c];
                if (a.float_gate) static_cast<float*>(a.dgate)[span.item * a.channels + c] = v;
                else static_cast<T*>(a.dgate)[span.item * a.channels + c] = static_cast<T>(v);
            }
        }
    }
}

// ---- sums over workgroups -----------------------------------------------------------------------------------------
// Column sums of [workgroup][kSums][channels] in an order that only the sizes decide. blockIdx.y: which sum; from kSums on the gate's of item
// blockIdx.y - kSums, over its own workgroups. A workgroup takes 32 columns, 32 threads side by side down the workgroups.
template <class T>
__global__ void __launch_bounds__(1024) join_rows_kernel(Rows<T> a, RowGrads out) {
    __shared__ float part[32][33];
    const int x = threadIdx.x % 32, y = threadIdx.x / 32, k = min(static_cast<int>(blockIdx.y), kSumGate);
    const int64_t item = static_cast<int64_t>(blockIdx.y) - kSumGate, c = blockIdx.x * 32ll + x;
    const bool of_item = a.gate_kind == kGateItem && k == kSumGate;
    void* const to = out.p[k];
    if (to == nullptr) return;
    const int64_t first = of_item ? item * a.plan.parts : 0, last = of_item ? first + a.plan.parts : a.plan.groups;
    float s = 0.0f;
    if (c < a.channels) {
#pragma unroll 8
        for (int64_t g = first + y; g < last; g += 32) s += a.sums[(g * kSums + k) * a.channels + c];
    }
    part[y][x] = s;
    __syncthreads();
    if (y == 0 && c < a.channels) {
        s = 0.0f;
        for (int i = 0; i < 32; ++i) s += part[i][x];
        const bool is_float = k == kSumGate ? a.float_gate : a.float_params;
        const int64_t i = of_item ? item * a.channels + c : c;
        if (is_float) static_cast<float*>(to)[i] = s;
        else static_cast<T*>(to)[i] = static_cast<T>(s);
    }
}

// ---- host -----------------------------------------------------------------------------------------------------------
template <class T>
Rows<T> rows_of(const ResidualNormCall& c) {
    Rows<T> a = {};
    a.x = static_cast<const T*>(c.x);
    a.residual = static_cast<const T*>(c.residual);
    a.gate = c.gate;
    a.after_weight = c.after_weight;
    a.after_bias = c.after_bias;
    a.before_weight = c.before_weight;
    a.before_bias = c.before_bias;
    a.channels = c.channels;
    a.gate_kind = c.gate_kind;
    a.after = c.after;
    a.before = c.before;
    a.centre = c.centre;
    a.float_params = c.float_params;
    a.float_gate = c.float_gate;
    a.scale = c.scale;
    a.eps = c.eps;
    a.pixels = c.gate_kind == kGateItem ? c.pixels : c.batch * c.pixels;
    return a;
}

}  // namespace

template <class T>
hipError_t residual_norm_forward(const ResidualNormCall& c, const ResidualNormOut& out, hipStream_t stream) {
    Rows<T> a = rows_of<T>(c);
    a.stream = static_cast<T*>(out.stream);
    (out.exponents != nullptr ? reinterpret_cast<void*&>(a.codes) : reinterpret_cast<void*&>(a.normed)) = out.normed;
    a.exponents = out.exponents;
    a.plan = plan_rows(c, 2048, 1);
    BOXCONV_LAUNCH("norm_rows", (norm_rows_any_kernel<T>), dim3(static_cast<unsigned>(a.plan.groups)), dim3(kAnyThreads), 0, stream, a);
    return hipGetLastError();
}

template <class T>
size_t residual_norm_workspace(const ResidualNormCall& c) {
    return static_cast<size_t>(plan_rows(c, 512, 1).groups) * kSums * c.channels * sizeof(float);
}

template <class T>
hipError_t residual_norm_backward(const ResidualNormCall& c, const ResidualNormGrads& g, void* workspace, hipStream_t stream) {
    Rows<T> a = rows_of<T>(c);
    a.dstream = static_cast<const T*>(g.dstream);
    a.dnormed = static_cast<const T*>(g.dnormed);
    a.dx = static_cast<T*>(g.dx);
    a.dresidual = static_cast<T*>(g.dresidual);
    a.plan = plan_rows(c, 512, 1);
    RowGrads to = {{g.dafter_weight, g.dafter_bias, g.dbefore_weight, g.dbefore_bias, c.gate_kind == kGateFull ? nullptr : g.dgate}};
    if (c.gate_kind == kGateFull) a.dgate_full = static_cast<T*>(g.dgate);
    bool any = false;
    for (void* p : to.p) any = any || p != nullptr;
    if (any) a.sums = static_cast<float*>(workspace);
    if (c.gate_kind == kGateItem && a.plan.parts == 1) {
        a.dgate = g.dgate;
        to.p[kSumGate] = nullptr;
    }
    BOXCONV_LAUNCH("norm_rows_grad", (norm_rows_any_grad_kernel<T>), dim3(static_cast<unsigned>(a.plan.groups)), dim3(kAnyThreads), 0, stream, a);
    any = false;
    for (void* p : to.p) any = any || p != nullptr;
    if (any) {
        const unsigned kinds = to.p[kSumGate] != nullptr && c.gate_kind == kGateItem ? kSumGate + static_cast<unsigned>(c.batch) : kSums;
        BOXCONV_LAUNCH("join_rows", (join_rows_kernel<T>), dim3(static_cast<unsigned>((c.channels + 31) / 32), kinds), dim3(1024), 0, stream, a, to);
    }
    return hipGetLastError();
}

template hipError_t residual_norm_forward<BOXCONV_INST_T>(const ResidualNormCall&, const ResidualNormOut&, hipStream_t);
template size_t residual_norm_workspace<BOXCONV_INST_T>(const ResidualNormCall&);
template hipError_t residual_norm_backward<BOXCONV_INST_T>(const ResidualNormCall&, const ResidualNormGrads&, void*, hipStream_t);

}  // namespace boxconv
