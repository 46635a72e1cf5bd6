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
// Statistics, sums over rows and every step between a load and a store are float32; what is stored is rounded once.
//
// Bound by memory: forward 20, backward 40 operations for each of 4 and 6 elements moved. Where a copy of 1 GiB reaches 5.2 TB/s (medians of a kernel trace):
//   forward   4 x 128 x 256 x 128 bfloat16, layer, gate per item   28 us 4.8 TB/s    8192 x 4096 bfloat16, rms   53 us 5.1 TB/s
//   backward                                                        41 us 4.9 TB/s                                 86 us 4.7 TB/s
//   2 x 301 x 767 x 52 float16, layer, gate per element             forward 57 us 4.2 TB/s, backward 91 to 93 us 4.1 to 4.2 TB/s
// and its sums' join 4 to 5 us. One row of 4096 without gradients 4.4 us. Rms without a gate: 16384 x 1000 bfloat16 28 and 37 us, x 1001 31 and 46.
// Still far from it: the backward of more than 4096 channels, whose sums leave the registers (4096 x 8190 bfloat16 134 us, 3.0 TB/s), and both passes of
// more than 8192, element by element (4096 x 12288 bfloat16 0.60 and 4.6 ms, where a copy of the same bytes takes 0.08 and 0.12).
#include <type_traits>

#include "float8_blocks.hpp"
#include "linear_tile.hpp"
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
    float* statistics;                 // written by the forward, read by the backward: a row's four
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
    int wanted;                        // bit k: sum k, over all the workgroup's rows
};

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
typedef float Four __attribute__((ext_vector_type(4)));

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
    // `kept`: the row's statistics, or null: formed here.
    __device__ __forceinline__ void measure(float* lds, const float* kept) {
        if (kept != nullptr) {
            x = {kept[0], kept[1]};
            s = {kept[2], kept[3]};
            return;
        }
        if (a.after) x = moments_any([&](int c) { return input(c); }, a.channels, a.centre, a.eps, lds);
        if (a.before) s = moments_any([&](int c) { return stream(c); }, a.channels, a.centre, a.eps, lds);
    }
    __device__ __forceinline__ float normed(int c) const { return (stream(c) - s.mean) * s.rstd * param(a.before_weight, c, 1.0f) + param(a.before_bias, c, 0.0f); }
};

template <class T>
__global__ void __launch_bounds__(kAnyThreads) norm_rows_any_kernel(Rows<T> a) {
    __shared__ float lds[kAnyThreads / 64];
    for (int64_t i = 0; i < items_of(a.plan, blockIdx.x); ++i) {
        const Span span = span_of(a.plan, a.pixels, blockIdx.x, i);
        for (int64_t row = span.first; row < span.last; ++row) {
            AnyRow<T> r = {a, row * a.channels, span.item};
            r.measure(lds, nullptr);
            if (a.statistics != nullptr && threadIdx.x == 0) *reinterpret_cast<Four*>(a.statistics + 4 * row) = Four{r.x.mean, r.x.rstd, r.s.mean, r.s.rstd};
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
    for (int64_t i = 0; i < items_of(a.plan, blockIdx.x); ++i) {
        const Span span = span_of(a.plan, a.pixels, blockIdx.x, i);
        for (int64_t row = span.first; row < span.last; ++row) {
            AnyRow<T> r = {a, row * a.channels, span.item};
            r.measure(lds, a.statistics == nullptr ? nullptr : a.statistics + 4 * row);
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

// ---- rows in registers ----------------------------------------------------------------------------------------------
// A team of lanes holds a row, kPerLane neighbouring elements a lane: LANES (a power of two) of a
// wave, or, LANES = 0 (WIDE), a whole workgroup. (With a number of lanes known at run time only, every step of a sum over them is a branch: backward of
// 4 x 128 x 256 x 128 bfloat16 74 us, 56 this way.) Every tensor is read once and written once; means and deviations are taken from registers. A team
// keeps its columns from row to row, so parameters stay in registers too, and so do the backward's sums over rows.
constexpr int kPerLane = 8, kNarrowThreads = 256, kWideThreads = 512;
constexpr int kMostRegisterChannels = kWideThreads * 2 * kPerLane;

template <class T, int LANES, int E, bool RAGGED>
struct Team {
    static constexpr bool WIDE = LANES == 0;
    static constexpr int V = Vec<T>::kLen, NV = E / V;
    int lane, channels;
    float inverse;                     // 1 / channels
    float (*exchange)[16][2];          // WIDE: [2][wave][2] in LDS, the two halves in turn
    int turn = 0;
    Chunk keep[RAGGED ? NV : 1];

    // columns of element k and of vector v: kPerLane neighbouring ones, and as many again behind those of all lanes
    __device__ __forceinline__ int column_at(int k) const { return k / kPerLane * static_cast<int>(blockDim.x) * kPerLane + lane * kPerLane + k % kPerLane; }
    __device__ __forceinline__ int column(int v) const { return column_at(v * V); }
    // whether element k of the lane's lies in the row (without RAGGED kPerLane of them lie there or none)
    __device__ __forceinline__ bool inside(int k) const { return column_at(RAGGED ? k : k / kPerLane * kPerLane) < channels; }

    // value of element k, 0 beyond the row
    __device__ __forceinline__ float within(float value, int k) const {
        if constexpr (!RAGGED) return inside(k) ? value : 0.0f;
        else {
            unsigned bits = keep[k / V][k % V * static_cast<int>(sizeof(T)) / 4];
            if constexpr (sizeof(T) == 2) bits = static_cast<unsigned>(static_cast<int>(k % 2 ? bits : bits << 16) >> 16);
            return __builtin_bit_cast(float, __builtin_bit_cast(unsigned, value) & bits);
        }
    }

    // Vectors of a row, as they lie in memory. RAGGED: the last one runs into the next row, whose elements settle() takes away; at the tensor's end,
    // where that would be out of bounds, it starts so much earlier, and mend() moves it. (Element by element such reads took a third of the
    // kernel's instructions, and their conditions drove the others out of the scalar registers: 16384 x 1001 bfloat16 forward 43 us, backward 57.)
    __device__ __forceinline__ int limit(int64_t row, int64_t elements) const {        // the last column that a vector of the row may start at
        return static_cast<int>(min<int64_t>(elements - V - row * channels, INT32_MAX));
    }
    __device__ __forceinline__ void request(const T* tensor, int64_t row, int last, Chunk (&raw)[NV]) const {
        if (tensor == nullptr) return;
        const T* p = tensor + row * channels;
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            const int c = column(v);
            if constexpr (RAGGED) raw[v] = __builtin_bit_cast(Chunk, *reinterpret_cast<const typename Vec<T>::Type*>(p + min(c < channels ? c : 0, last)));
            else raw[v] = c < channels ? __builtin_bit_cast(Chunk, *reinterpret_cast<const typename Vec<T>::Type*>(p + c)) : Chunk{0, 0, 0, 0};
        }
    }
    __device__ __forceinline__ void mend(int last, Chunk (&raw)[NV]) const {
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            Chunk& w = raw[v];
            const int c = column(v) < channels ? column(v) : 0, k = c - min(c, last);      // elements too early
            if (k * static_cast<int>(sizeof(T)) & 8) w = Chunk{w[2], w[3], 0, 0};
            if (k * static_cast<int>(sizeof(T)) & 4) w = Chunk{w[1], w[2], w[3], 0};
            if (sizeof(T) == 2 && (k & 1)) w = Chunk{w[0] >> 16 | w[1] << 16, w[1] >> 16 | w[2] << 16, w[2] >> 16 | w[3] << 16, w[3] >> 16};
        }
    }
    __device__ __forceinline__ bool clear_of_end(int64_t last_row, int64_t rows) const { return (rows - 1 - last_row) * channels >= V; }
    // What was requested, as floats; 0 beyond the row.
    __device__ __forceinline__ void settle(const Chunk (&raw)[NV], float (&out)[E]) const {
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            Chunk c = raw[v];
            if constexpr (RAGGED) c &= keep[v];
            const auto x = __builtin_bit_cast(typename Vec<T>::Type, c);
#pragma unroll
            for (int j = 0; j < V; ++j) out[v * V + j] = static_cast<float>(x[j]);
        }
    }
    // RAGGED: the bits of each vector that lie in the row.
    __device__ __forceinline__ void start() {
        if constexpr (RAGGED) {
#pragma unroll
            for (int v = 0; v < NV; ++v)
#pragma unroll
                for (int w = 0; w < 4; ++w) {
                    const int n = (channels - column(v)) * static_cast<int>(sizeof(T)) - 4 * w;        // bytes from here to the row's end
                    keep[v][w] = n >= 4 ? 0xffffffffu : n <= 0 ? 0u : (1u << 8 * n) - 1;
                }
        }
    }
    __device__ __forceinline__ void store(T* tensor, int64_t row, const float (&value)[E]) const {
        typedef typename Vec<T>::Type Packed;
        T* p = tensor + row * channels;
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            Packed out;
#pragma unroll
            for (int j = 0; j < V; ++j) out[j] = static_cast<T>(value[v * V + j]);
            T* to = p + column(v);
            const int n = channels - column(v);
            if (n >= V || (!RAGGED && n > 0)) *reinterpret_cast<Packed*>(to) = out;
            else if (RAGGED && n > 0) {
                // the row's last elements: as many as for every row, in pieces of 4, 2 and 1
                constexpr int B = sizeof(T);
                typedef T Two __attribute__((ext_vector_type(2), aligned(B)));
                typedef T Several __attribute__((ext_vector_type(4), aligned(B)));
                if constexpr (V == 8) {
                    if (channels & 4) {
                        *reinterpret_cast<Several*>(to) = Several{out[0], out[1], out[2], out[3]};
                        to += 4;
                        out[0] = out[4];
                        out[1] = out[5];
                        out[2] = out[6];
                    }
                }
                if (channels & 2) {
                    *reinterpret_cast<Two*>(to) = Two{out[0], out[1]};
                    to += 2;
                    out[0] = out[2];
                }
                if (channels & 1) *to = out[0];
            }
        }
    }
    // Values per column, of the parameters' type or float; `none` without a vector. RAGGED: 0 beyond the row (so that products with weight and gate
    // are 0 there, whatever was normalised).
    __device__ __forceinline__ void params(const void* p, bool is_float, float none, float (&out)[E]) const {
#pragma unroll
        for (int i = 0; i < E; ++i) out[i] = !RAGGED ? none : p == nullptr ? within(none, i) : 0.0f;
        if (p == nullptr) return;
        if (is_float) run(static_cast<const float*>(p), out);
        else run(static_cast<const T*>(p), out);
    }
    template <class P>
    __device__ __forceinline__ void run(const P* p, float (&out)[E]) const {
        typedef P Run __attribute__((ext_vector_type(kPerLane), aligned(sizeof(P))));
#pragma unroll
        for (int k = 0; k < E; k += kPerLane) {
            const int c = column_at(k);
            if (c + kPerLane <= channels) {
                const Run v = *reinterpret_cast<const Run*>(p + c);
#pragma unroll
                for (int j = 0; j < kPerLane; ++j) out[k + j] = static_cast<float>(v[j]);
            } else if (RAGGED) {
#pragma unroll
                for (int j = 0; j < kPerLane; ++j)
                    if (c + j < channels) out[k + j] = static_cast<float>(p[c + j]);
            }
        }
    }
    // Over the row: the sums of a and b, the same in all its lanes.
    template <bool BOTH = true>
    __device__ __forceinline__ void pair_sum(float& a, float& b) {         // (without BOTH only b's)
        if constexpr (!WIDE) {
            if constexpr (BOTH) a = sum_of_lanes(a, LANES);
            b = sum_of_lanes(b, LANES);
        } else {
            if constexpr (BOTH) a = sum_of_lanes(a, 64);
            b = sum_of_lanes(b, 64);
            swap(a, b);
            a = b = 0.0f;
            for (int w = 0; w < static_cast<int>(blockDim.x) / 64; ++w) {
                a += exchange[turn ^ 1][w][0];
                b += exchange[turn ^ 1][w][1];
            }
        }
    }
    // WIDE: a and b of every wave to the half of `exchange` that is now turn ^ 1. (One barrier: a wave that is a call ahead writes the
    // other half, and none gets two ahead.)
    __device__ __forceinline__ void swap(float a, float b) {
        if (threadIdx.x % 64 == 0) {
            exchange[turn][threadIdx.x / 64][0] = a;
            exchange[turn][threadIdx.x / 64][1] = b;
        }
        __syncthreads();
        turn ^= 1;
    }
    // Mean (0 unless centred) and 1/sqrt(variance + eps) of the row.
    __device__ __forceinline__ Moments moments(const float (&value)[E], bool centre, float eps) {
        Moments m = {0.0f, 0.0f};
        float sum = 0.0f, square = 0.0f;
        if (!centre) {
#pragma unroll
            for (int i = 0; i < E; ++i) square += value[i] * value[i];
            pair_sum(square, sum);
        } else {
            // within a wave first the mean, then the deviations from it
#pragma unroll
            for (int i = 0; i < E; ++i) sum += value[i];
            sum = sum_of_lanes(sum, WIDE ? 64 : LANES);
            float part = inverse;
            int count = channels;
            if constexpr (WIDE) {
                count = in_wave(threadIdx.x / 64);
                part = 1.0f / static_cast<float>(max(count, 1));
            }
            m.mean = sum * part;
#pragma unroll
            for (int i = 0; i < E; ++i) {
                const float d = RAGGED ? within(value[i] - m.mean, i) : value[i] - (inside(i) ? m.mean : 0.0f);
                square += d * d;
            }
            square = sum_of_lanes(square, WIDE ? 64 : LANES);
            if constexpr (WIDE) {
                // the waves' means before their deviations: nothing cancels however far the mean is from zero
                const int waves = blockDim.x / 64;
                swap(m.mean, square);
                float mean = 0.0f;
                for (int w = 0; w < waves; ++w) mean += static_cast<float>(in_wave(w)) * exchange[turn ^ 1][w][0];
                m.mean = mean * inverse;
                square = 0.0f;
                for (int w = 0; w < waves; ++w) {
                    const float d = exchange[turn ^ 1][w][0] - m.mean;
                    square += exchange[turn ^ 1][w][1] + static_cast<float>(in_wave(w)) * d * d;
                }
            }
        }
        m.rstd = rsqrtf(square * inverse + eps);
        return m;
    }
    // (value - mean) * rstd; 0 beyond the row (whose values are 0), but for RAGGED.
    __device__ __forceinline__ void normalise(float (&value)[E], const Moments& m) const {
#pragma unroll
        for (int i = 0; i < E; ++i) {
            const bool in = inside(i);
            value[i] = RAGGED ? (value[i] - m.mean) * m.rstd : (value[i] - (in ? m.mean : 0.0f)) * (in ? m.rstd : 0.0f);
        }
    }
    // Elements of the row in wave w.
    __device__ __forceinline__ int in_wave(int w) const {
        constexpr int kWave = 64 * kPerLane;
        int n = 0;
#pragma unroll
        for (int k = 0; k < E; k += kPerLane) n += min(max(channels - k * static_cast<int>(blockDim.x) - w * kWave, 0), kWave);
        return n;
    }
};

// The team of this thread, the first row of its wave's next ones (from 0 on), its own place among them, and how far apart they are.
template <class T, int LANES, int E, bool RAGGED>
struct Place {
    static constexpr bool WIDE = LANES == 0;
    Team<T, LANES, E, RAGGED> team;
    int first, own, step, teams;       // teams: of a wave
    __device__ __forceinline__ Place(const Rows<T>& a, float (*exchange)[16][2]) {
        constexpr int lanes = WIDE ? 64 : LANES;
        team.lane = WIDE ? threadIdx.x : threadIdx.x % lanes;
        team.channels = a.channels;
        team.inverse = 1.0f / static_cast<float>(a.channels);
        team.exchange = exchange;
        team.start();
        teams = WIDE ? 1 : 64 / lanes;
        first = WIDE ? 0 : __builtin_amdgcn_readfirstlane(threadIdx.x / 64) * teams;
        own = WIDE ? 0 : threadIdx.x % 64 / lanes;
        step = WIDE ? 1 : kNarrowThreads / 64 * teams;
    }
};

// g: the gate times the scale, the scale alone without one; of a gate per element whenever it is settled.
template <class T, int E>
__device__ __forceinline__ void scaled(const Rows<T>& a, float (&g)[E]) {
#pragma unroll
    for (int i = 0; i < E; ++i) g[i] *= a.scale;
}
template <class T, int LANES, int E, bool RAGGED>
__device__ __forceinline__ void item_gate(const Team<T, LANES, E, RAGGED>& team, const Rows<T>& a, int64_t item, float (&g)[E]) {
    if (a.gate_kind == kGateFull) return;
    const int64_t at = a.gate_kind == kGateItem ? item * a.channels : 0;
    const void* const gate = a.gate_kind != kGateChannel && a.gate_kind != kGateItem ? nullptr :
                             a.float_gate ? static_cast<const void*>(static_cast<const float*>(a.gate) + at) : static_cast<const void*>(static_cast<const T*>(a.gate) + at);
    team.params(gate, a.float_gate, 1.0f, g);
    scaled(a, g);
}

// CODES: the normed rows leave in 8 bits. A block of 128 lies in 128 / kPerLane neighbouring lanes.
// Four waves a SIMD, as forward_plan counts on: rows of odd length would take 133 registers otherwise, and leave three (4096 x 4095 bfloat16 43 us, 32 with
// four, a few values in scratch among the cost; 16384 x 1001 36 and 30; float32 the same within 5 %).
template <class T, int LANES, int E, bool RAGGED, bool CODES>
__global__ void __launch_bounds__(LANES == 0 ? kWideThreads : kNarrowThreads, E > kPerLane ? 2 : 4) norm_rows_kernel(Rows<T> a) {
    typedef Team<T, LANES, E, RAGGED> Row;
    constexpr int NV = Row::NV;
    __shared__ float exchange[2][16][2];
    Place<T, LANES, E, RAGGED> place(a, exchange);
    Row& team = place.team;
    float wa[E], ba[E], wb[E], bb[E], g[E];
    const T* const full = a.gate_kind == kGateFull ? static_cast<const T*>(a.gate) : nullptr;
    const int64_t rows = a.plan.batch * a.pixels, elements = rows * a.channels;
    bool loaded = false;
    for (int64_t i = 0; i < items_of(a.plan, blockIdx.x); ++i) {
        const Span span = span_of(a.plan, a.pixels, blockIdx.x, i);
        Chunk xs[NV] = {}, rs[NV] = {}, gs[NV] = {};
        const auto request = [&](int64_t base) {
            const int64_t row = min(base + place.own, span.last - 1);
            const int last = RAGGED ? team.limit(row, elements) : 0;
            team.request(a.x, row, last, xs);
            team.request(a.residual, row, last, rs);
            team.request(full, row, last, gs);
        };
        const auto mend = [&](int64_t base) {
            if (!RAGGED || team.clear_of_end(min(base + place.teams, span.last) - 1, rows)) return;
            const int last = team.limit(min(base + place.own, span.last - 1), elements);
            team.mend(last, xs);
            team.mend(last, rs);
            team.mend(last, gs);
        };
        int64_t base = span.first + place.first;
        if (base < span.last) request(base);
        if (!loaded) {
            team.params(a.after_weight, a.float_params, 1.0f, wa);
            team.params(a.after_bias, a.float_params, 0.0f, ba);
            team.params(a.before_weight, a.float_params, 1.0f, wb);
            team.params(a.before_bias, a.float_params, 0.0f, bb);
            loaded = true;
        }
        item_gate(team, a, span.item, g);
        for (; base < span.last; base += place.step) {
            const int64_t row = base + place.own;
            const bool live = row < span.last;
            float x[E], r[E];
            mend(base);
            team.settle(xs, x);
            team.settle(rs, r);
            if (full != nullptr) {
                team.settle(gs, g);
                scaled(a, g);
            }
            if (base + place.step < span.last) request(base + place.step);
            Four kept = {0.0f, 1.0f, 0.0f, 1.0f};
            if (a.after) {
                const Moments m = team.moments(x, a.centre, a.eps);
                team.normalise(x, m);
                if (LANES == 0) kept = Four{m.mean, m.rstd, 0.0f, 1.0f};
#pragma unroll
                for (int k = 0; k < E; ++k) x[k] = x[k] * wa[k] + ba[k];
            }
            // (0 beyond the row, where x, the residual and the bias are)
#pragma unroll
            for (int k = 0; k < E; ++k) x[k] = r[k] + x[k] * g[k];
            if (a.stream != nullptr && live) team.store(a.stream, row, x);
            Moments m = {0.0f, 1.0f};
            if (a.before) m = team.moments(x, a.centre, a.eps);
            if constexpr (LANES == 0) {
                if (a.statistics != nullptr && threadIdx.x == 0) *reinterpret_cast<Four*>(a.statistics + 4 * row) = Four{kept[0], kept[1], m.mean, m.rstd};
            }
            if (a.normed == nullptr && !CODES) continue;
            team.normalise(x, m);
#pragma unroll
            for (int k = 0; k < E; ++k) x[k] = x[k] * wb[k] + bb[k];
            if constexpr (!CODES) {
                if (live) team.store(a.normed, row, x);
            } else {
                const int blocks = blocks_of(a.channels), words = exponents_of(a.channels);
#pragma unroll
                for (int k = 0; k < E; k += kPerLane) {
                    float part[kPerLane];
#pragma unroll
                    for (int j = 0; j < kPerLane; ++j) part[j] = RAGGED ? team.within(x[k + j], k + j) : x[k + j];
                    const int e = block_exponent(most_of_lanes(largest(part), kBlock / kPerLane)), c = team.column_at(k), b = c / kBlock;
                    const Codes<kPerLane> codes = to_codes(part, e);
                    if (live && b < blocks) {
                        typedef unsigned Words __attribute__((ext_vector_type(kPerLane / 4)));
                        *reinterpret_cast<Words*>(a.codes + row * blocks * kBlock + c) = __builtin_bit_cast(Words, codes);
                        if (c % kBlock == 0) {
                            a.exponents[row * words + b] = static_cast<uint8_t>(e);
                            if (b == blocks - 1)
                                for (int w = blocks; w < words; ++w) a.exponents[row * words + w] = 127;
                        }
                    }
                }
            }
        }
    }
}

// LAYER: whether the norms centre or have biases: sums, means and values that root-mean-square norms do without (8192 x 4096 bfloat16
// 95 us with them, 88 without; 4096 x 4096 46 and 42, 4096 x 8190 205 and 145).
// Two rows ahead are on their way while one is worked on (4 x 128 x 256 x 128 bfloat16 56 us with one, 48 with two; 16384 x 1024 92 and 62). With twice the
// elements a lane (BIG) there are no registers for that, nor for the parameters, which come from the caches again for every row. Workgroups that
// hold a row (WIDE) take its means from the forward: each would cost two barriers a row (8192 x 4096 bfloat16 128 us, 95 this way).
template <class T, int LANES, int E, bool RAGGED, bool LAYER>
__global__ void __launch_bounds__(LANES == 0 ? kWideThreads : kNarrowThreads, 2) norm_rows_grad_kernel(Rows<T> a) {
    typedef Team<T, LANES, E, RAGGED> Row;
    constexpr bool WIDE = LANES == 0, BIG = E > kPerLane;
    constexpr int NV = Row::NV;
    __shared__ float exchange[2][16][2];
    __shared__ float gather[WIDE ? 1 : kNarrowThreads / 64][WIDE ? 1 : 64 * kPerLane];
    Place<T, LANES, E, RAGGED> place(a, exchange);
    Row& team = place.team;
    float sum[kSums][E] = {};
    const T* const full = a.gate_kind == kGateFull ? static_cast<const T*>(a.gate) : nullptr;
    float wa[E], ba[E] = {}, wb[E], g[E];
    const bool centre = LAYER && a.centre;
    const auto after_parameters = [&] {
        team.params(a.after_weight, a.float_params, 1.0f, wa);
        if constexpr (LAYER) team.params(a.after_bias, a.float_params, 0.0f, ba);
    };
    const auto before_parameters = [&] { team.params(a.before_weight, a.float_params, 1.0f, wb); };
    if constexpr (!BIG) {
        after_parameters();
        before_parameters();
    }
    const bool has_dh = a.before && a.dnormed != nullptr;
    const int64_t rows = a.plan.batch * a.pixels, elements = rows * a.channels;
    // sum k of the workgroup's teams to memory
    const auto put = [&](const float (&v)[E], void* to, int64_t at, bool is_float) {
        const auto write = [&](int c, float s) {
            if (is_float) static_cast<float*>(to)[at + c] = s;
            else static_cast<T*>(to)[at + c] = static_cast<T>(s);
        };
        if constexpr (WIDE) {
#pragma unroll
            for (int k = 0; k < E; ++k)
                if (team.inside(k)) write(team.column_at(k), v[k]);
        } else {
            __syncthreads();
#pragma unroll
            for (int k = 0; k < E; ++k) {
                float s = v[k];
                for (int d = LANES; d < 64; d <<= 1) s += __shfl_xor(s, d);
                if (static_cast<int>(threadIdx.x) % 64 < LANES) gather[threadIdx.x / 64][team.column(0) + k] = s;
            }
            __syncthreads();
            for (int c = threadIdx.x; c < a.channels; c += kNarrowThreads) {
                float s = 0.0f;
#pragma unroll
                for (int w = 0; w < kNarrowThreads / 64; ++w) s += gather[w][c];
                write(c, s);
            }
        }
    };
    for (int64_t i = 0; i < items_of(a.plan, blockIdx.x); ++i) {
        const Span span = span_of(a.plan, a.pixels, blockIdx.x, i);
        struct Raw { Chunk x[NV], r[NV], g[NV], d[NV], h[NV]; Four kept; } ahead[BIG ? 1 : 2] = {};
        const auto request = [&](int64_t base, Raw& raw) {
            const int64_t row = min(base + place.own, span.last - 1);
            const int last = RAGGED ? team.limit(row, elements) : 0;
            team.request(a.x, row, last, raw.x);
            if (a.before) team.request(a.residual, row, last, raw.r);
            team.request(full, row, last, raw.g);
            team.request(a.dstream, row, last, raw.d);
            if (a.before) team.request(a.dnormed, row, last, raw.h);
            if constexpr (WIDE) {
                if (a.statistics != nullptr) raw.kept = *reinterpret_cast<const Four*>(a.statistics + 4 * row);
            }
        };
        const auto mend = [&](int64_t base, Raw& raw) {
            if (!RAGGED || team.clear_of_end(min(base + place.teams, span.last) - 1, rows)) return;
            const int last = team.limit(min(base + place.own, span.last - 1), elements);
            team.mend(last, raw.x);
            team.mend(last, raw.r);
            team.mend(last, raw.g);
            team.mend(last, raw.d);
            team.mend(last, raw.h);
        };
        const auto work = [&](int64_t base, Raw& raw) {
            const int64_t row = base + place.own;
            const bool live = row < span.last;
            if constexpr (BIG) {
                request(base, raw);
                after_parameters();
                item_gate(team, a, span.item, g);
            }
            float p[E], q[E], d[E], h[E];                              // normalised x, normalised s, gradients of s and h; later what they become
            mend(base, raw);
            team.settle(raw.x, p);
            team.settle(raw.r, q);
            team.settle(raw.d, d);
            team.settle(raw.h, h);
            if (full != nullptr) {
                team.settle(raw.g, g);
                scaled(a, g);
            }
            const Four kept = raw.kept;
            const bool again = !WIDE || a.statistics == nullptr;
            if constexpr (!BIG) {
                if (base + 2 * place.step < span.last) request(base + 2 * place.step, raw);
            }
            Moments mx = {0.0f, 1.0f};
            if (a.after) {
                mx = again ? team.moments(p, centre, a.eps) : Moments{centre ? kept[0] : 0.0f, kept[1]};
                team.normalise(p, mx);
            }
            if (has_dh) {
#pragma unroll
                for (int k = 0; k < E; ++k) {
                    const float u = a.after ? LAYER ? p[k] * wa[k] + ba[k] : p[k] * wa[k] : p[k];
                    q[k] += u * g[k];
                }
                const Moments ms = again ? team.moments(q, centre, a.eps) : Moments{centre ? kept[2] : 0.0f, kept[3]};
                team.normalise(q, ms);
                if (live) {
#pragma unroll
                    for (int k = 0; k < E; ++k) {
                        sum[2][k] += h[k] * q[k];
                        if constexpr (LAYER) sum[3][k] += h[k];
                    }
                }
                if constexpr (BIG) before_parameters();
                float e1 = 0.0f, e2 = 0.0f;
#pragma unroll
                for (int k = 0; k < E; ++k) {
                    h[k] *= wb[k];                                      // (0 beyond the row)
                    if constexpr (LAYER) e1 += h[k];
                    e2 += h[k] * q[k];
                }
                team.template pair_sum<LAYER>(e1, e2);
                e1 = centre ? e1 * team.inverse : 0.0f;
                e2 *= team.inverse;
#pragma unroll
                for (int k = 0; k < E; ++k) {
                    const float through = h[k] - e1 - q[k] * e2;
                    d[k] += RAGGED ? ms.rstd * through : (team.inside(k) ? ms.rstd : 0.0f) * through;
                }
            }
            if (a.dresidual != nullptr && live) team.store(a.dresidual, row, d);
            if constexpr (BIG) {                                       // (again: they would wait in registers, or in memory)
                asm volatile("" ::: "memory");
                after_parameters();
                item_gate(team, a, span.item, g);
            }
            // d: gradient of s, then of u; h: of the gate, over the scale
#pragma unroll
            for (int k = 0; k < E; ++k) {
                h[k] = (a.after ? LAYER ? p[k] * wa[k] + ba[k] : p[k] * wa[k] : p[k]) * d[k];
                d[k] *= g[k];
            }
            if (a.dgate_full != nullptr && live) {
                float out[E];
#pragma unroll
                for (int k = 0; k < E; ++k) out[k] = h[k] * a.scale;
                team.store(a.dgate_full, row, out);
            }
            if (live) {
#pragma unroll
                for (int k = 0; k < E; ++k) {
                    sum[kSumGate][k] += h[k];
                    sum[0][k] += d[k] * p[k];
                    if constexpr (LAYER) sum[1][k] += d[k];
                }
            }
            if (a.after) {
                float f1 = 0.0f, f2 = 0.0f;
#pragma unroll
                for (int k = 0; k < E; ++k) {
                    d[k] *= wa[k];
                    if constexpr (LAYER) f1 += d[k];
                    f2 += d[k] * p[k];
                }
                team.template pair_sum<LAYER>(f1, f2);
                f1 = centre ? f1 * team.inverse : 0.0f;
                f2 *= team.inverse;
#pragma unroll
                for (int k = 0; k < E; ++k) d[k] = mx.rstd * (d[k] - f1 - p[k] * f2);
            }
            if (a.dx != nullptr && live) team.store(a.dx, row, d);
        };
        int64_t base = span.first + place.first;
        if constexpr (BIG) {
            for (; base < span.last; base += place.step) work(base, ahead[0]);
        } else {
            if (base < span.last) request(base, ahead[0]);
            if (base + place.step < span.last) request(base + place.step, ahead[1]);
            item_gate(team, a, span.item, g);
            for (; base < span.last; base += 2 * place.step) {
                work(base, ahead[0]);
                if (base + place.step < span.last) work(base + place.step, ahead[1]);
            }
        }
        if (a.gate_kind == kGateItem && (a.dgate != nullptr || a.sums != nullptr) && span.last > span.first) {
            scaled(a, sum[kSumGate]);
            if (a.dgate != nullptr) put(sum[kSumGate], a.dgate, span.item * a.channels, a.float_gate);
            else put(sum[kSumGate], a.sums, (static_cast<int64_t>(blockIdx.x) * kSums + kSumGate) * a.channels, true);
#pragma unroll
            for (int k = 0; k < E; ++k) sum[kSumGate][k] = 0.0f;
        }
    }
    if (a.wanted >> kSumGate & 1) scaled(a, sum[kSumGate]);
#pragma unroll
    for (int k = 0; k < kSums; ++k)
        if ((LAYER || k % 2 == 0) && (a.wanted >> k & 1)) put(sum[k], a.sums, (static_cast<int64_t>(blockIdx.x) * kSums + k) * a.channels, true);
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

// How the rows of a call are dealt out: lanes of a team, its workgroup's threads, and rows that a workgroup takes at once. big: twice
// kPerLane elements a lane. No lanes: rows of more channels than the registers of a workgroup hold, and tensors smaller than a vector.
struct Shape { bool wide; int lanes, threads, rows; bool big; };
template <class T>
Shape shape_of(const ResidualNormCall& c, bool codes) {
    const int channels = c.channels;
    if (channels > kMostRegisterChannels || c.batch * c.pixels * channels < kPerLane) return {true, 0, kAnyThreads, 1, false};
    const int columns = codes ? blocks_of(channels) * kBlock : channels;           // (codes are written to the end of the last block)
    int lanes = codes ? kBlock / kPerLane : 1;        // (more lanes without a share add zeros: the sums are the same to the bit)
    while (lanes < 64 && lanes * kPerLane < columns) lanes *= 2;
    if (lanes * kPerLane >= columns) return {false, lanes, kNarrowThreads, kNarrowThreads / lanes, false};
    const int each = columns > kWideThreads * kPerLane ? 2 * kPerLane : kPerLane;
    lanes = (columns + 64 * each - 1) / (64 * each) * 64;
    return {true, lanes, lanes, 1, each > kPerLane};
}

// f(value) with the value known to the compiler: true or false; LANES from `least` on, 0 for a workgroup.
template <class F>
void known(bool value, F f) {
    if (value) f(std::true_type());
    else f(std::false_type());
}
template <int LEAST, class F>
void known_lanes(const Shape& s, F f) {
    typedef std::integral_constant<int, kPerLane> Each;
    if (s.wide && s.big) return f(std::integral_constant<int, 0>(), std::integral_constant<int, 2 * kPerLane>());
    if (s.wide) return f(std::integral_constant<int, 0>(), Each());
    if constexpr (LEAST < 64) {
        if (s.lanes > LEAST) return known_lanes<LEAST * 2>(s, f);
    }
    f(std::integral_constant<int, LEAST>(), Each());
}

// As many workgroups as the chip holds at once: the forward's kernels leave room for four waves a SIMD, the backward's for two, and a workgroup is on one
// compute unit whole: counted in waves, workgroups of 3, 5, 6 or 7 came in two rounds (8192 x 3500 bfloat16 forward 71 us, backward 139; 53 and 82 this way;
// 4096 x 6400 backward 162 and 101; with 4 or 8 waves the count is the same). (Fewer where the backward's sums are long and in memory, read and written
// for every row: 4096 x 12288 bfloat16 takes it 4.7 ms with 128 workgroups, 2.4 with 256, 512 or 1024; 2048 x 16384 3.2 and 1.6; 64 x 16384 0.16 with any number.
// Their workspace grows with them, 20 bytes a channel and workgroup.)
int64_t resident(const Shape& s, int waves) { return 256 * std::max(1, waves * 64 / s.threads); }
RowPlan forward_plan(const ResidualNormCall& c, const Shape& s) { return plan_rows(c, resident(s, s.big ? 8 : 16), s.rows); }
RowPlan backward_plan(const ResidualNormCall& c, const Shape& s) { return plan_rows(c, backward_target(c, s.rows, s.lanes == 0 ? 128 : resident(s, 8)), s.rows); }

}  // namespace

template <class T>
hipError_t residual_norm_forward(const ResidualNormCall& c, const ResidualNormOut& out, hipStream_t stream) {
    Rows<T> a = rows_of<T>(c);
    a.stream = static_cast<T*>(out.stream);
    a.exponents = out.exponents;
    a.statistics = out.statistics;
    const bool coded = out.exponents != nullptr;
    if (coded) a.codes = static_cast<uint8_t*>(out.normed);
    else a.normed = static_cast<T*>(out.normed);
    const Shape s = shape_of<T>(c, coded);
    a.plan = forward_plan(c, s);
    const dim3 grid(static_cast<unsigned>(a.plan.groups)), block(s.threads);
    if (s.lanes == 0) BOXCONV_LAUNCH("norm_rows", (norm_rows_any_kernel<T>), grid, block, 0, stream, a);
    else
        known(c.channels % kPerLane != 0, [&](auto ragged) {
            constexpr bool R = decltype(ragged)::value;
            if (coded)
                known_lanes<kBlock / kPerLane>(s, [&](auto lanes, auto each) { BOXCONV_LAUNCH("norm_rows", (norm_rows_kernel<T, decltype(lanes)::value, decltype(each)::value, R, true>), grid, block, 0, stream, a); });
            else known_lanes<1>(s, [&](auto lanes, auto each) { BOXCONV_LAUNCH("norm_rows", (norm_rows_kernel<T, decltype(lanes)::value, decltype(each)::value, R, false>), grid, block, 0, stream, a); });
        });
    return hipGetLastError();
}

template <class T>
size_t residual_norm_workspace(const ResidualNormCall& c) {
    return static_cast<size_t>(backward_plan(c, shape_of<T>(c, false)).groups) * kSums * c.channels * sizeof(float);
}

template <class T>
hipError_t residual_norm_backward(const ResidualNormCall& c, const ResidualNormGrads& g, void* workspace, hipStream_t stream) {
    Rows<T> a = rows_of<T>(c);
    a.statistics = const_cast<float*>(g.statistics);
    a.dstream = static_cast<const T*>(g.dstream);
    a.dnormed = static_cast<const T*>(g.dnormed);
    a.dx = static_cast<T*>(g.dx);
    a.dresidual = static_cast<T*>(g.dresidual);
    const Shape s = shape_of<T>(c, false);
    a.plan = backward_plan(c, s);
    RowGrads to = {{g.dafter_weight, g.dafter_bias, g.dbefore_weight, g.dbefore_bias, c.gate_kind == kGateFull ? nullptr : g.dgate}};
    if (c.gate_kind == kGateFull) a.dgate_full = static_cast<T*>(g.dgate);
    for (int k = 0; k < kSums; ++k) {
        if (to.p[k] == nullptr) continue;
        a.sums = static_cast<float*>(workspace);
        if (k != kSumGate || c.gate_kind != kGateItem) a.wanted |= 1 << k;
    }
    if (c.gate_kind == kGateItem && a.plan.parts == 1) {
        a.dgate = g.dgate;
        to.p[kSumGate] = nullptr;
    }
    const dim3 grid(static_cast<unsigned>(a.plan.groups)), block(s.threads);
    if (s.lanes == 0) BOXCONV_LAUNCH("norm_rows_grad", (norm_rows_any_grad_kernel<T>), grid, block, 0, stream, a);
    else
        known(c.channels % kPerLane != 0, [&](auto ragged) {
            constexpr bool R = decltype(ragged)::value;
            known(c.centre || c.after_bias != nullptr || c.before_bias != nullptr, [&](auto layer) {
                known_lanes<1>(s, [&](auto lanes, auto each) {
                    BOXCONV_LAUNCH("norm_rows_grad", (norm_rows_grad_kernel<T, decltype(lanes)::value, decltype(each)::value, R, decltype(layer)::value>), grid, block, 0,
                                   stream, a);
                });
            });
        });
    bool any = false;
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
