// Group norm with a residual and an activation on channels-last data, forward and backward.
//
//   m = pixels * channels / groups values per (batch item b, group g);  mean, var over them;  rstd = 1/sqrt(var + eps)
//   u = (x - mean) * rstd;  z = u * weight[c] + bias[c] + residual;  y = act(z)
//   dz = dy * act'(z);  dweight[c] = sum dz*u;  dbias[c] = sum dz;  dresidual = dz
//   dx = rstd * (weight[c]*dz - (s1 + u*s2)/m),  s1, s2 = sums over the group of weight*dz and weight*dz*u
//
// A batch item is one run of pixels * channels elements. Lane t of a workgroup takes 16-byte vectors t, t + T, t + 2T, ... of
// it, with T (at most the workgroup's threads) a multiple of the vectors after which the channels repeat: the channels of a
// lane's elements then never change, so per-channel values and sums sit in registers, whatever the number of channels.
#include "activation.hpp"
#include "boxconv_host.hpp"
#include "operators_host.hpp"

namespace boxconv {

namespace {

constexpr int kUnroll = 8;             // vectors a lane requests before it uses the first one, in the statistics

// How a workgroup's lanes lie over one batch item (or, in the one-launch kernels, over `slab` of its channels).
struct Lanes {
    int64_t total;        // elements of a batch item
    int64_t stride;       // elements from a lane's vector to its next one
    int channels, slab;   // channels in all; channels a workgroup covers (all of them, or whole groups and whole vectors)
    int active;           // lanes that take part
    int phase;            // lanes after which the channels repeat
};

template <class T>
struct Item {
    static constexpr int V = Vec<T>::kLen;
    typedef typename Vec<T>::Type Packed;
    // First element of lane t (relative to the batch item), channels [c0, c0 + slab).
    static __device__ __forceinline__ int64_t offset(const Lanes& L, int t, int c0) {
        return static_cast<int64_t>(t / L.phase) * (L.slab == L.channels ? L.phase * V : L.channels) + c0 + (t % L.phase) * V;
    }
    // Channel of its first element.
    static __device__ __forceinline__ int channel(const Lanes& L, int t, int c0) { return (c0 + t % L.phase * V) % L.channels; }
    // Elements [off, off + V) of an item of `total`: V of them, fewer at its end, zeros beyond it.
    static __device__ __forceinline__ Packed load(const T* p, int64_t off, int64_t total) {
        if (off + V <= total) return *reinterpret_cast<const Packed*>(p + off);
        Packed v = {};
        for (int j = 0; j < V; ++j)
            if (off + j < total) v[j] = p[off + j];
        return v;
    }
    static __device__ __forceinline__ void store(T* p, int64_t off, int64_t total, Packed v) {
        if (off + V <= total) {
            *reinterpret_cast<Packed*>(p + off) = v;
            return;
        }
        for (int j = 0; j < V; ++j)
            if (off + j < total) p[off + j] = v[j];
    }
};

// The channel and group of a lane's elements one after the other (divisions take dozens of instructions, a step three).
struct Walk {
    int c, g, rest;       // channel, its group, its place in the group
    __device__ __forceinline__ Walk(int channel, int per_group) : c(channel), g(channel / per_group), rest(channel - g * per_group) {}
    __device__ __forceinline__ void next(int channels, int per_group) {
        if (++rest == per_group) {
            rest = 0;
            ++g;
        }
        if (++c == channels) c = g = rest = 0;
    }
};

// weight and bias of a lane's V channels from `at` on (1 and 0 where there are none): all requested before any is used.
template <class T, int V>
__device__ __forceinline__ void lane_params(const void* weight, const void* bias, bool is_float, Walk at, int channels, int per_group, float (&w)[V], float (&b)[V]) {
    int c[V];
#pragma unroll
    for (int j = 0; j < V; ++j) {
        c[j] = at.c;
        at.next(channels, per_group);
        w[j] = 1.0f;
        b[j] = 0.0f;
    }
    const auto get = [&](const void* p, float (&v)[V]) {
        if (p == nullptr) return;
        if (is_float) {
#pragma unroll
            for (int j = 0; j < V; ++j) v[j] = static_cast<const float*>(p)[c[j]];
        } else {
#pragma unroll
            for (int j = 0; j < V; ++j) v[j] = static_cast<float>(static_cast<const T*>(p)[c[j]]);
        }
    };
    get(weight, w);
    get(bias, b);
}

// u and z of one element, step by step as the formulas stand, each step rounded: forward and backward kernels form the very same
// z, so that relu's derivative is 0 exactly where its value is. ((x - mean) comes first: x * scale + shift would lose what a
// mean far from zero takes of the digits.)
struct Formed { float u, z; };
__device__ __forceinline__ Formed form(float x, float mean, float rstd, float w, float b, float r) {
#pragma clang fp contract(off)
    const float u = (x - mean) * rstd;
    const float scaled = u * w;
    const float shifted = scaled + b;
    return {u, shifted + r};
}
// 1/sqrt(variance + eps), rounded once.
__device__ __forceinline__ float inverse_deviation(float variance, float eps) { return static_cast<float>(1.0 / sqrt(static_cast<double>(variance + eps))); }

// Sum over `width` (a power of two, at most 64) neighbouring lanes.
__device__ __forceinline__ float sum_over(float v, int width) {
    for (int d = width >> 1; d > 0; d >>= 1) v += __shfl_xor(v, d);
    return v;
}

// Lanes that share a group when the workgroup's threads walk over `groups` of them: a power of two.
__device__ __forceinline__ int lanes_per_group(int threads, int groups) {
    int w = 64;
    while (w > 1 && w * groups > threads) w >>= 1;
    return w;
}

// Where LDS keeps slot f = V * lane + element: the lanes of one element side by side, so that neither the lanes' writes nor the
// reads of one channel (every slab-th slot) meet in a bank, and 32 / V words between the elements, so that those of neighbouring
// channels do not either where the lanes are a multiple of 64 (without: 77 % of the LDS cycles of norm_statistics were conflicts, now 33 %; 4 x 128 x 256 x 128 bfloat16 forward with a residual 33.4 and 32.3 us).
constexpr int kept_words(int active, int V) { return active * V + 32; }
template <int V>
__device__ __forceinline__ int kept_at(int lane, int element, int active) { return element * (active + 32 / V) + lane; }
template <int V>
__device__ __forceinline__ int kept_at(int f, int active) { return kept_at<V>(f / V, f % V, active); }

// Per-slot statistics of a workgroup's lanes to per-group ones: count, mean and sum of squared deviations. Means are joined
// before deviations, so nothing cancels however far the mean is from zero. `put(g, n, mean, m2)` gets the groups that start
// at channel c0, counted from 0.
template <int V, class Put>
__device__ __forceinline__ void join_statistics(const float (&mean)[V], const float (&m2)[V], const float (&count)[V], float* lds,
                                                const Lanes& L, int per_group, Put put) {
    const int t = threadIdx.x, slots = L.active * V;
    float *smean = lds, *sm2 = lds + kept_words(L.active, V), *sn = sm2 + kept_words(L.active, V);
    if (t < L.active) {
#pragma unroll
        for (int j = 0; j < V; ++j) {
            smean[kept_at<V>(t, j, L.active)] = mean[j];
            sm2[kept_at<V>(t, j, L.active)] = m2[j];
            sn[kept_at<V>(t, j, L.active)] = count[j];
        }
    }
    __syncthreads();
    // slots t*V + j with (t % phase)*V + j = c (mod slab) hold channel c: slot c + slab*k for every k. A group's `width` lanes
    // share its channels, `across` at a time, and where there are fewer of those the k
    const int groups = L.slab / per_group, width = lanes_per_group(blockDim.x, groups);
    int across = width;
    while (across > per_group) across >>= 1;
    const int first = t % width % across, row = t % width / across * L.slab, step = width / across * L.slab;
    for (int g0 = 0; g0 < groups; g0 += blockDim.x / width) {
        const int g = g0 + t / width;
        const bool live = g < groups;
        float n = 0.0f, sum = 0.0f;
        if (live)
            for (int c = first; c < per_group; c += across)
                for (int f = g * per_group + c + row; f < slots; f += step) {
                    const int s = kept_at<V>(f, L.active);
                    n += sn[s];
                    sum = fmaf(sn[s], smean[s], sum);
                }
        n = sum_over(n, width);
        const float mu = n > 0.0f ? sum_over(sum, width) / n : 0.0f;
        float dev = 0.0f;
        if (live)
            for (int c = first; c < per_group; c += across)
                for (int f = g * per_group + c + row; f < slots; f += step) {
                    const int s = kept_at<V>(f, L.active);
                    const float d = smean[s] - mu;
                    dev += sm2[s] + sn[s] * d * d;
                }
        dev = sum_over(dev, width);
        if (live && t % width == 0) put(g, n, mu, dev);
    }
}

// Sums per slot to sums per channel of the slab (channel counted from 0): put(c, sum a, sum b).
template <int V, class Put>
__device__ __forceinline__ void join_channels(const float (&a)[V], const float (&b)[V], float* lds, const Lanes& L, Put put) {
    const int t = threadIdx.x, slots = L.active * V;
    float *sa = lds, *sb = lds + kept_words(L.active, V);
    if (t < L.active) {
#pragma unroll
        for (int j = 0; j < V; ++j) {
            sa[kept_at<V>(t, j, L.active)] = a[j];
            sb[kept_at<V>(t, j, L.active)] = b[j];
        }
    }
    __syncthreads();
    for (int c = t; c < L.slab; c += blockDim.x) {
        float x = 0.0f, y = 0.0f;
#pragma unroll 4
        for (int f = c; f < slots; f += L.slab) {
            const int s = kept_at<V>(f, L.active);
            x += sa[s];
            y += sb[s];
        }
        put(c, x, y);
    }
}

// Sums per slot to sums per group of the slab: out[group] = result(sum), visible to the whole workgroup.
template <int V, class F>
__device__ __forceinline__ void join_groups(const float (&v)[V], float* lds, float* out, const Lanes& L, int per_group, F result) {
    const int t = threadIdx.x, slots = L.active * V;
    if (t < L.active) {
#pragma unroll
        for (int j = 0; j < V; ++j) lds[kept_at<V>(t, j, L.active)] = v[j];
    }
    __syncthreads();
    const int groups = L.slab / per_group, width = lanes_per_group(blockDim.x, groups);
    int across = width;
    while (across > per_group) across >>= 1;
    const int first = t % width % across, row = t % width / across * L.slab, step = width / across * L.slab;
    for (int g0 = 0; g0 < groups; g0 += blockDim.x / width) {
        const int g = g0 + t / width;
        float sum = 0.0f;
        if (g < groups)
            for (int c = first; c < per_group; c += across) {
#pragma unroll 4
                for (int f = g * per_group + c + row; f < slots; f += step) sum += lds[kept_at<V>(f, L.active)];
            }
        sum = sum_over(sum, width);
        if (g < groups && t % width == 0) out[g] = result(sum);
    }
    __syncthreads();
}

// ---- statistics of large items: partial results per workgroup --------------------------------------
// partial[(b * groups + g) * chunks + chunk] = (mean, sum of squared deviations) of a chunk of whole pixels. Every batch of kUnroll vectors is
// reduced around its own mean and joined to the lane's running one (the formula of Chan, Golub and LeVeque), so the sums
// are as good for a channel with a large mean as for one without. Bound by reading x: 8 x 128 x 256 x 128 bfloat16 (67 MB) 14 us,
// 2 x 512 x 1024 x 128 float (537 MB) 89 us, 6.0 TB/s.
template <class T>
__global__ void __launch_bounds__(1024)
norm_statistics_kernel(const T* __restrict__ x, float2* __restrict__ partial, Lanes L, int64_t chunk_steps, int chunks,
                       int groups, int per_group) {
    constexpr int V = Vec<T>::kLen;
    extern __shared__ float lds[];
    const int t = threadIdx.x;
    const unsigned chunk = blockIdx.x % static_cast<unsigned>(chunks);
    const int64_t b = blockIdx.x / static_cast<unsigned>(chunks);
    const T* item = x + b * L.total;
    float mean[V], m2[V], count[V];
#pragma unroll
    for (int j = 0; j < V; ++j) mean[j] = m2[j] = count[j] = 0.0f;
    if (t < L.active) {
        int64_t off = Item<T>::offset(L, t, 0) + chunk * chunk_steps * L.stride;
        const int64_t end = min(L.total, (chunk + 1) * chunk_steps * L.stride);    // the chunk's elements: a multiple of stride, or the item's end
        float n = 0.0f;
        for (; off + (kUnroll - 1) * L.stride + V <= end; off += kUnroll * L.stride) {
            typename Vec<T>::Type v[kUnroll];
#pragma unroll
            for (int k = 0; k < kUnroll; ++k) v[k] = *reinterpret_cast<const typename Vec<T>::Type*>(item + off + k * L.stride);
            const float inv = 1.0f / (n + kUnroll), share = kUnroll * inv, joint = n * share;
#pragma unroll
            for (int j = 0; j < V; ++j) {
                float s = 0.0f, d2 = 0.0f;
#pragma unroll
                for (int k = 0; k < kUnroll; ++k) s += static_cast<float>(v[k][j]);
                const float mu = s * (1.0f / kUnroll);
#pragma unroll
                for (int k = 0; k < kUnroll; ++k) {
                    const float d = static_cast<float>(v[k][j]) - mu;
                    d2 = fmaf(d, d, d2);
                }
                const float delta = mu - mean[j];
                mean[j] = fmaf(delta, share, mean[j]);
                m2[j] += fmaf(delta * delta, joint, d2);
            }
            n += kUnroll;
        }
#pragma unroll
        for (int j = 0; j < V; ++j) count[j] = n;
        for (; off < end; off += L.stride) {
            const auto v = Item<T>::load(item, off, L.total);
#pragma unroll
            for (int j = 0; j < V; ++j) {
                if (off + j >= L.total) continue;
                const float delta = static_cast<float>(v[j]) - mean[j], share = 1.0f / (count[j] + 1.0f);
                mean[j] = fmaf(delta, share, mean[j]);
                m2[j] = fmaf(delta * delta, count[j] * share, m2[j]);
                count[j] += 1.0f;
            }
        }
    }
    float2* out = partial + b * groups * chunks + chunk;
    join_statistics<V>(mean, m2, count, lds, L, per_group, [&](int g, float, float mu, float dev) { out[static_cast<int64_t>(g) * chunks] = {mu, dev}; });
}

// Sum over a workgroup of 256.
__device__ __forceinline__ float sum_of_workgroup(float v, float* lds) {
    v = sum_over(v, 64);
    __syncthreads();
    if (threadIdx.x % 64 == 0) lds[threadIdx.x / 64] = v;
    __syncthreads();
    return lds[0] + lds[1] + lds[2] + lds[3];
}

// One workgroup per (batch item, group): the results of all its chunks (at most kMostChunks), in their order. A chunk has
// `in_chunk` values of the group, the last one `in_last`. A launch and three sums one after the other: 3 to 5 us. (The pass that follows
// can join them itself, in every workgroup: 21 instead of 23.5 us for small images, but 35 instead of 33 at 4 x 128 x 256 x 128 bfloat16 and
// 40 instead of 26 where many groups meet many chunks. Forward in one pass, with x held on the chip between two halves joined by words
// in memory, took 37 + 2 us instead of 41 at 8 x 128 x 256 x 128, and 51 + 2 instead of 47 with a residual.)
constexpr int kMostChunks = 2048;
__global__ void __launch_bounds__(256)
norm_join_kernel(const float2* __restrict__ partial, float* __restrict__ mean, float* __restrict__ rstd, int chunks, float in_chunk,
                 float in_last, float eps) {
    __shared__ float lds[4];
    const int64_t pair = blockIdx.x;
    float2 v[kMostChunks / 256];
    float n[kMostChunks / 256], sum = 0.0f, total = 0.0f;
#pragma unroll
    for (int k = 0; k < kMostChunks / 256; ++k) {
        const int i = threadIdx.x + 256 * k;
        n[k] = i < chunks - 1 ? in_chunk : i == chunks - 1 ? in_last : 0.0f;
        v[k] = i < chunks ? partial[pair * chunks + i] : float2{0.0f, 0.0f};
        total += n[k];
        sum = fmaf(n[k], v[k].x, sum);
    }
    total = sum_of_workgroup(total, lds);
    const float mu = sum_of_workgroup(sum, lds) / total;
    float dev = 0.0f;
#pragma unroll
    for (int k = 0; k < kMostChunks / 256; ++k) {
        const float d = v[k].x - mu;
        dev += n[k] > 0.0f ? fmaf(n[k] * d, d, v[k].y) : 0.0f;
    }
    dev = sum_of_workgroup(dev, lds);
    if (threadIdx.x == 0) {
        mean[pair] = mu;
        rstd[pair] = inverse_deviation(dev / total, eps);
    }
}

template <class T>
struct NormArgs {
    const T *x, *residual;
    const void *weight, *bias;
    T* y;
    bool float_params;
    int groups, per_group;
    float eps;
};

// ---- y from the statistics -------------------------------------------------------------------------
// Bound by memory: x again, the residual, y (stored past the caches: nothing here reads it). 8 x 128 x 256 x 128 bfloat16 (134 MB) 27 us,
// 5.0 TB/s; 2 x 512 x 1024 x 128 float (1074 MB) 191 us, 5.6 TB/s.
template <class T, int ACT>
__global__ void __launch_bounds__(1024)
norm_apply_kernel(NormArgs<T> a, const float* __restrict__ mean, const float* __restrict__ rstd, Lanes L,
                  int64_t chunk_steps, int chunks, int total_workgroups) {
    constexpr int V = Vec<T>::kLen, U = 4;
    typedef typename Vec<T>::Type Packed;
    const int t = threadIdx.x;
    if (t >= L.active) return;
    // last to first: the end of x is what the statistics left in the memory-side cache
    const unsigned id = total_workgroups - 1 - blockIdx.x, chunk = id % static_cast<unsigned>(chunks);
    const int64_t b = id / static_cast<unsigned>(chunks);
    const T *x = a.x + b * L.total, *r = a.residual ? a.residual + b * L.total : nullptr;
    T* y = a.y + b * L.total;
    int64_t off = Item<T>::offset(L, t, 0);
    float mu[V], rs[V], w[V], bias[V];
    Walk at(Item<T>::channel(L, t, 0), a.per_group);
    lane_params<T, V>(a.weight, a.bias, a.float_params, at, L.channels, a.per_group, w, bias);
#pragma unroll
    for (int j = 0; j < V; ++j) {
        const int64_t pair = b * a.groups + at.g;
        mu[j] = mean[pair];
        rs[j] = rstd[pair];
        at.next(L.channels, a.per_group);
    }
    off += chunk * chunk_steps * L.stride;
    const int64_t end = min(L.total, (chunk + 1) * chunk_steps * L.stride);
    for (; off + (U - 1) * L.stride + V <= end; off += U * L.stride) {
        Packed v[U], q[U];
#pragma unroll
        for (int k = 0; k < U; ++k) v[k] = *reinterpret_cast<const Packed*>(x + off + k * L.stride);
        if (r != nullptr) {
#pragma unroll
            for (int k = 0; k < U; ++k) q[k] = *reinterpret_cast<const Packed*>(r + off + k * L.stride);
        } else {
#pragma unroll
            for (int k = 0; k < U; ++k) q[k] = Packed{};
        }
#pragma unroll
        for (int k = 0; k < U; ++k) {
            Packed o;
#pragma unroll
            for (int j = 0; j < V; ++j) {
                o[j] = static_cast<T>(activate<ACT>(form(static_cast<float>(v[k][j]), mu[j], rs[j], w[j], bias[j], static_cast<float>(q[k][j])).z));
            }
            __builtin_nontemporal_store(o, reinterpret_cast<Packed*>(y + off + k * L.stride));
        }
    }
    for (; off < end; off += L.stride) {
        const Packed v = Item<T>::load(x, off, L.total);
        Packed q = {}, o;
        if (r != nullptr) q = Item<T>::load(r, off, L.total);
#pragma unroll
        for (int j = 0; j < V; ++j) {
            o[j] = static_cast<T>(activate<ACT>(form(static_cast<float>(v[j]), mu[j], rs[j], w[j], bias[j], static_cast<float>(q[j])).z));
        }
        Item<T>::store(y, off, L.total, o);
    }
}

// ---- backward, first pass: per-channel sums of dz and dz*u -------------------------------------------
// Bound by reading x, dy and the residual: 4 x 128 x 256 x 128 bfloat16 with a residual (101 MB) 22 us, 4.6 TB/s; 2 x 512 x 1024 x 128 float
// (1074 MB) 174 us, 6.2 TB/s.
template <class T>
struct NormBackwardArgs {
    const T *x, *residual, *dy;
    const void *weight, *bias;
    const float *mean, *rstd;
    T *dx, *dresidual;
    void *dweight, *dbias;
    bool float_params;
    int groups, per_group;
};

template <class T, int ACT>
__global__ void __launch_bounds__(1024)
norm_sums_kernel(NormBackwardArgs<T> a, float* __restrict__ partial, Lanes L, int64_t chunk_steps, int chunks) {
    constexpr int V = Vec<T>::kLen, U = 2;
    typedef typename Vec<T>::Type Packed;
    extern __shared__ float lds[];
    const int t = threadIdx.x;
    const unsigned chunk = blockIdx.x % static_cast<unsigned>(chunks);
    const int64_t b = blockIdx.x / static_cast<unsigned>(chunks);
    float sum[V], dot[V];
#pragma unroll
    for (int j = 0; j < V; ++j) sum[j] = dot[j] = 0.0f;
    if (t < L.active) {
        const T *x = a.x + b * L.total, *dy = a.dy + b * L.total;
        const T* r = ACT != kActNone && a.residual ? a.residual + b * L.total : nullptr;
        int64_t off = Item<T>::offset(L, t, 0);
        float mu[V], rs[V], w[V], bias[V];
        Walk at(Item<T>::channel(L, t, 0), a.per_group);
        lane_params<T, V>(a.weight, a.bias, a.float_params, at, L.channels, a.per_group, w, bias);
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const int64_t pair = b * a.groups + at.g;
            mu[j] = a.mean[pair];
            rs[j] = a.rstd[pair];
            at.next(L.channels, a.per_group);
        }
        off += chunk * chunk_steps * L.stride;
        const int64_t end = min(L.total, (chunk + 1) * chunk_steps * L.stride);
        auto add = [&](const Packed& v, const Packed& g, const Packed& q) {      // (beyond the end g is zero)
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const auto [u, z] = form(static_cast<float>(v[j]), mu[j], rs[j], w[j], bias[j], static_cast<float>(q[j]));
                float dz = static_cast<float>(g[j]);
                if constexpr (ACT != kActNone) dz *= slope<ACT>(z);
                sum[j] += dz;
                dot[j] = fmaf(dz, u, dot[j]);
            }
        };
        for (; off + (U - 1) * L.stride + V <= end; off += U * L.stride) {
            Packed v[U], g[U], q[U];
#pragma unroll
            for (int k = 0; k < U; ++k) {
                v[k] = *reinterpret_cast<const Packed*>(x + off + k * L.stride);
                g[k] = *reinterpret_cast<const Packed*>(dy + off + k * L.stride);
                q[k] = Packed{};
            }
            if (r != nullptr) {
#pragma unroll
                for (int k = 0; k < U; ++k) q[k] = *reinterpret_cast<const Packed*>(r + off + k * L.stride);
            }
#pragma unroll
            for (int k = 0; k < U; ++k) add(v[k], g[k], q[k]);
        }
        for (; off < end; off += L.stride) {
            const Packed v = Item<T>::load(x, off, L.total), g = Item<T>::load(dy, off, L.total);
            Packed q = {};
            if (r != nullptr) q = Item<T>::load(r, off, L.total);
#pragma unroll
            for (int j = 0; j < V; ++j) {
                if (off + j >= L.total) continue;
                const auto [u, z] = form(static_cast<float>(v[j]), mu[j], rs[j], w[j], bias[j], static_cast<float>(q[j]));
                float dz = static_cast<float>(g[j]);
                if constexpr (ACT != kActNone) dz *= slope<ACT>(z);
                sum[j] += dz;
                dot[j] = fmaf(dz, u, dot[j]);
            }
        }
    }
    float* out = partial + blockIdx.x * static_cast<int64_t>(L.channels) * 2;
    join_channels<V>(sum, dot, lds, L, [&](int c, float s, float d) {
        out[2 * c] = s;
        out[2 * c + 1] = d;
    });
}

// The sums of rows [first, last) of [..][channels] pairs, channel c of 16 side by side (threadIdx.x % 16): a workgroup's 64 rows of threads
// walk down, then a tree, always in the same order. The result is in the first row of threads.
__device__ __forceinline__ float2 sum_rows(const float2* __restrict__ rows, int64_t first, int64_t last, int channels, int c, float2 (*part)[17]) {
    const int row = threadIdx.x / 16;
    float2 s = {0.0f, 0.0f};
    if (c < channels) {
#pragma unroll 4
        for (int64_t i = first + row; i < last; i += 64) {
            const float2 v = rows[i * channels + c];
            s.x += v.x;
            s.y += v.y;
        }
    }
    part[row][threadIdx.x % 16] = s;
    __syncthreads();
    for (int half = 32; half > 0; half >>= 1) {
        if (row < half) {
            const float2 v = part[row + half][threadIdx.x % 16];
            s.x += v.x;
            s.y += v.y;
            part[row][threadIdx.x % 16] = s;
        }
        __syncthreads();
    }
    return s;
}

// totals[p][c] = the sums of rows [p * per, (p + 1) * per) of `rows`: of an item's workgroups, or of some of the batch items. 5 us, most of
// it the launch and the chain of sums.
__global__ void __launch_bounds__(1024)
norm_join_sums_kernel(const float2* __restrict__ partial, float2* __restrict__ totals, int channels, int64_t per, int64_t rows, int tiles) {
    __shared__ float2 part[64][17];
    const int64_t p = blockIdx.x / static_cast<unsigned>(tiles);
    const int c = blockIdx.x % static_cast<unsigned>(tiles) * 16 + threadIdx.x % 16;
    const float2 s = sum_rows(partial, p * per, min(rows, (p + 1) * per), channels, c, part);
    if (threadIdx.x < 16 && c < channels) totals[p * channels + c] = s;
}

// s1/m and s2/m of the groups of `slab` channels from c0 on, in LDS, from per-channel totals.
template <class T, class Total>
__device__ __forceinline__ void group_terms(float2* terms, Total total, const NormBackwardArgs<T>& a, int c0, int slab, float inv_m) {
    const int groups = slab / a.per_group, width = lanes_per_group(blockDim.x, groups), t = threadIdx.x;
    for (int g0 = 0; g0 < groups; g0 += blockDim.x / width) {
        const int g = g0 + t / width;
        float s1 = 0.0f, s2 = 0.0f;
        if (g < groups)
            for (int i = t % width; i < a.per_group; i += width) {
                const int c = g * a.per_group + i;
                const float2 v = total(c);
                const float w = a.weight ? load_param<T>(a.weight, a.float_params, c0 + c) : 1.0f;
                s1 = fmaf(w, v.x, s1);
                s2 = fmaf(w, v.y, s2);
            }
        s1 = sum_over(s1, width);
        s2 = sum_over(s2, width);
        if (g < groups && t % width == 0) terms[g] = {s1 * inv_m, s2 * inv_m};
    }
}

// dweight, dbias: the totals of a few batch items, one after the other.
constexpr int64_t kFewItems = 64;
template <class T>
__device__ __forceinline__ void parameter_sums(const NormBackwardArgs<T>& a, const float2* totals, int64_t batch, int channels, int c) {
    float s = 0.0f, d = 0.0f;
    for (int64_t b = 0; b < batch; ++b) {
        const float2 v = totals[b * channels + c];
        s += v.x;
        d += v.y;
    }
    if (a.dbias) store_param<T>(a.dbias, a.float_params, c, s);
    if (a.dweight) store_param<T>(a.dweight, a.float_params, c, d);
}

// The same of many items (or of sums over some of them each).
template <class T>
__global__ void __launch_bounds__(1024) norm_parameter_kernel(const float2* __restrict__ totals, int64_t rows, int channels, void* dweight,
                                                                    void* dbias, bool float_params) {
    __shared__ float2 part[64][17];
    const int c = blockIdx.x * 16 + threadIdx.x % 16;
    const float2 s = sum_rows(totals, 0, rows, channels, c, part);
    if (threadIdx.x >= 16 || c >= channels) return;
    if (dbias) store_param<T>(dbias, float_params, c, s.x);
    if (dweight) store_param<T>(dweight, float_params, c, s.y);
}

// ---- backward, second pass: dx and dresidual -----------------------------------------------------------
// Bound by memory: x, dy and the residual again, dx and dresidual. 4 x 128 x 256 x 128 bfloat16 with a residual (168 MB) 31 us, 5.4 TB/s;
// 2 x 512 x 1024 x 128 float (1611 MB) 311 us, 5.2 TB/s. It walks from the last chunk to the first, as the pass that forms y does.
template <class T, int ACT>
__global__ void __launch_bounds__(1024)
norm_grad_kernel(NormBackwardArgs<T> a, const float2* __restrict__ totals, Lanes L, int64_t chunk_steps, int chunks,
                 int64_t batch, float inv_m, int total_workgroups) {
    constexpr int V = Vec<T>::kLen, U = 2;
    typedef typename Vec<T>::Type Packed;
    extern __shared__ float lds[];
    const int t = threadIdx.x;
    // the first workgroups add up the parameter gradients of a small batch on the side
    if (batch <= kFewItems)
        for (int64_t c = blockIdx.x * static_cast<int64_t>(blockDim.x) + t; c < L.channels; c += static_cast<int64_t>(total_workgroups) * blockDim.x)
            parameter_sums(a, totals, batch, L.channels, static_cast<int>(c));
    if (a.dx == nullptr && a.dresidual == nullptr) return;
    const unsigned id = total_workgroups - 1 - blockIdx.x, chunk = id % static_cast<unsigned>(chunks);   // last to first, as in norm_apply_kernel
    const int64_t b = id / static_cast<unsigned>(chunks);
    float2* terms = reinterpret_cast<float2*>(lds);
    group_terms(terms, [&](int c) { return totals[b * L.channels + c]; }, a, 0, L.channels, inv_m);
    __syncthreads();
    if (t >= L.active) return;
    const T *x = a.x + b * L.total, *dy = a.dy + b * L.total;
    const T* r = ACT != kActNone && a.residual ? a.residual + b * L.total : nullptr;
    T *dx = a.dx ? a.dx + b * L.total : nullptr, *dr = a.dresidual ? a.dresidual + b * L.total : nullptr;
    int64_t off = Item<T>::offset(L, t, 0);
    // dx = rstd w dz + D + E u
    float mu[V], rs[V], w[V], D[V], E[V], bias[V];
    Walk at(Item<T>::channel(L, t, 0), a.per_group);
    lane_params<T, V>(a.weight, a.bias, a.float_params, at, L.channels, a.per_group, w, bias);
#pragma unroll
    for (int j = 0; j < V; ++j) {
        const int g = at.g;
        rs[j] = a.rstd[b * a.groups + g];
        mu[j] = a.mean[b * a.groups + g];
        D[j] = -rs[j] * terms[g].x;
        E[j] = -rs[j] * terms[g].y;
        at.next(L.channels, a.per_group);
    }
    off += chunk * chunk_steps * L.stride;
    const int64_t end = min(L.total, (chunk + 1) * chunk_steps * L.stride);
    auto gradients = [&](const Packed& v, const Packed& g, const Packed& q, Packed& o, Packed& p) {
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const auto [u, z] = form(static_cast<float>(v[j]), mu[j], rs[j], w[j], bias[j], static_cast<float>(q[j]));
            float dz = static_cast<float>(g[j]);
            if constexpr (ACT != kActNone) dz *= slope<ACT>(z);
            o[j] = static_cast<T>(fmaf(rs[j] * w[j], dz, fmaf(E[j], u, D[j])));
            p[j] = static_cast<T>(dz);
        }
    };
    for (; off + (U - 1) * L.stride + V <= end; off += U * L.stride) {
        Packed v[U], g[U], q[U];
#pragma unroll
        for (int k = 0; k < U; ++k) {
            v[k] = *reinterpret_cast<const Packed*>(x + off + k * L.stride);
            g[k] = *reinterpret_cast<const Packed*>(dy + off + k * L.stride);
            q[k] = Packed{};
        }
        if (r != nullptr) {
#pragma unroll
            for (int k = 0; k < U; ++k) q[k] = *reinterpret_cast<const Packed*>(r + off + k * L.stride);
        }
#pragma unroll
        for (int k = 0; k < U; ++k) {
            Packed o, p;
            gradients(v[k], g[k], q[k], o, p);
            if (dx != nullptr) __builtin_nontemporal_store(o, reinterpret_cast<Packed*>(dx + off + k * L.stride));
            if (dr != nullptr) __builtin_nontemporal_store(p, reinterpret_cast<Packed*>(dr + off + k * L.stride));
        }
    }
    for (; off < end; off += L.stride) {
        const Packed v = Item<T>::load(x, off, L.total), g = Item<T>::load(dy, off, L.total);
        Packed q = {}, o, p;
        if (r != nullptr) q = Item<T>::load(r, off, L.total);
        gradients(v, g, q, o, p);
        if (dx != nullptr) Item<T>::store(dx, off, L.total, o);
        if (dr != nullptr) Item<T>::store(dr, off, L.total, p);
    }
}

// ---- items that one workgroup's registers hold: one launch -----------------------------------------------
// One compute unit does all of an item's work, so what counts is instructions: with WHOLE (items of whole vectors) no element
// is looked at alone, offsets are 32 bits wide, and a group's quotients and root are taken once. One 28 x 28 x 40 bfloat16 item in 8 groups 10.4
// us, eight of 28 x 28 x 64 16.6 us; x is 63 KB, so neither bytes nor operations matter. (16 vectors per lane: 27 us, the registers spill.)
template <class T, int ACT, int N, bool WHOLE>
__global__ void __launch_bounds__(1024)
norm_small_kernel(NormArgs<T> a, float* __restrict__ mean_out, float* __restrict__ rstd_out, Lanes L, int slabs, float m) {
    constexpr int V = Vec<T>::kLen;
    typedef typename Vec<T>::Type Packed;
    extern __shared__ float lds[];
    const int t = threadIdx.x, c0 = blockIdx.x % static_cast<unsigned>(slabs) * L.slab, total = static_cast<int>(L.total), stride = static_cast<int>(L.stride);
    const int64_t b = blockIdx.x / static_cast<unsigned>(slabs);
    const T *x = a.x + b * L.total, *r = a.residual ? a.residual + b * L.total : nullptr;
    const bool live = t < L.active;
    const int off = live ? static_cast<int>(Item<T>::offset(L, t, c0)) : total;
    // (requested without a branch, so that all are on their way at once; an item has at least one vector)
    Packed v[N];
#pragma unroll
    for (int k = 0; k < N; ++k) v[k] = *reinterpret_cast<const Packed*>(x + (off + k * stride + V <= total ? off + k * stride : 0));
#pragma unroll
    for (int k = 0; k < N; ++k)
        if (off + k * stride + V > total) v[k] = WHOLE ? Packed{} : Item<T>::load(x, off + k * stride, total);
    // the mean, then the deviations from it: both from registers
    const int groups = L.slab / a.per_group, g0 = c0 / a.per_group;
    float *means = lds + kept_words(L.active, V), *rstds = means + groups;
    float v1[V], mean[V], rs[V], w[V], bias[V];
    Walk walk(Item<T>::channel(L, t, c0), a.per_group);
    lane_params<T, V>(a.weight, a.bias, a.float_params, walk, L.channels, a.per_group, w, bias);
#pragma unroll
    for (int j = 0; j < V; ++j) {
        v1[j] = 0.0f;
#pragma unroll
        for (int k = 0; k < N; ++k) v1[j] += static_cast<float>(v[k][j]);    // (zeros beyond the end)
    }
    join_groups<V>(v1, lds, means, L, a.per_group, [&](float sum) { return sum / m; });   // (a product with 1/m would be off where all values are the same)
    int group[V];
#pragma unroll
    for (int j = 0; j < V; ++j) {
        group[j] = live ? walk.g - g0 : 0;
        mean[j] = means[group[j]];
        v1[j] = 0.0f;
        walk.next(L.channels, a.per_group);
    }
#pragma unroll
    for (int k = 0; k < N; ++k) {
        if (WHOLE && off + k * stride >= total) continue;
#pragma unroll
        for (int j = 0; j < V; ++j) {
            if (!WHOLE && off + k * stride + j >= total) continue;
            const float d = static_cast<float>(v[k][j]) - mean[j];
            v1[j] = fmaf(d, d, v1[j]);
        }
    }
    join_groups<V>(v1, lds, rstds, L, a.per_group, [&](float sum) { return inverse_deviation(sum / m, a.eps); });
    if (mean_out != nullptr)
        for (int g = t; g < groups; g += blockDim.x) {
            mean_out[b * a.groups + g0 + g] = means[g];
            rstd_out[b * a.groups + g0 + g] = rstds[g];
        }
#pragma unroll
    for (int j = 0; j < V; ++j) rs[j] = rstds[group[j]];
    T* y = a.y + b * L.total;
#pragma unroll
    for (int k = 0; k < N; ++k) {
        const int at = off + k * stride;
        if (at >= total) continue;
        Packed q = {}, o;
        if (r != nullptr) q = WHOLE ? *reinterpret_cast<const Packed*>(r + at) : Item<T>::load(r, at, total);
#pragma unroll
        for (int j = 0; j < V; ++j)
            o[j] = static_cast<T>(activate<ACT>(form(static_cast<float>(v[k][j]), mean[j], rs[j], w[j], bias[j], static_cast<float>(q[j])).z));
        if (WHOLE) *reinterpret_cast<Packed*>(y + at) = o;
        else Item<T>::store(y, at, total, o);
    }
}

// The backward reads its tensors twice, the second time from the L2: x and dy would not fit a lane's registers beside the
// per-channel values of its elements. Bound by the chain load, sums, join, load: one 28 x 28 x 40 bfloat16 item 20 us, eight of 28 x 28 x
// 64 29 us.
template <class T, int ACT>
__global__ void __launch_bounds__(1024)
norm_small_grad_kernel(NormBackwardArgs<T> a, float2* __restrict__ totals, Lanes L, int slabs, float inv_m, bool only_item) {
    constexpr int V = Vec<T>::kLen;
    typedef typename Vec<T>::Type Packed;
    extern __shared__ float lds[];
    const int t = threadIdx.x, c0 = blockIdx.x % slabs * L.slab, g0 = c0 / a.per_group;
    const int64_t b = blockIdx.x / slabs;
    const T *x = a.x + b * L.total, *dy = a.dy + b * L.total;
    const T* r = ACT != kActNone && a.residual ? a.residual + b * L.total : nullptr;
    const int64_t off = Item<T>::offset(L, t, c0);
    const int64_t end = t < L.active ? L.total : 0;
    float mu[V], rs[V], w[V], bias[V], sum[V], dot[V];
    Walk walk(Item<T>::channel(L, t, c0), a.per_group);
    lane_params<T, V>(a.weight, a.bias, a.float_params, walk, L.channels, a.per_group, w, bias);
#pragma unroll
    for (int j = 0; j < V; ++j) {
        const int64_t pair = b * a.groups + walk.g;
        sum[j] = dot[j] = 0.0f;
        mu[j] = a.mean[pair];
        rs[j] = a.rstd[pair];
        walk.next(L.channels, a.per_group);
    }
    T* dr = a.dresidual ? a.dresidual + b * L.total : nullptr;
#pragma unroll 1
    for (int64_t at = off; at < end; at += L.stride) {
        const Packed v = Item<T>::load(x, at, L.total), g = Item<T>::load(dy, at, L.total);
        Packed q = {}, p;
        if (r != nullptr) q = Item<T>::load(r, at, L.total);
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const auto [u, z] = form(static_cast<float>(v[j]), mu[j], rs[j], w[j], bias[j], static_cast<float>(q[j]));
            float dz = static_cast<float>(g[j]);
            if constexpr (ACT != kActNone) dz *= slope<ACT>(z);
            p[j] = static_cast<T>(dz);
            if (at + j < L.total) {
                sum[j] += dz;
                dot[j] = fmaf(dz, u, dot[j]);
            }
        }
        if (dr != nullptr) Item<T>::store(dr, at, L.total, p);
    }
    float2* chan = reinterpret_cast<float2*>(lds + 2 * kept_words(L.active, V));
    float2* terms = chan + L.slab;
    join_channels<V>(sum, dot, lds, L, [&](int ch, float s, float d) {
        chan[ch] = {s, d};
        totals[b * L.channels + c0 + ch] = {s, d};
        if (only_item) {
            if (a.dbias) store_param<T>(a.dbias, a.float_params, c0 + ch, s);
            if (a.dweight) store_param<T>(a.dweight, a.float_params, c0 + ch, d);
        }
    });
    __syncthreads();
    group_terms(terms, [&](int ch) { return chan[ch]; }, a, c0, L.slab, inv_m);
    __syncthreads();
    if (a.dx == nullptr || end == 0) return;
    T* dx = a.dx + b * L.total;
    float t1[V], t2[V];
    Walk again(Item<T>::channel(L, t, c0), a.per_group);
#pragma unroll
    for (int j = 0; j < V; ++j) {
        const float2 s = terms[again.g - g0];
        t1[j] = s.x;
        t2[j] = s.y;
        again.next(L.channels, a.per_group);
    }
#pragma unroll 1
    for (int64_t at = off; at < end; at += L.stride) {
        const Packed v = Item<T>::load(x, at, L.total), g = Item<T>::load(dy, at, L.total);
        Packed q = {}, o;
        if (r != nullptr) q = Item<T>::load(r, at, L.total);
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const auto [u, z] = form(static_cast<float>(v[j]), mu[j], rs[j], w[j], bias[j], static_cast<float>(q[j]));
            float dz = static_cast<float>(g[j]);
            if constexpr (ACT != kActNone) dz *= slope<ACT>(z);
            o[j] = static_cast<T>(rs[j] * (fmaf(w[j], dz, -t1[j]) - u * t2[j]));
        }
        Item<T>::store(dx, at, L.total, o);
    }
}

// ---- channels that no workgroup's lanes can repeat over --------------------------------------------------------
// (odd numbers of them above 1024, multiples of 8 above 8192 in 16-bit types and of 4 above 4096 in float, the like between), and items of fewer
// elements than a vector. A workgroup takes a chunk of whole pixels of one (batch item, group), element by element. Bound by the index arithmetic
// and loads of two or four bytes: 2 x 64 x 64 x 1031 float16 in one group (17 MB) statistics 16 us, y 17, input gradient 21; the channel sums of the
// backward, which walk down single channels, 88 us.
struct AnyChunk { int64_t base; int g; unsigned elements; };     // of the group: its first element, and how many there are
__device__ __forceinline__ AnyChunk any_chunk(int64_t pixels, int channels, int groups, int per_group, int64_t chunk_pixels, int chunks) {
    const unsigned chunk = blockIdx.x % static_cast<unsigned>(chunks), pair = blockIdx.x / static_cast<unsigned>(chunks);
    const int64_t b = pair / static_cast<unsigned>(groups), first = chunk * chunk_pixels;
    const int g = static_cast<int>(pair % static_cast<unsigned>(groups));
    return {(b * pixels + first) * channels + static_cast<int64_t>(g) * per_group, g, static_cast<unsigned>(min(chunk_pixels, pixels - first)) * per_group};
}
// f(place in memory, channel) of this thread's elements of the chunk
template <class F>
__device__ __forceinline__ void any_elements(const AnyChunk& c, int channels, int per_group, F f) {
    const unsigned width = static_cast<unsigned>(per_group);
    for (unsigned i = threadIdx.x; i < c.elements; i += 256) {
        const unsigned pixel = i / width, channel = i - pixel * width;
        f(c.base + static_cast<int64_t>(pixel) * channels + channel, static_cast<int>(c.g * width + channel));
    }
}

__device__ __forceinline__ float workgroup_sum(float v, float* lds) {
    v = sum_over(v, 64);
    __syncthreads();
    if (threadIdx.x % 64 == 0) lds[threadIdx.x / 64] = v;
    __syncthreads();
    v = 0.0f;
    for (unsigned i = 0; i < blockDim.x / 64; ++i) v += lds[i];
    return v;
}

template <class T>
__global__ void __launch_bounds__(256)
norm_any_statistics_kernel(const T* __restrict__ x, float2* __restrict__ partial, int64_t pixels, int channels, int groups, int per_group,
                           int64_t chunk_pixels, int chunks) {
    __shared__ float lds[4];
    const AnyChunk chunk = any_chunk(pixels, channels, groups, per_group, chunk_pixels, chunks);
    float s = 0.0f;
    any_elements(chunk, channels, per_group, [&](int64_t at, int) { s += static_cast<float>(x[at]); });
    const float mu = workgroup_sum(s, lds) / static_cast<float>(chunk.elements);
    s = 0.0f;
    any_elements(chunk, channels, per_group, [&](int64_t at, int) {
        const float d = static_cast<float>(x[at]) - mu;
        s = fmaf(d, d, s);
    });
    s = workgroup_sum(s, lds);
    if (threadIdx.x == 0) partial[blockIdx.x] = {mu, s};
}

template <class T, int ACT>
__global__ void __launch_bounds__(256)
norm_any_apply_kernel(NormArgs<T> a, const float* __restrict__ mean, const float* __restrict__ rstd, int64_t pixels, int channels, int64_t chunk_pixels,
                      int chunks) {
    const AnyChunk chunk = any_chunk(pixels, channels, a.groups, a.per_group, chunk_pixels, chunks);
    const unsigned pair = blockIdx.x / static_cast<unsigned>(chunks);
    const float mu = mean[pair], rs = rstd[pair];
    any_elements(chunk, channels, a.per_group, [&](int64_t at, int c) {
        const float w = a.weight ? load_param<T>(a.weight, a.float_params, c) : 1.0f, shift = a.bias ? load_param<T>(a.bias, a.float_params, c) : 0.0f;
        a.y[at] = static_cast<T>(activate<ACT>(form(static_cast<float>(a.x[at]), mu, rs, w, shift, a.residual ? static_cast<float>(a.residual[at]) : 0.0f).z));
    });
}

struct AnyElement { float u, w, dz; };
template <class T, int ACT>
__device__ __forceinline__ AnyElement any_element(const NormBackwardArgs<T>& a, int64_t at, int c, float mu, float rs) {
    const float w = a.weight ? load_param<T>(a.weight, a.float_params, c) : 1.0f, shift = a.bias ? load_param<T>(a.bias, a.float_params, c) : 0.0f;
    const auto [u, z] = form(static_cast<float>(a.x[at]), mu, rs, w, shift, ACT != kActNone && a.residual ? static_cast<float>(a.residual[at]) : 0.0f);
    return {u, w, static_cast<float>(a.dy[at]) * slope<ACT>(z)};
}

// One workgroup per (batch item, channel).
template <class T, int ACT>
__global__ void __launch_bounds__(256)
norm_any_sums_kernel(NormBackwardArgs<T> a, float2* __restrict__ totals, int64_t pixels, int channels) {
    __shared__ float lds[4];
    const int64_t b = blockIdx.x / channels;
    const int c = blockIdx.x % channels;
    const int64_t pair = b * a.groups + c / a.per_group;
    const float mu = a.mean[pair], rs = a.rstd[pair];
    float s = 0.0f, d = 0.0f;
    for (int64_t i = threadIdx.x; i < pixels; i += 256) {
        const int64_t at = (b * pixels + i) * channels + c;
        const AnyElement e = any_element<T, ACT>(a, at, c, mu, rs);
        s += e.dz;
        d = fmaf(e.dz, e.u, d);
        if (a.dresidual) a.dresidual[at] = static_cast<T>(e.dz);
    }
    s = workgroup_sum(s, lds);
    d = workgroup_sum(d, lds);
    if (threadIdx.x == 0) totals[blockIdx.x] = {s, d};
}

template <class T, int ACT>
__global__ void __launch_bounds__(256)
norm_any_grad_kernel(NormBackwardArgs<T> a, const float2* __restrict__ totals, int64_t pixels, int channels, int64_t chunk_pixels, int chunks, float inv_m) {
    __shared__ float lds[4];
    const AnyChunk chunk = any_chunk(pixels, channels, a.groups, a.per_group, chunk_pixels, chunks);
    const unsigned pair = blockIdx.x / static_cast<unsigned>(chunks);
    const float2* of_group = totals + static_cast<int64_t>(pair) * a.per_group;             // (batch item by batch item, group by group)
    float s1 = 0.0f, s2 = 0.0f;
    for (int i = threadIdx.x; i < a.per_group; i += 256) {
        const float w = a.weight ? load_param<T>(a.weight, a.float_params, chunk.g * a.per_group + i) : 1.0f;
        s1 = fmaf(w, of_group[i].x, s1);
        s2 = fmaf(w, of_group[i].y, s2);
    }
    s1 = workgroup_sum(s1, lds) * inv_m;
    s2 = workgroup_sum(s2, lds) * inv_m;
    const float mu = a.mean[pair], rs = a.rstd[pair];
    any_elements(chunk, channels, a.per_group, [&](int64_t at, int c) {
        const AnyElement e = any_element<T, ACT>(a, at, c, mu, rs);
        a.dx[at] = static_cast<T>(rs * (fmaf(e.w, e.dz, -s1) - e.u * s2));
    });
}

// ---- plans -------------------------------------------------------------------------------------------------
int gcd(int a, int b) { while (b) { const int r = a % b; a = b; b = r; } return a; }

struct NormPlan {
    bool any;                  // the element-by-element kernels
    int small;                 // > 0: one launch, so many vectors per lane
    int threads, slabs, chunks;
    int64_t chunk_steps;
    int pieces;                // the same for the passes that write: workgroups per item, steps of each
    int64_t piece_steps;
    Lanes L;
};

constexpr int kPieces = 4;             // of a chunk in the passes that write, while they have 16 steps each (537 MB of float32: 201 us with 1024 workgroups, 190 with 4096)
constexpr int kMostVectors = 8;        // of a lane of the one-launch kernels: what its registers hold of x

// per_lane: vectors that a lane of a one-launch kernel should rather take than leave to more lanes. Forward: 8, all on their way at
// once (one 28 x 28 x 40 item: 1024 lanes with 4 each take 11.8 us, half of it the instructions that every wave repeats). Backward: 1, its
// loop waits for every vector.
NormPlan plan_norm(int64_t batch, int64_t pixels, int channels, int groups, int V, int per_lane) {
    NormPlan p = {};
    Lanes& L = p.L;
    L.channels = L.slab = channels;
    L.total = pixels * channels;
    const int per_group = channels / groups;
    L.phase = channels / gcd(channels, V);
    p.slabs = 1;
    if (L.phase > 1024 || L.total < V) {
        p.any = true;                                      // chunks of whole pixels of a group, chunk_steps of them
        const int64_t want = std::min<int64_t>(kMostChunks, std::max<int64_t>(1, 2048 / std::max<int64_t>(1, batch * groups)));
        p.chunk_steps = std::max<int64_t>((pixels + want - 1) / want, (2047 + per_group) / per_group);
        p.chunks = static_cast<int>((pixels + p.chunk_steps - 1) / p.chunk_steps);
        return p;
    }
    // one launch where a workgroup of at most 1024 lanes can hold an item, or whole groups of it that are at least 64 bytes
    // wide (narrower pieces of a pixel's channels would fetch the same cache lines from several workgroups)
    for (int groups_in_slab = groups; groups_in_slab >= 1; --groups_in_slab) {
        if (groups % groups_in_slab) continue;
        const int slab = groups_in_slab * per_group;
        if (groups_in_slab < groups && (channels % V || slab % V || slab < 4 * V)) continue;
        const int phase = slab == channels ? L.phase : slab / V;
        const int64_t vectors = slab == channels ? (L.total + V - 1) / V : pixels * phase;
        if (phase > 1024 || vectors > static_cast<int64_t>(1024 / phase * phase) * kMostVectors || L.total > 0x7fffffff) continue;
        int threads = 64;
        while (threads < 1024 && (threads < phase || vectors > static_cast<int64_t>(threads / phase * phase) * per_lane)) threads *= 2;
        const int active = threads / phase * phase;
        if (static_cast<size_t>(2) * kept_words(active, V) * 4 + static_cast<size_t>(slab + groups_in_slab) * 8 > kMaxDynamicLds) continue;   // (the backward's)
        p.threads = threads;
        p.slabs = groups / groups_in_slab;
        L.slab = slab;
        L.phase = phase;
        L.active = threads / phase * phase;
        L.stride = slab == channels ? static_cast<int64_t>(L.active) * V : static_cast<int64_t>(L.active / phase) * channels;
        int n = 1;
        while (static_cast<int64_t>(L.active) * n < vectors) n *= 2;
        p.small = n;
        return p;
    }
    p.threads = 256;
    while (p.threads < L.phase) p.threads *= 2;
    if (p.threads < 1024 && p.threads / L.phase * L.phase * 4 < p.threads * 3) p.threads *= 2;   // fewer idle lanes
    L.active = p.threads / L.phase * L.phase;
    L.stride = static_cast<int64_t>(L.active) * V;
    const int64_t steps = (L.total + L.stride - 1) / L.stride;
    const int64_t want = std::max<int64_t>(1, (512 * 256 / p.threads + batch - 1) / batch);    // workgroups per item: two waves per SIMD in all. What a
    // workgroup does before and after its rows costs as much as 4 to 8 of its steps (33.5 M bfloat16 elements: statistics 20 us with 2048 workgroups, 17
    // with 1024, 15 with 512; y 30, 26 and 27, and 46 with 4096)
    p.chunk_steps = (steps + want - 1) / want;
    if (p.chunk_steps < kUnroll) p.chunk_steps = kUnroll;
    p.chunks = static_cast<int>((steps + p.chunk_steps - 1) / p.chunk_steps);
    p.piece_steps = std::min(p.chunk_steps, std::max<int64_t>((steps + kPieces * want - 1) / (kPieces * want), 16));
    p.pieces = static_cast<int>((steps + p.piece_steps - 1) / p.piece_steps);
    return p;
}

// How the parameters' gradients are summed over the batch: in pieces of `per` items, whose sums are added by another launch. A thread adds 64
// to 512 values one after the other up to half a billion items, and a tree joins the threads' sums. (One chain over all items loses digits
// with their number: 100000 times the same gradient 1.1 was off by 9e-4 of the sum.) One piece up to 4096 items.
struct ItemsPlan { int64_t pieces, per; };
ItemsPlan plan_items(int64_t batch) {
    const int64_t per = std::max<int64_t>(4096, (batch + 16383) / 16384);
    return {(batch + per - 1) / per, per};
}

template <int ACT> struct ActTag { static constexpr int value = ACT; };
template <class F>
hipError_t with_activation(int act, F f) {
    switch (act) {
        case kActRelu: return f(ActTag<kActRelu>());
        case kActSilu: return f(ActTag<kActSilu>());
        case kActGelu: return f(ActTag<kActGelu>());
        default: return f(ActTag<kActNone>());
    }
}
template <int N> struct CountTag { static constexpr int value = N; };
template <class F>
hipError_t with_count(int n, F f) {
    switch (n) {
        case 1: return f(CountTag<1>());
        case 2: return f(CountTag<2>());
        case 4: return f(CountTag<4>());
        default: return f(CountTag<8>());
    }
}

// Items that one launch takes: a grid has fewer than 2^32 threads. (What a workgroup does depends on the plan for all items, not on the launch.)
int64_t items_per_launch(const NormPlan& p, int64_t channels, int64_t groups) {
    const int64_t widest = p.any     ? std::max(channels, groups * p.chunks) * 256
                           : p.small ? static_cast<int64_t>(p.slabs) * p.threads
                                     : std::max({static_cast<int64_t>(std::max(p.chunks, p.pieces)) * p.threads, groups * 256, (channels + 15) / 16 * 1024});
    return std::max<int64_t>(1, kMostThreads / widest);
}
template <class T, class P>
P* from_item(P* p, int64_t elements) { return p == nullptr ? nullptr : reinterpret_cast<P*>(reinterpret_cast<uintptr_t>(p) + elements * sizeof(T)); }

template <class T>
hipError_t forward_items(const NormCall& n, const NormPlan& p, void* workspace, hipStream_t stream) {
    constexpr int V = Vec<T>::kLen;
    NormArgs<T> a;
    a.x = static_cast<const T*>(n.x);
    a.residual = static_cast<const T*>(n.residual);
    a.weight = n.weight;
    a.bias = n.bias;
    a.y = static_cast<T*>(n.y);
    a.float_params = n.float_params;
    a.groups = n.groups;
    a.per_group = n.channels / n.groups;
    a.eps = n.eps;
    const Lanes L = p.L;
    if (p.small)
        return with_activation(n.activation, [&](auto act) {
            const size_t lds = static_cast<size_t>(kept_words(L.active, V)) * 4 + static_cast<size_t>(L.slab / a.per_group) * 8;
            const dim3 grid(static_cast<unsigned>(n.batch * p.slabs));
            const float m = static_cast<float>(n.pixels * a.per_group);
            if (L.total % V != 0) {
                BOXCONV_LAUNCH("norm_small", (norm_small_kernel<T, decltype(act)::value, kMostVectors, false>), grid, dim3(p.threads), lds, stream, a, n.mean,
                               n.rstd, L, p.slabs, m);
                return hipGetLastError();
            }
            return with_count(p.small, [&](auto count) {
                BOXCONV_LAUNCH("norm_small", (norm_small_kernel<T, decltype(act)::value, decltype(count)::value, true>), grid, dim3(p.threads), lds, stream, a,
                               n.mean, n.rstd, L, p.slabs, m);
                return hipGetLastError();
            });
        });
    float2* partial = static_cast<float2*>(workspace);
    float *mean = n.mean, *rstd = n.rstd;
    const int64_t pairs = n.batch * n.groups;
    if (mean == nullptr) {
        mean = reinterpret_cast<float*>(partial + n.batch * p.chunks * n.groups);
        rstd = mean + pairs;
    }
    const int64_t chunk_pixels = p.any ? p.chunk_steps : p.chunk_steps * L.stride / L.channels, last_pixels = n.pixels - (p.chunks - 1) * chunk_pixels;
    const dim3 any_grid(static_cast<unsigned>(pairs * p.chunks));
    const int workgroups = static_cast<int>(n.batch * p.pieces);
    if (p.any)
        BOXCONV_LAUNCH("norm_any_statistics", (norm_any_statistics_kernel<T>), any_grid, dim3(256), 0, stream, a.x, partial, n.pixels, n.channels, a.groups,
                       a.per_group, chunk_pixels, p.chunks);
    else
        BOXCONV_LAUNCH("norm_statistics", (norm_statistics_kernel<T>), dim3(static_cast<unsigned>(n.batch * p.chunks)), dim3(p.threads),
                       static_cast<size_t>(3) * kept_words(L.active, V) * 4, stream, a.x, partial, L, p.chunk_steps, p.chunks, a.groups, a.per_group);
    BOXCONV_LAUNCH("norm_join", norm_join_kernel, dim3(static_cast<unsigned>(pairs)), dim3(256), 0, stream, partial, mean, rstd, p.chunks,
                   static_cast<float>(chunk_pixels * a.per_group), static_cast<float>(last_pixels * a.per_group), a.eps);
    return with_activation(n.activation, [&](auto act) {
        if (p.any)
            BOXCONV_LAUNCH("norm_any_apply", (norm_any_apply_kernel<T, decltype(act)::value>), any_grid, dim3(256), 0, stream, a, mean, rstd, n.pixels,
                           n.channels, chunk_pixels, p.chunks);
        else
            BOXCONV_LAUNCH("norm_apply", (norm_apply_kernel<T, decltype(act)::value>), dim3(workgroups), dim3(p.threads), 0, stream, a, mean, rstd, L,
                           p.piece_steps, p.pieces, workgroups);
        return hipGetLastError();
    });
}

// dweight and dbias from the items' totals; `spare`: room for the sums of several pieces.
template <class T>
void parameter_gradients(const NormGradCall& n, const float2* totals, float2* spare, int64_t batch, hipStream_t stream) {
    if (n.dweight == nullptr && n.dbias == nullptr) return;
    const ItemsPlan p = plan_items(batch);
    const int tiles = (n.channels + 15) / 16;
    if (p.pieces > 1)
        BOXCONV_LAUNCH("norm_join_sums", norm_join_sums_kernel, dim3(static_cast<unsigned>(p.pieces * tiles)), dim3(1024), 0, stream, totals, spare, n.channels,
                       p.per, batch, tiles);
    BOXCONV_LAUNCH("norm_parameter", (norm_parameter_kernel<T>), dim3(static_cast<unsigned>(tiles)), dim3(1024), 0, stream, p.pieces > 1 ? spare : totals,
                   p.pieces > 1 ? p.pieces : batch, n.channels, n.dweight, n.dbias, n.float_params);
}

template <class T>
hipError_t forward(NormCall n, void* workspace, hipStream_t stream) {
    const NormPlan p = plan_norm(n.batch, n.pixels, n.channels, n.groups, Vec<T>::kLen, kMostVectors);
    const int64_t most = items_per_launch(p, n.channels, n.groups);
    for (int64_t left = n.batch; left > 0; left -= n.batch) {
        n.batch = std::min(left, most);
        if (const hipError_t e = forward_items<T>(n, p, workspace, stream); e != hipSuccess) return e;
        const int64_t elements = n.batch * p.L.total, pairs = n.batch * n.groups;
        n.x = from_item<T>(n.x, elements);
        n.residual = from_item<T>(n.residual, elements);
        n.y = from_item<T>(n.y, elements);
        n.mean = from_item<float>(n.mean, pairs);
        n.rstd = from_item<float>(n.rstd, pairs);
    }
    return hipSuccess;
}

// dx, dresidual and the items' totals; of `all_items` up to kFewItems dweight and dbias too (then this is all of them).
template <class T>
hipError_t backward_items(const NormGradCall& n, const NormPlan& p, int64_t all_items, float2* totals, float2* partial, hipStream_t stream) {
    constexpr int V = Vec<T>::kLen;
    NormBackwardArgs<T> a;
    a.x = static_cast<const T*>(n.x);
    a.residual = static_cast<const T*>(n.residual);
    a.dy = static_cast<const T*>(n.dy);
    a.weight = n.weight;
    a.bias = n.bias;
    a.mean = n.mean;
    a.rstd = n.rstd;
    a.dx = static_cast<T*>(n.dx);
    a.dresidual = static_cast<T*>(n.dresidual);
    a.dweight = n.dweight;
    a.dbias = n.dbias;
    a.float_params = n.float_params;
    a.groups = n.groups;
    a.per_group = n.channels / n.groups;
    const Lanes L = p.L;
    const float inv_m = static_cast<float>(1.0 / (static_cast<double>(n.pixels) * a.per_group));
    if (p.any)
        return with_activation(n.activation, [&](auto act) {
            BOXCONV_LAUNCH("norm_any_sums", (norm_any_sums_kernel<T, decltype(act)::value>), dim3(static_cast<unsigned>(n.batch * n.channels)), dim3(256), 0,
                           stream, a, totals, n.pixels, n.channels);
            if (a.dx != nullptr)
                BOXCONV_LAUNCH("norm_any_grad", (norm_any_grad_kernel<T, decltype(act)::value>), dim3(static_cast<unsigned>(n.batch * n.groups * p.chunks)),
                               dim3(256), 0, stream, a, totals, n.pixels, n.channels, p.chunk_steps, p.chunks, inv_m);
            return hipGetLastError();
        });
    if (p.small)
        return with_activation(n.activation, [&](auto act) {
            const size_t lds = static_cast<size_t>(2) * kept_words(L.active, V) * 4 + static_cast<size_t>(L.slab) * 8 + static_cast<size_t>(L.slab / a.per_group) * 8;
            BOXCONV_LAUNCH("norm_small_grad", (norm_small_grad_kernel<T, decltype(act)::value>), dim3(static_cast<unsigned>(n.batch * p.slabs)),
                           dim3(p.threads), lds, stream, a, totals, L, p.slabs, inv_m, all_items == 1);
            return hipGetLastError();
        });
    const int workgroups = static_cast<int>(n.batch * p.pieces), tiles = (n.channels + 15) / 16;
    return with_activation(n.activation, [&](auto act) {
        BOXCONV_LAUNCH("norm_sums", (norm_sums_kernel<T, decltype(act)::value>), dim3(static_cast<unsigned>(n.batch * p.chunks)), dim3(p.threads), static_cast<size_t>(2) * kept_words(L.active, V) * 4,
                       stream, a, reinterpret_cast<float*>(partial), L, p.chunk_steps, p.chunks);
        BOXCONV_LAUNCH("norm_join_sums", norm_join_sums_kernel, dim3(static_cast<unsigned>(n.batch * tiles)), dim3(1024), 0, stream, partial, totals,
                       n.channels, p.chunks, n.batch * p.chunks, tiles);
        BOXCONV_LAUNCH("norm_grad", (norm_grad_kernel<T, decltype(act)::value>), dim3(workgroups), dim3(p.threads), static_cast<size_t>(a.groups) * 8, stream,
                       a, totals, L, p.piece_steps, p.pieces, all_items, inv_m, workgroups);
        return hipGetLastError();
    });
}

template <class T>
hipError_t backward(NormGradCall n, void* workspace, hipStream_t stream) {
    const NormPlan p = plan_norm(n.batch, n.pixels, n.channels, n.groups, Vec<T>::kLen, 1);
    const int64_t batch = n.batch, most = items_per_launch(p, n.channels, n.groups);
    float2* totals = static_cast<float2*>(workspace);
    float2 *partial = totals + batch * n.channels, *spare = partial + (p.any || p.small ? 0 : batch * p.chunks * n.channels);
    float2* of_items = totals;
    for (int64_t left = batch; left > 0; left -= n.batch) {
        n.batch = std::min(left, most);
        if (const hipError_t e = backward_items<T>(n, p, batch, of_items, partial, stream); e != hipSuccess) return e;
        const int64_t elements = n.batch * p.L.total, pairs = n.batch * n.groups;
        n.x = from_item<T>(n.x, elements);
        n.residual = from_item<T>(n.residual, elements);
        n.dy = from_item<T>(n.dy, elements);
        n.dx = from_item<T>(n.dx, elements);
        n.dresidual = from_item<T>(n.dresidual, elements);
        n.mean = from_item<float>(n.mean, pairs);
        n.rstd = from_item<float>(n.rstd, pairs);
        of_items += n.batch * n.channels;
    }
    const bool done = p.small ? batch == 1 : !p.any && batch <= kFewItems;     // by the launches above
    if (!done) parameter_gradients<T>(n, totals, spare, batch, stream);
    return hipGetLastError();
}

}  // namespace

size_t norm_workspace_bytes(int64_t batch, int64_t pixels, int channels, int groups, int dtype, bool backward_pass) {
    const NormPlan p = plan_norm(batch, pixels, channels, groups, dtype == kF32 ? 4 : 8, backward_pass ? 1 : kMostVectors);
    const int64_t chunks = p.small || (p.any && backward_pass) ? 0 : batch * p.chunks;
    const ItemsPlan items = plan_items(batch);
    if (backward_pass) return static_cast<size_t>(batch + chunks + (items.pieces > 1 ? items.pieces : 0)) * channels * 8;
    return chunks ? static_cast<size_t>(chunks * groups * 2 + batch * groups * 2) * 4 : 0;
}

hipError_t norm_forward_launch(const NormCall& n, void* workspace, hipStream_t stream) {
    if (n.dtype == kF32) return forward<float>(n, workspace, stream);
    if (n.dtype == kF16) return forward<_Float16>(n, workspace, stream);
    return forward<__bf16>(n, workspace, stream);
}

hipError_t norm_backward_launch(const NormGradCall& n, void* workspace, hipStream_t stream) {
    if (n.dtype == kF32) return backward<float>(n, workspace, stream);
    if (n.dtype == kF16) return backward<_Float16>(n, workspace, stream);
    return backward<__bf16>(n, workspace, stream);
}

}  // namespace boxconv
