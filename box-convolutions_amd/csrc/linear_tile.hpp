// The tile that the pointwise products share: out[m][n] = sum over k of A(m, k) * B(n, k) by matrix instructions, with both
// operands staged through LDS.
//
// Each operand lies in memory either with k contiguous ("K-major": x and weight in the forward) or with k as its slow index
// (the weight in dx = dz W, both operands in dW = dz^T x). A K-major operand is staged as rows of 64 or 128 bytes of k; the other
// kind as rows of one k, and its fragments are read transposed (ds_read_b64_tr_b16: 16 lanes read a block of 4 k by 16
// columns and each ends up with the 4 k of one column), so no operand is ever transposed in memory.
//
// B is the first operand of the matrix instruction and A the second: of the 32 x 32 block a lane then holds 16 values of
// one output row m, and with B's rows taken in the order of `column_of` they are 16 consecutive n. They leave as whole runs of a row, turned
// through LDS (store_blocks); the narrow backward stores a lane's 16 values as they are.
#pragma once

#include "activation.hpp"
#include "boxconv_host.hpp"
#include "operators_host.hpp"

namespace boxconv {

namespace {

typedef float Acc16 __attribute__((ext_vector_type(16)));
typedef unsigned Chunk __attribute__((ext_vector_type(4)));            // 16 bytes of an operand

// A chunk of `valid` elements (none where it is <= 0, all where it is >= the vector's length) and zeros beyond, in two parts.
// What is requested does not depend on a branch, so that many can be on their way at once: the end of a row is read as the row's last
// whole vector (rows have at least one) and shifted down, nothing as `safe`, any whole vector.
template <class T, class I>
__device__ __forceinline__ Chunk request_chunk(const T* p, I valid, const T* safe) {
    constexpr int V = Vec<T>::kLen;
    const T* from = valid <= 0 ? safe : p - (valid < V ? V - static_cast<int>(valid) : 0);
    return __builtin_bit_cast(Chunk, *reinterpret_cast<const typename Vec<T>::Type*>(from));
}
template <class T, class I>
__device__ __forceinline__ void settle_chunk(Chunk& c, I valid) {
    constexpr int V = Vec<T>::kLen;
    if (valid <= 0) c = Chunk{0, 0, 0, 0};
    if (valid > 0 && valid < V) {
        typedef uint64_t Halves __attribute__((ext_vector_type(2)));
        Halves h = __builtin_bit_cast(Halves, c);
        const int bits = (V - static_cast<int>(valid)) * static_cast<int>(sizeof(T)) * 8;        // 16 to 112
        h = bits >= 64 ? Halves{h.y >> (bits - 64), 0} : Halves{h.x >> bits | h.y << (64 - bits), h.y >> bits};
        c = __builtin_bit_cast(Chunk, h);
    }
}
// The same where rows are shorter than a vector.
template <class T>
__device__ __forceinline__ Chunk short_chunk(const T* p, int valid) {
    typename Vec<T>::Type v = {};
#pragma unroll
    for (int j = 0; j < Vec<T>::kLen; ++j)
        if (j < valid) v[j] = p[j];
    return __builtin_bit_cast(Chunk, v);
}

// Row of a 32-row block of B that row r of the matrix instruction's result stands for: result element i of lane l is row
// 8 (i/4) + 4 (l/32) + i%4, which this maps to column 16 (l/32) + i.
__device__ __forceinline__ int column_of(int r) { return 16 * ((r >> 2) & 1) + 4 * (r >> 3) + (r & 3); }

// Shape of one operand's tile in LDS: X rows (m or n) by KT values of k, CH chunks of 16 bytes.
template <class T, bool K_MAJOR, int X, int CH>
struct TileShape {
    static constexpr int V = Vec<T>::kLen;
    static constexpr int KT = CH * V;
    static constexpr int kSteps = CH / 2;                                 // of the matrix instructions: 16 values of k in 16-bit types, 8 in float
    static constexpr int kRowChunks = K_MAJOR ? CH : X / V;               // 16-byte chunks in a row of the tile
    static constexpr int kRows = K_MAJOR ? X : KT;
    static constexpr int kChunks = kRows * kRowChunks;
    // Position of chunk c of row r: exclusive-or with a few bits of r, so that the lanes of one LDS access spread over the
    // 64 banks. PERM: fragments of B take rows in the order of column_of (bits 0, 1, 4 and 2 of the row count the lanes of an
    // access), those of A in natural order (bits 0 to 3).
    template <bool PERM>
    static __device__ __forceinline__ int place(int r, int c) {
        if constexpr (K_MAJOR && CH == 8) return r * 8 + (c ^ (PERM ? ((r >> 1) & 3) | ((r >> 2) & 4) : (r >> 1) & 7));
        else if constexpr (K_MAJOR) return r * 4 + (c ^ (PERM ? ((r >> 2) & 1) | ((r >> 3) & 2) : (r >> 2) & 3));
        else if constexpr (sizeof(T) == 2) return r * kRowChunks + (kRowChunks >= 16 ? c ^ (4 * (r & 3)) : kRowChunks == 8 ? c ^ (2 * (r & 2)) : c);
        else return r * kRowChunks + (kRowChunks >= 16 ? c ^ (2 * (r & 4)) : c);
    }
};

// One operand in memory: element (i, k), i counting m or n. `extent` rows i, `depth` values of k.
template <class T>
struct Operand {
    const T* p;
    int64_t ld;            // elements from one row of memory to the next
    int64_t extent, depth;
};

// The chunks of a tile that one thread of THREADS stages, through registers and with every bound checked.
template <class T, bool K_MAJOR, int X, int THREADS, bool PERM>
struct Stage {
    typedef TileShape<T, K_MAJOR, X, 8> Shape;
    static constexpr int N = Shape::kChunks / THREADS;
    Chunk v[N];
    static_assert(Shape::kChunks % THREADS == 0, "whole chunks per thread");
    static_assert(!K_MAJOR || THREADS % Shape::kRowChunks == 0, "a thread's chunks of a K-major tile all have the same k");
    const T* at[N];            // the thread's chunks in the tile that was last asked for
    int room[N];               // elements of them inside the operand's extent, at most a vector
    const T* safe;             // null: the operand's rows are shorter than a vector, and there is no safe place to read one from
    bool inner;                // no chunk ends inside the extent: with KT values of k left, all that is read is used as it lies in memory.
                               // (Rows beyond the extent of a K-major operand hold anything then: sums that nobody stores. 90022 rows, 431 -> 149
                               // bfloat16 68 us with every chunk masked, 63 so; 8000 rows, 1001 -> 999 47 and 43.)
    int64_t step;

    // The tile with rows from i0 and k from k0 on; `step`: k from one tile asked for to the next, in tiles.
    __device__ __forceinline__ void start(const Operand<T>& o, int64_t i0, int64_t k0, int tiles) {
        safe = (K_MAJOR ? o.depth : o.extent) >= Shape::V ? o.p : nullptr;
        inner = safe != nullptr && (K_MAJOR || i0 + X <= o.extent);
        step = K_MAJOR ? static_cast<int64_t>(tiles) * Shape::KT : tiles * Shape::KT * o.ld;
#pragma unroll
        for (int s = 0; s < N; ++s) {
            const int id = threadIdx.x % THREADS + s * THREADS, r = id / Shape::kRowChunks, c = id % Shape::kRowChunks;
            const int64_t i = i0 + (K_MAJOR ? r : c * Shape::V), k = k0 + (K_MAJOR ? c * Shape::V : r);
            at[s] = o.p + (K_MAJOR ? i * o.ld + k : k * o.ld + i);
            room[s] = static_cast<int>(min<int64_t>(max<int64_t>(o.extent - i, 0), Shape::V));
            if (K_MAJOR && room[s] > 0) room[s] = Shape::V;
        }
    }
    // Elements of chunk s, with k_left values of k from the tile's corner on.
    __device__ __forceinline__ int valid(int s, int k_left) const {
        const int id = threadIdx.x % THREADS + s * THREADS, r = id / Shape::kRowChunks, c = id % Shape::kRowChunks;
        if constexpr (K_MAJOR) return min(room[s], k_left - c * Shape::V);
        else return r < k_left ? room[s] : 0;
    }
    __device__ __forceinline__ void request(int k_left) {
        if (inner && k_left >= Shape::KT) {
#pragma unroll
            for (int s = 0; s < N; ++s) v[s] = __builtin_bit_cast(Chunk, *reinterpret_cast<const typename Vec<T>::Type*>(room[s] > 0 ? at[s] : safe));
            return;
        }
#pragma unroll
        for (int s = 0; s < N; ++s) v[s] = Chunk{0, 0, 0, 0};
        if (safe != nullptr) {
#pragma unroll
            for (int s = 0; s < N; ++s) v[s] = request_chunk(at[s], valid(s, k_left), safe);
        }
    }
    __device__ __forceinline__ void settle(int k_left) {
        if (inner && k_left >= Shape::KT) return;
#pragma unroll
        for (int s = 0; s < N; ++s) settle_chunk<T>(v[s], valid(s, k_left));
        if (safe == nullptr) {
#pragma unroll
            for (int s = 0; s < N; ++s) v[s] = short_chunk(at[s], valid(s, k_left));
        }
    }
    __device__ __forceinline__ void advance() {
#pragma unroll
        for (int s = 0; s < N; ++s) at[s] += step;
    }
    __device__ __forceinline__ void store(Chunk* tile) const {
#pragma unroll
        for (int s = 0; s < N; ++s) {
            const int id = threadIdx.x % THREADS + s * THREADS, r = id / Shape::kRowChunks, c = id % Shape::kRowChunks;
            tile[Shape::template place<PERM>(r, c)] = v[s];
        }
    }
};

// The fragment of 32 rows from `i` on and k step ks.
template <class T, bool K_MAJOR, int X, int CH, bool PERM>
__device__ __forceinline__ Chunk fragment(const Chunk* tile, int i, int ks) {
    typedef TileShape<T, K_MAJOR, X, CH> Shape;
    const int l = threadIdx.x % 64;
    if constexpr (K_MAJOR) {
        const int r = i + (PERM ? column_of(l % 32) : l % 32);
        return tile[Shape::template place<PERM>(r, 2 * ks + l / 32)];
    } else if constexpr (sizeof(T) == 2) {
        typedef short Four __attribute__((ext_vector_type(4)));
        typedef __attribute__((address_space(3))) Four* LdsPtr;
        // lane s of a group of 16 fetches columns 4 (s%4) .. +3 (in the order of the fragment's rows) of k row s/4
        const int s = l % 16, q = l / 16, four = 4 * (q & 1) + s % 4;
        const int col = i + (PERM ? 16 * (four & 1) + 4 * (four >> 1) : 4 * four);
        // (`place` looks at two bits of the row: the rows of a later k step and of the second half are as far on for every lane)
        const char* base = reinterpret_cast<const char*>(tile) + (Shape::template place<PERM>(8 * (q >> 1) + s / 4, col / 8) * 16 + col % 8 * 2);
        constexpr int kRow = Shape::kRowChunks * 16;
        Four lo, hi;
        lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LdsPtr)(base + 16 * ks * kRow));
        hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LdsPtr)(base + (16 * ks + 4) * kRow));
        typedef short Eight __attribute__((ext_vector_type(8)));
        return __builtin_bit_cast(Chunk, Eight(__builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7)));
    } else {
        const int col = i + (PERM ? column_of(l % 32) : l % 32), k = 8 * ks + 4 * (l / 32);
        const float* base = reinterpret_cast<const float*>(tile);
        typedef float Four __attribute__((ext_vector_type(4)));
        Four v;
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = base[Shape::template place<PERM>(k + j, col / 4) * 4 + col % 4];
        return __builtin_bit_cast(Chunk, v);
    }
}

template <class T> __device__ __forceinline__ Acc16 multiply_add(Chunk b, Chunk a, Acc16 c);
template <> __device__ __forceinline__ Acc16 multiply_add<__bf16>(Chunk b, Chunk a, Acc16 c) {
    typedef __bf16 Eight __attribute__((ext_vector_type(8)));
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(Eight, b), __builtin_bit_cast(Eight, a), c, 0, 0, 0);
}
template <> __device__ __forceinline__ Acc16 multiply_add<_Float16>(Chunk b, Chunk a, Acc16 c) {
    typedef _Float16 Eight __attribute__((ext_vector_type(8)));
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(Eight, b), __builtin_bit_cast(Eight, a), c, 0, 0, 0);
}
template <> __device__ __forceinline__ Acc16 multiply_add<float>(Chunk b, Chunk a, Acc16 c) {
    typedef float Four __attribute__((ext_vector_type(4)));
    const Four x = __builtin_bit_cast(Four, b), y = __builtin_bit_cast(Four, a);
#pragma unroll
    for (int j = 0; j < 4; ++j) c = __builtin_amdgcn_mfma_f32_32x32x2f32(x[j], y[j], c, 0, 0, 0);
    return c;
}

// ---- epilogue ------------------------------------------------------------------------------------------------
// act'(z) kept for the backward: float, or for 16-bit types a 16-bit number, 16400 plus or minus m, 65535 for NaN. From |act'| = 2^-5 on m counts steps of
// 2^-15; below, it is 13100 (32 |act'|)^(1/4), so that small derivatives keep their digits. (The derivatives of silu and gelu lie in
// [-0.13, 1.13]: m reaches 16305 downwards and 49071 upwards. 0 and 1 are exact.) What is read back is off by 2^-16 at most, and below 2^-5 by
// 2^-13.9 |act'|^(3/4), down to 2^-40: 2^-12.6 of act' at 2^-5, 2^-10.9 at 2^-12, to be compared with the rounding of the gradient, 2^-11 in float16 and 2^-8 in
// bfloat16. Steps of 2^-15 all the way lost gelu' from z = -5 on and a third of it at -4.6; float would double what is kept.
template <class T> struct SlopeOf { typedef uint16_t Type; };
template <> struct SlopeOf<float> { typedef float Type; };
constexpr float kRootSteps = 13100.0f;
__device__ __forceinline__ void keep_slope(float d, float& o) { o = d; }
__device__ __forceinline__ void keep_slope(float d, uint16_t& o) {
    const float a = fabsf(d), root = __builtin_amdgcn_sqrtf(__builtin_amdgcn_sqrtf(32.0f * a));
    const float m = a < 0.03125f ? kRootSteps * root : fmaf(a, 32768.0f, kRootSteps - 1024.0f);
    o = d != d ? 65535 : static_cast<uint16_t>(static_cast<int>(rintf(copysignf(m, d))) + 16400);
}
__device__ __forceinline__ float kept_slope(float v) { return v; }
__device__ __forceinline__ float kept_slope(uint16_t v) {
    const float m = static_cast<float>(static_cast<int>(v) - 16400), root = m * (1.0f / kRootSteps), square = root * root;
    const float a = fabsf(m) < kRootSteps ? 0.03125f * square * square : fmaf(fabsf(m), 1.0f / 32768.0f, (1024.0f - kRootSteps) / 32768.0f);
    return v == 65535 ? __builtin_nanf("") : copysignf(a, m);
}

// What becomes of a sum: y = act(sum + bias[n] + residual[m][n]). Null pointers leave their piece out.
template <class T>
struct Tail {
    T* out;
    int64_t rows, cols;
    const T *bias, *residual;
    int64_t ld_residual;
    typename SlopeOf<T>::Type* slope;
    int activation;
    float* partial;            // split products: the sums go here as they are, [split][rows][cols]
};

template <class T, int ACT, bool KEEP, int LEN>
__device__ __forceinline__ void finish(const float (&z)[LEN], T (&y)[LEN], typename SlopeOf<T>::Type (&d)[LEN]) {
#pragma unroll
    for (int i = 0; i < LEN; ++i) {
        y[i] = static_cast<T>(activate<ACT>(z[i]));
        if constexpr (KEEP) keep_slope(slope<ACT>(z[i]), d[i]);
    }
}

// f(0), ..., f(N - 1) written out. (A loop over single elements that ends at a number known at run time becomes a copy
// through the stack, whatever the unrolling.)
template <int N, int I = 0, class F>
__device__ __forceinline__ void each(F f) {
    if constexpr (I < N) {
        f(I);
        each<N, I + 1>(f);
    }
}

// LEN consecutive elements of a row to or from memory, `valid` of them, 16 bytes at a time.
template <class E, int LEN>
__device__ __forceinline__ void load_run(const E* p, E (&v)[LEN], int64_t valid) {
    constexpr int P = LEN * sizeof(E) < 16 ? LEN : 16 / static_cast<int>(sizeof(E));
    typedef E Packed __attribute__((ext_vector_type(P), aligned(sizeof(E))));
    if (valid >= LEN) {
#pragma unroll
        for (int k = 0; k < LEN; k += P) {
            const Packed q = *reinterpret_cast<const Packed*>(p + k);
#pragma unroll
            for (int i = 0; i < P; ++i) v[k + i] = q[i];
        }
    } else {
        each<LEN>([&](int i) { v[i] = i < valid ? p[i] : E(0); });
    }
}
template <class E, int LEN>
__device__ __forceinline__ void store_run(E* p, const E (&v)[LEN], int64_t valid) {
    constexpr int P = LEN * sizeof(E) < 16 ? LEN : 16 / static_cast<int>(sizeof(E));
    typedef E Packed __attribute__((ext_vector_type(P), aligned(sizeof(E))));
    if (valid >= LEN) {
#pragma unroll
        for (int k = 0; k < LEN; k += P) {
            Packed q;
#pragma unroll
            for (int i = 0; i < P; ++i) q[i] = v[k + i];
            *reinterpret_cast<Packed*>(p + k) = q;
        }
    } else {
        each<LEN>([&](int i) {
            if (i < valid) p[i] = v[i];
        });
    }
}

template <class T, int LEN>
__device__ __forceinline__ void finish_tail(const Tail<T>& t, float (&z)[LEN], int64_t m, int64_t n) {
    typedef typename SlopeOf<T>::Type S;
    const int64_t valid = t.cols - n;
    T v[LEN];
    S d[LEN];
    const bool keep = t.slope != nullptr;
    // (asked here and not element by element: those branches kept the elements' instructions from overlapping:
    // 895560 x 32 -> 88 with gelu and a kept slope 190 us, 172 without them, 175 with gelu's tail and small slopes kept; 48552 x 208 -> 456
    // float 158 and 144)
    if (keep) {
        if (t.activation == kActSilu) finish<T, kActSilu, true>(z, v, d);
        else finish<T, kActGelu, true>(z, v, d);
    } else {
        switch (t.activation) {
            case kActRelu: finish<T, kActRelu, false>(z, v, d); break;
            case kActSilu: finish<T, kActSilu, false>(z, v, d); break;
            case kActGelu: finish<T, kActGelu, false>(z, v, d); break;
            default: finish<T, kActNone, false>(z, v, d);
        }
    }
    store_run<T, LEN>(t.out + m * t.cols + n, v, valid);
    if (keep) store_run<S, LEN>(t.slope + m * t.cols + n, d, valid);
}

// All of it at once, at the ends of rows too.
template <class T, int LEN>
__device__ __forceinline__ void apply_tail(const Tail<T>& t, float (&z)[LEN], int64_t m, int64_t n) {
    if (m >= t.rows || n >= t.cols) return;
    const int64_t valid = t.cols - n;
    T v[LEN];
    if (t.bias != nullptr) {
        load_run<T, LEN>(t.bias + n, v, valid);
#pragma unroll
        for (int i = 0; i < LEN; ++i) z[i] += static_cast<float>(v[i]);
    }
    if (t.residual != nullptr) {
        load_run<T, LEN>(t.residual + m * t.ld_residual + n, v, valid);
#pragma unroll
        for (int i = 0; i < LEN; ++i) z[i] += static_cast<float>(v[i]);
    }
    finish_tail<T, LEN>(t, z, m, n);
}

// Where LDS keeps 16-byte chunk c of row r of a wave's 32 x 32 FN sums. Neither the 16 lanes that write one chunk each of as many rows
// nor those that read rows along, one or two chunks each, meet in a bank.
template <int FN>
__device__ __forceinline__ int turned(int r, int c) { return r * 8 * FN + (FN == 1 ? c ^ (r / 2 % 8) : c ^ (r % 16) ^ (c / 16)); }

// What a wave's lanes wrote to LDS is there for its other lanes (its LDS instructions run in their order), and what they read was read.
__device__ __forceinline__ void wave_in_step() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// The blocks of a wave's part of a tile, from row m0 and column n0 on, to memory: sums as they are, or through the tail. A lane's sums
// are 16 columns of one row, and stores of 16 bytes each to 32 rows are as many requests to the L2 as lanes: 513323 x 136 -> 144
// bfloat16 with a residual and a kept slope took 277 us, 239 this way; 8192 x 2048 -> 4096 with gelu 146 and 140. So 32 rows at a time pass through `lds` (256 FN chunks of this wave's own, free when
// this is called) and leave as runs of 64 FN bytes (of float: 128 FN).
template <class T, int FN, int FM>
__device__ __forceinline__ void store_blocks(const Tail<T>& t, const Acc16 (&acc)[FN][FM], int64_t m0, int64_t n0, int64_t part, Chunk* lds) {
    typedef typename Vec<T>::Type Packed;
    typedef float Four __attribute__((ext_vector_type(4)));
    const int l = threadIdx.x % 64;
    const auto turn = [&](int i) {
        wave_in_step();
#pragma unroll
        for (int f = 0; f < FN; ++f)
#pragma unroll
            for (int q = 0; q < 4; ++q)
                lds[turned<FN>(l % 32, 8 * f + 4 * (l / 32) + q)] =
                    __builtin_bit_cast(Chunk, Four{acc[f][i][4 * q], acc[f][i][4 * q + 1], acc[f][i][4 * q + 2], acc[f][i][4 * q + 3]});
        wave_in_step();
    };
    if (t.partial != nullptr) {
        constexpr int ROWS = 8 / FN;                           // that an instruction covers
        const int r = l / (8 * FN), c = l % (8 * FN);
        const int64_t n = n0 + 4 * c;
        each<FM>([&](int i) {
            turn(i);
            for (int s = 0; s < 32 / ROWS; ++s) {
                const Four v = __builtin_bit_cast(Four, lds[turned<FN>(r + ROWS * s, c)]);
                const float z[4] = {v[0], v[1], v[2], v[3]};
                const int64_t m = m0 + 32 * i + r + ROWS * s;
                if (m < t.rows && n < t.cols) store_run<float, 4>(t.partial + (part * t.rows + m) * t.cols + n, z, t.cols - n);
            }
        });
        return;
    }
    constexpr int V = Vec<T>::kLen, LANES = 32 * FN / V, ROWS = 64 / LANES, STEPS = 32 / ROWS, D = STEPS < 4 ? STEPS : 4, GROUPS = STEPS / D;
    const int r = l / LANES, c = l % LANES * (V / 4);
    const int64_t n = n0 + l % LANES * V;
    const bool whole = n + V <= t.cols;                        // (else the tail goes element by element)
    const auto row = [&](int group, int d) { return m0 + 32 * (group / GROUPS) + r + ROWS * (group % GROUPS * D + d); };
    Packed bias = {}, ahead[D] = {};                           // (the residual is requested D steps ahead)
    if (whole && t.bias != nullptr) bias = *reinterpret_cast<const Packed*>(t.bias + n);
    const auto request = [&](int group) {
        if (t.residual == nullptr || !whole) return;
#pragma unroll
        for (int d = 0; d < D; ++d)
            if (row(group, d) < t.rows) ahead[d] = *reinterpret_cast<const Packed*>(t.residual + row(group, d) * t.ld_residual + n);
    };
    request(0);
    each<FM>([&](int i) {
        turn(i);
#pragma unroll 1
        for (int g = 0; g < GROUPS; ++g) {
            const int group = i * GROUPS + g;
            Packed residual[D];
#pragma unroll
            for (int d = 0; d < D; ++d) residual[d] = ahead[d];
            if (group + 1 < FM * GROUPS) request(group + 1);
#pragma unroll
            for (int d = 0; d < D; ++d) {
                float z[V];
#pragma unroll
                for (int k = 0; k < V / 4; ++k) {
                    const Four v = __builtin_bit_cast(Four, lds[turned<FN>(r + ROWS * (g * D + d), c + k)]);
#pragma unroll
                    for (int e = 0; e < 4; ++e) z[4 * k + e] = v[e];
                }
                const int64_t m = row(group, d);
                if (whole && m < t.rows) {
                    if (t.bias != nullptr) {
#pragma unroll
                        for (int e = 0; e < V; ++e) z[e] += static_cast<float>(bias[e]);
                    }
                    if (t.residual != nullptr) {
#pragma unroll
                        for (int e = 0; e < V; ++e) z[e] += static_cast<float>(residual[d][e]);
                    }
                    finish_tail<T, V>(t, z, m, n);
                } else {
                    apply_tail<T, V>(t, z, m, n);
                }
            }
        }
    });
}

}  // namespace

}  // namespace boxconv
