// Blocks of 128 values in 8-bit floating point (e4m3: one sign bit, four of exponent, three of mantissa, largest value 448, no
// infinity) with a power of two each: value = code * 2^(exponent - 127). And sums over a wave's lanes.
//
// The power is the least, not below 2^-126, that keeps the block's largest finite magnitude at or below 448 times it; a block of
// zeros has exponent 127. Scaling by it is exact, so a code is its value rounded once, to nearest, ties to even. A power of two costs nothing
// against a finer scale (the format's relative precision is the same wherever a value lies in its range) and the matrix instructions
// multiply by it themselves. NaN and infinities become NaN and leave the rest of their block alone.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace boxconv {

constexpr int kBlock = 128;
constexpr int64_t blocks_of(int64_t columns) { return (columns + kBlock - 1) / kBlock; }
constexpr int64_t exponents_of(int64_t columns) { return (blocks_of(columns) + 3) / 4 * 4; }       // of a row, padded to whole words
constexpr int blocks_of(int columns) { return (columns + kBlock - 1) / kBlock; }
constexpr int exponents_of(int columns) { return (blocks_of(columns) + 3) / 4 * 4; }

namespace {

// The value of a lane's partner: the neighbour, the other pair, the other four, the other eight, ... All of them pair lanes that
// hold the same thing so far, so after every step twice as many lanes do, to the bit. (Moves within the vector unit: no LDS.)
template <int STEP>
__device__ __forceinline__ float partner(float v) {
    const int i = __builtin_bit_cast(int, v);
    if constexpr (STEP == 1) return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(i, i, 0xb1, 0xf, 0xf, true));       // quad_perm 1 0 3 2
    if constexpr (STEP == 2) return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(i, i, 0x4e, 0xf, 0xf, true));       // quad_perm 2 3 0 1
    if constexpr (STEP == 4) return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(i, i, 0x141, 0xf, 0xf, true));      // row_half_mirror
    if constexpr (STEP == 8) return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(i, i, 0x140, 0xf, 0xf, true));      // row_mirror
    if constexpr (STEP == 16) {
        const auto r = __builtin_amdgcn_permlane16_swap(i, i, false, false);
        return __builtin_bit_cast(float, static_cast<int>(threadIdx.x & 16 ? r[0] : r[1]));
    }
    if constexpr (STEP == 32) {
        const auto r = __builtin_amdgcn_permlane32_swap(i, i, false, false);
        return __builtin_bit_cast(float, static_cast<int>(threadIdx.x & 32 ? r[0] : r[1]));
    }
}

// f over `lanes` neighbouring lanes (a power of two, the same in the whole wave), every lane of which is active.
template <class F>
__device__ __forceinline__ float over_lanes(float v, int lanes, F f) {
    if (lanes > 1) v = f(v, partner<1>(v));
    if (lanes > 2) v = f(v, partner<2>(v));
    if (lanes > 4) v = f(v, partner<4>(v));
    if (lanes > 8) v = f(v, partner<8>(v));
    if (lanes > 16) v = f(v, partner<16>(v));
    if (lanes > 32) v = f(v, partner<32>(v));
    return v;
}
__device__ __forceinline__ float sum_of_lanes(float v, int lanes) {
    return over_lanes(v, lanes, [](float a, float b) { return a + b; });
}
__device__ __forceinline__ float most_of_lanes(float v, int lanes) {
    return over_lanes(v, lanes, [](float a, float b) { return a < b ? b : a; });
}

// The largest finite magnitude.
template <int N>
__device__ __forceinline__ float largest(const float (&v)[N]) {
    float most = 0.0f;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const float a = fabsf(v[i]);
        most = a < __builtin_inff() && a > most ? a : most;
    }
    return most;
}

// The stored exponent of a block whose largest magnitude is `most`: 448 = 1.75 * 2^8.
__device__ __forceinline__ int block_exponent(float most) {
    const unsigned bits = __builtin_bit_cast(unsigned, most);
    const int e = static_cast<int>(bits >> 23) - 8 + ((bits & 0x7fffff) > 0x600000 ? 1 : 0);
    return bits == 0 ? 127 : e < 1 ? 1 : e;
}

// N values (a multiple of 4, or 2) as codes, four in a word.
template <int N>
struct Codes {
    unsigned word[(N + 3) / 4];
    __device__ __forceinline__ unsigned operator[](int i) const { return word[i]; }
};
template <int N>
__device__ __forceinline__ Codes<N> to_codes(const float (&v)[N], int exponent) {
    const float by = __builtin_bit_cast(float, static_cast<unsigned>(254 - exponent) << 23);       // 2^(127 - exponent), from 2^-119 to 2^126
    float u[N];
#pragma unroll
    for (int i = 0; i < N; ++i) u[i] = fabsf(v[i]) < __builtin_inff() ? v[i] * by : __builtin_nanf("");
    Codes<N> c = {};
#pragma unroll
    for (int i = 0; i < N; i += 2)
        c.word[i / 4] = i % 4 == 0 ? __builtin_amdgcn_cvt_pk_fp8_f32(u[i], u[i + 1], c.word[i / 4], false)
                                   : __builtin_amdgcn_cvt_pk_fp8_f32(u[i], u[i + 1], c.word[i / 4], true);
    return c;
}

}  // namespace

}  // namespace boxconv
