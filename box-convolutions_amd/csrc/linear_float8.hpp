// The pointwise product of rows in 8-bit blocks of 128 (float8_blocks.hpp): y = act(x W^T + bias + residual), both operands K-major.
// The matrix instructions multiply by the blocks' powers of two themselves: each lane gives one exponent for the 32 values that it holds
// of a row.
#pragma once

#include "float8_blocks.hpp"
#include "linear_wide.hpp"

namespace boxconv {

namespace {

// One operand: [extent] rows of `blocks` blocks of codes, and `padded` exponents each.
struct Coded {
    const uint8_t *codes, *exponents;
    int64_t extent;
    int blocks, padded;
};

// 32 codes of a row: a lane's share of 64 values of k.
struct Codes32 { Chunk lo, hi; };

// The 8-bit instructions cut every product of 8 neighbouring k down to a multiple of 2^-13 of the largest of them before they add (found
// with products of one large and one small pair: one 2^13 times smaller is kept, one 2^14 times smaller is lost, from the ninth k on nothing
// is). That is 1e-5 to 4e-5 of a sum of random signs, far below half a step of the 16-bit types. Results in float32 take the bfloat16
// instructions instead, at half the rate: codes and powers of two fit that type, and its products add up in float32.
typedef int Eight __attribute__((ext_vector_type(8)));
template <class T>
__device__ __forceinline__ Acc16 multiply_add8(const Codes32& b, int eb, const Codes32& a, int ea, Acc16 c) {
    typedef __bf16 Pair __attribute__((ext_vector_type(2)));
    typedef __bf16 Run __attribute__((ext_vector_type(8)));
    if constexpr (sizeof(T) == 2) {
        const auto join = [](const Codes32& v) { return __builtin_bit_cast(Eight, v); };
        return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(join(b), join(a), c, 0, 0, 0, eb, 0, ea);
    } else {
        const auto wide = [](const Codes32& v, int e, int i) {             // eight codes as bfloat16
            const float power = __builtin_bit_cast(float, static_cast<unsigned>(e) << 23);
            const Chunk from = i < 2 ? v.lo : v.hi;
            Run out;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const unsigned word = from[i % 2 * 2 + j / 2];
                const Pair two = j % 2 == 0 ? __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(word, power, false) : __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(word, power, true);
                out[2 * j] = two[0];
                out[2 * j + 1] = two[1];
            }
            return out;
        };
#pragma unroll
        for (int i = 0; i < 4; ++i) c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(wide(b, eb, i), wide(a, ea, i), c, 0, 0, 0);
        return c;
    }
}

// A wave computes a 32 x 32 block, fragments straight from memory.
template <class T>
__global__ void __launch_bounds__(256) product_float8_kernel(Coded a, Coded b, Tail<T> tail, int64_t tiles_n, int64_t tiles) {
    __shared__ Chunk lds[4 * 256];
    const int l = threadIdx.x % 64, wave = threadIdx.x / 64;
    const int64_t id = min(blockIdx.x * 4ll + wave, tiles - 1), m0 = id / tiles_n * 32, n0 = id % tiles_n * 32;
    const int64_t m = min(m0 + l % 32, a.extent - 1), n = min(n0 + column_of(l % 32), b.extent - 1);
    const uint8_t *x = a.codes + m * a.blocks * kBlock + l / 32 * 32, *w = b.codes + n * b.blocks * kBlock + l / 32 * 32;
    Acc16 acc[1][1] = {};
    for (int s = 0; s < a.blocks; ++s) {
        const int ea = a.exponents[m * a.padded + s], eb = b.exponents[n * b.padded + s];
        for (int h = 0; h < 2; ++h)
            acc[0][0] = multiply_add8<T>(*reinterpret_cast<const Codes32*>(w + s * kBlock + h * 64), eb, *reinterpret_cast<const Codes32*>(x + s * kBlock + h * 64), ea, acc[0][0]);
    }
    store_blocks<T, 1, 1>(tail, acc, m0, n0, 0, lds + wave * 256);
}

}  // namespace

template <class T>
hipError_t linear_float8_forward(const LinearFloat8Call& c, void* workspace, hipStream_t stream) {
    QuantizeCall q = {c.x, c.ld_x, c.input_dtype, c.rows, c.K, nullptr, nullptr};
    Coded a = {static_cast<const uint8_t*>(c.x), c.x_exponents, c.rows, static_cast<int>(blocks_of(c.K)), static_cast<int>(exponents_of(c.K))}, b = a;
    if (c.input_dtype != kE4M3) {
        q.codes = static_cast<uint8_t*>(workspace);
        q.exponents = q.codes + c.rows * a.blocks * kBlock;
        a.codes = q.codes;
        a.exponents = q.exponents;
        if (const hipError_t e = quantize_launch(q, stream); e != hipSuccess) return e;
    }
    b.codes = c.weight;
    b.exponents = c.weight_exponents;
    b.extent = c.N;
    Tail<T> tail = {};
    tail.out = static_cast<T*>(c.y);
    tail.rows = c.rows;
    tail.cols = c.N;
    tail.bias = static_cast<const T*>(c.bias);
    tail.residual = static_cast<const T*>(c.residual);
    tail.ld_residual = c.ld_residual;
    tail.activation = c.activation;
    const int64_t tm = (c.rows + 31) / 32, tn = (c.N + 31) / 32;
    BOXCONV_LAUNCH("linear_float8", (product_float8_kernel<T>), dim3(static_cast<unsigned>((tm * tn + 3) / 4)), dim3(256), 0, stream, a, b, tail, tn, tm * tn);
    return hipGetLastError();
}

template <class T>
size_t linear_float8_workspace(int64_t rows, int64_t K, int64_t N, bool values) {
    return values ? static_cast<size_t>(rows) * (blocks_of(K) * kBlock + exponents_of(K)) : 0;
}

}  // namespace boxconv
