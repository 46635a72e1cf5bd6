// Rows of values to blocks of 128 in 8-bit floating point (float8_blocks.hpp has the format).
#include "activation.hpp"
#include "boxconv_host.hpp"
#include "float8_blocks.hpp"
#include "operators_host.hpp"

namespace boxconv {

namespace {

// Eight lanes take a block, a lane 16 neighbouring values: whole 16-byte vectors in and out, the largest magnitude over the eight by moves within the
// vector unit. kAhead blocks of a lane are requested before the first is used. I: a type that counts all blocks (64-bit divisions take dozens of
// instructions). Bound by memory: 8192 x 4096 bfloat16 17.4 to 17.9 us, 5.7 TB/s (one block at a time 48 us; part of it comes from the caches), 4096 x 2048 float32
// 8.2 to 8.6 us, 36993 x 502 bfloat16 12.4.
template <class T, class I>
__global__ void __launch_bounds__(256) quantize_kernel(QuantizeCall q, I blocks, I padded, I total) {
    constexpr int V = Vec<T>::kLen, PER = 16, NV = PER / V, kAhead = NV == 2 ? 4 : 2;
    typedef typename Vec<T>::Type Packed;
    const int sub = threadIdx.x % 8;
    const I step = static_cast<I>(gridDim.x) * 32;
    for (I first = blockIdx.x * static_cast<I>(32) + threadIdx.x / 8; first < total; first += kAhead * step) {
        Packed raw[kAhead][NV] = {};
        int64_t row[kAhead];
        I block[kAhead];
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
            const I id = first + i * step;
            if (id >= total) break;
            row[i] = id / blocks;
            block[i] = id - static_cast<I>(row[i]) * blocks;
            const int64_t c = static_cast<int64_t>(block[i]) * kBlock + sub * PER, left = q.columns - c;
            const T* p = static_cast<const T*>(q.x) + row[i] * q.ld + c;
            // the last values of a row: whole vectors that run into what follows, while that is inside the tensor, and a mask (element by element
            // every wave waits for them in turn: 36993 x 502 bfloat16 23 us, 12 this way)
            const bool clear = (q.rows - 1 - row[i]) * q.ld + q.columns >= static_cast<int64_t>(blocks) * kBlock;
            if (left >= PER || (clear && left > 0)) {
#pragma unroll
                for (int v = 0; v < NV; ++v) raw[i][v] = *reinterpret_cast<const Packed*>(p + v * V);
            } else if (left > 0) {
#pragma unroll
                for (int v = 0; v < NV; ++v) {
                    Packed part = {};
#pragma unroll
                    for (int j = 0; j < V; ++j)
                        if (v * V + j < left) part[j] = p[v * V + j];
                    raw[i][v] = part;
                }
            }
        }
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
            if (first + i * step >= total) break;                  // (the same for all eight)
            // (here, and not where they are requested: the mask waits for them)
            if (const int64_t left = q.columns - static_cast<int64_t>(block[i]) * kBlock - sub * PER; left < PER) {
                typedef unsigned Words __attribute__((ext_vector_type(4)));
                const int bytes = static_cast<int>(max<int64_t>(left, 0)) * static_cast<int>(sizeof(T));
#pragma unroll
                for (int v = 0; v < NV; ++v) {
                    Words w = __builtin_bit_cast(Words, raw[i][v]);
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const int n = bytes - 16 * v - 4 * j;                  // from this word to the row's end
                        w[j] &= n >= 4 ? 0xffffffffu : n <= 0 ? 0u : (1u << 8 * n) - 1;
                    }
                    raw[i][v] = __builtin_bit_cast(Packed, w);
                }
            }
            float x[PER];
#pragma unroll
            for (int j = 0; j < PER; ++j) x[j] = static_cast<float>(raw[i][j / V][j % V]);
            const int e = block_exponent(most_of_lanes(largest(x), 8));
            typedef unsigned Four __attribute__((ext_vector_type(4)));
            const Codes<PER> codes = to_codes(x, e);
            *reinterpret_cast<Four*>(q.codes + (row[i] * blocks + block[i]) * kBlock + sub * PER) = __builtin_bit_cast(Four, codes);
            uint8_t* to = q.exponents + row[i] * padded + block[i];
            if (sub == 0) to[0] = static_cast<uint8_t>(e);
            else if (block[i] == blocks - 1 && block[i] + sub < padded) to[sub] = 127;
        }
    }
}

}  // namespace

namespace {

template <class T>
void quantize(const QuantizeCall& q, hipStream_t stream) {
    const int64_t blocks = blocks_of(q.columns), padded = exponents_of(q.columns), total = q.rows * blocks;
    const dim3 grid(static_cast<unsigned>(std::min<int64_t>((total + 31) / 32, 4096)));
    if (total < (int64_t(1) << 30))
        BOXCONV_LAUNCH("quantize", (quantize_kernel<T, unsigned>), grid, dim3(256), 0, stream, q, static_cast<unsigned>(blocks), static_cast<unsigned>(padded),
                       static_cast<unsigned>(total));
    else BOXCONV_LAUNCH("quantize", (quantize_kernel<T, int64_t>), grid, dim3(256), 0, stream, q, blocks, padded, total);
}

}  // namespace

hipError_t quantize_launch(const QuantizeCall& q, hipStream_t stream) {
    if (q.dtype == kF32) quantize<float>(q, stream);
    else if (q.dtype == kF16) quantize<_Float16>(q, stream);
    else quantize<__bf16>(q, stream);
    return hipGetLastError();
}

}  // namespace boxconv
