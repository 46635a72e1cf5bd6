// Rows of values to blocks of 128 in 8-bit floating point (float8_blocks.hpp has the format).
#include "activation.hpp"
#include "boxconv_host.hpp"
#include "float8_blocks.hpp"
#include "operators_host.hpp"

namespace boxconv {

namespace {

// A wave takes a block, a lane two of its values.
template <class T>
__global__ void __launch_bounds__(256) quantize_kernel(QuantizeCall q, int64_t blocks, int64_t padded) {
    const int l = threadIdx.x % 64;
    for (int64_t id = blockIdx.x * 4ll + threadIdx.x / 64; id < q.rows * blocks; id += gridDim.x * 4ll) {
        const int64_t row = id / blocks, b = id % blocks, c = b * kBlock + 2 * l;
        const T* p = static_cast<const T*>(q.x) + row * q.ld;
        const float v[2] = {c < q.columns ? static_cast<float>(p[c]) : 0.0f, c + 1 < q.columns ? static_cast<float>(p[c + 1]) : 0.0f};
        const int e = block_exponent(most_of_lanes(largest(v), 64));
        *reinterpret_cast<uint16_t*>(q.codes + id * kBlock + 2 * l) = static_cast<uint16_t>(to_codes(v, e)[0]);
        if (l == 0) q.exponents[row * padded + b] = static_cast<uint8_t>(e);
        if (b == blocks - 1 && l > 0 && b + l < padded) q.exponents[row * padded + b + l] = 127;
    }
}

}  // namespace

hipError_t quantize_launch(const QuantizeCall& q, hipStream_t stream) {
    const int64_t blocks = blocks_of(q.columns), padded = exponents_of(q.columns), groups = std::min<int64_t>((q.rows * blocks + 3) / 4, 8192);
    const dim3 grid(static_cast<unsigned>(groups));
    if (q.dtype == kF32) BOXCONV_LAUNCH("quantize", (quantize_kernel<float>), grid, dim3(256), 0, stream, q, blocks, padded);
    else if (q.dtype == kF16) BOXCONV_LAUNCH("quantize", (quantize_kernel<_Float16>), grid, dim3(256), 0, stream, q, blocks, padded);
    else BOXCONV_LAUNCH("quantize", (quantize_kernel<__bf16>), grid, dim3(256), 0, stream, q, blocks, padded);
    return hipGetLastError();
}

}  // namespace boxconv
