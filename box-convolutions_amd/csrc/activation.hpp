// Activations at the end of the pointwise product and of group norm, and their derivatives; 16-byte vectors of
// the three element types.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace boxconv {

// BOXCONV_ACT_* of include/boxconv.h
enum Activation : int { kActNone = 0, kActRelu = 1, kActSilu = 2, kActGelu = 3 };

namespace {

// 1 / (1 + exp(-z)). exp overflows to infinity from z = -88.7 on, where the quotient is 0 as it should be.
__device__ __forceinline__ float sigmoid(float z) { return __builtin_amdgcn_rcpf(1.0f + __expf(-z)); }

// The normal distribution's probability below z, and its density. With t = 1/(1 + 0.3039 |z|) the probability beyond |z| is q(t) exp(-z*z/2),
// q the polynomial of eight terms that fits it best relatively (weighted least squares, the weights raised where the error is largest): within
// 8.3e-8 from z = 0 to 13.3, where the exponential leaves float32. In float32 it is within 4e-7, and the exponential adds its argument's
// rounding, z*z * 1e-7: digits are kept as far as the value is a normal number. One exponential serves both.
struct Normal { float below, density; };
__device__ __forceinline__ Normal normal(float z) {
    const float e = __builtin_amdgcn_exp2f(z * z * (-0.5f * 1.44269504089f));
    const float t = __builtin_amdgcn_rcpf(fmaf(0.3039f, fabsf(z), 1.0f));
    float q = fmaf(0.036879742f, t, -0.155553320f);
    q = fmaf(q, t, 0.192881254f);
    q = fmaf(q, t, -0.043691076f);
    q = fmaf(q, t, 0.123832448f);
    q = fmaf(q, t, 0.102314367f);
    q = fmaf(q, t, 0.122142549f);
    q = fmaf(q, t, 0.121194078f);
    const float tail = q * t * e;
    return {z > 0.0f ? 1.0f - tail : tail, 0.39894228040f * e};
}

// NaN stays NaN in all of them (relu: the comparison is false for it).
template <int ACT>
__device__ __forceinline__ float activate(float z) {
    if constexpr (ACT == kActRelu) return z < 0.0f ? 0.0f : z;
    if constexpr (ACT == kActSilu) return z * sigmoid(z);
    if constexpr (ACT == kActGelu) return z * normal(z).below;
    return z;
}

// d activate / dz. relu: 0 at z = 0.
template <int ACT>
__device__ __forceinline__ float slope(float z) {
    if constexpr (ACT == kActRelu) return z > 0.0f ? 1.0f : 0.0f;
    if constexpr (ACT == kActSilu) {
        const float s = sigmoid(z);
        return fmaf(z * s, 1.0f - s, s);
    }
    if constexpr (ACT == kActGelu) {
        const Normal n = normal(z);
        return fmaf(z, n.density, n.below);
    }
    return 1.0f;
}

// 16 bytes of T: what a lane loads or stores at once. Declared with the alignment of one element: rows of odd length start
// anywhere, and the vector memory instructions take any address.
template <class T> struct Vec;
template <> struct Vec<float> { static constexpr int kLen = 4; typedef float Type __attribute__((ext_vector_type(4), aligned(4))); };
template <> struct Vec<_Float16> { static constexpr int kLen = 8; typedef _Float16 Type __attribute__((ext_vector_type(8), aligned(2))); };
template <> struct Vec<__bf16> { static constexpr int kLen = 8; typedef __bf16 Type __attribute__((ext_vector_type(8), aligned(2))); };

// A parameter vector in float or in T.
template <class T>
__device__ __forceinline__ float load_param(const void* p, bool is_float, int i) {
    return is_float ? static_cast<const float*>(p)[i] : static_cast<float>(static_cast<const T*>(p)[i]);
}
template <class T>
__device__ __forceinline__ void store_param(void* p, bool is_float, int i, float v) {
    if (is_float) static_cast<float*>(p)[i] = v;
    else static_cast<T*>(p)[i] = static_cast<T>(v);
}

}  // namespace

}  // namespace boxconv
