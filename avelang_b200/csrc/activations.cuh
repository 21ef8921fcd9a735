// Activations of the integer, gated and gradient kernels: values and slopes in fp32.  (The FP4 tiles' epilogue keeps the forms in
// gemm_fp4_sm100.cuh, with a bound on gelu's absolute error; there relu of a NaN is 0, here it is a NaN.)
//
// erf enters through erfcx(z) = exp(z^2) erfc(z), z >= 0, as t P(t) with t = 1 / (1 + 0.6 z) and a degree-7 P fitted
// to the smallest relative error over 0 <= z <= 13.5 (3.5e-7 as a polynomial, 4.4e-7 evaluated in fp32).  A bound on the
// *relative* error keeps the far negative tail of gelu, where the value itself goes to zero, as exact as the rest.
#pragma once

#include <cstdint>
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include "../../include/ave_fp4.h"

namespace avefp4 {

// 0.5 erfc(z / sqrt 2) for z = |x|: the probability of the normal tail beyond |x|
__device__ __forceinline__ float normal_tail(float ax) {
    const float z = ax * 0.70710678118654752f;
    const float t = __fdividef(1.0f, fmaf(0.6f, z, 1.0f));
    float p = fmaf(-0.0911727f, t, 0.40852696f);
    p = fmaf(p, t, -0.6392193f);
    p = fmaf(p, t, 0.27956369f);
    p = fmaf(p, t, 0.07530976f);
    p = fmaf(p, t, 0.29112424f);
    p = fmaf(p, t, 0.33731033f);
    p = fmaf(p, t, 0.33855701f);
    return 0.5f * p * t * __expf(-0.5f * ax * ax);
}

__device__ __forceinline__ float exp2_approx(float x) {
    float y;
    asm("ex2.approx.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// 1 / (1 + e^-x) with numerator and denominator taken 2^-8 times: __fdividef gives 0 for a divisor beyond 2^126, which 1 + e^-x passes
// at x = -87.3, where silu is still -1e-36.  So every silu in the normal range of fp32 (to x = -91.9) keeps its relative error; below, 0.
__device__ __forceinline__ float sigmoid(float x) {
    constexpr float kLog2E = 1.44269504088896341f, kPart = 0.00390625f;
    return __fdividef(kPart, kPart + exp2_approx(fmaf(x, -kLog2E, -8.0f)));
}

// twice the argument of the tanh form: 0.5 (1 + tanh u) = sigmoid(2u)
__device__ __forceinline__ float gelu_tanh_arg(float x) { return 1.59576912160573071f * fmaf(0.044715f * x * x, x, x); }

template <int ACT>
__device__ __forceinline__ float act_value(float x) {
    if constexpr (ACT == AVE_FP4_ACT_RELU) {
        return x < 0.0f ? 0.0f : x;      // a NaN stays one
    } else if constexpr (ACT == AVE_FP4_ACT_GELU) {
        const float tail = normal_tail(fabsf(x));
        return x < 0.0f ? x * tail : x * (1.0f - tail);
    } else if constexpr (ACT == AVE_FP4_ACT_GELU_TANH) {
        return x * sigmoid(gelu_tanh_arg(x));
    } else if constexpr (ACT == AVE_FP4_ACT_SILU) {
        return x * sigmoid(x);
    } else {
        return x;
    }
}

// Value and slope together (they share the exponential).
template <int ACT>
__device__ __forceinline__ void act_value_slope(float x, float& value, float& slope) {
    if constexpr (ACT == AVE_FP4_ACT_RELU) {
        value = x < 0.0f ? 0.0f : x;
        slope = x > 0.0f ? 1.0f : 0.0f;
    } else if constexpr (ACT == AVE_FP4_ACT_GELU) {
        const float tail = normal_tail(fabsf(x));
        const float cdf = x < 0.0f ? tail : 1.0f - tail;
        value = x * cdf;
        slope = fmaf(x, 0.39894228040143268f * __expf(-0.5f * x * x), cdf);
    } else if constexpr (ACT == AVE_FP4_ACT_GELU_TANH) {
        const float s = sigmoid(gelu_tanh_arg(x));
        const float q = s * (1.0f - s);
        value = x * s;
        // where s has run into 0 or 1 the second term is 0, whatever x * x has become
        slope = q == 0.0f ? s : fmaf(x * q, 1.59576912160573071f * fmaf(0.134145f * x, x, 1.0f), s);
    } else if constexpr (ACT == AVE_FP4_ACT_SILU) {
        const float s = sigmoid(x);
        value = x * s;
        slope = s * fmaf(x, 1.0f - s, 1.0f);
    } else {
        value = x;
        slope = 1.0f;
    }
}

__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
    __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<uint32_t*>(&h);
}
__device__ __forceinline__ float bf16_lo(uint32_t w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float bf16_hi(uint32_t w) { return __uint_as_float(w & 0xffff0000u); }

}  // namespace avefp4
