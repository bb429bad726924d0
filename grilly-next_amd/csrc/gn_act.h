// gn_act.h — activations and their slopes in the fewest instructions, for the epilogues of bf16 products (gn_linear_act_core.h; the
// passes behind fp32 ones, gn_linear_act.hip, have forms of their own).
#pragma once

#include <type_traits>

#include "gn_math.h"

namespace gn {
namespace {

// With the hardware's exponential and reciprocal (1 ulp), not the correctly rounded division of six more instructions,
// and in the fewest full-rate instructions: a 256 x 128 tile has 128 elements a lane, 0.25 us of the tile for each
// instruction of an element.
__device__ __forceinline__ float rcp(float x) { return __builtin_amdgcn_rcpf(x); }
constexpr float kLog2e = 1.4426950408889634f;
__device__ __forceinline__ float sigmoid_of(float x) { return rcp(1.0f + __builtin_amdgcn_exp2f(x * -kLog2e)); }
// (1 + tanh z) / 2 = sigmoid(2 z), 2 z = 2 sqrt(2 / pi) (x + 0.044715 x^3)
constexpr float kG1 = 2.0f * kSqrt2OverPi, kG3 = 2.0f * kSqrt2OverPi * kGeluC;
__device__ __forceinline__ float gelu_gate(float x, float xx) {
    return rcp(1.0f + __builtin_amdgcn_exp2f(x * fmaf(xx, -kLog2e * kG3, -kLog2e * kG1)));
}

// 1 - 2 / (1 + e^2x), which is good to 2^-22 of 1: towards 0, where that is too little of x, the series, whose next term is 62/2835 x^8
// (4096 x 5632 x 2048: 104 us for 99 without)
__device__ __forceinline__ float tanh_of(float x) {
    const float xx = x * x, far = fmaf(-2.0f, rcp(1.0f + __builtin_amdgcn_exp2f(x * (2.0f * kLog2e))), 1.0f);
    return fabsf(x) < 0.25f ? x * fmaf(xx, fmaf(xx, fmaf(xx, -17.0f / 315.0f, 2.0f / 15.0f), -1.0f / 3.0f), 1.0f) : far;
}

template <int KIND>
__device__ __forceinline__ float act_of(float x) {
    if constexpr (KIND == GN_ACT_RELU) return x < 0.f ? 0.f : x;  // a NaN stays
    else if constexpr (KIND == GN_ACT_GELU_TANH) return x * gelu_gate(x, x * x);
    else if constexpr (KIND == GN_ACT_GELU_ERF) return 0.5f * x * (1.0f + erff(x * 0.70710678118654752f));
    else if constexpr (KIND == GN_ACT_SILU) return x * sigmoid_of(x);
    else if constexpr (KIND == GN_ACT_TANH) return tanh_of(x);
    else return sigmoid_of(x);
}
// tanh and sigmoid at their output; of x sigmoid(u): s + x s (1 - s) u' = s (1 + (1 - s) x u')
template <int KIND>
__device__ __forceinline__ float slope_of(float x) {
    if constexpr (KIND == GN_ACT_GELU_TANH) {
        // from |x| = 20 on the gate is 0 or 1, and the slope: without the limit x u' overflows, and 0 times inf is NaN.  The gate
        // takes x itself, so that a NaN stays one.
        const float c = __builtin_amdgcn_fmed3f(x, -20.f, 20.f), xx = c * c, s = gelu_gate(x, xx);
        return s * fmaf(1.0f - s, c * fmaf(xx, 3.0f * kG3, kG1), 1.0f);
    } else if constexpr (KIND == GN_ACT_SILU) {
        const float s = sigmoid_of(x);
        return s * fmaf(1.0f - s, x, 1.0f);
    } else {
        return act_grad<KIND>(x);
    }
}

// f(its compile-time number) for an activation: KIND, or kAny: of the number at run time
constexpr int kAny = -2;
template <int KIND, bool NONE, typename F>
__device__ __forceinline__ void by_act(int kind, F&& f) {
    using std::integral_constant;
    if constexpr (KIND != kAny) {
        f(integral_constant<int, KIND>{});
        return;
    } else switch (kind) {
        case GN_ACT_RELU: f(integral_constant<int, GN_ACT_RELU>{}); break;
        case GN_ACT_GELU_TANH: f(integral_constant<int, GN_ACT_GELU_TANH>{}); break;
        case GN_ACT_GELU_ERF: f(integral_constant<int, GN_ACT_GELU_ERF>{}); break;
        case GN_ACT_SILU: f(integral_constant<int, GN_ACT_SILU>{}); break;
        case GN_ACT_TANH: f(integral_constant<int, GN_ACT_TANH>{}); break;
        default:
            if (!NONE || kind == GN_ACT_SIGMOID) f(integral_constant<int, GN_ACT_SIGMOID>{});
            else f(integral_constant<int, GN_ACT_NONE>{});
    }
}

}  // namespace
}  // namespace gn
