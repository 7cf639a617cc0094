// Activations of the fused linear layer and their slopes, on FP32 values.
//
//   relu       max(z, 0); slope 1 for z > 0, else 0
//   gelu       z Phi(z), Phi the normal distribution function; slope Phi(z) + z phi(z)
//   gelu_tanh  z s(2 c (z + 0.044715 z^3)), c = sqrt(2 / pi), s the logistic function: 0.5 z (1 + tanh(..)) written
//              without the cancellation of 1 + tanh
//   silu       z s(z); slope s(z) (1 + z (1 - s(z)))
//
// kExact (results kept in FP32): the CUDA library's erfcf / expf and IEEE division.  Otherwise the result is rounded to
// 16 bits and the special-function unit's 2^x and 1/x (relative error about 2^-22) serve, with Phi from formula 7.1.26 of
// Abramowitz and Stegun (absolute error 1.5e-7): far below half a step of BF16 (2^-9) or FP16 (2^-12) of every value
// that is not itself below 1e-4.
#pragma once

#include "../../common/common.h"

namespace ko {

enum Activation : int { kActNone = 0, kActRelu = 1, kActGelu = 2, kActGeluTanh = 3, kActSilu = 4, kActCount = 5 };

constexpr float kLog2e = 1.44269504088896341f;

template <bool kExact>
__device__ __forceinline__ float exp_of(float x) {
    if constexpr (kExact) return expf(x);
    return exp2_approx(x * kLog2e);
}
template <bool kExact>
__device__ __forceinline__ float reciprocal(float x) {
    if constexpr (kExact) return 1.0f / x;
    return rcp_approx(x);
}
// 1 / (1 + e^-v)
template <bool kExact>
__device__ __forceinline__ float logistic(float v) {
    return reciprocal<kExact>(1.0f + exp_of<kExact>(-v));
}
// Phi(z); `bell` receives e^(-z^2 / 2)
template <bool kExact>
__device__ __forceinline__ float normal_cdf(float z, float &bell) {
    constexpr float kSqrtHalf = 0.70710678118654752f;
    bell = exp_of<kExact>(-0.5f * z * z);
    if constexpr (kExact) {
        return 0.5f * erfcf(-z * kSqrtHalf);
    } else {
        const float t = rcp_approx(fmaf(0.3275911f * kSqrtHalf, fabsf(z), 1.0f));
        float poly = fmaf(t, 1.061405429f, -1.453152027f);
        poly = fmaf(t, poly, 1.421413741f);
        poly = fmaf(t, poly, -0.284496736f);
        poly = fmaf(t, poly, 0.254829592f);
        const float tail = 0.5f * t * poly * bell;  // Phi(-|z|)
        return z > 0.f ? 1.0f - tail : tail;
    }
}

template <int kAct, bool kExact>
__device__ __forceinline__ float activate(float z) {
    if constexpr (kAct == kActRelu) {
        return z < 0.f ? 0.f : z;  // NaN stays NaN
    } else if constexpr (kAct == kActGelu) {
        float bell;
        return z * normal_cdf<kExact>(z, bell);
    } else if constexpr (kAct == kActGeluTanh) {
        constexpr float c2 = 2.0f * 0.79788456080286536f;
        return z * logistic<kExact>(z * fmaf(c2 * 0.044715f, z * z, c2));
    } else if constexpr (kAct == kActSilu) {
        return z * logistic<kExact>(z);
    }
    return z;
}

template <int kAct, bool kExact>
__device__ __forceinline__ float activation_slope(float z) {
    if constexpr (kAct == kActRelu) {
        return z > 0.f ? 1.f : 0.f;
    } else if constexpr (kAct == kActGelu) {
        float bell;
        const float cdf = normal_cdf<kExact>(z, bell);
        return fmaf(z * 0.39894228040143268f, bell, cdf);
    } else if constexpr (kAct == kActGeluTanh) {
        constexpr float c2 = 2.0f * 0.79788456080286536f;
        const float s = logistic<kExact>(z * fmaf(c2 * 0.044715f, z * z, c2));
        return fmaf(z * s * (1.0f - s), fmaf(3.0f * c2 * 0.044715f, z * z, c2), s);
    } else if constexpr (kAct == kActSilu) {
        const float s = logistic<kExact>(z);
        return s * fmaf(z, 1.0f - s, 1.0f);
    }
    return 1.f;
}

// f(std::integral_constant<int, act>) for the activation chosen at run time
template <class F>
__device__ __forceinline__ void with_activation(int act, F &&f) {
    switch (act) {
        case kActRelu: f(std::integral_constant<int, kActRelu>{}); break;
        case kActGelu: f(std::integral_constant<int, kActGelu>{}); break;
        case kActGeluTanh: f(std::integral_constant<int, kActGeluTanh>{}); break;
        case kActSilu: f(std::integral_constant<int, kActSilu>{}); break;
        default: f(std::integral_constant<int, kActNone>{}); break;
    }
}

}  // namespace ko
