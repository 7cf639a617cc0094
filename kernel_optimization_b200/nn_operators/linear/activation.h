// Activations of the fused linear layer and their slopes, on FP32 values.
//
//   relu       max(z, 0); slope 1 for z > 0, else 0
//   gelu       z Phi(z), Phi the normal distribution function; slope Phi(z) + z phi(z)
//   gelu_tanh  z s(2 c (z + 0.044715 z^3)), c = sqrt(2 / pi), s the logistic function: 0.5 z (1 + tanh(..)) written
//              without the cancellation of 1 + tanh
//   silu       z s(z); slope s(z) (1 + z (1 - s(z)))
//
// Two forms.  kExact, for results kept in FP32: the CUDA library's erfcf / expf and IEEE division, one value at a time.
// Fast, for results rounded to 16 bits, where the epilogue's instruction slots count: two values at a time on packed FP32
// arithmetic, with the special-function unit's 2^x and 1/x (relative error about 2^-22) used as little as possible -- it
// takes four times as long as an FMA:
//   gelu        Phi(-a) = 2^p(a) for a = |z|, Phi(a) = 1 - Phi(-a).  p is log2 Phi(-a), almost a parabola, as a polynomial of
//               degree 7 (least maximal error on [0, 5.5], found by linear programming on 4000 Chebyshev nodes): 5e-6 relative
//               in Phi up to there, and it falls on below the FP32 range, so a gelu is off by at most 6e-7
//   its slope   g(-a) = Phi(-a) - a phi(a) = e^(-a^2 / 2) r(a), g(a) = 1 - g(-a).  r is of degree 9, fitted on [0, 5.5] by linear
//               programming (20000 Chebyshev nodes) to an error that is small both ways: 8e-7 of g absolutely and, from a = 2 on, 7.5e-4
//               of g itself; beyond, g is below 6e-7 and off by at most 1.1e-9.  So gradients through z = -5 keep their size:
//               degree 8 with an absolute bound of 1e-6 was off by 8 % at -4.9 and by several times the slope at -6.  Every further
//               degree costs 1.5 % of a product (16384 x 1024 x 4096: degree 8 125 us, 9 127, 10 130; Phi and phi apart, two powers of 2,
//               good to 1.4e-4 as far as -13, 134)
//   logistic    one ex2 and one reciprocal a value; arguments are held above -200 (silu) and -40 (gelu_tanh), where it is 0
// Limits are put with max.NaN / min.NaN: a NaN stays one; an infinity gives the limit, inf or 0, and a slope of 1 or 0.  A value's
// result depends on nothing but the value: every form of the epilogue gives the same bits for the same sums.
// Half a step of FP16 is 2.4e-4 of a value.
#pragma once

#include <type_traits>

#include "../../common/common.h"

namespace ko {

enum Activation : int { kActNone = 0, kActRelu = 1, kActGelu = 2, kActGeluTanh = 3, kActSilu = 4, kActCount = 5 };

constexpr float kLog2e = 1.44269504088896341f;
constexpr float kTwoRoot2OverPi = 2.0f * 0.79788456080286536f;

__device__ __forceinline__ float max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float min_nan(float a, float b) {
    float r;
    asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}

// ---- exact forms ----
// (__fmul_rn, __fadd_rn: no contraction with what the library functions begin or end with, so that they give the same bits
// wherever they are expanded)
__device__ __forceinline__ float logistic_exact(float v) { return 1.0f / __fadd_rn(1.0f, expf(-v)); }
__device__ __forceinline__ float normal_cdf_exact(float z) { return 0.5f * erfcf(__fmul_rn(-z, 0.70710678118654752f)); }

// At an infinity the limit: z is held (as far out as where the other factor is 0 or 1 in FP32) wherever it would meet a 0.
template <int kAct>
__device__ __forceinline__ float activate_exact(float z) {
    if constexpr (kAct == kActRelu) return z < 0.f ? 0.f : z;  // NaN stays NaN
    if constexpr (kAct == kActGelu) {
        const float t = max_nan(z, -40.f);
        return t * normal_cdf_exact(t);
    }
    if constexpr (kAct == kActGeluTanh) {
        const float t = max_nan(z, -40.f);
        return t * logistic_exact(t * fmaf(kTwoRoot2OverPi * 0.044715f, t * t, kTwoRoot2OverPi));
    }
    if constexpr (kAct == kActSilu) {
        const float t = max_nan(z, -200.f);
        return t * logistic_exact(t);
    }
    return z;
}
template <int kAct>
__device__ __forceinline__ float slope_exact(float z) {
    if constexpr (kAct == kActRelu) return z > 0.f ? 1.f : 0.f;
    if constexpr (kAct == kActGelu) {
        const float t = min_nan(max_nan(z, -40.f), 40.f);
        return fmaf(t * 0.39894228040143268f, expf(-0.5f * t * t), normal_cdf_exact(t));
    }
    if constexpr (kAct == kActGeluTanh) {
        const float s = logistic_exact(z * fmaf(kTwoRoot2OverPi * 0.044715f, z * z, kTwoRoot2OverPi));
        // s (1 - s) first: 0 for large |z|, where z^2 may be infinite
        const float bend = s * (1.0f - s);
        return bend == 0.f ? s : fmaf(z * bend, fmaf(3.0f * kTwoRoot2OverPi * 0.044715f, z * z, kTwoRoot2OverPi), s);
    }
    if constexpr (kAct == kActSilu) {
        const float t = min_nan(max_nan(z, -200.f), 200.f), s = logistic_exact(t);
        return s * fmaf(t, 1.0f - s, 1.0f);
    }
    return 1.f;
}

// ---- fast forms, two values ----
__device__ __forceinline__ f32x2 both(float v) { return pair_of(v, v); }

__device__ __forceinline__ f32x2 at_least_pair(f32x2 z, float limit) {
    float a, b;
    pair_split(z, a, b);
    return pair_of(max_nan(a, limit), max_nan(b, limit));
}
__device__ __forceinline__ f32x2 at_most_pair(f32x2 z, float limit) {
    float a, b;
    pair_split(z, a, b);
    return pair_of(min_nan(a, limit), min_nan(b, limit));
}

// |z|, at most `limit`
__device__ __forceinline__ f32x2 magnitude_pair(f32x2 z, float limit) {
    float a, b;
    pair_split(z, a, b);
    return pair_of(min_nan(fabsf(a), limit), min_nan(fabsf(b), limit));
}

// 1 / (1 + 2^x), x = -v log2(e) for the logistic function of v; 0 where 2^x is infinite.  Each value has a reciprocal of its own: one for
// both, 1 / u = v / (u v), makes the last bit of a value depend on which other one it is paired with, and the forms of the epilogue
// pair columns, rows, or a value with itself.
__device__ __forceinline__ f32x2 logistic_pair(f32x2 x) {
    float x0, x1, u, v;
    pair_split(x, x0, x1);
    const f32x2 d = pair_add(pair_of(exp2_approx(x0), exp2_approx(x1)), both(1.f));
    pair_split(d, u, v);
    return pair_of(rcp_approx(u), rcp_approx(v));
}
// f(-|z|) where z is negative, else 1 - f(-|z|)
__device__ __forceinline__ f32x2 reflect_pair(f32x2 z, f32x2 low) {
    float z0, z1, a, b;
    pair_split(z, z0, z1);
    pair_split(low, a, b);
    return pair_of(z0 > 0.f ? 1.f - a : a, z1 > 0.f ? 1.f - b : b);
}

template <int kAct>
__device__ __forceinline__ f32x2 activate_pair(f32x2 z) {
    if constexpr (kAct == kActRelu) {
        float a, b;
        pair_split(z, a, b);
        return pair_of(a < 0.f ? 0.f : a, b < 0.f ? 0.f : b);
    } else if constexpr (kAct == kActGelu) {
        // z Phi(z) = max(z, 0) - |z| Phi(-|z|)
        const f32x2 a = magnitude_pair(z, 32.f);
        f32x2 p = pair_fma(a, both(-1.7937167058e-06f), both(6.0908834712e-05f));
        p = pair_fma(a, p, both(-9.2606159160e-04f));
        p = pair_fma(a, p, both(8.4938677028e-03f));
        p = pair_fma(a, p, both(-5.3938016295e-02f));
        p = pair_fma(a, p, both(-4.5848044753e-01f));
        p = pair_fma(a, p, both(-1.1512467861e+00f));
        p = pair_fma(a, p, both(-9.9999547005e-01f));
        float p0, p1, z0, z1;
        pair_split(p, p0, p1);
        pair_split(z, z0, z1);
        return pair_fma(a, pair_of(-exp2_approx(p0), -exp2_approx(p1)), pair_of(fmaxf(z0, 0.f), fmaxf(z1, 0.f)));
    } else if constexpr (kAct == kActGeluTanh) {
        const f32x2 t = at_least_pair(z, -40.f);
        const f32x2 u = pair_fma(both(-kLog2e * kTwoRoot2OverPi * 0.044715f), pair_mul(t, t), both(-kLog2e * kTwoRoot2OverPi));
        return pair_mul(t, logistic_pair(pair_mul(t, u)));
    } else if constexpr (kAct == kActSilu) {
        const f32x2 t = at_least_pair(z, -200.f);
        return pair_mul(t, logistic_pair(pair_mul(t, both(-kLog2e))));
    }
    return z;
}

template <int kAct>
__device__ __forceinline__ f32x2 slope_pair(f32x2 z) {
    if constexpr (kAct == kActRelu) {
        float a, b;
        pair_split(z, a, b);
        return pair_of(a > 0.f ? 1.f : 0.f, b > 0.f ? 1.f : 0.f);
    } else if constexpr (kAct == kActGelu) {
        float e0, e1;
        const f32x2 a = magnitude_pair(z, 16.f);  // e^-128 = 0; the polynomial stays finite
        pair_split(pair_mul(pair_mul(a, a), both(-0.5f * kLog2e)), e0, e1);
        f32x2 r = pair_fma(a, both(-3.9254905460e-06f), both(9.0380679467e-05f));
        r = pair_fma(a, r, both(-9.0088939760e-04f));
        r = pair_fma(a, r, both(5.2183372900e-03f));
        r = pair_fma(a, r, both(-2.0162180066e-02f));
        r = pair_fma(a, r, both(5.7404585183e-02f));
        r = pair_fma(a, r, both(-1.3062055409e-01f));
        r = pair_fma(a, r, both(2.4944375455e-01f));
        r = pair_fma(a, r, both(-7.9783397913e-01f));
        r = pair_fma(a, r, both(4.9999925494e-01f));
        return reflect_pair(z, pair_mul(r, pair_of(exp2_approx(e0), exp2_approx(e1))));
    } else if constexpr (kAct == kActGeluTanh) {
        // the slope is 1 beyond 16; held there, z^2 times nothing stays nothing
        const f32x2 t = at_most_pair(at_least_pair(z, -40.f), 16.f), t2 = pair_mul(t, t);
        const f32x2 u = pair_fma(both(-kLog2e * kTwoRoot2OverPi * 0.044715f), t2, both(-kLog2e * kTwoRoot2OverPi));
        const f32x2 s = logistic_pair(pair_mul(t, u));
        const f32x2 bend = pair_mul(t, pair_fma(pair_mul(s, both(-1.f)), s, s));
        return pair_fma(bend, pair_fma(both(3.0f * kTwoRoot2OverPi * 0.044715f), t2, both(kTwoRoot2OverPi)), s);
    } else if constexpr (kAct == kActSilu) {
        // 1 beyond 20 (to 4e-8); held there, t times the last bit of s, which the reciprocal may leave below 1, stays 2e-6
        const f32x2 t = at_most_pair(at_least_pair(z, -200.f), 20.f), s = logistic_pair(pair_mul(t, both(-kLog2e)));
        return pair_mul(s, pair_fma(t, pair_fma(s, both(-1.f), both(1.f)), both(1.f)));
    }
    return both(1.f);
}

// one value in either form
template <int kAct, bool kExact>
__device__ __forceinline__ float activate(float z) {
    if constexpr (kExact) return activate_exact<kAct>(z);
    float lo, hi;
    pair_split(activate_pair<kAct>(both(z)), lo, hi);
    return lo;
}
template <int kAct, bool kExact>
__device__ __forceinline__ float activation_slope(float z) {
    if constexpr (kExact) return slope_exact<kAct>(z);
    float lo, hi;
    pair_split(slope_pair<kAct>(both(z)), lo, hi);
    return lo;
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
