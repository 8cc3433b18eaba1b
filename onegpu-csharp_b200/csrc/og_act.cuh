// The activations that the product's epilogue and the mixture-of-experts layer apply to a float32 value
// (og_activation of the C ABI):
//   none       v
//   relu       max(v, 0), NaN stays NaN
//   gelu       v * Phi(v) = v / 2 * (1 + erf(v / sqrt 2))
//   gelu_tanh  v / 2 * (1 + tanh(u)), u = sqrt(2 / pi) * (v + 0.044715 v^3), formed as v / (1 + exp(-2 u)): the same
//              value, with no cancellation for negative v
//   silu       v / (1 + exp(-v))
// Errors relative to the result, negative tails included: silu 2^-21, gelu 26 x 2^-24, gelu_tanh (5 + 9 |u|) 2^-23, whose
// exponential's argument 2 u is itself a rounded one. Quotients are the fast ones (2 units in the last place for divisors
// of this size), exponentials expf's; for tanh GELU the fast one (2 + 1.173 |2 u| units), which adds less than the argument's
// rounding does: with expf 8192 x 8192 x 2048 into float32 took 199 us, so 187, and the results' distance from 64 bits is
// 6.0e-8 with either.
#pragma once

#include <cuda_runtime.h>

namespace og {

enum Activation : int { ACT_NONE = 0, ACT_RELU = 1, ACT_GELU = 2, ACT_GELU_TANH = 3, ACT_SILU = 4 };

// v / (1 + exp(-t)) for v and t of one sign: with the exponential of -|t| the divisor stays between 1 and 2.
template <bool FAST>
__device__ __forceinline__ float logistic_times(float v, float t) {
    const float e = FAST ? __expf(-fabsf(t)) : expf(-fabsf(t));
    return __fdividef(t < 0.0f ? v * e : v, 1.0f + e);
}

// v * Phi(v). Phi(-a) = exp(-a^2 / 2) g(a) for a = |v|, with g(a) = exp(a^2 / 2) erfc(a / sqrt 2) / 2 as a polynomial of degree
// 8 in t = 1 / (1 + 0.31 a) without a constant term: fitted to g in 64 bits (least relative error over 0 .. 14.6, 2.9 x 2^-24
// with these coefficients). The square's rounding is put back by its rest l, and no digit cancels on either side of zero. A
// third of the instructions of erfcf on both sides of its branches; the 1955 rational approximation that was here, good to
// 1.5e-7 absolutely, was off by 5e-5 of the result at v = -3 and 2e-3 at -5.
__device__ __forceinline__ float gelu(float v) {
    const float a = fminf(fabsf(v), 15.0f);  // past it Phi(-a) is 0 in float32
    const float h = a * a, l = fmaf(a, a, -h);
    float e = expf(-0.5f * h);
    e = fmaf(e, -0.5f * l, e);
    const float t = __fdividef(1.0f, fmaf(0.31f, a, 1.0f));
    float g = 0.0358747765f;
    g = fmaf(g, t, -0.141749799f);
    g = fmaf(g, t, 0.155332953f);
    g = fmaf(g, t, -0.0151631441f);
    g = fmaf(g, t, 0.110257111f);
    g = fmaf(g, t, 0.107723266f);
    g = fmaf(g, t, 0.124068588f);
    g = fmaf(g, t, 0.123656332f);
    const float tail = g * t * e;  // Phi(-a)
    return v * (v < 0.0f ? tail : 1.0f - tail);
}

template <int KIND>
__device__ __forceinline__ float activate(float v) {
    if constexpr (KIND == ACT_RELU) {
        return v < 0.0f ? 0.0f : v;
    } else if constexpr (KIND == ACT_GELU) {
        return gelu(v);
    } else if constexpr (KIND == ACT_GELU_TANH) {
        return logistic_times<true>(v, 1.5957691f * v * fmaf(0.044715f * v, v, 1.0f));
    } else if constexpr (KIND == ACT_SILU) {
        return logistic_times<false>(v, v);
    } else {
        return v;
    }
}

template <int N, int KIND>
__device__ __forceinline__ void activate_each(float (&f)[N]) {
#pragma unroll
    for (int i = 0; i < N; i++) f[i] = activate<KIND>(f[i]);
}

// The activation `kind` (the same for a whole launch) applied to N values: one branch per N of them.
template <int N>
__device__ __forceinline__ void activate_all(float (&f)[N], int kind) {
    if (kind == ACT_NONE) return;
    if (kind == ACT_SILU)
        activate_each<N, ACT_SILU>(f);
    else if (kind == ACT_GELU_TANH)
        activate_each<N, ACT_GELU_TANH>(f);
    else if (kind == ACT_GELU)
        activate_each<N, ACT_GELU>(f);
    else
        activate_each<N, ACT_RELU>(f);
}

}  // namespace og
