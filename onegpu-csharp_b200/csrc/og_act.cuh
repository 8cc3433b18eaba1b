// The activations that the product's epilogue and the mixture-of-experts layer apply to a float32 value
// (og_activation of the C ABI):
//   none       v
//   relu       max(v, 0), NaN stays NaN
//   gelu       v * Phi(v) = v / 2 * (1 + erf(v / sqrt 2))
//   gelu_tanh  v / 2 * (1 + tanh(u)), u = sqrt(2 / pi) * (v + 0.044715 v^3), formed as v / (1 + exp(-2 u)): the same
//              value, with no cancellation for negative v
//   silu       v / (1 + exp(-v))
// The exponentials and quotients use the fast forms (ex2.approx, rcp.approx): their relative error of a few 2^-23 is
// the size of the float32 rounding of the result itself.
#pragma once

#include <cuda_runtime.h>

namespace og {

enum Activation : int { ACT_NONE = 0, ACT_RELU = 1, ACT_GELU = 2, ACT_GELU_TANH = 3, ACT_SILU = 4 };

// v / (1 + exp(-t)). For exp(-t) past 2^126 the quotient is 0, as it should be.
__device__ __forceinline__ float logistic_times(float v, float t) { return __fdividef(v, 1.0f + __expf(-t)); }

// v * Phi(v) with erf by the rational approximation of Hastings, "Approximations for Digital Computers" (1955), 7.1.26 in
// Abramowitz and Stegun: erfc(z) = (a1 t + .. + a5 t^5) exp(-z^2), t = 1 / (1 + p z), z >= 0, off by at most 1.5e-7. With
// z = |v| / sqrt 2, Phi(-|v|) = erfc(z) / 2 directly and Phi(|v|) = 1 - that: no cancellation on either side. A third of
// erff's instructions.
__device__ __forceinline__ float gelu(float v) {
    const float z = fabsf(v) * 0.70710678f;
    const float t = __fdividef(1.0f, fmaf(0.3275911f, z, 1.0f));
    const float poly =
        t * fmaf(t, fmaf(t, fmaf(t, fmaf(t, 0.5f * 1.061405429f, 0.5f * -1.453152027f), 0.5f * 1.421413741f), 0.5f * -0.284496736f),
                 0.5f * 0.254829592f);
    const float tail = poly * __expf(-z * z);  // Phi(-|v|)
    return v * (v < 0.0f ? tail : 1.0f - tail);
}

template <int KIND>
__device__ __forceinline__ float activate(float v) {
    if constexpr (KIND == ACT_RELU) {
        return v < 0.0f ? 0.0f : v;
    } else if constexpr (KIND == ACT_GELU) {
        return gelu(v);
    } else if constexpr (KIND == ACT_GELU_TANH) {
        return logistic_times(v, 1.5957691f * v * fmaf(0.044715f * v, v, 1.0f));
    } else if constexpr (KIND == ACT_SILU) {
        return logistic_times(v, v);
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
