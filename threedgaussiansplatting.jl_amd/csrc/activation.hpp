// activation.hpp — the activations of group norm and of linear layers, with their derivatives.
#pragma once

#include "common.hpp"

namespace tdgs {

// act(z), and its derivative in *slope where wanted. SiLU: z s, s + y (1 - s) with s = 1 / (1 + e^-z).
// GELU: z cdf(z), cdf + z e^(-z^2 / 2) / sqrt(2 pi); the normal distribution's tail is
// erfc(x) = (a1 t + .. + a5 t^5) e^(-x^2), t = 1 / (1 + p x), off by 1.5e-7 at most (Abramowitz & Stegun
// 7.1.26), which takes the exponential that the derivative needs anyway: 0.8e-7 in cdf, one rounding.
template <int ACT, bool SLOPE>
__device__ __forceinline__ float act_value(float z, float* slope) {
    if constexpr (ACT == TDGS_ACT_IDENTITY) {
        if (SLOPE) *slope = 1.0f;
        return z;
    } else if constexpr (ACT == TDGS_ACT_RELU) {
        if (SLOPE) *slope = z > 0.0f ? 1.0f : 0.0f;
        return z < 0.0f ? 0.0f : z;   // (NaN stays)
    } else if constexpr (ACT == TDGS_ACT_SILU) {
        const float s = __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-kLog2e * z));
        const float y = z * s;
        // (infinities, as which float16 keeps a z past its range, have slopes of 0 and 1: at both ends a factor is zero,
        // which the largest magnitudes that are taken leave zero; NaN is s's)
        if (SLOPE) *slope = __builtin_fmaf(__builtin_amdgcn_fmed3f(z, -1e30f, 1e30f) * s, 1.0f - s, s);
        return y;
    } else {
        const float ax = fabsf(z) * 0.70710678118654752f;
        const float t = __builtin_amdgcn_rcpf(__builtin_fmaf(0.3275911f, ax, 1.0f));
        const float e = __builtin_amdgcn_exp2f(-0.5f * kLog2e * z * z);
        float a = __builtin_fmaf(1.061405429f, t, -1.453152027f);
        a = __builtin_fmaf(a, t, 1.421413741f);
        a = __builtin_fmaf(a, t, -0.284496736f);
        a = __builtin_fmaf(a, t, 0.254829592f);
        const float tail = 0.5f * a * t * e;
        const float cdf = z < 0.0f ? tail : 1.0f - tail;
        if (SLOPE) *slope = __builtin_fmaf(z * 0.39894228040143268f, e, cdf);
        return z * cdf;
    }
}

}  // namespace tdgs
