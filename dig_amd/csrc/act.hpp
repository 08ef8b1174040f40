// Activations of the trainable block operators and their slopes, fp32.
#pragma once
#include "common.hpp"

// a launch holds fewer than 2^32 threads
inline bool grid_fits(long long blocks, int threads) { return blocks * threads < (1ll << 32); }

enum { ACT_NONE = DIG_ACT_NONE, ACT_RELU = DIG_ACT_RELU, ACT_GELU = DIG_ACT_GELU, ACT_SILU = DIG_ACT_SILU };

// Phi(u) of the standard normal and E = exp(-u^2 / 2): Phi(-a) = E erfcx(a / sqrt 2) / 2 with erfcx as a polynomial in t = 1 / (1 + 0.42 a / sqrt 2),
// degree 8, fitted here for the least relative error over 0 <= a <= 13 (1.7e-7; 6e-7 evaluated in fp32) - one exp and one rcp serve the
// value and the slope, and the lower tail keeps its relative accuracy, which (1 + erf) / 2 does not.  For values that end in bf16; erff
// itself costs three times as many instructions.
__device__ __forceinline__ void normal_cdf(float u, float& cdf, float& e) {
    const float a = fabsf(u), t = __builtin_amdgcn_rcpf(fmaf(0.29698484809834996f, a, 1.f));
    float h = fmaf(t, 0.03510759562954625f, -0.16009482814557335f);
    h = fmaf(h, t, 0.22027828479590017f);
    h = fmaf(h, t, -0.06520910496275273f);
    h = fmaf(h, t, 0.1343422932710867f);
    h = fmaf(h, t, 0.09737201127785354f);
    h = fmaf(h, t, 0.1197914483732252f);
    h = fmaf(h, t, 0.11841221521044045f);
    e = __builtin_amdgcn_exp2f(u * u * -0.72134752044448170f);
    h *= t * e;
    cdf = u > 0.f ? 1.f - h : h;
}

template <typename T, int ACT> __device__ __forceinline__ float act_val(float u) {
    if constexpr (ACT == ACT_RELU) return u < 0.f ? 0.f : u;  // keeps a NaN
    else if constexpr (ACT == ACT_GELU) {
        if constexpr (sizeof(T) == 2) {
            float c, e;
            normal_cdf(u, c, e);
            return u * c;
        } else {
            return gelu_erf_f(u);
        }
    } else if constexpr (ACT == ACT_SILU) return silu_f(u);
    else return u;
}
template <typename T, int ACT> __device__ __forceinline__ float act_slope(float u) {
    if constexpr (ACT == ACT_RELU) return u > 0.f ? 1.f : 0.f;
    else if constexpr (ACT == ACT_GELU) {
        if constexpr (sizeof(T) == 2) {
            float c, e;
            normal_cdf(u, c, e);
            return fmaf(u * e, 0.39894228040143268f, c);
        } else {
            return 0.5f * (1.f + erff(u * 0.70710678118654752f)) + u * __expf(-0.5f * u * u) * 0.39894228040143268f;
        }
    } else if constexpr (ACT == ACT_SILU) {
        const float s = __builtin_amdgcn_rcpf(1.0f + __expf(-u));
        return s * fmaf(u, 1.f - s, 1.f);
    } else return 1.f;
}
