// The activations that group norm and the dense layer apply in their own kernels, and their slopes.
#pragma once

#include <type_traits>

#include "common.h"

namespace dopt {

inline bool known_activation(int act) { return act >= DOPT_HIP_ACT_NONE && act <= DOPT_HIP_ACT_SILU; }

// exp(x) by the hardware's 2^x: within 2^-23 (1 + |x|) of it.
__device__ __forceinline__ float fast_exp(float x) { return __builtin_amdgcn_exp2f(x * 1.44269504f); }

// 1 - Phi(t) = exp(-t^2 / 2) R(t) for t >= 0, Phi the normal distribution function.  R falls smoothly from 1/2 like 0.4 / t; in
// s = 1 / (1 + 0.27 t) a polynomial of nine terms fits it to 2.6e-8 of itself up to t = 6 and to 3.1e-8 up to 13.5, where the density leaves fp32's range
// (least squares of the relative error, weighted towards the largest; the form is that of Abramowitz and Stegun 26.2.17).  Far
// below zero Phi keeps its relative accuracy so, but for what fast_exp leaves of it, where 1 + erf would cancel.  `density` receives exp(-z^2 / 2).
__device__ __forceinline__ float normal_cdf(float z, float &density)
{
    const float t = __builtin_fabsf(z), s = __builtin_amdgcn_rcpf(__builtin_fmaf(0.27f, t, 1.0f));
    float r = 0.028914351f;
    r = __builtin_fmaf(r, s, -0.126250967f);
    r = __builtin_fmaf(r, s, 0.169282883f);
    r = __builtin_fmaf(r, s, -0.0686115995f);
    r = __builtin_fmaf(r, s, 0.107393175f);
    r = __builtin_fmaf(r, s, 0.0722428784f);
    r = __builtin_fmaf(r, s, 0.101758517f);
    r = __builtin_fmaf(r, s, 0.107550599f);
    r = __builtin_fmaf(r, s, 0.107720174f);
    density = fast_exp(-0.5f * z * z);
    const float tail = density * (r * s);
    return z > 0.0f ? 1.0f - tail : tail;
}

__device__ __forceinline__ float sigmoid(float z) { return __builtin_amdgcn_rcpf(1.0f + fast_exp(-z)); }

template <int kAct>
__device__ __forceinline__ float act_value(float z)
{
    if constexpr (kAct == DOPT_HIP_ACT_RELU) return z < 0.0f ? 0.0f : z;   // NaN stays, as dopt_hip_relu_fwd
    if constexpr (kAct == DOPT_HIP_ACT_GELU) {
        float density;
        return z * normal_cdf(z, density);
    }
    if constexpr (kAct == DOPT_HIP_ACT_SILU) return z * sigmoid(z);
    return z;
}

// dy times the activation's slope at z.
template <int kAct>
__device__ __forceinline__ float act_grad(float dy, float z)
{
    if constexpr (kAct == DOPT_HIP_ACT_RELU) return z > 0.0f ? dy : 0.0f;   // as dopt_hip_relu_bwd
    if constexpr (kAct == DOPT_HIP_ACT_GELU) {
        float density;
        const float cdf = normal_cdf(z, density);
        return dy * __builtin_fmaf(z, 0.39894228f * density, cdf);
    }
    if constexpr (kAct == DOPT_HIP_ACT_SILU) {
        const float s = sigmoid(z);
        return dy * (s * __builtin_fmaf(z, 1.0f - s, 1.0f));
    }
    return dy;
}

// Calls f with the activation as a compile-time constant (f takes a std::integral_constant).
template <class F>
__host__ __device__ __forceinline__ auto with_activation(int act, F &&f)
{
    switch (act) {
    case DOPT_HIP_ACT_RELU: return f(std::integral_constant<int, DOPT_HIP_ACT_RELU>{});
    case DOPT_HIP_ACT_GELU: return f(std::integral_constant<int, DOPT_HIP_ACT_GELU>{});
    case DOPT_HIP_ACT_SILU: return f(std::integral_constant<int, DOPT_HIP_ACT_SILU>{});
    default: return f(std::integral_constant<int, DOPT_HIP_ACT_NONE>{});
    }
}

}  // namespace dopt
