// The activations that group norm and the dense layer apply in their own kernels, and their slopes.
#pragma once

#include "common.h"

namespace dopt {

inline bool known_activation(int act) { return act >= DOPT_HIP_ACT_NONE && act <= DOPT_HIP_ACT_SILU; }

// Phi(z), the normal distribution function: erfc keeps its relative accuracy far below zero, where 1 + erf would cancel.
__device__ inline float normal_cdf(float z) { return 0.5f * erfcf(z * -0.70710678f); }

template <int kAct>
__device__ inline float act_value(float z)
{
    if constexpr (kAct == DOPT_HIP_ACT_RELU) return z < 0.0f ? 0.0f : z;   // NaN stays, as dopt_hip_relu_fwd
    if constexpr (kAct == DOPT_HIP_ACT_GELU) return z * normal_cdf(z);
    if constexpr (kAct == DOPT_HIP_ACT_SILU) return z / (1.0f + expf(-z));
    return z;
}

// dy times the activation's slope at z.
template <int kAct>
__device__ inline float act_grad(float dy, float z)
{
    if constexpr (kAct == DOPT_HIP_ACT_RELU) return z > 0.0f ? dy : 0.0f;   // as dopt_hip_relu_bwd
    if constexpr (kAct == DOPT_HIP_ACT_GELU) return dy * (normal_cdf(z) + z * (0.39894228f * expf(-0.5f * z * z)));
    if constexpr (kAct == DOPT_HIP_ACT_SILU) {
        const float s = 1.0f / (1.0f + expf(-z));
        return dy * (s * (1.0f + z * (1.0f - s)));
    }
    return dy;
}

// Calls f with the activation as a compile-time constant (f takes a std::integral_constant).
template <class F>
auto with_activation(int act, F &&f)
{
    switch (act) {
    case DOPT_HIP_ACT_RELU: return f(std::integral_constant<int, DOPT_HIP_ACT_RELU>{});
    case DOPT_HIP_ACT_GELU: return f(std::integral_constant<int, DOPT_HIP_ACT_GELU>{});
    case DOPT_HIP_ACT_SILU: return f(std::integral_constant<int, DOPT_HIP_ACT_SILU>{});
    default: return f(std::integral_constant<int, DOPT_HIP_ACT_NONE>{});
    }
}

}  // namespace dopt
