// Activations of the pointwise linear layer and their derivatives, in fp32.
#pragma once

#include "common.cuh"

namespace spconv {

template <int ACT>
__device__ __forceinline__ float act_value(float z) {
    if constexpr (ACT == SPCONV_ACT_RELU) return z < 0.f ? 0.f : z;          // NaN stays NaN
    if constexpr (ACT == SPCONV_ACT_GELU) return 0.5f * z * (1.f + erff(z * 0.70710678f));
    if constexpr (ACT == SPCONV_ACT_SILU) return z / (1.f + expf(-z));
    return z;
}

template <int ACT>
__device__ __forceinline__ float act_slope(float z) {
    if constexpr (ACT == SPCONV_ACT_RELU) return z > 0.f ? 1.f : 0.f;
    if constexpr (ACT == SPCONV_ACT_GELU)
        return 0.5f * (1.f + erff(z * 0.70710678f)) + z * 0.39894228f * expf(-0.5f * z * z);
    if constexpr (ACT == SPCONV_ACT_SILU) {
        const float s = 1.f / (1.f + expf(-z));
        return s * (1.f + z * (1.f - s));
    }
    return 1.f;
}

// Calls f with the activation as a compile-time constant.
template <typename F>
inline int act_dispatch(int activation, F f) {
    switch (activation) {
        case SPCONV_ACT_RELU: return f(std::integral_constant<int, SPCONV_ACT_RELU>{});
        case SPCONV_ACT_GELU: return f(std::integral_constant<int, SPCONV_ACT_GELU>{});
        case SPCONV_ACT_SILU: return f(std::integral_constant<int, SPCONV_ACT_SILU>{});
        default: return f(std::integral_constant<int, SPCONV_ACT_NONE>{});
    }
}

}  // namespace spconv
