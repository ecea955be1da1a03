// Activations of the gated and the linear projections: value and slope in float32.
#pragma once

#include <hip/hip_runtime.h>

#include <type_traits>

#include "common.hpp"

namespace zcgvs_hip {
namespace {

// 1 / (1 + exp(-x)): exp2 and the reciprocal of the hardware, each within 1 ulp. The reciprocal gives zeros in the
// place of results below 2^-126, so it is taken of 2^-32 of the sum.
__device__ __forceinline__ float logistic(float x) {
    constexpr float kSmall = 0x1p-32f;
    return kSmall * __builtin_amdgcn_rcpf(fmaf(__builtin_amdgcn_exp2f(-1.44269504f * x), kSmall, kSmall));
}

// The activation's value and slope at g.
template <int kActivation>
__device__ __forceinline__ float activate(float g) {
    if constexpr (kActivation == ZCGVS_ACT_NONE) {
        return g;
    } else if constexpr (kActivation == ZCGVS_ACT_SILU) {
        return g * logistic(g);
    } else if constexpr (kActivation == ZCGVS_ACT_GELU) {
        return 0.5f * g * (1.0f + erff(g * 0.70710678f));
    } else {
        // 0.5 (1 + tanh(z)) is the logistic function of 2 z
        return g * logistic(1.59576912f * (g + 0.044715f * g * g * g));
    }
}

template <int kActivation>
__device__ __forceinline__ void activateBoth(float g, float& value, float& slope) {
    if constexpr (kActivation == ZCGVS_ACT_NONE) {
        value = g;
        slope = 1.0f;
    } else if constexpr (kActivation == ZCGVS_ACT_SILU) {
        const float y = logistic(g);
        value = g * y;
        slope = y + value * (1.0f - y);
    } else if constexpr (kActivation == ZCGVS_ACT_GELU) {
        const float y = 0.5f * (1.0f + erff(g * 0.70710678f));
        value = g * y;
        slope = y + g * 0.39894228f * __builtin_amdgcn_exp2f(-0.72134752f * g * g);
    } else {
        const float y = logistic(1.59576912f * (g + 0.044715f * g * g * g));
        value = g * y;
        // value * (1 - y) is 0 long before |g| is 100; the square must not make an infinity of it
        const float square = fminf(g * g, 1.0e4f);
        slope = y + value * (1.0f - y) * (1.59576912f * (1.0f + 0.134145f * square));
    }
}

// Calls body(std::integral_constant<int, activation>).
template <typename Body>
int withActivation(int activation, Body&& body) {
    switch (activation) {
        case ZCGVS_ACT_GELU:
            return body(std::integral_constant<int, ZCGVS_ACT_GELU>{});
        case ZCGVS_ACT_GELU_TANH:
            return body(std::integral_constant<int, ZCGVS_ACT_GELU_TANH>{});
        default:
            return body(std::integral_constant<int, ZCGVS_ACT_SILU>{});
    }
}

}  // namespace
}  // namespace zcgvs_hip
