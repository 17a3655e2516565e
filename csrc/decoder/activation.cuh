/**
 * The activations of feed-forward layers and their derivatives, in fp32.
 */
#pragma once
#include "decoder_ops.hpp"
#include <cuda_runtime.h>
#include <type_traits>

namespace dccl {

__device__ __forceinline__ float sigmoid(float v) { return __fdividef(1.0f, 1.0f + __expf(-v)); }

constexpr float kTanhScale = 1.5957691216057308f, kTanhCubic = 0.044715f;      // 2 sqrt(2 / pi)

/** 0.5 g (1 + tanh(z)) = g sigmoid(2 z). */
template <int ACT> __device__ __forceinline__ float activate(float g) {
    if constexpr (ACT == DCCL_ACT_SILU) return g * sigmoid(g);
    else if constexpr (ACT == DCCL_ACT_GELU) return 0.5f * g * (1.0f + erff(g * 0.70710678118654752f));
    else return g * sigmoid(kTanhScale * fmaf(kTanhCubic * g * g, g, g));
}

/** The activation and its derivative. */
template <int ACT> __device__ __forceinline__ void activate_grad(float g, float& a, float& da) {
    if constexpr (ACT == DCCL_ACT_SILU) {
        const float s = sigmoid(g);
        a = g * s;
        da = s * fmaf(g, 1.0f - s, 1.0f);
    } else if constexpr (ACT == DCCL_ACT_GELU) {
        const float cdf = 0.5f * (1.0f + erff(g * 0.70710678118654752f));
        a = g * cdf;
        da = fmaf(g * 0.3989422804014327f, __expf(-0.5f * g * g), cdf);
    } else {
        const float s = sigmoid(kTanhScale * fmaf(kTanhCubic * g * g, g, g));
        a = g * s;
        da = fmaf(g * s * (1.0f - s), kTanhScale * fmaf(3.0f * kTanhCubic * g, g, 1.0f), s);
    }
}

/** f with the activation as a constant: one choice for many elements. */
template <typename F> __device__ __forceinline__ void with_activation(int act, F&& f) {
    if (act == DCCL_ACT_SILU) f(std::integral_constant<int, DCCL_ACT_SILU>{});
    else if (act == DCCL_ACT_GELU) f(std::integral_constant<int, DCCL_ACT_GELU>{});
    else f(std::integral_constant<int, DCCL_ACT_GELU_TANH>{});
}

} // namespace dccl
