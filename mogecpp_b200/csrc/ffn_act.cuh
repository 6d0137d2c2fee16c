// Activations of the gated feed-forward block and their derivatives.
#pragma once

#include "ffn.h"

#include <cuda_runtime.h>

namespace msc {

// sigma(v) = 1 / (1 + 2^(-v log2 e)) with the hardware exp2 and reciprocal
// (relative error ~1e-6; the fp32 sums of the bias gradients stay at fp32's
// own accuracy).
__device__ __forceinline__ float sigmoid_fast(float v) {
    float e, r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(v * -1.4426950408889634f));
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.0f + e));
    return r;
}

// GELU's tanh form as g sigma(2 z), z = sqrt(2/pi) (g + 0.044715 g^3): the
// same function without the cancellation of 1 + tanh in the negative tail.
constexpr float kGelu0 = 1.5957691216057308f;   // 2 sqrt(2/pi)
constexpr float kGelu1 = 0.07135481282553484f;  // 2 sqrt(2/pi) 0.044715

template <int ACT>
__device__ __forceinline__ float act_value(float g) {
    if constexpr (ACT == ACT_SILU) return g * sigmoid_fast(g);
    if constexpr (ACT == ACT_GELU) return g * sigmoid_fast(g * fmaf(kGelu1, g * g, kGelu0));
    return 0.5f * g * (1.0f + erff(g * 0.7071067811865476f));
}

template <int ACT>
__device__ __forceinline__ void act_both(float g, float& v, float& dv) {
    if constexpr (ACT == ACT_SILU) {
        const float s = sigmoid_fast(g);
        v = g * s;
        dv = s * fmaf(g, 1.0f - s, 1.0f);
    } else if constexpr (ACT == ACT_GELU) {
        const float s = sigmoid_fast(g * fmaf(kGelu1, g * g, kGelu0));
        v = g * s;
        dv = s * fmaf(g * fmaf(3.0f * kGelu1, g * g, kGelu0), 1.0f - s, 1.0f);
    } else {
        const float p = 0.5f * (1.0f + erff(g * 0.7071067811865476f));
        v = g * p;
        dv = fmaf(g * 0.3989422804014327f, __expf(-0.5f * g * g), p);
    }
}

template <int N>
__device__ __forceinline__ void gate_chunk(int act, float (&g)[N], const float (&u)[N]) {
    if (act == ACT_SILU) {
#pragma unroll
        for (int e = 0; e < N; ++e) g[e] = act_value<ACT_SILU>(g[e]) * u[e];
    } else if (act == ACT_GELU) {
#pragma unroll
        for (int e = 0; e < N; ++e) g[e] = act_value<ACT_GELU>(g[e]) * u[e];
    } else {
#pragma unroll
        for (int e = 0; e < N; ++e) g[e] = act_value<ACT_GELU_ERF>(g[e]) * u[e];
    }
}

// (g, u, dh) -> (dg, du, h)
template <int ACT, int N>
__device__ __forceinline__ void gate_back(float (&g)[N], float (&u)[N], float (&dh)[N]) {
#pragma unroll
    for (int e = 0; e < N; ++e) {
        float v, dv;
        act_both<ACT>(g[e], v, dv);
        const float h = v * u[e];
        g[e] = dh[e] * u[e] * dv;
        u[e] = dh[e] * v;
        dh[e] = h;
    }
}

template <int N>
__device__ __forceinline__ void gate_back_chunk(int act, float (&g)[N], float (&u)[N], float (&dh)[N]) {
    if (act == ACT_SILU) gate_back<ACT_SILU>(g, u, dh);
    else if (act == ACT_GELU) gate_back<ACT_GELU>(g, u, dh);
    else gate_back<ACT_GELU_ERF>(g, u, dh);
}

}  // namespace msc
