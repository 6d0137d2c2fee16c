// Activations of the gated feed-forward block and their derivatives, two
// elements at a time.
//
// The special-function unit bounds these epilogues first (16 results a cycle
// and SM): an exp2 and a reciprocal an element would take it longer than the
// tensor cores take for the products at 64 or 128 channels.  So two elements
// share one reciprocal.  Scalar fp32 throughout: the packed f32x2 forms spend
// as many register moves as they save operations between the special-function
// results (measured: 14 instructions an element against 9).
#pragma once

#include "common.cuh"
#include "ffn.h"

namespace msc {

// 2^v (relative error 2^-22; underflow gives 0).
__device__ __forceinline__ float exp2_fast(float v) {
    float e;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(v));
    return e;
}

// 1 / d of two values from the reciprocal of their product, r = 1 / (d0 d1):
// 1 / d0 = r d1, 1 / d1 = r d0 (a few ulp).  1 <= d <= 2^63, so that the
// product stays finite.
__device__ __forceinline__ void reciprocals(float& d0, float& d1) {
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(d0 * d1));
    const float t = r * d1;
    d1 = r * d0;
    d0 = t;
}

// sigma(v) = 1 / (1 + 2^(-v log2 e)).  The exponent is held at 62, where
// sigma is 2^-62 in place of less: v sigma(v) is then off by |v| 2^-62 at
// most.
__device__ __forceinline__ void sigmoids(float v0, float v1, float& s0, float& s1) {
    s0 = 1.0f + exp2_fast(fminf(v0 * -1.4426950408889634f, 62.0f));
    s1 = 1.0f + exp2_fast(fminf(v1 * -1.4426950408889634f, 62.0f));
    reciprocals(s0, s1);
}

// GELU's tanh form as g sigma(2 z), z = sqrt(2/pi) (g + 0.044715 g^3): the
// same function without the cancellation of 1 + tanh in the negative tail.
constexpr float kGelu0 = 1.5957691216057308f;   // 2 sqrt(2/pi)
constexpr float kGelu1 = 0.07135481282553484f;  // 2 sqrt(2/pi) 0.044715
__device__ __forceinline__ float gelu_arg(float g) { return g * fmaf(kGelu1, g * g, kGelu0); }

// Phi(g) = (1 + erf(g / sqrt 2)) / 2 by Abramowitz and Stegun's 7.1.26
// (|error| <= 1.5e-7 in erf): erfc(z) = (a1 t + ... + a5 t^5) e^(-z^2), t =
// 1 / (1 + p z), for z = |g| / sqrt 2, reflected for g > 0.  e is
// e^(-g^2 / 2), which the derivative needs too.
__device__ __forceinline__ void normal_cdfs(float g0, float g1, float& p0, float& p1, float& e0, float& e1) {
    auto poly = [](float g, float t, float e) {
        // 1/2 - erfc / 2, then the sign of g
        float p = fmaf(t, -0.5f * 1.061405429f, 0.5f * 1.453152027f);
        p = fmaf(t, p, -0.5f * 1.421413741f);
        p = fmaf(t, p, 0.5f * 0.284496736f);
        p = fmaf(t, p, -0.5f * 0.254829592f);
        return 0.5f + copysignf(fmaf(t * p, e, 0.5f), g);
    };
    const float z0 = fminf(fabsf(g0), 20.0f), z1 = fminf(fabsf(g1), 20.0f);
    float t0 = fmaf(z0, 0.3275911f * 0.7071067811865476f, 1.0f), t1 = fmaf(z1, 0.3275911f * 0.7071067811865476f, 1.0f);
    reciprocals(t0, t1);
    e0 = exp2_fast(z0 * z0 * -0.7213475204444817f);  // -log2(e) / 2
    e1 = exp2_fast(z1 * z1 * -0.7213475204444817f);
    p0 = poly(g0, t0, e0);
    p1 = poly(g1, t1, e1);
}

template <int ACT>
__device__ __forceinline__ void act_values(float& g0, float& g1) {
    float s0, s1;
    if constexpr (ACT == ACT_SILU) {
        sigmoids(g0, g1, s0, s1);
    } else if constexpr (ACT == ACT_GELU) {
        sigmoids(gelu_arg(g0), gelu_arg(g1), s0, s1);
    } else {
        float e0, e1;
        normal_cdfs(g0, g1, s0, s1, e0, e1);
    }
    g0 *= s0;
    g1 *= s1;
}

// Activations v and their derivatives d.
template <int ACT>
__device__ __forceinline__ void act_both(float g0, float g1, float& v0, float& v1, float& d0, float& d1) {
    float s0, s1;
    if constexpr (ACT == ACT_SILU) {
        sigmoids(g0, g1, s0, s1);
        v0 = g0 * s0, v1 = g1 * s1;
        d0 = fmaf(v0, 1.0f - s0, s0), d1 = fmaf(v1, 1.0f - s1, s1);
    } else if constexpr (ACT == ACT_GELU) {
        sigmoids(gelu_arg(g0), gelu_arg(g1), s0, s1);
        v0 = g0 * s0, v1 = g1 * s1;
        d0 = fmaf(v0 * (1.0f - s0), fmaf(3.0f * kGelu1, g0 * g0, kGelu0), s0);
        d1 = fmaf(v1 * (1.0f - s1), fmaf(3.0f * kGelu1, g1 * g1, kGelu0), s1);
    } else {
        float e0, e1;
        normal_cdfs(g0, g1, s0, s1, e0, e1);
        v0 = g0 * s0, v1 = g1 * s1;
        d0 = fmaf(g0 * 0.3989422804014327f, e0, s0);
        d1 = fmaf(g1 * 0.3989422804014327f, e1, s1);
    }
}

template <int ACT, int N>
__device__ __forceinline__ void gate_values(float (&g)[N], const float (&u)[N]) {
#pragma unroll
    for (int e = 0; e < N; e += 2) {
        act_values<ACT>(g[e], g[e + 1]);
        g[e] *= u[e];
        g[e + 1] *= u[e + 1];
    }
}

// g <- act(g) * u; N even.
template <int N>
__device__ __forceinline__ void gate_chunk(int act, float (&g)[N], const float (&u)[N]) {
    if (act == ACT_SILU) gate_values<ACT_SILU>(g, u);
    else if (act == ACT_GELU) gate_values<ACT_GELU>(g, u);
    else gate_values<ACT_GELU_ERF>(g, u);
}

template <int ACT, int N>
__device__ __forceinline__ void gate_back(float (&g)[N], float (&u)[N], float (&dh)[N]) {
#pragma unroll
    for (int e = 0; e < N; e += 2) {
        float v[2], dv[2];
        act_both<ACT>(g[e], g[e + 1], v[0], v[1], dv[0], dv[1]);
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            const float h = v[k] * u[e + k];
            g[e + k] = dh[e + k] * u[e + k] * dv[k];
            u[e + k] = dh[e + k] * v[k];
            dh[e + k] = h;
        }
    }
}

// (g, u, dh) -> (dg, du, h); N even.
template <int N>
__device__ __forceinline__ void gate_back_chunk(int act, float (&g)[N], float (&u)[N], float (&dh)[N]) {
    if (act == ACT_SILU) gate_back<ACT_SILU>(g, u, dh);
    else if (act == ACT_GELU) gate_back<ACT_GELU>(g, u, dh);
    else gate_back<ACT_GELU_ERF>(g, u, dh);
}

}  // namespace msc
