// Activations of the gated feed-forward block and their derivatives, on
// packed f32 pairs.
//
// The special-function unit would bound the epilogues (one exp2 and one
// reciprocal an element, 16 a cycle and SM), so that only the exp2 runs
// there; the reciprocal is Newton's method on packed fused multiply-adds.
#pragma once

#include "common.cuh"
#include "ffn.h"

namespace msc {

// 2^v of both lanes (relative error 2^-22; underflow gives 0).
__device__ __forceinline__ uint64_t exp2_2(uint64_t v) {
    float a, b;
    unpack2(v, a, b);
    asm("ex2.approx.ftz.f32 %0, %0;" : "+f"(a));
    asm("ex2.approx.ftz.f32 %0, %0;" : "+f"(b));
    return pack2(a, b);
}

__device__ __forceinline__ uint64_t min2(uint64_t v, float m) {
    float a, b;
    unpack2(v, a, b);
    return pack2(fminf(a, m), fminf(b, m));
}

// 1 / d from nd = -d, 1 <= d <= 2^101.  A float's bits are, up to a linear
// interpolation within each octave, 2^23 times its logarithm, so that a
// constant minus them is a first reciprocal y; the constant (found by search
// over an octave) leaves |r| = |1 - d y| <= 0.0506.  One third-order step
// y (1 + r + r^2) leaves r^3 = 1.3e-4, one Newton step its square, 1.7e-8.
__device__ __forceinline__ uint64_t reciprocal2(uint64_t nd) {
    constexpr uint32_t kSeed = 0x7ef31000u + 0x80000000u;  // the sign of nd cancels
    const uint64_t one = both(1.0f);
    float a, b;
    unpack2(nd, a, b);
    uint64_t y = pack2(__uint_as_float(kSeed - __float_as_uint(a)), __uint_as_float(kSeed - __float_as_uint(b)));
    uint64_t r = fma2(nd, y, one);
    y = fma2(y, fma2(r, r, r), y);
    r = fma2(nd, y, one);
    return fma2(y, r, y);
}

// sigma(v) = 1 / (1 + 2^(-v log2 e)).  The exponent is held at 100, where
// sigma is 2^-100 in place of less: nothing next to the smallest value that
// a 16-bit result distinguishes from zero at any magnitude of v.
__device__ __forceinline__ uint64_t sigmoid2(uint64_t v) {
    const uint64_t e = exp2_2(min2(mul2(v, both(-1.4426950408889634f)), 100.0f));
    return reciprocal2(fma2(e, both(-1.0f), both(-1.0f)));
}

// GELU's tanh form as g sigma(2 z), z = sqrt(2/pi) (g + 0.044715 g^3): the
// same function without the cancellation of 1 + tanh in the negative tail.
constexpr float kGelu0 = 1.5957691216057308f;   // 2 sqrt(2/pi)
constexpr float kGelu1 = 0.07135481282553484f;  // 2 sqrt(2/pi) 0.044715

// Phi(g) = (1 + erf(g / sqrt 2)) / 2 by Abramowitz and Stegun's 7.1.26
// (|error| <= 1.5e-7 in erf): erfc(z) = (a1 t + ... + a5 t^5) e^(-z^2), t =
// 1 / (1 + p z), for z = |g| / sqrt 2, reflected for g > 0.  gauss is
// e^(-g^2 / 2), which the derivative needs too.
__device__ __forceinline__ uint64_t normal_cdf2(uint64_t g, uint64_t& gauss) {
    constexpr uint64_t kSigns = 0x8000000080000000ull;
    const uint64_t z = min2(g & ~kSigns, 20.0f);
    const uint64_t t = reciprocal2(fma2(z, both(-0.3275911f * 0.7071067811865476f), both(-1.0f)));
    gauss = exp2_2(mul2(mul2(z, z), both(-0.7213475204444817f)));  // -log2(e) / 2
    // the polynomial's coefficients halved: Phi(-|g|) = erfc / 2
    uint64_t p = fma2(t, both(0.5f * 1.061405429f), both(-0.5f * 1.453152027f));
    p = fma2(t, p, both(0.5f * 1.421413741f));
    p = fma2(t, p, both(-0.5f * 0.284496736f));
    p = fma2(t, p, both(0.5f * 0.254829592f));
    p = mul2(mul2(t, p), gauss);
    float p0, p1, g0, g1;
    unpack2(p, p0, p1);
    unpack2(g, g0, g1);
    return pack2(g0 > 0.f ? 1.f - p0 : p0, g1 > 0.f ? 1.f - p1 : p1);
}

template <int ACT>
__device__ __forceinline__ uint64_t act_value(uint64_t g) {
    if constexpr (ACT == ACT_SILU) {
        return mul2(g, sigmoid2(g));
    } else if constexpr (ACT == ACT_GELU) {
        return mul2(g, sigmoid2(mul2(g, fma2(mul2(g, g), both(kGelu1), both(kGelu0)))));
    } else {
        uint64_t gauss;
        return mul2(g, normal_cdf2(g, gauss));
    }
}

// Activation v and its derivative dv.
template <int ACT>
__device__ __forceinline__ void act_both(uint64_t g, uint64_t& v, uint64_t& dv) {
    const uint64_t one = both(1.0f), minus = both(-1.0f);
    if constexpr (ACT == ACT_SILU) {
        const uint64_t s = sigmoid2(g);
        v = mul2(g, s);
        dv = fma2(v, fma2(s, minus, one), s);
    } else if constexpr (ACT == ACT_GELU) {
        const uint64_t gg = mul2(g, g);
        const uint64_t s = sigmoid2(mul2(g, fma2(gg, both(kGelu1), both(kGelu0))));
        v = mul2(g, s);
        dv = fma2(mul2(v, fma2(s, minus, one)), fma2(gg, both(3.0f * kGelu1), both(kGelu0)), s);
    } else {
        uint64_t gauss;
        const uint64_t p = normal_cdf2(g, gauss);
        v = mul2(g, p);
        dv = fma2(mul2(g, both(0.3989422804014327f)), gauss, p);
    }
}

template <int ACT, int N>
__device__ __forceinline__ void gate_pairs(uint64_t (&g)[N], const uint64_t (&u)[N]) {
#pragma unroll
    for (int e = 0; e < N; ++e) g[e] = mul2(act_value<ACT>(g[e]), u[e]);
}

// g <- act(g) * u over N pairs.
template <int N>
__device__ __forceinline__ void gate_chunk(int act, uint64_t (&g)[N], const uint64_t (&u)[N]) {
    if (act == ACT_SILU) gate_pairs<ACT_SILU>(g, u);
    else if (act == ACT_GELU) gate_pairs<ACT_GELU>(g, u);
    else gate_pairs<ACT_GELU_ERF>(g, u);
}

template <int ACT, int N>
__device__ __forceinline__ void gate_back(uint64_t (&g)[N], uint64_t (&u)[N], uint64_t (&dh)[N]) {
#pragma unroll
    for (int e = 0; e < N; ++e) {
        uint64_t v, dv;
        act_both<ACT>(g[e], v, dv);
        const uint64_t h = mul2(v, u[e]);
        g[e] = mul2(mul2(dh[e], u[e]), dv);
        u[e] = mul2(dh[e], v);
        dh[e] = h;
    }
}

// (g, u, dh) -> (dg, du, h) over N pairs.
template <int N>
__device__ __forceinline__ void gate_back_chunk(int act, uint64_t (&g)[N], uint64_t (&u)[N], uint64_t (&dh)[N]) {
    if (act == ACT_SILU) gate_back<ACT_SILU>(g, u, dh);
    else if (act == ACT_GELU) gate_back<ACT_GELU>(g, u, dh);
    else gate_back<ACT_GELU_ERF>(g, u, dh);
}

}  // namespace msc
