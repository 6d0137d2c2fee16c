// Activations of the gated feed-forward block and their derivatives, on
// packed f32 pairs.
//
// The special-function unit bounds these epilogues first (16 results a cycle
// and SM): an exp2 and a reciprocal an element would take it longer than the
// tensor cores take for the products at 64 or 128 channels.  So two elements
// share one reciprocal.
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

// 1 / d of both lanes from the reciprocal of their product, r = 1 / (d0 d1):
// 1 / d0 = r d1, 1 / d1 = r d0 (a few ulp).  1 <= d <= 2^63, so that the
// product stays finite.
__device__ __forceinline__ uint64_t reciprocal2(uint64_t d) {
    float a, b, r;
    unpack2(d, a, b);
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(a * b));
    return pack2(r * b, r * a);
}

// e = 2^(-v log2 e) of sigma(v) = 1 / (1 + e).  The exponent is held at 62,
// where sigma is 2^-62 in place of less: v sigma(v) is then off by |v| 2^-62 at
// most, so that the activations hold their gates where that is nothing
// (floor2).  NaN comes out as the floor too, and leaves the neighbour alone.
__device__ __forceinline__ uint64_t sigmoid_exp2(uint64_t v) {
    return exp2_2(min2(mul2(v, both(-1.4426950408889634f)), 62.0f));
}
__device__ __forceinline__ uint64_t sigmoid2(uint64_t v) { return reciprocal2(add2(sigmoid_exp2(v), both(1.0f))); }

// sigma(v), and rest = 1 - sigma(v) as e sigma(v): it goes to exactly 0 with e
// far above zero, where 1 - s would keep the last bits of s (which depend on
// the lane's neighbour), for the derivatives to multiply by v or more.
__device__ __forceinline__ uint64_t sigmoid2(uint64_t v, uint64_t& rest) {
    const uint64_t e = sigmoid_exp2(v);
    const uint64_t s = reciprocal2(add2(e, both(1.0f)));
    rest = mul2(e, s);
    return s;
}

// GELU's tanh form as g sigma(2 z), z = sqrt(2/pi) (g + 0.044715 g^3): the
// same function without the cancellation of 1 + tanh in the negative tail.
constexpr float kGelu0 = 1.5957691216057308f;   // 2 sqrt(2/pi)
constexpr float kGelu1 = 0.07135481282553484f;  // 2 sqrt(2/pi) 0.044715

// The lanes held at m from below / above; NaN stays.
__device__ __forceinline__ uint64_t floor2(uint64_t v, float m) {
    float a, b;
    unpack2(v, a, b);
    asm("max.NaN.f32 %0, %0, %1;" : "+f"(a) : "f"(m));
    asm("max.NaN.f32 %0, %0, %1;" : "+f"(b) : "f"(m));
    return pack2(a, b);
}
__device__ __forceinline__ uint64_t ceiling2(uint64_t v, float m) {
    float a, b;
    unpack2(v, a, b);
    asm("min.NaN.f32 %0, %0, %1;" : "+f"(a) : "f"(m));
    asm("min.NaN.f32 %0, %0, %1;" : "+f"(b) : "f"(m));
    return pack2(a, b);
}

// Gates are held where sigma reaches its floor and the activation and its
// derivative are under 2^-55 (SiLU; 2^-300 GELU): further out the floor times
// the gate, or GELU's cube, would grow again.
constexpr float kSiluFloor = -43.0f, kGeluFloor = -15.0f;
// GELU's derivative takes its polynomials at min(g, 15): from there on e is
// exactly 0 (2^-380), and g^3 stays finite.
constexpr float kGeluCeiling = 15.0f;

// Phi(g) = (1 + erf(g / sqrt 2)) / 2 by Abramowitz and Stegun's 7.1.26
// (|error| <= 1.5e-7 in erf): erfc(z) = (a1 t + ... + a5 t^5) e^(-z^2), t =
// 1 / (1 + p z), for z = |g| / sqrt 2, reflected for g > 0.  gauss is
// e^(-g^2 / 2), which the derivative needs too.
__device__ __forceinline__ uint64_t normal_cdf2(uint64_t g, uint64_t& gauss) {
    constexpr uint64_t kSigns = 0x8000000080000000ull;
    const uint64_t z = min2(g & ~kSigns, 20.0f);
    const uint64_t t = reciprocal2(fma2(z, both(0.3275911f * 0.7071067811865476f), both(1.0f)));
    gauss = exp2_2(mul2(mul2(z, z), both(-0.7213475204444817f)));  // -log2(e) / 2
    // the polynomial's coefficients halved and negated: Phi(|g|) - 1/2 = 1/2 - erfc / 2
    uint64_t p = fma2(t, both(-0.5f * 1.061405429f), both(0.5f * 1.453152027f));
    p = fma2(t, p, both(-0.5f * 1.421413741f));
    p = fma2(t, p, both(0.5f * 0.284496736f));
    p = fma2(t, p, both(-0.5f * 0.254829592f));
    p = fma2(mul2(t, p), gauss, both(0.5f));
    return add2((p & ~kSigns) | (g & kSigns), both(0.5f));
}

template <int ACT>
__device__ __forceinline__ uint64_t act_value(uint64_t g) {
    if constexpr (ACT == ACT_SILU) {
        g = floor2(g, kSiluFloor);
        return mul2(g, sigmoid2(g));
    } else if constexpr (ACT == ACT_GELU) {
        g = floor2(g, kGeluFloor);
        return mul2(g, sigmoid2(mul2(g, fma2(mul2(g, g), both(kGelu1), both(kGelu0)))));
    } else {
        uint64_t gauss;
        return mul2(g, normal_cdf2(g, gauss));
    }
}

// Activation v and its derivative dv: s + v (1 - s) (slope of sigma's argument).
template <int ACT>
__device__ __forceinline__ void act_both(uint64_t g, uint64_t& v, uint64_t& dv) {
    if constexpr (ACT == ACT_SILU) {
        g = floor2(g, kSiluFloor);
        uint64_t rest;
        const uint64_t s = sigmoid2(g, rest);
        v = mul2(g, s);
        dv = fma2(v, rest, s);
    } else if constexpr (ACT == ACT_GELU) {
        g = floor2(g, kGeluFloor);
        const uint64_t gc = ceiling2(g, kGeluCeiling), gg = mul2(gc, gc);
        uint64_t rest;
        const uint64_t s = sigmoid2(mul2(gc, fma2(gg, both(kGelu1), both(kGelu0))), rest);
        v = mul2(g, s);
        dv = fma2(mul2(v, rest), fma2(gg, both(3.0f * kGelu1), both(kGelu0)), s);
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

template <int N>
__device__ __forceinline__ void to_pairs(const float (&v)[N], uint64_t (&p)[N / 2]) {
#pragma unroll
    for (int e = 0; e < N / 2; ++e) p[e] = pack2(v[2 * e], v[2 * e + 1]);
}
template <int N>
__device__ __forceinline__ void from_pairs(const uint64_t (&p)[N / 2], float (&v)[N]) {
#pragma unroll
    for (int e = 0; e < N / 2; ++e) unpack2(p[e], v[2 * e], v[2 * e + 1]);
}

// g <- act(g) * u; N even.
template <int N>
__device__ __forceinline__ void gate_chunk(int act, float (&g)[N], const float (&u)[N]) {
    uint64_t pg[N / 2], pu[N / 2];
    to_pairs(g, pg);
    to_pairs(u, pu);
    if (act == ACT_SILU) gate_pairs<ACT_SILU>(pg, pu);
    else if (act == ACT_GELU) gate_pairs<ACT_GELU>(pg, pu);
    else gate_pairs<ACT_GELU_ERF>(pg, pu);
    from_pairs(pg, g);
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

// (g, u, dh) -> (dg, du, h); N even.
template <int N>
__device__ __forceinline__ void gate_back_chunk(int act, float (&g)[N], float (&u)[N], float (&dh)[N]) {
    uint64_t pg[N / 2], pu[N / 2], pd[N / 2];
    to_pairs(g, pg);
    to_pairs(u, pu);
    to_pairs(dh, pd);
    if (act == ACT_SILU) gate_back<ACT_SILU>(pg, pu, pd);
    else if (act == ACT_GELU) gate_back<ACT_GELU>(pg, pu, pd);
    else gate_back<ACT_GELU_ERF>(pg, pu, pd);
    from_pairs(pg, g);
    from_pairs(pu, u);
    from_pairs(pd, dh);
}

}  // namespace msc
