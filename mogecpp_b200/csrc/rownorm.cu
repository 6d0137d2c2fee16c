// Norms before and after a residual block, fused with the block's gate and
// residual scale, one pass over the rows each way.
//
// Forward, per row (all in fp32, one rounding per output):
//   t = Norm_post(f)             or f
//   r = s x + gate * t           the new residual stream
//   h = Norm_pre(r)              the next block's input, from the unrounded r
// Norm: LayerNorm (v - mean) / sqrt(var + eps) or RMSNorm v / sqrt(mean v^2 +
// eps), times w, plus b.  The gate is one weight per channel, or per sample
// and channel (the sample is field 3 of the row's coordinates).
//
// Backward, from dr (gradient of r) and dh, with v^ the normalised row and k
// its scale 1 / sqrt(...):
//   norm'(d; v) = k (d w - [mean(d w)] - v^ mean(d w v^))   [LayerNorm only]
//   dr += norm'_pre(dh; r);  dx = s dr;  dt = gate dr;  df = norm'_post(dt; f)
//   gate: sum dr t;  post: w sum dt f^, b sum dt;  pre: w sum dh r^, b sum dh
//
// Both are bound by HBM: a row's tensors are read and written once (8 B an
// element forward and 12 B backward for 16-bit tensors) for some 20-40 fp32
// operations an element.  A row is held in registers by T threads, 8 columns
// (16 bytes of a 16-bit tensor) each: 8 to 32 lanes of a warp up to 256
// channels, so that a row's means are shuffles alone and a warp has up to
// four rows in flight; a block per row beyond (one shared-memory exchange
// per mean).  A thread keeps its 8 columns of every weight in registers over
// all its rows.
//
// The backward column sums are kept in fp32 registers over a unit's (warp's
// or block's) run of rows, written once per unit, and added over the units in
// double in a fixed order by a second kernel: no atomics, the same bits every
// time.  A per-sample gate adds its sums to the unit's own slab whenever the
// sample changes (rows are normally sorted by sample; any order is right).
#include "rownorm.h"

#include "common.cuh"
#include "conv.h"

#include <algorithm>
#include <mutex>

namespace msc {
namespace {

template <int DT>
struct Raw8 {
    uint4 q[DT == DT_F32 ? 2 : 1];
};

template <int DT>
__device__ __forceinline__ Raw8<DT> load8(const void* p, int64_t off) {
    Raw8<DT> r;
    const uint4* s = reinterpret_cast<const uint4*>(static_cast<const uint8_t*>(p) + off * (DT == DT_F32 ? 4 : 2));
#pragma unroll
    for (int i = 0; i < (DT == DT_F32 ? 2 : 1); ++i) r.q[i] = s[i];
    return r;
}

template <int DT>
__device__ __forceinline__ void zero8(Raw8<DT>& r) {
#pragma unroll
    for (int i = 0; i < (DT == DT_F32 ? 2 : 1); ++i) r.q[i] = make_uint4(0u, 0u, 0u, 0u);
}

template <int DT>
__device__ __forceinline__ void unpack8(const Raw8<DT>& r, float* v) {
    if constexpr (DT == DT_F32) {
        const uint32_t w[8] = {r.q[0].x, r.q[0].y, r.q[0].z, r.q[0].w, r.q[1].x, r.q[1].y, r.q[1].z, r.q[1].w};
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = __uint_as_float(w[e]);
    } else {
        const uint32_t w[4] = {r.q[0].x, r.q[0].y, r.q[0].z, r.q[0].w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            float2 t;
            if constexpr (DT == DT_F16)
                t = __half22float2(*reinterpret_cast<const __half2*>(&w[e]));
            else
                t = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&w[e]));
            v[2 * e] = t.x, v[2 * e + 1] = t.y;
        }
    }
}

template <int DT>
__device__ __forceinline__ void store8(void* p, int64_t off, const float* v) {
    if constexpr (DT == DT_F32) {
        float4* d = reinterpret_cast<float4*>(static_cast<float*>(p) + off);
        d[0] = make_float4(v[0], v[1], v[2], v[3]);
        d[1] = make_float4(v[4], v[5], v[6], v[7]);
    } else {
        uint32_t w[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            if constexpr (DT == DT_F16) {
                const __half2 h = __floats2half2_rn(v[2 * e], v[2 * e + 1]);
                w[e] = *reinterpret_cast<const uint32_t*>(&h);
            } else {
                const __nv_bfloat162 h = __floats2bfloat162_rn(v[2 * e], v[2 * e + 1]);
                w[e] = *reinterpret_cast<const uint32_t*>(&h);
            }
        }
        *reinterpret_cast<uint4*>(static_cast<uint8_t*>(p) + off * 2) = make_uint4(w[0], w[1], w[2], w[3]);
    }
}

// 8 columns of a weight vector (fill where it is absent).
__device__ __forceinline__ void load_param(const float* p, int col, float fill, float* v) {
    if (p) {
        const float4 a = __ldg(reinterpret_cast<const float4*>(p + col));
        const float4 b = __ldg(reinterpret_cast<const float4*>(p + col) + 1);
        v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = fill;
    }
}

// Sums of a and b over the T threads of a row.  Beyond a warp the partial
// sums cross through shared memory; `turn` alternates between two buffers, so
// that one barrier per exchange orders both its own reads and the reuse.
template <int T>
__device__ __forceinline__ void row_sum2(float& a, float& b, float2 (*buf)[T > 32 ? T / 32 : 1], int& turn) {
#pragma unroll
    for (int o = (T < 32 ? T : 32) / 2; o >= 1; o >>= 1) {
        a += __shfl_xor_sync(0xffffffffu, a, o);
        b += __shfl_xor_sync(0xffffffffu, b, o);
    }
    if constexpr (T > 32) {
        if ((threadIdx.x & 31) == 0) buf[turn][threadIdx.x >> 5] = make_float2(a, b);
        __syncthreads();
        a = 0.f, b = 0.f;
#pragma unroll
        for (int w = 0; w < T / 32; ++w) {
            a += buf[turn][w].x;
            b += buf[turn][w].y;
        }
        turn ^= 1;
    }
}

template <int T>
constexpr int block_threads() {
    return T > 32 ? T : 256;
}

// The row's gate: per channel, or of the row's sample.  An index outside the
// samples is a device failure and gates the branch off.
__device__ __forceinline__ int row_sample(const RowNormArgs& a, int64_t row, bool live) {
    if (!a.nsamples) return 0;
    const int s = live ? __ldg(a.coords + row * 4 + 3) : 0;
    if (static_cast<unsigned>(s) < static_cast<unsigned>(a.nsamples)) return s;
    set_status(a.status, MSC_DEV_BAD_COORD);
    return -1;
}

template <int XT, int FT, int T, int V>
__global__ void __launch_bounds__(block_threads<T>()) rownorm_kernel(const RowNormArgs a) {
    constexpr int R = T > 32 ? 1 : 32 / T;  // rows per unit and step
    __shared__ float2 buf[2][T > 32 ? T / 32 : 1];
    int turn = 0;
    const int t = T > 32 ? threadIdx.x : threadIdx.x & (T - 1);
    const int sub = T > 32 ? 0 : (threadIdx.x & 31) / T;
    const int64_t unit = T > 32 ? blockIdx.x : blockIdx.x * (block_threads<T>() / 32) + (threadIdx.x >> 5);
    const int64_t units = T > 32 ? gridDim.x : static_cast<int64_t>(gridDim.x) * (block_threads<T>() / 32);
    const int chunks = a.c / 8;
    const float inv_c = 1.0f / static_cast<float>(a.c);
    float post_w[8], post_b[8], pre_w[8], pre_b[8], gate[8];
    int gate_of = -2;  // sample whose gate is held
    auto params = [&](int v) {
        const int col = min(t + v * T, chunks - 1) * 8;
        load_param(a.post.w, col, 1.f, post_w);
        load_param(a.post.b, col, 0.f, post_b);
        load_param(a.pre.w, col, 1.f, pre_w);
        load_param(a.pre.b, col, 0.f, pre_b);
    };
    if constexpr (V == 1) params(0);
    for (int64_t row0 = unit * R; row0 < a.n; row0 += units * R) {
        const int64_t row = row0 + sub;
        const bool live = row < a.n;
        Raw8<XT> xr[V];
        Raw8<FT> fr[V];
#pragma unroll
        for (int v = 0; v < V; ++v) {
            zero8(xr[v]);
            zero8(fr[v]);
            const int j = t + v * T;
            if (live && j < chunks) {
                xr[v] = load8<XT>(a.x, row * a.c + j * 8);
                if (a.f) fr[v] = load8<FT>(a.f, row * a.c + j * 8);
            }
        }
        const int s = a.gate ? row_sample(a, row, live) : 0;
        float r[V * 8];
        float mean = 0.f, k = 1.f;
        if (a.f && a.post.kind != NORM_NONE) {
            float s1 = 0.f, s2 = 0.f;
#pragma unroll
            for (int v = 0; v < V; ++v) {
                unpack8(fr[v], r + 8 * v);
#pragma unroll
                for (int e = 0; e < 8; ++e) s1 += r[8 * v + e], s2 += r[8 * v + e] * r[8 * v + e];
            }
            if (a.post.kind == NORM_LAYER) {
                // two passes over the registers: the variance of the centred values
                float dummy = 0.f;
                row_sum2<T>(s1, dummy, buf, turn);
                mean = s1 * inv_c;
                s2 = 0.f;
#pragma unroll
                for (int v = 0; v < V; ++v)
                    if (t + v * T < chunks) {
#pragma unroll
                        for (int e = 0; e < 8; ++e) s2 += (r[8 * v + e] - mean) * (r[8 * v + e] - mean);
                    }
            }
            row_sum2<T>(s1, s2, buf, turn);
            k = rsqrtf(s2 * inv_c + a.post.eps);
        }
        float s1 = 0.f, s2 = 0.f;
#pragma unroll
        for (int v = 0; v < V; ++v) {
            const int j = t + v * T;
            if constexpr (V > 1) params(v);
            if (a.gate && (V > 1 || s != gate_of)) {
                load_param(s < 0 ? nullptr : a.gate + static_cast<int64_t>(s) * a.c, min(j, chunks - 1) * 8, 0.f, gate);
                gate_of = s;
            }
            float x[8], f[8];
            unpack8(xr[v], x);
            unpack8(fr[v], f);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                float q = f[e];
                if (a.post.kind != NORM_NONE) q = fmaf((q - mean) * k, post_w[e], post_b[e]);
                if (a.gate) q *= gate[e];
                q = a.f ? fmaf(a.res_scale, x[e], q) : a.res_scale * x[e];
                r[8 * v + e] = j < chunks ? q : 0.f;
                s1 += r[8 * v + e];
                s2 += r[8 * v + e] * r[8 * v + e];
            }
            if (a.r && live && j < chunks) store8<XT>(a.r, row * a.c + j * 8, r + 8 * v);
        }
        if (a.pre.kind == NORM_NONE) {
            // no norm: h, where asked for, is r in the branch's type
            if (a.h && live) {
#pragma unroll
                for (int v = 0; v < V; ++v)
                    if (t + v * T < chunks) store8<FT>(a.h, row * a.c + (t + v * T) * 8, r + 8 * v);
            }
            continue;
        }
        mean = 0.f;
        if (a.pre.kind == NORM_LAYER) {
            float dummy = 0.f;
            row_sum2<T>(s1, dummy, buf, turn);
            mean = s1 * inv_c;
            s2 = 0.f;
#pragma unroll
            for (int v = 0; v < V; ++v)
                if (t + v * T < chunks) {
#pragma unroll
                    for (int e = 0; e < 8; ++e) s2 += (r[8 * v + e] - mean) * (r[8 * v + e] - mean);
                }
        }
        row_sum2<T>(s1, s2, buf, turn);
        k = rsqrtf(s2 * inv_c + a.pre.eps);
#pragma unroll
        for (int v = 0; v < V; ++v) {
            const int j = t + v * T;
            if constexpr (V > 1) params(v);
            float h[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) h[e] = fmaf((r[8 * v + e] - mean) * k, pre_w[e], pre_b[e]);
            if (live && j < chunks) store8<FT>(a.h, row * a.c + j * 8, h);
        }
    }
}

// Slab rows of a unit: pre_w, pre_b, post_w, post_b, then the gate's.
enum SlabRow : int { SLAB_PRE_W = 0, SLAB_PRE_B = 1, SLAB_POST_W = 2, SLAB_POST_B = 3, SLAB_GATE = 4 };

template <int XT, int FT, int T, int V>
__global__ void __launch_bounds__(block_threads<T>(), T > 32 ? 512 / T : 2) rownorm_backward_kernel(const RowNormArgs a) {
    constexpr int R = T > 32 ? 1 : 32 / T;
    __shared__ float2 buf[2][T > 32 ? T / 32 : 1];
    int turn = 0;
    const int t = T > 32 ? threadIdx.x : threadIdx.x & (T - 1);
    const int sub = T > 32 ? 0 : (threadIdx.x & 31) / T;
    const int64_t unit = T > 32 ? blockIdx.x : blockIdx.x * (block_threads<T>() / 32) + (threadIdx.x >> 5);
    if (unit >= a.units) return;  // whole warps (T <= 32, no block barrier) or whole blocks
    const int chunks = a.c / 8;
    const float inv_c = 1.0f / static_cast<float>(a.c);
    const int gate_rows = !a.gate ? 0 : (a.nsamples ? a.nsamples : 1);
    float* slab = a.partial + unit * (SLAB_GATE + gate_rows) * a.c;
    const bool has_pre = a.pre.kind != NORM_NONE, has_post = a.post.kind != NORM_NONE;
    float pre_w[8], post_w[8], post_b[8], gate[8];
    int gate_of = -2;
    auto params = [&](int v) {
        const int col = min(t + v * T, chunks - 1) * 8;
        load_param(a.pre.w, col, 1.f, pre_w);
        load_param(a.post.w, col, 1.f, post_w);
        load_param(a.post.b, col, 0.f, post_b);
    };
    auto load_gate = [&](int v, int s) {
        if (a.gate && (V > 1 || s != gate_of)) {
            load_param(s < 0 ? nullptr : a.gate + static_cast<int64_t>(s) * a.c, min(t + v * T, chunks - 1) * 8, 0.f, gate);
            gate_of = s;
        }
    };
    if constexpr (V == 1) params(0);
    float acc_pre_w[V * 8] = {}, acc_pre_b[V * 8] = {}, acc_post_w[V * 8] = {}, acc_post_b[V * 8] = {},
          acc_gate[V * 8] = {};
    int cur = -1;  // sample of the rows in acc_gate
    // adds the rows held in acc_gate to the slab of their sample and clears them
    auto flush_gate = [&]() {
#pragma unroll
        for (int v = 0; v < V; ++v)
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                float q = acc_gate[8 * v + e];
                acc_gate[8 * v + e] = 0.f;
                if constexpr (T < 32) {
#pragma unroll
                    for (int o = T; o < 32; o <<= 1) q += __shfl_xor_sync(0xffffffffu, q, o);
                }
                if (cur >= 0 && sub == 0 && t + v * T < chunks) {
                    float* p = slab + static_cast<int64_t>(SLAB_GATE + cur) * a.c + (t + v * T) * 8 + e;
                    *p += q;
                }
            }
        if constexpr (T <= 32) __syncwarp();
    };
    const int64_t row_end = min(a.n, (unit + 1) * a.rows_per_unit);
    for (int64_t row0 = unit * a.rows_per_unit; row0 < row_end; row0 += R) {
        const int64_t row = row0 + sub;
        const bool live = row < row_end;
        Raw8<XT> rr[V], gr[V];
        Raw8<FT> fr[V], hr[V];
#pragma unroll
        for (int v = 0; v < V; ++v) {
            zero8(rr[v]), zero8(gr[v]), zero8(fr[v]), zero8(hr[v]);
            const int j = t + v * T;
            if (live && j < chunks) {
                const int64_t off = row * a.c + j * 8;
                if (has_pre) rr[v] = load8<XT>(a.x, off);
                if (a.dh) hr[v] = load8<FT>(a.dh, off);
                if (a.dr) gr[v] = load8<XT>(a.dr, off);
                if (a.f) fr[v] = load8<FT>(a.f, off);
            }
        }
        const int s = a.gate ? row_sample(a, row, live) : 0;
        // both norms' statistics together: means, then centred squares
        float r_mean = 0.f, f_mean = 0.f, s1 = 0.f, s2 = 0.f;
        float r[V * 8], f[V * 8];
#pragma unroll
        for (int v = 0; v < V; ++v) {
            unpack8(rr[v], r + 8 * v);
            unpack8(fr[v], f + 8 * v);
#pragma unroll
            for (int e = 0; e < 8; ++e) s1 += r[8 * v + e], s2 += f[8 * v + e];
        }
        if (a.pre.kind == NORM_LAYER || a.post.kind == NORM_LAYER) {
            row_sum2<T>(s1, s2, buf, turn);
            if (a.pre.kind == NORM_LAYER) r_mean = s1 * inv_c;
            if (a.post.kind == NORM_LAYER) f_mean = s2 * inv_c;
        }
        s1 = s2 = 0.f;
#pragma unroll
        for (int v = 0; v < V; ++v)
            if (t + v * T < chunks) {
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    r[8 * v + e] -= r_mean;
                    if (has_post) f[8 * v + e] -= f_mean;
                    s1 += r[8 * v + e] * r[8 * v + e];
                    s2 += f[8 * v + e] * f[8 * v + e];
                }
            }
        row_sum2<T>(s1, s2, buf, turn);
        const float r_k = rsqrtf(s1 * inv_c + a.pre.eps);
        const float f_k = has_post ? rsqrtf(s2 * inv_c + a.post.eps) : 1.f;
        // dr = dr + norm'_pre(dh; r)
        float d[V * 8];
        s1 = s2 = 0.f;
#pragma unroll
        for (int v = 0; v < V; ++v) {
            if constexpr (V > 1) params(v);
            float g[8];
            unpack8(hr[v], g);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const int i = 8 * v + e;
                r[i] *= r_k;
                if (has_pre) {
                    acc_pre_w[i] = fmaf(g[e], r[i], acc_pre_w[i]);
                    acc_pre_b[i] += g[e];
                }
                d[i] = has_pre ? g[e] * pre_w[e] : g[e];
                s1 += d[i];
                s2 = fmaf(d[i], r[i], s2);
            }
        }
        if (has_pre) row_sum2<T>(s1, s2, buf, turn);
        const float m1 = a.pre.kind == NORM_LAYER ? s1 * inv_c : 0.f, m2 = s2 * inv_c;
        float q1 = 0.f, q2 = 0.f;
#pragma unroll
        for (int v = 0; v < V; ++v) {
            const int j = t + v * T;
            if constexpr (V > 1) params(v);
            load_gate(v, s);
            float g[8], o[8];
            unpack8(gr[v], g);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const int i = 8 * v + e;
                g[e] = has_pre ? fmaf(r_k, d[i] - m1 - r[i] * m2, g[e]) : g[e] + d[i];
                o[e] = a.res_scale * g[e];
                f[i] *= f_k;  // f^, or f without a norm
                const float tt = has_post ? fmaf(f[i], post_w[e], post_b[e]) : f[i];
                r[i] = g[e] * tt;  // this row's gate gradient
                const float dt = a.gate ? gate[e] * g[e] : g[e];
                acc_post_w[i] = fmaf(dt, f[i], acc_post_w[i]);
                acc_post_b[i] += dt;
                d[i] = has_post ? dt * post_w[e] : dt;
                q1 += d[i];
                q2 = fmaf(d[i], f[i], q2);
            }
            if (a.dx && live && j < chunks) store8<XT>(a.dx, row * a.c + j * 8, o);
        }
        if (a.f) {
            if (has_post) row_sum2<T>(q1, q2, buf, turn);
            const float n1 = a.post.kind == NORM_LAYER ? q1 * inv_c : 0.f, n2 = q2 * inv_c;
#pragma unroll
            for (int v = 0; v < V; ++v) {
                const int j = t + v * T;
                float o[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const int i = 8 * v + e;
                    o[e] = has_post ? f_k * (d[i] - n1 - f[i] * n2) : d[i];
                }
                if (a.df && live && j < chunks) store8<FT>(a.df, row * a.c + j * 8, o);
            }
        }
        if (a.gate) {
            if (a.nsamples) {
                int first = s;
                bool mixed = false;
                if constexpr (T < 32) {
                    first = __shfl_sync(0xffffffffu, s, 0);  // the first row of a step is always live
                    mixed = !__all_sync(0xffffffffu, !live || s == first);
                }
                if (mixed || first != cur) {
                    flush_gate();
                    cur = mixed ? -1 : first;
                }
                if (mixed) {
                    // the step's rows belong to different samples: one row after the other
                    for (int g = 0; g < R; ++g) {
                        if (sub == g && live && s >= 0) {
#pragma unroll
                            for (int v = 0; v < V; ++v)
                                if (t + v * T < chunks) {
                                    float* p = slab + static_cast<int64_t>(SLAB_GATE + s) * a.c + (t + v * T) * 8;
#pragma unroll
                                    for (int e = 0; e < 8; ++e) p[e] += r[8 * v + e];
                                }
                        }
                        __syncwarp();
                    }
                } else {
#pragma unroll
                    for (int i = 0; i < V * 8; ++i) acc_gate[i] += live ? r[i] : 0.f;
                }
            } else {
#pragma unroll
                for (int i = 0; i < V * 8; ++i) acc_gate[i] += r[i];
            }
        }
    }
    if (a.gate) {
        if (!a.nsamples) cur = 0;
        flush_gate();
    }
    auto put = [&](float* acc, int slab_row) {
#pragma unroll
        for (int v = 0; v < V; ++v)
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                float q = acc[8 * v + e];
                if constexpr (T < 32) {
#pragma unroll
                    for (int o = T; o < 32; o <<= 1) q += __shfl_xor_sync(0xffffffffu, q, o);
                }
                if (sub == 0 && t + v * T < chunks)
                    slab[static_cast<int64_t>(slab_row) * a.c + (t + v * T) * 8 + e] = q;
            }
    };
    put(acc_pre_w, SLAB_PRE_W);
    put(acc_pre_b, SLAB_PRE_B);
    put(acc_post_w, SLAB_POST_W);
    put(acc_post_b, SLAB_POST_B);
}

// Column sums over the units, 32 columns a block, in double and in a fixed order.
__global__ void __launch_bounds__(1024) slab_sum_kernel(const float* part, int64_t units, int slab_rows, int c,
                                                        RowNormGrads g) {
    __shared__ double red[32][33];
    const int col = blockIdx.x * 32 + threadIdx.x;
    const int srow = blockIdx.y;
    float* dst = nullptr;
    if (srow == SLAB_PRE_W) dst = g.pre_w;
    else if (srow == SLAB_PRE_B) dst = g.pre_b;
    else if (srow == SLAB_POST_W) dst = g.post_w;
    else if (srow == SLAB_POST_B) dst = g.post_b;
    else if (g.gate) dst = g.gate + static_cast<int64_t>(srow - SLAB_GATE) * c;
    if (!dst) return;
    double s = 0.0;
    if (col < c)
        for (int64_t u = threadIdx.y; u < units; u += 32) s += part[(u * slab_rows + srow) * c + col];
    red[threadIdx.y][threadIdx.x] = s;
    __syncthreads();
    for (int o = 16; o >= 1; o >>= 1) {
        if (threadIdx.y < o) red[threadIdx.y][threadIdx.x] += red[threadIdx.y + o][threadIdx.x];
        __syncthreads();
    }
    if (threadIdx.y == 0 && col < c) dst[col] = static_cast<float>(red[0][threadIdx.x]);
}

int sm_count() {
    static std::mutex mu;
    static int sms[64] = {0};
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 148;
    std::lock_guard<std::mutex> lk(mu);
    if (!sms[dev]) {
        int count = 0;
        if (cudaDeviceGetAttribute(&count, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) count = 148;
        sms[dev] = count;
    }
    return sms[dev];
}

// Threads a row: 8 columns each up to 2048 channels, 16 beyond.
int row_threads(int c) {
    int t = 8;
    while (t < 256 && t * 8 < c) t *= 2;
    return c > 2048 ? 512 : t;
}

// Units of the backward pass: enough to fill the GPU, at least four steps of
// rows each where there are that many, and few enough that the slabs stay
// within 64 MiB however many samples have a gate.
void backward_units(int64_t n, int c, int nsamples, int64_t* units, int64_t* rows_per_unit) {
    const int t = row_threads(c);
    const int64_t r = t > 32 ? 1 : 32 / t;
    constexpr int64_t kSms = 148;  // B200; a fixed count keeps the workspace size and the sums the same everywhere
    int64_t u = t > 32 ? kSms * (512 / t) : kSms * 16;
    const int64_t slab = static_cast<int64_t>(4 + std::max(nsamples, 1)) * c * 4;
    u = std::min(u, std::max<int64_t>((int64_t(64) << 20) / slab, 1));
    u = std::min(u, std::max<int64_t>((n + 4 * r - 1) / (4 * r), 1));
    int64_t rows = (n + u - 1) / u;
    rows = (rows + r - 1) / r * r;
    *rows_per_unit = std::max<int64_t>(rows, r);
    *units = std::max<int64_t>((n + *rows_per_unit - 1) / *rows_per_unit, 1);
}

template <int XT, int FT, int T, int V>
cudaError_t launch_fwd(const RowNormArgs& a, cudaStream_t st) {
    constexpr int threads = block_threads<T>();
    constexpr int rows = T > 32 ? 1 : threads / T;  // rows a block and step
    const int64_t blocks = (a.n + rows - 1) / rows;
    const int64_t cap = static_cast<int64_t>(sm_count()) * (2048 / threads);
    rownorm_kernel<XT, FT, T, V><<<static_cast<unsigned>(std::min(blocks, cap)), threads, 0, st>>>(a);
    return cudaGetLastError();
}

template <int XT, int FT, int T, int V>
cudaError_t launch_bwd(const RowNormArgs& a, cudaStream_t st) {
    constexpr int threads = block_threads<T>();
    constexpr int per_block = T > 32 ? 1 : threads / 32;
    rownorm_backward_kernel<XT, FT, T, V>
        <<<static_cast<unsigned>((a.units + per_block - 1) / per_block), threads, 0, st>>>(a);
    return cudaGetLastError();
}

template <int XT, int FT>
cudaError_t launch_c(const RowNormArgs& a, bool backward, cudaStream_t st) {
#define MSC_ROWNORM_CASE(T, V) return backward ? launch_bwd<XT, FT, T, V>(a, st) : launch_fwd<XT, FT, T, V>(a, st)
    switch (row_threads(a.c)) {
        case 8: MSC_ROWNORM_CASE(8, 1);
        case 16: MSC_ROWNORM_CASE(16, 1);
        case 32: MSC_ROWNORM_CASE(32, 1);
        case 64: MSC_ROWNORM_CASE(64, 1);
        case 128: MSC_ROWNORM_CASE(128, 1);
        default: break;
    }
    if (a.c <= 2048) MSC_ROWNORM_CASE(256, 1);
    MSC_ROWNORM_CASE(512, 2);
#undef MSC_ROWNORM_CASE
}

cudaError_t launch_any(const RowNormArgs& a, bool backward, cudaStream_t st) {
    if (a.x_dtype == DT_F32) {
        if (a.f_dtype == DT_F32) return launch_c<DT_F32, DT_F32>(a, backward, st);
        if (a.f_dtype == DT_F16) return launch_c<DT_F32, DT_F16>(a, backward, st);
        return launch_c<DT_F32, DT_BF16>(a, backward, st);
    }
    if (a.x_dtype == DT_F16) return launch_c<DT_F16, DT_F16>(a, backward, st);
    return launch_c<DT_BF16, DT_BF16>(a, backward, st);
}

}  // namespace

bool rownorm_dtypes_supported(int x_dtype, int f_dtype) { return x_dtype == f_dtype || x_dtype == DT_F32; }

cudaError_t launch_rownorm(const RowNormArgs& a, cudaStream_t st) {
    return a.n ? launch_any(a, false, st) : cudaSuccess;
}

size_t rownorm_backward_workspace_bytes(int64_t n, int c, int nsamples) {
    int64_t units = 0, rows = 0;
    backward_units(n, c, nsamples, &units, &rows);
    return static_cast<size_t>(units) * (SLAB_GATE + std::max(nsamples, 1)) * c * sizeof(float);
}

cudaError_t launch_rownorm_backward(RowNormArgs a, const RowNormGrads& g, void* ws, cudaStream_t st) {
    a.partial = static_cast<float*>(ws);
    backward_units(a.n, a.c, a.nsamples, &a.units, &a.rows_per_unit);
    const int slab_rows = SLAB_GATE + (!a.gate ? 0 : (a.nsamples ? a.nsamples : 1));
    // the gate rows are added to, so they start at zero (all rows do where n = 0)
    if (a.gate || a.n == 0) {
        cudaError_t e = cudaMemsetAsync(ws, 0, static_cast<size_t>(a.units) * slab_rows * a.c * sizeof(float), st);
        if (e != cudaSuccess) return e;
    }
    if (a.n) {
        cudaError_t e = launch_any(a, true, st);
        if (e != cudaSuccess) return e;
    }
    slab_sum_kernel<<<dim3((a.c + 31) / 32, slab_rows), dim3(32, 32), 0, st>>>(a.partial, a.units, slab_rows, a.c, g);
    return cudaGetLastError();
}

}  // namespace msc
