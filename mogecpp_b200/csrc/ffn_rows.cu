// Gated feed-forward block of a few rows (a global token, single tokens of a
// batch): bound by reading the weights once.
//
// Two kernels of dot products on the CUDA cores (packed f32x2, fp32
// throughout; h stays fp32 between them).  The first gives each hidden unit
// to a warp, which holds its rows of both projections and all input rows'
// sums; the second splits each output's hidden sum over the warps of a block
// (about 1024 weights a warp) and joins them in a fixed order.  The second is
// launched with the first (programmatic dependent launch): it fetches its
// weights while the first still runs and only then waits for h.
//
// Measured: one row of 1024 -> 4096 bf16 6.8 us for 25 MB of weights (3.7 TB/s
// with both launches; the weights stay in L2 when the same block runs again);
// the tensor-core path takes 19 us.
//
// A tensor-core tile would be 128 rows high for these few, and its CTAs too
// few to draw the whole memory bandwidth.
#include "ffn.h"

#include "common.cuh"
#include "conv.h"
#include "ffn_act.cuh"
#include "ffn_rows.h"

namespace msc {
namespace {

constexpr int kWarps = 8;
constexpr int kWarpSpan = 1024;  // weights a warp holds at once: 4 x 16 bytes a lane

template <bool BF16>
__device__ __forceinline__ void unpack_w(const uint4& q, uint64_t (&v)[4]) {
    const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        if constexpr (BF16) {
            v[e] = pack2(__uint_as_float(w[e] << 16), __uint_as_float(w[e] & 0xffff0000u));
        } else {
            const float2 t = __half22float2(*reinterpret_cast<const __half2*>(&w[e]));
            v[e] = pack2(t.x, t.y);
        }
    }
}

__device__ __forceinline__ uint4 load_stream(const void* p, int64_t off) {
    uint4 q;
    asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(q.x), "=r"(q.y), "=r"(q.z), "=r"(q.w)
                 : "l"(static_cast<const uint16_t*>(p) + off));
    return q;
}

__device__ __forceinline__ float warp_total(uint64_t v) {
    float a, b;
    unpack2(v, a, b);
    a += b;
#pragma unroll
    for (int o = 16; o >= 1; o >>= 1) a += __shfl_xor_sync(0xffffffffu, a, o);
    return a;
}

template <int NR, bool BF16>
__global__ void __launch_bounds__(32 * kWarps) rows_hidden_kernel(const void* x, int n, int c, int hidden, FfnWeights w,
                                                                  int act, float* h) {
    launch_dependents();
    const int lane = threadIdx.x & 31;
    const int j = blockIdx.x * kWarps + (threadIdx.x >> 5);
    if (j >= hidden) return;
    const int64_t row = static_cast<int64_t>(j) * c;
    uint64_t g[NR], u[NR];
#pragma unroll
    for (int r = 0; r < NR; ++r) g[r] = u[r] = 0ull;
    for (int base = 0; base < c; base += kWarpSpan) {
        uint4 qg[4], qu[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int k = base + (i * 32 + lane) * 8;
            qg[i] = qu[i] = make_uint4(0u, 0u, 0u, 0u);
            if (k < c) {
                qg[i] = load_stream(w.w_gate, row + k);
                qu[i] = load_stream(w.w_up, row + k);
            }
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int k = base + (i * 32 + lane) * 8;
            if (k < c) {
                uint64_t vg[4], vu[4];
                unpack_w<BF16>(qg[i], vg);
                unpack_w<BF16>(qu[i], vu);
#pragma unroll
                for (int r = 0; r < NR; ++r) {
                    uint64_t vx[4];
                    const int64_t rr = min(r, n - 1);
                    unpack_w<BF16>(*reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(x) + rr * c + k), vx);
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        g[r] = fma2(vg[e], vx[e], g[r]);
                        u[r] = fma2(vu[e], vx[e], u[r]);
                    }
                }
            }
        }
    }
    const float bg = w.b_gate ? __ldg(w.b_gate + j) : 0.f, bu = w.b_up ? __ldg(w.b_up + j) : 0.f;
#pragma unroll
    for (int r = 0; r < NR; ++r) {
        const float tg = warp_total(g[r]) + bg, tu = warp_total(u[r]) + bu;
        if (r < n && lane == r) {
            float a[2] = {tg, 0.f};
            const float b[2] = {tu, 0.f};
            gate_chunk(act, a, b);
            h[static_cast<int64_t>(r) * hidden + j] = a[0];
        }
    }
}

template <int NR, bool BF16, int SLICES>
__global__ void __launch_bounds__(32 * kWarps) rows_down_kernel(const float* h, int n, int c, int hidden, FfnWeights w,
                                                                void* y) {
    __shared__ float part[kWarps][NR];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int i = blockIdx.x * (kWarps / SLICES) + warp / SLICES;
    const int per = (hidden / 8 + SLICES - 1) / SLICES * 8;
    const int k0 = (warp % SLICES) * per, k1 = i < c ? min(k0 + per, hidden) : 0;
    const int64_t row = static_cast<int64_t>(i) * hidden;
    uint64_t s[NR];
#pragma unroll
    for (int r = 0; r < NR; ++r) s[r] = 0ull;
    bool waited = false;
    for (int base = k0; base < k1 || !waited; base += kWarpSpan) {
        uint4 q[4];
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            const int k = base + (t * 32 + lane) * 8;
            q[t] = make_uint4(0u, 0u, 0u, 0u);
            if (k < k1) q[t] = load_stream(w.w_down, row + k);
        }
        if (!waited) wait_dependency();
        waited = true;
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            const int k = base + (t * 32 + lane) * 8;
            if (k < k1) {
                uint64_t v[4];
                unpack_w<BF16>(q[t], v);
#pragma unroll
                for (int r = 0; r < NR; ++r) {
                    const float4* p = reinterpret_cast<const float4*>(h + static_cast<int64_t>(min(r, n - 1)) * hidden + k);
                    const float4 a = p[0], b = p[1];
                    s[r] = fma2(v[0], pack2(a.x, a.y), s[r]);
                    s[r] = fma2(v[1], pack2(a.z, a.w), s[r]);
                    s[r] = fma2(v[2], pack2(b.x, b.y), s[r]);
                    s[r] = fma2(v[3], pack2(b.z, b.w), s[r]);
                }
            }
        }
    }
#pragma unroll
    for (int r = 0; r < NR; ++r) {
        const float t = warp_total(s[r]);
        if (lane == 0) part[warp][r] = t;
    }
    __syncthreads();
    if (warp % SLICES == 0 && i < c && lane < n && lane < NR) {
        float t = 0.f;
#pragma unroll
        for (int k = 0; k < SLICES; ++k) t += part[warp + k][lane];
        if (w.b_down) t += __ldg(w.b_down + i);
        const int64_t o = static_cast<int64_t>(lane) * c + i;
        if constexpr (BF16)
            static_cast<__nv_bfloat16*>(y)[o] = __float2bfloat16_rn(t);
        else
            static_cast<__half*>(y)[o] = __float2half_rn(t);
    }
}

template <int NR, bool BF16, int SLICES>
cudaError_t launch_down(const FfnShape& s, const FfnWeights& w, void* y, const float* h, cudaStream_t st) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((s.c + kWarps / SLICES - 1) / (kWarps / SLICES));
    cfg.blockDim = dim3(32 * kWarps);
    cfg.stream = st;
    cudaLaunchAttribute at{};
    at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &at;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, rows_down_kernel<NR, BF16, SLICES>, h, static_cast<int>(s.n), s.c, s.hidden, w, y);
}

template <int NR, bool BF16>
cudaError_t launch_nr(const FfnShape& s, const void* x, const FfnWeights& w, void* y, float* h, cudaStream_t st) {
    rows_hidden_kernel<NR, BF16><<<(s.hidden + kWarps - 1) / kWarps, 32 * kWarps, 0, st>>>(
        x, static_cast<int>(s.n), s.c, s.hidden, w, s.act, h);
    const cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) return e;
    if (s.hidden > 4 * kWarpSpan) return launch_down<NR, BF16, 8>(s, w, y, h, st);
    if (s.hidden > kWarpSpan) return launch_down<NR, BF16, 4>(s, w, y, h, st);
    return launch_down<NR, BF16, 1>(s, w, y, h, st);
}

template <bool BF16>
cudaError_t launch_dt(const FfnShape& s, const void* x, const FfnWeights& w, void* y, float* h, cudaStream_t st) {
    if (s.n == 1) return launch_nr<1, BF16>(s, x, w, y, h, st);
    if (s.n == 2) return launch_nr<2, BF16>(s, x, w, y, h, st);
    if (s.n <= 4) return launch_nr<4, BF16>(s, x, w, y, h, st);
    return launch_nr<8, BF16>(s, x, w, y, h, st);
}

}  // namespace

cudaError_t launch_ffn_rows(const FfnShape& s, const void* x, const FfnWeights& w, void* y, float* h, cudaStream_t st) {
    return s.dtype == DT_BF16 ? launch_dt<true>(s, x, w, y, h, st) : launch_dt<false>(s, x, w, y, h, st);
}

}  // namespace msc
