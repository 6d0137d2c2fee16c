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
// A row's tensors are read and written once (8 B an element forward and 12 B
// backward for 16-bit tensors) for some 20-40 fp32 operations an element:
// HBM's work, if the instructions do not get in its way.  A row is held in
// registers by T threads, 8 columns (16 bytes of a 16-bit tensor) each: 8 to
// 32 lanes of a warp up to 256 channels, so that a row's means are shuffles
// alone and a warp has up to four rows in flight; a block per row beyond (one
// shared-memory exchange per mean; 16 columns a thread beyond 2048).  A thread
// keeps its columns of every weight in registers over all its rows, works on
// packed f32 pairs, and its rows come through a cp.async ring up to four
// steps deep.  Measured at 402,131 x 128 bf16 with a gate per sample: forward
// 178 us as first written, 101 with packed arithmetic and the gate folded into
// the post norm, 90 with unpredicated loads, 73.5 with the ring (5.7 TB/s, 87 %
// of the copy rate); backward 255, 206, 164 and 128 us (4.9 TB/s; issue slots
// 63 %: the row sums' shuffles at the 16 warps that 128 registers allow).
// Above 2048 channels the backward pass spills (436 to 564 bytes a thread):
// 20,000 x 4096 bf16 takes 1,026 us, x 8192 954, x 2048 171.
//
// The backward column sums are kept in fp32 registers over a unit's (warp's
// or block's) run of rows, at most 1,024 steps, written once per unit, and
// added over the units (and passes over them, where the rows are more) in
// double in a fixed order by a second kernel: no atomics, the same bits every
// time.  A per-sample gate adds its sums (fp32) to the unit's own slab whenever
// the sample changes (rows are normally sorted by sample; any order is right).
#include "rownorm.h"

#include "common.cuh"
#include "conv.h"

#include <algorithm>
#include <atomic>
#include <mutex>
#include <type_traits>

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
__device__ __forceinline__ Raw8<DT> zero8() {
    Raw8<DT> r;
#pragma unroll
    for (int i = 0; i < (DT == DT_F32 ? 2 : 1); ++i) r.q[i] = make_uint4(0u, 0u, 0u, 0u);
    return r;
}

// Rows on their way from global memory: a ring of up to four steps in shared
// memory, filled by 16-byte cp.async.  Every thread copies and reads its own
// pieces alone, so that no barrier is needed, only its own wait.  BYTES is a
// thread's share of the SM's shared memory at the kernel's occupancy.

template <int DT>
constexpr int pieces() {
    return DT == DT_F32 ? 2 : 1;
}

// [step][piece][thread] 16-byte pieces, then [step][thread] sample indices.
template <int THREADS, int PIECES, int BYTES>
struct Ring {
    uint32_t base;  // shared-window address of this thread's first piece
    static constexpr int FIT = BYTES / (PIECES * 16 + 4);
    static constexpr int DEPTH = FIT > 4 ? 4 : FIT;
    static_assert(DEPTH >= 1, "one step fits");
    static constexpr size_t bytes() { return static_cast<size_t>(DEPTH) * THREADS * (PIECES * 16 + 4); }
    __device__ __forceinline__ explicit Ring(void* smem) : base(smem_u32(smem) + threadIdx.x * 16) {}
    __device__ __forceinline__ uint32_t at(int slot, int piece) const {
        return base + static_cast<uint32_t>((slot * PIECES + piece) * THREADS * 16);
    }
    __device__ __forceinline__ uint32_t sample_at(int slot) const {
        return base - threadIdx.x * 12 + static_cast<uint32_t>(DEPTH * PIECES * THREADS * 16 + slot * THREADS * 4);
    }
    template <int DT>
    __device__ __forceinline__ void put(int slot, int piece, const void* p, int64_t off) const {
        const uint8_t* src = static_cast<const uint8_t*>(p) + off * (DT == DT_F32 ? 4 : 2);
#pragma unroll
        for (int i = 0; i < pieces<DT>(); ++i) cp_async16(at(slot, piece + i), src + 16 * i, 16);
    }
    template <int DT>
    __device__ __forceinline__ Raw8<DT> get(int slot, int piece) const {
        Raw8<DT> r;
#pragma unroll
        for (int i = 0; i < pieces<DT>(); ++i)
            asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
                         : "=r"(r.q[i].x), "=r"(r.q[i].y), "=r"(r.q[i].z), "=r"(r.q[i].w)
                         : "r"(at(slot, piece + i)));
        return r;
    }
    __device__ __forceinline__ void put_sample(int slot, const int32_t* p) const {
        asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(sample_at(slot)), "l"(p) : "memory");
    }
    __device__ __forceinline__ int get_sample(int slot) const {
        int s;
        asm volatile("ld.shared.s32 %0, [%1];" : "=r"(s) : "r"(sample_at(slot)));
        return s;
    }
};

// The 8 values as four f32 pairs (packed f32x2 arithmetic from here on: the
// forward pass spends its instruction slots, not its memory time, on scalar
// arithmetic otherwise).
template <int DT>
__device__ __forceinline__ void unpack8(const Raw8<DT>& r, uint64_t* v) {
    if constexpr (DT == DT_F32) {
        v[0] = pack2(__uint_as_float(r.q[0].x), __uint_as_float(r.q[0].y));
        v[1] = pack2(__uint_as_float(r.q[0].z), __uint_as_float(r.q[0].w));
        v[2] = pack2(__uint_as_float(r.q[1].x), __uint_as_float(r.q[1].y));
        v[3] = pack2(__uint_as_float(r.q[1].z), __uint_as_float(r.q[1].w));
    } else {
        const uint32_t w[4] = {r.q[0].x, r.q[0].y, r.q[0].z, r.q[0].w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            if constexpr (DT == DT_F16) {
                const float2 t = __half22float2(*reinterpret_cast<const __half2*>(&w[e]));
                v[e] = pack2(t.x, t.y);
            } else {
                v[e] = pack2(__uint_as_float(w[e] << 16), __uint_as_float(w[e] & 0xffff0000u));
            }
        }
    }
}

template <int DT>
__device__ __forceinline__ void store8(void* p, int64_t off, const uint64_t* v) {
    float f[8];
#pragma unroll
    for (int e = 0; e < 4; ++e) unpack2(v[e], f[2 * e], f[2 * e + 1]);
    if constexpr (DT == DT_F32) {
        float4* d = reinterpret_cast<float4*>(static_cast<float*>(p) + off);
        d[0] = make_float4(f[0], f[1], f[2], f[3]);
        d[1] = make_float4(f[4], f[5], f[6], f[7]);
    } else {
        uint32_t w[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            if constexpr (DT == DT_F16) {
                const __half2 h = __floats2half2_rn(f[2 * e], f[2 * e + 1]);
                w[e] = *reinterpret_cast<const uint32_t*>(&h);
            } else {
                const __nv_bfloat162 h = __floats2bfloat162_rn(f[2 * e], f[2 * e + 1]);
                w[e] = *reinterpret_cast<const uint32_t*>(&h);
            }
        }
        *reinterpret_cast<uint4*>(static_cast<uint8_t*>(p) + off * 2) = make_uint4(w[0], w[1], w[2], w[3]);
    }
}

__device__ __forceinline__ float sum_pair(uint64_t v) {
    float a, b;
    unpack2(v, a, b);
    return a + b;
}

// 8 columns of a weight vector (fill where it is absent).
__device__ __forceinline__ void load_param(const float* p, int col, float fill, uint64_t* v) {
    if (p) {
        const float4 a = __ldg(reinterpret_cast<const float4*>(p + col));
        const float4 b = __ldg(reinterpret_cast<const float4*>(p + col) + 1);
        v[0] = pack2(a.x, a.y), v[1] = pack2(a.z, a.w), v[2] = pack2(b.x, b.y), v[3] = pack2(b.z, b.w);
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = both(fill);
    }
}

// Sums of a (and b) over the T threads of a row.  Beyond a warp the partial
// sums cross through shared memory; `turn` alternates between two buffers, so
// that one barrier per exchange orders both its own reads and the reuse.
template <int T, int N>
__device__ __forceinline__ void row_sum(float (&v)[N], float2 (*buf)[T > 32 ? T / 32 : 1], int& turn) {
#pragma unroll
    for (int o = (T < 32 ? T : 32) / 2; o >= 1; o >>= 1) {
#pragma unroll
        for (int k = 0; k < N; ++k) v[k] += __shfl_xor_sync(0xffffffffu, v[k], o);
    }
    if constexpr (T > 32) {
        if ((threadIdx.x & 31) == 0) buf[turn][threadIdx.x >> 5] = make_float2(v[0], v[N - 1]);
        __syncthreads();
        float2 s = make_float2(0.f, 0.f);
#pragma unroll
        for (int w = 0; w < T / 32; ++w) {
            s.x += buf[turn][w].x;
            s.y += buf[turn][w].y;
        }
        v[0] = s.x;
        if constexpr (N > 1) v[1] = s.y;
        turn ^= 1;
    }
}

template <int T>
constexpr int block_threads() {
    return T > 32 ? T : 256;
}

// 0 where the gate is not per sample, -1 where the index is outside the
// samples: a device failure that gates the branch off.
__device__ __forceinline__ int checked_sample(const RowNormArgs& a, int s) {
    return static_cast<unsigned>(s) < static_cast<unsigned>(a.nsamples) ? s : -1;
}

template <int XT, int FT, int T, int V>
using FwdRing = Ring<block_threads<T>(), V * (pieces<XT>() + pieces<FT>()), 290>;
template <int XT, int FT, int T, int V>
using BwdRing = Ring<block_threads<T>(), 2 * V * (pieces<XT>() + pieces<FT>()), 430>;

// Forward.  The gate folds into the post norm's weights (gate * (f^ w + b) =
// f^ (gate w) + gate b), which are multiplied only when the gate changes; the
// next step's row is on its way while this one is computed.
template <int XT, int FT, int T, int V, bool FULL>
__global__ void __launch_bounds__(block_threads<T>(), T > 32 ? (V > 1 ? 1 : 768 / T) : 3) rownorm_kernel(const RowNormArgs a) {
    constexpr int R = T > 32 ? 1 : 32 / T;  // rows per unit and step
    __shared__ float2 buf[2][T > 32 ? T / 32 : 1];
    int turn = 0;
    const int t = T > 32 ? threadIdx.x : threadIdx.x & (T - 1);
    const int sub = T > 32 ? 0 : (threadIdx.x & 31) / T;
    const int64_t unit = T > 32 ? blockIdx.x : blockIdx.x * (block_threads<T>() / 32) + (threadIdx.x >> 5);
    const int64_t units = T > 32 ? gridDim.x : static_cast<int64_t>(gridDim.x) * (block_threads<T>() / 32);
    const int chunks = a.c / 8;
    // FULL: every thread has all its columns (c = 8 T V)
    auto has = [&](int v) { return FULL || t + v * T < chunks; };
    auto column = [&](int v) { return (FULL ? t + v * T : min(t + v * T, chunks - 1)) * 8; };
    const float inv_c = 1.0f / static_cast<float>(a.c);
    const bool has_post = a.post.kind != NORM_NONE;
    uint64_t gate_w[V * 4], gate_b[V * 4];
    int gate_of = -2;  // sample whose gate is folded in
    const uint64_t scale = both(a.res_scale);
    auto load_gate = [&](int s) {
#pragma unroll
        for (int v = 0; v < V; ++v) {
            const int col = column(v);
            load_param(a.post.w, col, 1.f, gate_w + 4 * v);
            load_param(a.post.b, col, 0.f, gate_b + 4 * v);
            if (a.gate) {
                uint64_t g[4];
                load_param(s < 0 ? nullptr : a.gate + static_cast<int64_t>(s) * a.c, col, 0.f, g);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    gate_w[4 * v + e] = mul2(gate_w[4 * v + e], g[e]);
                    gate_b[4 * v + e] = mul2(gate_b[4 * v + e], g[e]);
                }
            }
        }
        gate_of = s;
    };
    uint64_t pre_w[V * 4], pre_b[V * 4];
#pragma unroll
    for (int v = 0; v < V; ++v) {
        const int col = column(v);
        load_param(a.pre.w, col, 1.f, pre_w + 4 * v);
        load_param(a.pre.b, col, 0.f, pre_b + 4 * v);
    }
    // loads run without predicates: rows past the last one read the last one
    // again, threads without a column the last columns, and both are left out
    // of sums and stores
    extern __shared__ uint4 ring_smem[];
    const FwdRing<XT, FT, T, V> ring(ring_smem);
    constexpr int D = FwdRing<XT, FT, T, V>::DEPTH;
    constexpr int PX = pieces<XT>(), PF = pieces<FT>();
    auto fetch = [&](int slot, int64_t row) {
        row = min(row, a.n - 1);
#pragma unroll
        for (int v = 0; v < V; ++v) {
            const int64_t off = row * a.c + column(v);
            ring.template put<XT>(slot, v * PX, a.x, off);
            if (a.f) ring.template put<FT>(slot, V * PX + v * PF, a.f, off);
        }
        if (a.nsamples) ring.put_sample(slot, a.coords + row * 4 + 3);
        cp_async_commit();
    };
#pragma unroll
    for (int k = 0; k < D - 1; ++k) fetch(k, (unit + k * units) * R + sub);
    int slot = 0;
    for (int64_t row0 = unit * R; row0 < a.n; row0 += units * R, slot = (slot + 1) % D) {
        const int64_t row = row0 + sub;
        const bool live = row < a.n;
        fetch((slot + D - 1) % D, row + (D - 1) * units * R);
        cp_async_wait<D - 1>();
        uint64_t f[V * 4], r[V * 4];
#pragma unroll
        for (int v = 0; v < V; ++v) {
            unpack8(ring.template get<XT>(slot, v * PX), r + 4 * v);
            unpack8(a.f ? ring.template get<FT>(slot, V * PX + v * PF) : zero8<FT>(), f + 4 * v);
        }
        const int s = a.nsamples ? checked_sample(a, ring.get_sample(slot)) : 0;
        if (s != gate_of) load_gate(s);
        if (s < 0) set_status(a.status, MSC_DEV_BAD_COORD);
        if (a.f) {
            if (has_post) {
                // two passes over the registers: the variance of the centred values
                float q[1] = {0.f};
                if (a.post.kind == NORM_LAYER) {
#pragma unroll
                    for (int v = 0; v < V; ++v) {
                        uint64_t acc = 0ull;
#pragma unroll
                        for (int e = 0; e < 4; ++e) acc = add2(acc, f[4 * v + e]);
                        if (has(v)) q[0] += sum_pair(acc);
                    }
                    row_sum<T>(q, buf, turn);
                    const uint64_t m = both(-q[0] * inv_c);
#pragma unroll
                    for (int i = 0; i < V * 4; ++i) f[i] = add2(f[i], m);
                }
                q[0] = 0.f;
#pragma unroll
                for (int v = 0; v < V; ++v) {
                    uint64_t acc = 0ull;
#pragma unroll
                    for (int e = 0; e < 4; ++e) acc = fma2(f[4 * v + e], f[4 * v + e], acc);
                    if (has(v)) q[0] += sum_pair(acc);
                }
                row_sum<T>(q, buf, turn);
                const uint64_t k = both(rsqrtf(q[0] * inv_c + a.post.eps));
#pragma unroll
                for (int i = 0; i < V * 4; ++i) f[i] = mul2(f[i], k);
            }
#pragma unroll
            for (int i = 0; i < V * 4; ++i) r[i] = fma2(scale, r[i], fma2(f[i], gate_w[i], gate_b[i]));
            if (s < 0) {
                // the branch of a row without a sample stays out, whatever it holds
#pragma unroll
                for (int v = 0; v < V; ++v)
                    if (live && has(v)) {
                        unpack8(load8<XT>(a.x, row * a.c + (t + v * T) * 8), r + 4 * v);
#pragma unroll
                        for (int e = 0; e < 4; ++e) r[4 * v + e] = mul2(scale, r[4 * v + e]);
                    }
            }
        } else {
#pragma unroll
            for (int i = 0; i < V * 4; ++i) r[i] = mul2(scale, r[i]);
        }
        if (a.r && live) {
#pragma unroll
            for (int v = 0; v < V; ++v)
                if (has(v)) store8<XT>(a.r, row * a.c + (t + v * T) * 8, r + 4 * v);
        }
        if (a.pre.kind != NORM_NONE) {
            float q[1] = {0.f};
            if (a.pre.kind == NORM_LAYER) {
#pragma unroll
                for (int v = 0; v < V; ++v) {
                    uint64_t acc = 0ull;
#pragma unroll
                    for (int e = 0; e < 4; ++e) acc = add2(acc, r[4 * v + e]);
                    if (has(v)) q[0] += sum_pair(acc);
                }
                row_sum<T>(q, buf, turn);
                const uint64_t m = both(-q[0] * inv_c);
#pragma unroll
                for (int i = 0; i < V * 4; ++i) r[i] = add2(r[i], m);
            }
            q[0] = 0.f;
#pragma unroll
            for (int v = 0; v < V; ++v) {
                uint64_t acc = 0ull;
#pragma unroll
                for (int e = 0; e < 4; ++e) acc = fma2(r[4 * v + e], r[4 * v + e], acc);
                if (has(v)) q[0] += sum_pair(acc);
            }
            row_sum<T>(q, buf, turn);
            const uint64_t k = both(rsqrtf(q[0] * inv_c + a.pre.eps));
#pragma unroll
            for (int i = 0; i < V * 4; ++i) r[i] = fma2(mul2(r[i], k), pre_w[i], pre_b[i]);
        }
        // without a norm h, where asked for, is r in the branch's type
        if (a.h && live) {
#pragma unroll
            for (int v = 0; v < V; ++v)
                if (has(v)) store8<FT>(a.h, row * a.c + (t + v * T) * 8, r + 4 * v);
        }
    }
    // the copies past the last row have landed before the shared memory goes
    cp_async_wait_all();
}

// Slab rows of a unit: pre_w, pre_b, post_w, post_b, then the gate's.
enum SlabRow : int { SLAB_PRE_W = 0, SLAB_PRE_B = 1, SLAB_POST_W = 2, SLAB_POST_B = 3, SLAB_GATE = 4 };

// Backward.  With one gate over a run of rows, the sums A = sum dr f^ and B =
// sum dr give all three gradients of the branch (gate w A + b B, post norm's
// weight gate A, its bias gate B), so only A and B are kept per row; they are
// resolved into the unit's slab when the gate changes.
template <int XT, int FT, int T, int V, bool FULL>
__global__ void __launch_bounds__(block_threads<T>(), T > 32 ? 512 / T : 2) rownorm_backward_kernel(const RowNormArgs a) {
    constexpr int R = T > 32 ? 1 : 32 / T;
    __shared__ float2 buf[2][T > 32 ? T / 32 : 1];
    int turn = 0;
    const int t = T > 32 ? threadIdx.x : threadIdx.x & (T - 1);
    const int sub = T > 32 ? 0 : (threadIdx.x & 31) / T;
    const int64_t unit = T > 32 ? blockIdx.x : blockIdx.x * (block_threads<T>() / 32) + (threadIdx.x >> 5);
    if (unit >= a.units) return;  // whole warps (T <= 32, no block barrier) or whole blocks
    const int chunks = a.c / 8;
    // FULL: every thread has all its columns (c = 8 T V)
    auto has = [&](int v) { return FULL || t + v * T < chunks; };
    auto column = [&](int v) { return (FULL ? t + v * T : min(t + v * T, chunks - 1)) * 8; };
    const float inv_c = 1.0f / static_cast<float>(a.c);
    const int slab_rows = SLAB_GATE + (!a.gate ? 0 : (a.nsamples ? a.nsamples : 1));
    float* slab = a.partial + unit * slab_rows * a.c;
    const bool has_pre = a.pre.kind != NORM_NONE, has_post = a.post.kind != NORM_NONE;
    const bool pre_ln = a.pre.kind == NORM_LAYER, post_ln = a.post.kind == NORM_LAYER;
    const uint64_t scale = both(a.res_scale);
    auto clear8 = [&](int srow, int col) {
        float4* p = reinterpret_cast<float4*>(slab + static_cast<int64_t>(srow) * a.c + col);
        p[0] = p[1] = make_float4(0.f, 0.f, 0.f, 0.f);
    };
    if (sub == 0) {
#pragma unroll
        for (int v = 0; v < V; ++v)
            if (has(v)) {
#pragma unroll 1
                for (int q = SLAB_POST_W; q < a.slab_clear; ++q) clear8(q, (t + v * T) * 8);
            }
    }
    if constexpr (T <= 32) __syncwarp();
    uint64_t pre_w[V * 4], gate_w[V * 4];
#pragma unroll
    for (int v = 0; v < V; ++v) load_param(a.pre.w, column(v), 1.f, pre_w + 4 * v);
    auto load_gate8 = [&](int v, int s, uint64_t* g) {
        if (a.gate)
            load_param(s < 0 ? nullptr : a.gate + static_cast<int64_t>(s) * a.c, column(v), 0.f, g);
        else
            load_param(nullptr, 0, 1.f, g);
    };
    int gate_of = -2;
    auto fold_gate = [&](int s) {
#pragma unroll
        for (int v = 0; v < V; ++v) {
            uint64_t g[4];
            load_gate8(v, s, g);
            load_param(a.post.w, column(v), 1.f, gate_w + 4 * v);
#pragma unroll
            for (int e = 0; e < 4; ++e) gate_w[4 * v + e] = mul2(gate_w[4 * v + e], g[e]);
        }
        gate_of = s;
    };
    uint64_t acc_pre_w[V * 4], acc_pre_b[V * 4], acc_a[V * 4], acc_b[V * 4];
#pragma unroll
    for (int i = 0; i < V * 4; ++i) acc_pre_w[i] = acc_pre_b[i] = acc_a[i] = acc_b[i] = 0ull;
    auto add8 = [&](int srow, int col, const uint64_t* v) {
        float* p = slab + static_cast<int64_t>(srow) * a.c + col;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            float lo, hi;
            unpack2(v[e], lo, hi);
            p[2 * e] += lo;
            p[2 * e + 1] += hi;
        }
    };
    // adds A and B of rows of sample s to the slab (by the calling lanes)
    auto resolve = [&](int v, int s, const uint64_t* sa, const uint64_t* sb) {
        const int col = (t + v * T) * 8;
        if (!has(v) || s < 0) return;
        uint64_t g[4], w[4], o[4];
        load_gate8(v, s, g);
#pragma unroll
        for (int e = 0; e < 4; ++e) o[e] = mul2(g[e], sa[e]);
        add8(SLAB_POST_W, col, o);
#pragma unroll
        for (int e = 0; e < 4; ++e) o[e] = mul2(g[e], sb[e]);
        add8(SLAB_POST_B, col, o);
        if (!a.gate) return;
        load_param(a.post.b, col, 0.f, g);
        load_param(a.post.w, col, 1.f, w);
#pragma unroll
        for (int e = 0; e < 4; ++e) o[e] = fma2(w[e], sa[e], mul2(g[e], sb[e]));
        add8(SLAB_GATE + s, col, o);
    };
    auto over_rows = [&](uint64_t* v) {  // sum over the warp's rows
        if constexpr (T < 32) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
#pragma unroll
                for (int o = T; o < 32; o <<= 1) v[e] = add2(v[e], __shfl_xor_sync(0xffffffffu, v[e], o));
            }
        }
    };
    int cur = -1;  // sample of the rows in A and B
    auto flush = [&]() {
#pragma unroll
        for (int v = 0; v < V; ++v) {
            over_rows(acc_a + 4 * v);
            over_rows(acc_b + 4 * v);
            if (sub == 0) resolve(v, cur, acc_a + 4 * v, acc_b + 4 * v);
#pragma unroll
            for (int e = 0; e < 4; ++e) acc_a[4 * v + e] = acc_b[4 * v + e] = 0ull;
        }
        if constexpr (T <= 32) __syncwarp();
    };
    const int64_t row_end = min(a.n, (unit + 1) * a.rows_per_unit);
    extern __shared__ uint4 ring_smem[];
    const BwdRing<XT, FT, T, V> ring(ring_smem);
    constexpr int D = BwdRing<XT, FT, T, V>::DEPTH;
    constexpr int PX = pieces<XT>(), PF = pieces<FT>();
    constexpr int P_GR = V * PX, P_FR = 2 * V * PX, P_HR = P_FR + V * PF;
    auto fetch = [&](int slot, int64_t row) {
        row = min(row, row_end - 1);
#pragma unroll
        for (int v = 0; v < V; ++v) {
            const int64_t off = row * a.c + column(v);
            if (has_pre) ring.template put<XT>(slot, v * PX, a.x, off);
            if (a.dr) ring.template put<XT>(slot, P_GR + v * PX, a.dr, off);
            if (a.f) ring.template put<FT>(slot, P_FR + v * PF, a.f, off);
            if (a.dh) ring.template put<FT>(slot, P_HR + v * PF, a.dh, off);
        }
        if (a.nsamples) ring.put_sample(slot, a.coords + row * 4 + 3);
        cp_async_commit();
    };
#pragma unroll
    for (int k = 0; k < D - 1; ++k) fetch(k, unit * a.rows_per_unit + k * R + sub);
    int slot = 0;
    for (int64_t row0 = unit * a.rows_per_unit; row0 < row_end; row0 += R, slot = (slot + 1) % D) {
        const int64_t row = row0 + sub;
        const bool live = row < row_end;
        fetch((slot + D - 1) % D, row + (D - 1) * R);
        cp_async_wait<D - 1>();
        uint64_t r[V * 4], f[V * 4], d[V * 4], g[V * 4];
#pragma unroll
        for (int v = 0; v < V; ++v) {
            unpack8(has_pre ? ring.template get<XT>(slot, v * PX) : zero8<XT>(), r + 4 * v);
            unpack8(a.dr ? ring.template get<XT>(slot, P_GR + v * PX) : zero8<XT>(), g + 4 * v);
            unpack8(a.f ? ring.template get<FT>(slot, P_FR + v * PF) : zero8<FT>(), f + 4 * v);
            unpack8(a.dh ? ring.template get<FT>(slot, P_HR + v * PF) : zero8<FT>(), d + 4 * v);
        }
        const int s = a.nsamples ? checked_sample(a, ring.get_sample(slot)) : 0;
        if (!live) {
            // past the run: nothing to add
#pragma unroll
            for (int i = 0; i < V * 4; ++i) d[i] = g[i] = 0ull;
        }
        if (s != gate_of) fold_gate(s);
        if (s < 0) {
            // a row without a sample has no branch
            set_status(a.status, MSC_DEV_BAD_COORD);
#pragma unroll
            for (int i = 0; i < V * 4; ++i) f[i] = 0ull;
        }
        // the rows' gate changes: resolve the sums so far
        bool mixed = false;
        {
            int first = s;
            if constexpr (T < 32) {
                first = __shfl_sync(0xffffffffu, s, 0);  // the first row of a step is always live
                mixed = !__all_sync(0xffffffffu, s == first);
            }
            if (mixed || first != cur) {
                flush();
                cur = mixed ? -1 : first;
            }
        }
        // both norms' statistics together: means, then centred squares
        float q[2] = {0.f, 0.f};
        if (pre_ln || post_ln) {
#pragma unroll
            for (int v = 0; v < V; ++v) {
                uint64_t u0 = 0ull, u1 = 0ull;
#pragma unroll
                for (int e = 0; e < 4; ++e) u0 = add2(u0, r[4 * v + e]), u1 = add2(u1, f[4 * v + e]);
                if (has(v)) q[0] += sum_pair(u0), q[1] += sum_pair(u1);
            }
            row_sum<T>(q, buf, turn);
            const uint64_t rm = both(pre_ln ? -q[0] * inv_c : 0.f), fm = both(post_ln ? -q[1] * inv_c : 0.f);
#pragma unroll
            for (int i = 0; i < V * 4; ++i) r[i] = add2(r[i], rm), f[i] = add2(f[i], fm);
            q[0] = q[1] = 0.f;
        }
#pragma unroll
        for (int v = 0; v < V; ++v) {
            uint64_t u0 = 0ull, u1 = 0ull;
#pragma unroll
            for (int e = 0; e < 4; ++e)
                u0 = fma2(r[4 * v + e], r[4 * v + e], u0), u1 = fma2(f[4 * v + e], f[4 * v + e], u1);
            if (has(v)) q[0] += sum_pair(u0), q[1] += sum_pair(u1);
        }
        row_sum<T>(q, buf, turn);
        const float r_k = rsqrtf(q[0] * inv_c + a.pre.eps);
        const float f_k = has_post ? rsqrtf(q[1] * inv_c + a.post.eps) : 1.f;
        // dr = dr + norm'_pre(dh; r)
        if (has_pre) {
            const uint64_t k2 = both(r_k);
            q[0] = q[1] = 0.f;
#pragma unroll
            for (int v = 0; v < V; ++v) {
                uint64_t u0 = 0ull, u1 = 0ull;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int i = 4 * v + e;
                    r[i] = mul2(r[i], k2);
                    acc_pre_w[i] = fma2(d[i], r[i], acc_pre_w[i]);
                    acc_pre_b[i] = add2(acc_pre_b[i], d[i]);
                    d[i] = mul2(d[i], pre_w[i]);
                    u0 = add2(u0, d[i]);
                    u1 = fma2(d[i], r[i], u1);
                }
                if (has(v)) q[0] += sum_pair(u0), q[1] += sum_pair(u1);
            }
            row_sum<T>(q, buf, turn);
            const uint64_t m1 = both(pre_ln ? -q[0] * inv_c : 0.f), m2 = both(-q[1] * inv_c);
#pragma unroll
            for (int i = 0; i < V * 4; ++i) g[i] = fma2(k2, add2(fma2(r[i], m2, d[i]), m1), g[i]);
        } else {
#pragma unroll
            for (int i = 0; i < V * 4; ++i) g[i] = add2(g[i], d[i]);
        }
        if (a.dx && live) {
#pragma unroll
            for (int v = 0; v < V; ++v)
                if (has(v)) {
                    uint64_t o[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) o[e] = mul2(scale, g[4 * v + e]);
                    store8<XT>(a.dx, row * a.c + (t + v * T) * 8, o);
                }
        }
        if (!a.f) continue;
        const uint64_t k2 = both(f_k);
        q[0] = q[1] = 0.f;
#pragma unroll
        for (int v = 0; v < V; ++v) {
            uint64_t u0 = 0ull, u1 = 0ull;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int i = 4 * v + e;
                f[i] = mul2(f[i], k2);  // f^, or f without a norm
                d[i] = mul2(g[i], gate_w[i]);
                u0 = add2(u0, d[i]);
                u1 = fma2(d[i], f[i], u1);
            }
            if (has(v)) q[0] += sum_pair(u0), q[1] += sum_pair(u1);
        }
        if (mixed) {
            // the step's rows belong to different samples: one row after the other
            for (int k = 0; k < R; ++k) {
                if (sub == k && live) {
#pragma unroll
                    for (int v = 0; v < V; ++v) {
                        uint64_t u0[4];
#pragma unroll
                        for (int e = 0; e < 4; ++e) u0[e] = mul2(g[4 * v + e], f[4 * v + e]);
                        resolve(v, s, u0, g + 4 * v);
                    }
                }
                __syncwarp();
            }
        } else {
#pragma unroll
            for (int i = 0; i < V * 4; ++i) acc_a[i] = fma2(g[i], f[i], acc_a[i]), acc_b[i] = add2(acc_b[i], g[i]);
        }
        if (has_post) {
            row_sum<T>(q, buf, turn);
            const uint64_t n1 = both(post_ln ? -q[0] * inv_c : 0.f), n2 = both(-q[1] * inv_c);
#pragma unroll
            for (int i = 0; i < V * 4; ++i) d[i] = mul2(k2, add2(fma2(f[i], n2, d[i]), n1));
        }
        if (a.df && live) {
#pragma unroll
            for (int v = 0; v < V; ++v)
                if (has(v)) store8<FT>(a.df, row * a.c + (t + v * T) * 8, d + 4 * v);
        }
    }
    flush();
    auto put = [&](uint64_t* acc, int srow) {
#pragma unroll
        for (int v = 0; v < V; ++v) {
            over_rows(acc + 4 * v);
            if (sub == 0 && has(v)) {
                float o[8];
#pragma unroll
                for (int e = 0; e < 4; ++e) unpack2(acc[4 * v + e], o[2 * e], o[2 * e + 1]);
                float4* p = reinterpret_cast<float4*>(slab + static_cast<int64_t>(srow) * a.c + (t + v * T) * 8);
                p[0] = make_float4(o[0], o[1], o[2], o[3]);
                p[1] = make_float4(o[4], o[5], o[6], o[7]);
            }
        }
    };
    put(acc_pre_w, SLAB_PRE_W);
    put(acc_pre_b, SLAB_PRE_B);
    // the copies past the run have landed before the shared memory goes
    cp_async_wait_all();
}

// Column sums over the units, 8 columns (a 32-byte sector) a block, in double
// and in a fixed order, of the slab rows from row0 on.  Of several passes over
// the rows each adds its sums to `totals` [4][c], which the first one starts
// (pass 0), and the last one writes the gradients.
__global__ void __launch_bounds__(1024) slab_sum_kernel(const float* part, int64_t units, int slab_rows, int row0, int c,
                                                        double* totals, int64_t pass, bool last, RowNormGrads g) {
    __shared__ double red[128][9];
    const int tx = threadIdx.x & 7, ty = threadIdx.x >> 3;
    const int col = blockIdx.x * 8 + tx;
    const int srow = row0 + blockIdx.y;
    float* dst = nullptr;
    if (srow == SLAB_PRE_W) dst = g.pre_w;
    else if (srow == SLAB_PRE_B) dst = g.pre_b;
    else if (srow == SLAB_POST_W) dst = g.post_w;
    else if (srow == SLAB_POST_B) dst = g.post_b;
    else if (g.gate) dst = g.gate + static_cast<int64_t>(srow - SLAB_GATE) * c;
    if (!dst) return;
    double s = 0.0;
#pragma unroll 8
    for (int64_t u = ty; u < units; u += 128) s += part[(u * slab_rows + srow) * c + col];
    red[ty][tx] = s;
    __syncthreads();
    for (int o = 64; o >= 1; o >>= 1) {
        if (ty < o) red[ty][tx] += red[ty + o][tx];
        __syncthreads();
    }
    if (ty == 0) {
        double* total = totals + static_cast<int64_t>(srow) * c + col;
        const double sum = pass ? *total + red[0][tx] : red[0][tx];
        if (last) dst[col] = static_cast<float>(sum);
        else *total = sum;
    }
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
// rows each where there are that many; but no more than 64 MiB of slabs, since
// a gate per sample takes nsamples rows of each unit's.  Many samples therefore
// leave fewer units, and the pass slows down: 400,000 x 128 bf16 takes 144 us
// with 2 samples, 239 with 64, 987 with 512, 7,750 with 4,096 and 90,500 with
// 32,768.
//
// No unit's fp32 sums run over more than kRunSteps steps (an fp32 chain over
// the 100,000 rows that each of three units has left in the last of these was
// off by 3.5e-4 of a sum of one sign): more rows take several passes.
constexpr int kRunSteps = 1024;
struct BackwardPlan {
    int64_t units, rows_per_unit, passes;
};
BackwardPlan backward_plan(int64_t n, int c, int nsamples) {
    const int t = row_threads(c);
    const int64_t r = t > 32 ? 1 : 32 / t;
    constexpr int64_t kSms = 148;  // B200; a fixed count keeps the workspace size and the sums the same everywhere
    int64_t u = t > 32 ? kSms * (512 / t) : kSms * 16;
    const int64_t slab = static_cast<int64_t>(SLAB_GATE + std::max(nsamples, 1)) * c * 4;
    u = std::min(u, std::max<int64_t>((int64_t(64) << 20) / slab, 1));
    u = std::min(u, std::max<int64_t>((n + 4 * r - 1) / (4 * r), 1));
    const int64_t rows = (n + u - 1) / u, run = kRunSteps * r;
    const int64_t parts = std::max<int64_t>((rows + run - 1) / run, 1);
    BackwardPlan p{};
    p.rows_per_unit = std::max(((rows + parts - 1) / parts + r - 1) / r * r, r);
    const int64_t all = std::max<int64_t>((n + p.rows_per_unit - 1) / p.rows_per_unit, 1);
    p.units = std::min(u, all);
    p.passes = (all + p.units - 1) / p.units;
    return p;
}

// Shared-memory opt-in of a kernel, once per device.
cudaError_t smem_opt_in(const void* kern, size_t smem, std::atomic<uint64_t>& done) {
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (dev < 0 || dev >= 64) return cudaErrorInvalidDevice;
    if (done.load(std::memory_order_acquire) >> dev & 1) return cudaSuccess;
    e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem));
    if (e == cudaSuccess) done.fetch_or(uint64_t(1) << dev, std::memory_order_release);
    return e;
}

template <int XT, int FT, int T, int V, bool FULL>
cudaError_t launch_fwd(const RowNormArgs& a, cudaStream_t st) {
    constexpr int threads = block_threads<T>();
    constexpr size_t smem = FwdRing<XT, FT, T, V>::bytes();
    static std::atomic<uint64_t> done{0};
    const cudaError_t e = smem_opt_in(reinterpret_cast<const void*>(rownorm_kernel<XT, FT, T, V, FULL>), smem, done);
    if (e != cudaSuccess) return e;
    constexpr int rows = T > 32 ? 1 : threads / T;  // rows a block and step
    const int64_t blocks = (a.n + rows - 1) / rows;
    const int64_t cap = static_cast<int64_t>(sm_count()) * std::max(768 / threads, 1);
    rownorm_kernel<XT, FT, T, V, FULL><<<static_cast<unsigned>(std::min(blocks, cap)), threads, smem, st>>>(a);
    return cudaGetLastError();
}

template <int XT, int FT, int T, int V, bool FULL>
cudaError_t launch_bwd(const RowNormArgs& a, cudaStream_t st) {
    constexpr int threads = block_threads<T>();
    constexpr size_t smem = BwdRing<XT, FT, T, V>::bytes();
    static std::atomic<uint64_t> done{0};
    const cudaError_t e = smem_opt_in(reinterpret_cast<const void*>(rownorm_backward_kernel<XT, FT, T, V, FULL>), smem, done);
    if (e != cudaSuccess) return e;
    constexpr int per_block = T > 32 ? 1 : threads / 32;
    rownorm_backward_kernel<XT, FT, T, V, FULL>
        <<<static_cast<unsigned>((a.units + per_block - 1) / per_block), threads, smem, st>>>(a);
    return cudaGetLastError();
}

template <int XT, int FT>
cudaError_t launch_c(const RowNormArgs& a, bool backward, cudaStream_t st) {
#define MSC_ROWNORM_CASE(T, V)                                                                               \
    if (a.c == 8 * T * V)                                                                                    \
        return backward ? launch_bwd<XT, FT, T, V, true>(a, st) : launch_fwd<XT, FT, T, V, true>(a, st);     \
    return backward ? launch_bwd<XT, FT, T, V, false>(a, st) : launch_fwd<XT, FT, T, V, false>(a, st)
    switch (row_threads(a.c)) {
        case 8: MSC_ROWNORM_CASE(8, 1);
        case 16: MSC_ROWNORM_CASE(16, 1);
        case 32: MSC_ROWNORM_CASE(32, 1);
        case 64: MSC_ROWNORM_CASE(64, 1);
        case 128: MSC_ROWNORM_CASE(128, 1);
        default: break;
    }
    if (a.c <= 2048) {
        MSC_ROWNORM_CASE(256, 1);
    }
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
    const BackwardPlan p = backward_plan(n, c, nsamples);
    const size_t rows = SLAB_GATE + std::max(nsamples, 1);
    return p.units * rows * c * sizeof(float) + (p.passes > 1 ? SLAB_GATE * c * sizeof(double) : 0);
}

cudaError_t launch_rownorm_backward(RowNormArgs a, const RowNormGrads& g, void* ws, cudaStream_t st) {
    const BackwardPlan p = backward_plan(a.n, a.c, a.nsamples);
    const int slab_rows = SLAB_GATE + (!a.gate ? 0 : (a.nsamples ? a.nsamples : 1));
    double* const totals = static_cast<double*>(ws);  // where there are several passes
    a.partial = reinterpret_cast<float*>(totals + (p.passes > 1 ? SLAB_GATE * a.c : 0));
    a.rows_per_unit = p.rows_per_unit;
    const int64_t n = a.n, x_row = a.c * (a.x_dtype == DT_F32 ? 4 : 2), f_row = a.c * (a.f_dtype == DT_F32 ? 4 : 2);
    auto advance = [](auto*& q, int64_t bytes) {
        if (q) q = reinterpret_cast<std::remove_reference_t<decltype(q)>>(reinterpret_cast<uintptr_t>(q) + bytes);
    };
    for (int64_t pass = 0; pass < p.passes; ++pass) {
        const int64_t row0 = pass * p.units * p.rows_per_unit;
        RowNormArgs b = a;
        b.n = std::min(p.units * p.rows_per_unit, n - row0);
        b.units = std::max<int64_t>((b.n + p.rows_per_unit - 1) / p.rows_per_unit, 1);
        advance(b.x, row0 * x_row), advance(b.dr, row0 * x_row), advance(b.dx, row0 * x_row);
        advance(b.f, row0 * f_row), advance(b.dh, row0 * f_row), advance(b.df, row0 * f_row);
        advance(b.coords, row0 * 16);
        b.slab_clear = pass ? SLAB_GATE : slab_rows;
        const cudaError_t e =
            b.n ? launch_any(b, true, st)
                : cudaMemsetAsync(a.partial, 0, static_cast<size_t>(b.units) * slab_rows * a.c * sizeof(float), st);
        if (e != cudaSuccess) return e;
        const bool once = p.passes == 1, last = pass + 1 == p.passes;
        slab_sum_kernel<<<dim3(a.c / 8, once ? slab_rows : SLAB_GATE), 1024, 0, st>>>(
            a.partial, b.units, slab_rows, 0, a.c, totals, pass, last, g);
        // the gate's rows of all the units there were
        if (last && !once && slab_rows > SLAB_GATE)
            slab_sum_kernel<<<dim3(a.c / 8, slab_rows - SLAB_GATE), 1024, 0, st>>>(a.partial, p.units, slab_rows, SLAB_GATE,
                                                                                  a.c, totals, 0, true, g);
    }
    return cudaGetLastError();
}

}  // namespace msc
