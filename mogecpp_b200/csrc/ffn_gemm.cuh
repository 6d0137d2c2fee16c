// The matrix products of the gated feed-forward block as one persistent
// tcgen05 kernel, specialised by what its epilogue does (ffn.cu has the
// mathematics).
//
// Output tiles of 128 rows x HT columns; the K loop runs in steps of 64
// elements through a ring of shared-memory stages filled by TMA (128-byte
// swizzle; rows, columns and K past the extents read as zero, so every size
// that is a multiple of 8 is right without a special case).  Operands that
// are contiguous along K are K-major; the transposed products of the
// backward pass read the same row-major tensors MN-major, so that nothing is
// ever transposed in memory.
//
// Warps: 0 TMA producer, 1 MMA issuer (one thread each), 2 TMEM allocation,
// 4-11 epilogue (TMEM lane quarter x half of the columns).  Two accumulator
// slots in TMEM: a tile's epilogue runs under the next tile's products.
// 16-bit outputs leave through swizzled shared memory and TMA stores (which
// clip at the extents); fp32 partial sums of a K split are stored directly.
// Every wait is bounded: one that runs out sets MSC_DEV_TIMEOUT, and every
// role unwinds (the epilogue warps keep meeting at their barriers).
#pragma once

#include "common.cuh"
#include "conv_common.cuh"
#include "ffn.h"
#include "ffn_act.cuh"
#include "tma.cuh"

namespace msc {

enum FfnMode : int {
    FFN_HIDDEN = 0,  // h = act(x Wg^T + bg) * (x Wu^T + bu)
    FFN_PROJ = 1,    // y = h Wd^T + bd
    FFN_HBACK = 2,   // g, u again, dh = dy Wd -> dg, du, h (and the bias sums)
    FFN_DX = 3,      // dx = dg Wg + du Wu
    FFN_DW = 4,      // dWg = dg^T x, dWu = du^T x, dWd = dy^T h
};

struct alignas(64) FfnGemmArgs {
    CUtensorMap ma[3], mb[3], mo[3];
    int m_tiles[3], n_tiles[3];
    int rows[3], cols[3];  // output extents of each problem
    int nprob;
    int tiles;          // tiles of one split, all problems
    int ksteps[2];      // K steps of each segment
    int splits, ksplit;  // K split: ksplit steps each
    float* partial;     // fp32 partial sums [split][problem][rows][cols], or NULL
    int64_t partial_split, partial_prob[3];
    const float* bias0;
    const float* bias1;
    float* bias_part;   // HBACK: [m tile][2][hidden] column sums of dg, du, or NULL
    int act, bf16;
    uint32_t* status;
};

constexpr int kFfnThreads = 384;
constexpr int kFfnEpiWarps = 8;
constexpr int kFfnSmemMax = 227 * 1024;

template <int MODE, int HT>
struct FfnCfg {
    static constexpr bool GATED = MODE == FFN_HIDDEN || MODE == FFN_HBACK;
    static constexpr bool A_MN = MODE == FFN_DW;
    static constexpr bool b_mn(int seg) { return MODE == FFN_DX || MODE == FFN_DW || (MODE == FFN_HBACK && seg == 1); }
    static constexpr int b_rows(int seg) { return GATED && seg == 0 ? 2 * HT : HT; }
    static constexpr int ACC = MODE == FFN_HIDDEN ? 2 * HT : (MODE == FFN_HBACK ? 3 * HT : HT);
    static constexpr int SLOT = ACC <= 64 ? 64 : (ACC <= 128 ? 128 : 256);
    static constexpr int TMEM_COLS = 2 * SLOT;
    static constexpr int A_BYTES = 128 * 128;
    static constexpr int B_BYTES = b_rows(0) * 128;
    static constexpr int STAGE = A_BYTES + B_BYTES;
    static constexpr int UNITS = HT / 64;  // 64-column units of an output tile
    static constexpr int UNIT_BYTES = 128 * 128;
    static constexpr int OUT_UNITS = MODE == FFN_HBACK ? 3 : (UNITS < 2 ? 1 : 2);
    static constexpr int RED_BYTES = MODE == FFN_HBACK ? 4 * 2 * HT * 4 : 0;
    static constexpr int FIXED = 1024 + OUT_UNITS * UNIT_BYTES + RED_BYTES + 256;
    static constexpr int FIT = (kFfnSmemMax - FIXED) / STAGE;
    static constexpr int STAGES = FIT > 8 ? 8 : FIT;
    static constexpr int SMEM = FIXED + STAGES * STAGE;
    static_assert(ACC <= 256 && STAGES >= 3, "tile fits");
    static_assert(MODE != FFN_HBACK || HT == 64, "three accumulators side by side");
};

struct FfnTile {
    int prob, split, mt, nt, k0, k1;
};

// Tiles run in groups of 16 row blocks, column blocks outer, so that the
// CTAs in flight share both operands in L2; splits outermost.
__device__ __forceinline__ FfnTile ffn_tile(const FfnGemmArgs& a, int tile) {
    FfnTile t;
    t.split = tile / a.tiles;
    int r = tile - t.split * a.tiles;
    t.prob = 0;
    while (t.prob + 1 < a.nprob && r >= a.m_tiles[t.prob] * a.n_tiles[t.prob]) {
        r -= a.m_tiles[t.prob] * a.n_tiles[t.prob];
        ++t.prob;
    }
    constexpr int GM = 16;
    const int width = GM * a.n_tiles[t.prob];
    const int g = r / width;
    const int gm = min(a.m_tiles[t.prob] - g * GM, GM);
    r -= g * width;
    t.mt = g * GM + r % gm;
    t.nt = r / gm;
    t.k0 = t.split * a.ksplit;
    t.k1 = min(t.k0 + a.ksplit, a.ksteps[0] + a.ksteps[1]);
    return t;
}

struct FfnSmem {
    uint8_t* stages;
    uint8_t* out;
    float* red;       // HBACK: [4 lane quarters][2][HT]
    uint64_t* full;
    uint64_t* empty;
    uint64_t* acc_full;
    uint64_t* acc_empty;
    uint64_t* drained;
    uint32_t* tmem;
    int* abort;
};

template <int MODE, int HT>
__device__ void ffn_producer(const FfnGemmArgs& a, const FfnSmem& S) {
    using C = FfnCfg<MODE, HT>;
    int i = 0;
    bool ok = true;
    for (int tile = blockIdx.x; tile < a.tiles * a.splits && ok; tile += gridDim.x) {
        const FfnTile t = ffn_tile(a, tile);
        const int m0 = t.mt * 128, n0 = t.nt * HT;
        for (int kk = t.k0; kk < t.k1; ++kk, ++i) {
            const int seg = kk >= a.ksteps[0];
            const int k = (kk - (seg ? a.ksteps[0] : 0)) * 64;
            const int s = i % C::STAGES;
            if (i >= C::STAGES &&
                !wait_or_abort(&S.empty[s], static_cast<uint32_t>(i / C::STAGES - 1) & 1, S.abort, a.status)) {
                ok = false;
                break;
            }
            const uint32_t sa = smem_u32(S.stages + s * C::STAGE);
            const uint32_t sb = sa + C::A_BYTES;
            uint64_t* bar = &S.full[s];
            mbar_arrive_expect_tx(bar, C::A_BYTES + (seg ? C::b_rows(1) : C::b_rows(0)) * 128);
            if constexpr (C::A_MN) {
                const CUtensorMap* m = &a.ma[t.prob];
                tma_load_2d(sa, m, m0, k, bar);
                tma_load_2d(sa + 8192, m, m0 + 64, k, bar);
            } else {
                tma_load_2d(sa, &a.ma[seg], k, m0, bar);
            }
            if constexpr (MODE == FFN_HIDDEN) {
                tma_load_2d(sb, &a.mb[0], k, n0, bar);
                tma_load_2d(sb + HT * 128, &a.mb[1], k, n0, bar);
            } else if constexpr (MODE == FFN_PROJ) {
                tma_load_2d(sb, &a.mb[0], k, n0, bar);
            } else if constexpr (MODE == FFN_HBACK) {
                if (!seg) {
                    tma_load_2d(sb, &a.mb[0], k, n0, bar);
                    tma_load_2d(sb + HT * 128, &a.mb[1], k, n0, bar);
                } else {
                    tma_load_2d(sb, &a.mb[2], n0, k, bar);
                }
            } else {
                const CUtensorMap* m = &a.mb[MODE == FFN_DX ? seg : t.prob];
#pragma unroll
                for (int j = 0; j < HT / 64; ++j) tma_load_2d(sb + j * 8192, m, n0 + 64 * j, k, bar);
            }
        }
    }
    if (!ok) {
        // aborted: copies in flight land within microseconds; wait 100 us
        // before the CTA's shared memory can go away
        const uint64_t t_end = global_timer_ns() + 100000ull;
        while (global_timer_ns() < t_end) __nanosleep(1000);
    }
}

template <int MODE, int HT>
__device__ void ffn_issuer(const FfnGemmArgs& a, const FfnSmem& S, uint32_t tmem) {
    using C = FfnCfg<MODE, HT>;
    const uint32_t fmt = a.bf16 ? 1u : 0u;
    const uint32_t idesc0 = idesc_f16(128, C::b_rows(0), fmt) | (C::A_MN ? kIdescAMn : 0u) | (C::b_mn(0) ? kIdescBMn : 0u);
    const uint32_t idesc1 = idesc_f16(128, C::b_rows(1), fmt) | (C::A_MN ? kIdescAMn : 0u) | (C::b_mn(1) ? kIdescBMn : 0u);
    int i = 0, it = 0;
    for (int tile = blockIdx.x; tile < a.tiles * a.splits; tile += gridDim.x, ++it) {
        const FfnTile t = ffn_tile(a, tile);
        const int slot = it & 1;
        if (it >= 2 && !wait_or_abort(&S.acc_empty[slot], static_cast<uint32_t>((it >> 1) - 1) & 1, S.abort, a.status))
            return;
        tc_fence_after();
        for (int kk = t.k0; kk < t.k1; ++kk, ++i) {
            const int seg = kk >= a.ksteps[0];
            const int s = i % C::STAGES;
            if (!wait_or_abort(&S.full[s], static_cast<uint32_t>(i / C::STAGES) & 1, S.abort, a.status)) return;
            tc_fence_after();
            const uint32_t sa = smem_u32(S.stages + s * C::STAGE);
            const uint32_t sb = sa + C::A_BYTES;
            const uint32_t d = tmem + static_cast<uint32_t>(slot * C::SLOT + (MODE == FFN_HBACK && seg ? 2 * HT : 0));
            const bool fresh = kk == t.k0 || (MODE == FFN_HBACK && kk == a.ksteps[0]);
#pragma unroll
            for (int ks = 0; ks < 4; ++ks) {
                const uint64_t da = C::A_MN ? sdesc_mn_sw128(sa + ks * 2048, 8192) : sdesc_k_sw128(sa + ks * 32);
                const bool bmn = seg ? C::b_mn(1) : C::b_mn(0);
                const uint64_t db = bmn ? sdesc_mn_sw128(sb + ks * 2048, 8192) : sdesc_k_sw128(sb + ks * 32);
                umma_f16(d, da, db, seg ? idesc1 : idesc0, (ks > 0 || !fresh) ? 1u : 0u);
            }
            umma_commit(&S.empty[s]);
        }
        umma_commit(&S.acc_full[slot]);
    }
}

// N accumulator registers as pairs.
template <int N>
__device__ __forceinline__ void to_pairs(const uint32_t (&r)[N], uint64_t (&v)[N / 2]) {
#pragma unroll
    for (int e = 0; e < N / 2; ++e) v[e] = pack2(__uint_as_float(r[2 * e]), __uint_as_float(r[2 * e + 1]));
}

// N pairs of a bias from col on (columns past the end: nothing added).
template <int N>
__device__ __forceinline__ void add_bias(const float* b, int col, int cols, uint64_t (&v)[N]) {
    if (!b) return;
#pragma unroll
    for (int e = 0; e < N; e += 2)
        if (col + 2 * e < cols) {
            const float4 t = __ldg(reinterpret_cast<const float4*>(b + col + 2 * e));
            v[e] = add2(v[e], pack2(t.x, t.y));
            v[e + 1] = add2(v[e + 1], pack2(t.z, t.w));
        }
}

// N pairs (a multiple of 4) as 16-bit 16-byte chunks of row m of a swizzled
// unit, from 16-byte chunk `chunk` on.
template <int N>
__device__ __forceinline__ void put_unit(uint8_t* unit, int m, int chunk, const uint64_t (&v)[N], int bf16) {
    uint32_t w[N];
    if (bf16) {
#pragma unroll
        for (int e = 0; e < N; ++e) {
            float a, b;
            unpack2(v[e], a, b);
            const __nv_bfloat162 t = __floats2bfloat162_rn(a, b);
            w[e] = *reinterpret_cast<const uint32_t*>(&t);
        }
    } else {
#pragma unroll
        for (int e = 0; e < N; ++e) {
            float a, b;
            unpack2(v[e], a, b);
            const __half2 t = __floats2half2_rn(a, b);
            w[e] = *reinterpret_cast<const uint32_t*>(&t);
        }
    }
#pragma unroll
    for (int k = 0; k < N / 4; ++k)
        *reinterpret_cast<uint4*>(unit + sw128_offset(m, chunk + k)) = make_uint4(w[4 * k], w[4 * k + 1], w[4 * k + 2], w[4 * k + 3]);
}

__device__ __forceinline__ void named_bar(int id, int threads) {
    asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(threads) : "memory");
}

// Sums of 16 columns over the warp's 32 rows: each exchange halves the
// columns a lane holds; afterwards lane l holds the sum of column
// bits 4..1 of l (most significant first), both lanes of a pair the same.
__device__ __forceinline__ float column_sums16(float (&v)[16], int lane) {
#pragma unroll
    for (int o = 16; o >= 2; o >>= 1) {
        const int half = o / 2;  // columns kept
        const bool up = lane & o;
#pragma unroll
        for (int e = 0; e < 8; ++e)
            if (e < half) {
                const float send = up ? v[e] : v[e + half];
                const float keep = up ? v[e + half] : v[e];
                v[e] = keep + __shfl_xor_sync(0xffffffffu, send, o);
            }
    }
    return v[0] + __shfl_xor_sync(0xffffffffu, v[0], 1);
}

template <int MODE, int HT>
__device__ void ffn_epilogue(const FfnGemmArgs& a, const FfnSmem& S, uint32_t tmem) {
    using C = FfnCfg<MODE, HT>;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int q = warp & 3, half = (warp - 4) >> 2;
    const int m = q * 32 + lane;
    const uint32_t lane_addr = static_cast<uint32_t>(q * 32) << 16;
    constexpr bool SHARED = C::UNITS == 1;  // both halves fill the same unit
    const int bar_id = SHARED ? 1 : 1 + half;
    const int bar_threads = SHARED ? 256 : 128;
    const bool issuer = lane == 0 && warp == (SHARED ? 4 : 4 + 4 * half);
    bool ok = true;
    int it = 0;
    for (int tile = blockIdx.x; tile < a.tiles * a.splits; tile += gridDim.x, ++it) {
        const FfnTile t = ffn_tile(a, tile);
        const int slot = it & 1;
        const int m0 = t.mt * 128, n0 = t.nt * HT;
        const int rows = a.rows[t.prob], cols = a.cols[t.prob];
        ok = ok && wait_or_abort(&S.acc_full[slot], static_cast<uint32_t>(it >> 1) & 1, S.abort, a.status);
        ok = __all_sync(0xffffffffu, ok);
        tc_fence_after();
        const uint32_t acc = tmem + lane_addr + static_cast<uint32_t>(slot * C::SLOT);
        auto release = [&]() {
            tc_fence_before();
            warp_arrive(&S.acc_empty[slot]);
        };
        if constexpr (MODE == FFN_HBACK) {
            if (issuer) bulk_wait_read();
            named_bar(bar_id, bar_threads);
            if (ok) {
#pragma unroll
                for (int cc = 0; cc < 2; ++cc) {
                    const int c0 = half * 32 + cc * 16;
                    uint32_t rg[16], ru[16], rd[16];
                    tmem_ld16(acc + c0, rg);
                    tmem_ld16(acc + HT + c0, ru);
                    tmem_ld16(acc + 2 * HT + c0, rd);
                    tmem_wait_ld_regs(rg);
                    tmem_wait_ld_regs(ru);
                    tmem_wait_ld_regs(rd);
                    if (cc == 1) release();
                    uint64_t g[8], u[8], d[8];
                    to_pairs(rg, g);
                    to_pairs(ru, u);
                    to_pairs(rd, d);
                    add_bias(a.bias0, n0 + c0, cols, g);
                    add_bias(a.bias1, n0 + c0, cols, u);
                    gate_back_chunk(a.act, g, u, d);
                    put_unit(S.out, m, c0 / 8, g, a.bf16);
                    put_unit(S.out + C::UNIT_BYTES, m, c0 / 8, u, a.bf16);
                    put_unit(S.out + 2 * C::UNIT_BYTES, m, c0 / 8, d, a.bf16);
                    if (a.bias_part) {
                        const bool live = m0 + m < rows;
                        float fg[16], fu[16];
#pragma unroll
                        for (int e = 0; e < 8; ++e) {
                            unpack2(live ? g[e] : 0ull, fg[2 * e], fg[2 * e + 1]);
                            unpack2(live ? u[e] : 0ull, fu[2 * e], fu[2 * e + 1]);
                        }
                        const float sg = column_sums16(fg, lane), su = column_sums16(fu, lane);
                        if (!(lane & 1)) {
                            S.red[(q * 2 + 0) * HT + c0 + (lane >> 1 & 1) + (lane >> 2 & 1) * 2 + (lane >> 3 & 1) * 4 +
                                  (lane >> 4) * 8] = sg;
                            S.red[(q * 2 + 1) * HT + c0 + (lane >> 1 & 1) + (lane >> 2 & 1) * 2 + (lane >> 3 & 1) * 4 +
                                  (lane >> 4) * 8] = su;
                        }
                    }
                }
                fence_proxy_async();
            }
            named_bar(bar_id, bar_threads);
            if (ok && issuer) {
#pragma unroll
                for (int o = 0; o < 3; ++o) tma_store_2d(&a.mo[o], smem_u32(S.out + o * C::UNIT_BYTES), n0, m0);
                bulk_commit();
            }
            if (ok && a.bias_part) {
                const int e = static_cast<int>(threadIdx.x) - 128;  // 2 * HT columns
                if (e < 2 * HT) {
                    const int which = e / HT, col = e % HT;
                    if (n0 + col < cols) {
                        float s = 0.f;
#pragma unroll
                        for (int w = 0; w < 4; ++w) s += S.red[(w * 2 + which) * HT + col];
                        a.bias_part[(static_cast<int64_t>(t.mt) * 2 + which) * cols + n0 + col] = s;
                    }
                }
            }
        } else {
            // columns of this warp: units half, half + 2, ... or half of the only unit
            constexpr int NC = SHARED ? 32 : 64;
            constexpr int STEP = SHARED ? 64 : 128;
            const bool direct = (MODE != FFN_HIDDEN) && a.partial;
#pragma unroll 1
            for (int u0 = half * NC; u0 < HT; u0 += STEP) {
                const bool last = u0 + STEP >= HT;
                uint8_t* unit = S.out + (SHARED ? 0 : half) * C::UNIT_BYTES;
                if (!direct) {
                    if (issuer) bulk_wait_read();
                    named_bar(bar_id, bar_threads);
                }
                if (ok) {
#pragma unroll
                    for (int cc = 0; cc < NC; cc += 32) {
                        uint64_t v[16];
                        if constexpr (MODE == FFN_HIDDEN) {
                            uint32_t rg[32], ru[32];
                            tmem_ld32(acc + u0 + cc, rg);
                            tmem_ld32(acc + HT + u0 + cc, ru);
                            tmem_wait_ld_regs(rg);
                            tmem_wait_ld_regs(ru);
                            if (last && cc + 32 == NC) release();
                            uint64_t u[16];
                            to_pairs(rg, v);
                            to_pairs(ru, u);
                            add_bias(a.bias0, n0 + u0 + cc, cols, v);
                            add_bias(a.bias1, n0 + u0 + cc, cols, u);
                            gate_chunk(a.act, v, u);
                        } else {
                            uint32_t r[32];
                            tmem_ld32(acc + u0 + cc, r);
                            tmem_wait_ld_regs(r);
                            if (last && cc + 32 == NC) release();
                            to_pairs(r, v);
                            if (direct) {
                                if (m0 + m < rows) {
                                    float* p = a.partial + t.split * a.partial_split + a.partial_prob[t.prob] +
                                               static_cast<int64_t>(m0 + m) * cols + n0 + u0 + cc;
#pragma unroll
                                    for (int e = 0; e < 32; e += 4)
                                        if (n0 + u0 + cc + e < cols)
                                            *reinterpret_cast<ulonglong2*>(p + e) = make_ulonglong2(v[e / 2], v[e / 2 + 1]);
                                }
                                continue;
                            }
                            if constexpr (MODE == FFN_PROJ) add_bias(a.bias0, n0 + u0 + cc, cols, v);
                        }
                        put_unit(unit, m, ((SHARED ? u0 : 0) + cc) / 8, v, a.bf16);
                    }
                    fence_proxy_async();
                }
                if (!direct) {
                    named_bar(bar_id, bar_threads);
                    if (ok && issuer) {
                        const int col = n0 + (SHARED ? 0 : u0);
                        if (col < cols) tma_store_2d(&a.mo[t.prob], smem_u32(unit), col, m0);
                        bulk_commit();
                    }
                }
            }
        }
    }
    if (issuer) bulk_wait();
}

template <int MODE, int HT>
__global__ void __launch_bounds__(kFfnThreads, 1) ffn_gemm_kernel(const __grid_constant__ FfnGemmArgs a) {
    using C = FfnCfg<MODE, HT>;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* p = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    FfnSmem S;
    S.stages = p;
    p += C::STAGES * C::STAGE;
    S.out = p;
    p += C::OUT_UNITS * C::UNIT_BYTES;
    S.red = reinterpret_cast<float*>(p);
    p += C::RED_BYTES;
    S.full = reinterpret_cast<uint64_t*>(p);
    S.empty = S.full + C::STAGES;
    S.acc_full = S.empty + C::STAGES;
    S.acc_empty = S.acc_full + 2;
    S.drained = S.acc_empty + 2;
    S.tmem = reinterpret_cast<uint32_t*>(S.drained + 1);
    S.abort = reinterpret_cast<int*>(S.tmem + 1);

    const int warp = threadIdx.x >> 5;
    if (threadIdx.x == 0) {
        for (int s = 0; s < C::STAGES; ++s) {
            mbar_init(&S.full[s], 1);
            mbar_init(&S.empty[s], 1);
        }
        for (int s = 0; s < 2; ++s) {
            mbar_init(&S.acc_full[s], 1);
            mbar_init(&S.acc_empty[s], kFfnEpiWarps);
        }
        mbar_init(S.drained, 1);
        *S.abort = 0;
        fence_mbar_init();
    }
    if (warp == 2) {
        tmem_alloc(S.tmem, C::TMEM_COLS);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *S.tmem;

    if (warp == 0) {
        if ((threadIdx.x & 31) == 0) ffn_producer<MODE, HT>(a, S);
        __syncwarp();
    } else if (warp == 1) {
        if ((threadIdx.x & 31) == 0) ffn_issuer<MODE, HT>(a, S, tmem);
        __syncwarp();
    } else if (warp >= 4) {
        ffn_epilogue<MODE, HT>(a, S, tmem);
    }
    tc_fence_before();
    __syncthreads();
    if (*reinterpret_cast<volatile int*>(S.abort)) {
        // MMAs sent before the abort may still write TMEM: a commit tracks
        // them all; wait (bounded) before the columns go
        if (threadIdx.x == 32) {
            umma_commit(S.drained);
            (void)mbar_wait(S.drained, 0);
        }
        __syncthreads();
    }
    if (warp == 2) {
        tc_fence_after();
        tmem_dealloc(tmem, C::TMEM_COLS);
    }
}

}  // namespace msc
