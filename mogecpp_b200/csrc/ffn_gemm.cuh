// The matrix products of the gated feed-forward block as one persistent
// tcgen05 kernel, specialised by what its epilogue does (ffn.cu has the
// mathematics).
//
// Output tiles of 128 rows x HT columns of a CTA, or of 256 rows of a CTA
// pair (CG = 2: tcgen05's cta_group::2, each CTA holding its own 128 rows of
// A and half of B's, which halves B's copies and shared-memory reads); the K
// loop runs in steps of 64 elements through a ring of shared-memory stages filled by TMA (128-byte
// swizzle; rows, columns and K past the extents read as zero, so every size
// that is a multiple of 8 is right without a special case).  Operands that
// are contiguous along K are K-major; the transposed products of the
// backward pass read the same row-major tensors MN-major, so that nothing is
// ever transposed in memory.
//
// Warps: 0 TMA producer, 1 MMA issuer (one thread each; of a pair, the first
// CTA's issues for both), 2 TMEM allocation, 4 on epilogue (TMEM lane quarter
// x half of the columns).  Two accumulator slots in TMEM: a tile's epilogue
// runs under the next tile's products.  The backward pass's three
// accumulators (FFN_HBACK) of 128 hidden units fill 384 of the 512 columns,
// so that there dh comes first, into one of two banks, under the epilogue of
// the tile before, and g, u follow once that has read its own.
// 16-bit outputs leave through swizzled shared memory and TMA stores (which
// clip at the extents); fp32 partial sums of a K split are stored directly.
// Every wait is bounded: one that runs out sets MSC_DEV_TIMEOUT, and every
// role unwinds (the epilogue warps keep meeting at their barriers).
//
// Measured at 8192 x 1024 -> 4096 bf16 (single CTAs / pairs): hidden 100 / 92
// us, projection 59 / 52 us; backward dx 108 / 92 us, weights 160 / 136 us (92
// % of the tensor pipe's cycles), hidden gradients 310 (64 hidden units) / 236
// us.  A 128-column tile in place of 256 costs the projection a third (80 us),
// a 64-column one doubles it: the operand reads from shared memory bound it.
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

constexpr int kFfnSmemMax = 227 * 1024;

template <int MODE, int HT, int CG>
struct FfnCfg {
    static constexpr bool GATED = MODE == FFN_HIDDEN || MODE == FFN_HBACK;
    static constexpr bool A_MN = MODE == FFN_DW;
    // HBACK's segments: 0 dh (dy, Wd), 1 g and u (x, Wg and Wu)
    static constexpr bool b_mn(int seg) { return MODE == FFN_DX || MODE == FFN_DW || (MODE == FFN_HBACK && seg == 0); }
    static constexpr int n_cols(int seg) { return MODE == FFN_HIDDEN || (MODE == FFN_HBACK && seg == 1) ? 2 * HT : HT; }
    static constexpr int b_rows(int seg) { return n_cols(seg) / CG; }  // of this CTA
    static constexpr bool BANKS = MODE == FFN_HBACK && HT == 128;
    static constexpr int ACC = MODE == FFN_HIDDEN ? 2 * HT : (MODE == FFN_HBACK ? 3 * HT : HT);
    static constexpr int SLOT = ACC <= 64 ? 64 : (ACC <= 128 ? 128 : 256);
    static constexpr int TMEM_COLS = BANKS ? 512 : 2 * SLOT;
    static constexpr int EPI_WARPS = BANKS ? 16 : 8;
    static constexpr int THREADS = 32 * (4 + EPI_WARPS);
    static constexpr int A_BYTES = 128 * 128;
    static constexpr int B_BYTES = (b_rows(0) > b_rows(1) ? b_rows(0) : b_rows(1)) * 128;
    static constexpr int STAGE = A_BYTES + B_BYTES;
    static constexpr int UNITS = HT / 64;  // 64-column units of an output tile
    static constexpr int UNIT_BYTES = 128 * 128;
    static constexpr int OUT_UNITS = MODE == FFN_HBACK ? 3 * UNITS : (UNITS < 2 ? 1 : 2);
    static constexpr int RED_BYTES = MODE == FFN_HBACK ? 4 * 2 * HT * 4 : 0;
    static constexpr int FIXED = 1024 + OUT_UNITS * UNIT_BYTES + RED_BYTES + 256;
    static constexpr int FIT = (kFfnSmemMax - FIXED) / STAGE;
    static constexpr int STAGES = FIT > 8 ? 8 : FIT;
    static constexpr int SMEM = FIXED + STAGES * STAGE;
    static_assert(ACC <= (BANKS ? 384 : 256) && STAGES >= 3, "tile fits");
    static_assert(CG == 1 || HT >= 128, "a pair's MN-major half of B is whole 64-column groups");
    static_assert(MODE != FFN_HBACK || HT == 64 || CG == 2, "128 hidden units at a time by pairs alone");
    // TMEM column of a segment's accumulators in the it-th tile
    static __device__ __forceinline__ int column(int it, int seg) {
        if (BANKS) return seg == 0 ? 256 + (it & 1) * 128 : 0;
        return (it & 1) * SLOT + (MODE == FFN_HBACK && seg == 0 ? 2 * HT : 0);
    }
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
    t.mt = g * GM + r % gm;  // of 128 rows, or of 256 of a pair
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

template <int MODE, int HT, int CG>
__device__ void ffn_producer(const FfnGemmArgs& a, const FfnSmem& S, int rank) {
    using C = FfnCfg<MODE, HT, CG>;
    const int first = blockIdx.x / CG, step = gridDim.x / CG;
    int i = 0;
    bool ok = true;
    for (int tile = first; tile < a.tiles * a.splits && ok; tile += step) {
        const FfnTile t = ffn_tile(a, tile);
        const int m0 = (t.mt * CG + rank) * 128, n0 = t.nt * HT;
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
            const int b_rows = seg ? C::b_rows(1) : C::b_rows(0);
            // both CTAs' bytes complete on the first CTA's barrier
            uint32_t bar = 0;
            if constexpr (CG == 2) bar = map_rank(smem_u32(&S.full[s]), 0);
            if (rank == 0) mbar_arrive_expect_tx(&S.full[s], CG * (C::A_BYTES + b_rows * 128));
            auto load = [&](uint32_t dst, const CUtensorMap* map, int x, int y) {
                if constexpr (CG == 2)
                    tma_load_2d_pair(dst, map, x, y, bar);
                else
                    tma_load_2d(dst, map, x, y, &S.full[s]);
            };
            if constexpr (C::A_MN) {
                load(sa, &a.ma[t.prob], m0, k);
                load(sa + 8192, &a.ma[t.prob], m0 + 64, k);
            } else {
                load(sa, &a.ma[seg], k, m0);
            }
            if ((MODE == FFN_HIDDEN) || (MODE == FFN_HBACK && seg)) {
                // gate rows, then up rows: of a pair, one each
                if constexpr (CG == 2) {
                    load(sb, &a.mb[rank], k, n0);
                } else {
                    load(sb, &a.mb[0], k, n0);
                    load(sb + HT * 128, &a.mb[1], k, n0);
                }
            } else if constexpr (MODE == FFN_PROJ) {
                load(sb, &a.mb[0], k, n0 + rank * C::b_rows(0));
            } else {
                const CUtensorMap* m = &a.mb[MODE == FFN_HBACK ? 2 : (MODE == FFN_DX ? seg : t.prob)];
#pragma unroll
                for (int j = 0; j < C::b_rows(0) / 64; ++j) load(sb + j * 8192, m, n0 + rank * C::b_rows(0) + 64 * j, k);
            }
        }
    }
    if constexpr (CG == 2) {
        // the other CTA's products have read this one's last stages, and their
        // arrivals have landed here, before this shared memory can go away
        for (int e = i > C::STAGES ? i - C::STAGES : 0; ok && e < i; ++e)
            ok = wait_or_abort(&S.empty[e % C::STAGES], static_cast<uint32_t>(e / C::STAGES) & 1, S.abort, a.status);
    }
    if (!ok) {
        // aborted: copies in flight land within microseconds; wait 100 us
        // before the CTA's shared memory can go away
        const uint64_t t_end = global_timer_ns() + 100000ull;
        while (global_timer_ns() < t_end) __nanosleep(1000);
    }
}

template <int MODE, int HT, int CG>
__device__ void ffn_issuer(const FfnGemmArgs& a, const FfnSmem& S, uint32_t tmem) {
    using C = FfnCfg<MODE, HT, CG>;
    const int first = blockIdx.x / CG, step = gridDim.x / CG;
    const uint32_t fmt = a.bf16 ? 1u : 0u;
    const uint32_t idesc0 =
        idesc_f16(128 * CG, C::n_cols(0), fmt) | (C::A_MN ? kIdescAMn : 0u) | (C::b_mn(0) ? kIdescBMn : 0u);
    const uint32_t idesc1 =
        idesc_f16(128 * CG, C::n_cols(1), fmt) | (C::A_MN ? kIdescAMn : 0u) | (C::b_mn(1) ? kIdescBMn : 0u);
    auto commit = [&](uint64_t* bar) {
        if constexpr (CG == 2)
            umma_commit_pair(bar);
        else
            umma_commit(bar);
    };
    int i = 0, it = 0;
    for (int tile = first; tile < a.tiles * a.splits; tile += step, ++it) {
        const FfnTile t = ffn_tile(a, tile);
        const int slot = it & 1;
        auto acc_free = [&](int s, int use) {
            const bool ok = wait_or_abort(&S.acc_empty[s], static_cast<uint32_t>(use) & 1, S.abort, a.status);
            tc_fence_after();
            return ok;
        };
        if (!C::BANKS && it >= 2 && !acc_free(slot, (it >> 1) - 1)) return;
        for (int kk = t.k0; kk < t.k1; ++kk, ++i) {
            const int seg = kk >= a.ksteps[0];
            // g and u share their columns with the tile before
            if (C::BANKS && kk == a.ksteps[0] && it >= 1 && !acc_free(0, it - 1)) return;
            const int s = i % C::STAGES;
            if (!wait_or_abort(&S.full[s], static_cast<uint32_t>(i / C::STAGES) & 1, S.abort, a.status)) return;
            tc_fence_after();
            const uint32_t sa = smem_u32(S.stages + s * C::STAGE);
            const uint32_t sb = sa + C::A_BYTES;
            const uint32_t d = tmem + static_cast<uint32_t>(C::column(it, seg));
            const bool fresh = kk == t.k0 || (MODE == FFN_HBACK && kk == a.ksteps[0]);
#pragma unroll
            for (int ks = 0; ks < 4; ++ks) {
                const uint64_t da = C::A_MN ? sdesc_mn_sw128(sa + ks * 2048, 8192) : sdesc_k_sw128(sa + ks * 32);
                const bool bmn = seg ? C::b_mn(1) : C::b_mn(0);
                const uint64_t db = bmn ? sdesc_mn_sw128(sb + ks * 2048, 8192) : sdesc_k_sw128(sb + ks * 32);
                const uint32_t acc = (ks > 0 || !fresh) ? 1u : 0u;
                if constexpr (CG == 2)
                    umma_f16_pair(d, da, db, seg ? idesc1 : idesc0, acc);
                else
                    umma_f16(d, da, db, seg ? idesc1 : idesc0, acc);
            }
            commit(&S.empty[s]);
        }
        commit(&S.acc_full[slot]);
    }
}

template <int N>
__device__ __forceinline__ void to_floats(const uint32_t (&r)[N], float (&v)[N]) {
#pragma unroll
    for (int e = 0; e < N; ++e) v[e] = __uint_as_float(r[e]);
}

// N columns of a bias from col on (columns past the end: nothing added).
template <int N>
__device__ __forceinline__ void add_bias(const float* b, int col, int cols, float (&v)[N]) {
    if (!b) return;
#pragma unroll
    for (int e = 0; e < N; e += 4)
        if (col + e < cols) {
            const float4 t = __ldg(reinterpret_cast<const float4*>(b + col + e));
            v[e] += t.x, v[e + 1] += t.y, v[e + 2] += t.z, v[e + 3] += t.w;
        }
}

// N values (a multiple of 8) as 16-bit 16-byte chunks of row m of a swizzled
// unit, from 16-byte chunk `chunk` on.
template <int N>
__device__ __forceinline__ void put_unit(uint8_t* unit, int m, int chunk, const float (&v)[N], int bf16) {
    uint32_t w[N / 2];
    if (bf16) {
#pragma unroll
        for (int e = 0; e < N / 2; ++e) {
            const __nv_bfloat162 t = __floats2bfloat162_rn(v[2 * e], v[2 * e + 1]);
            w[e] = *reinterpret_cast<const uint32_t*>(&t);
        }
    } else {
#pragma unroll
        for (int e = 0; e < N / 2; ++e) {
            const __half2 t = __floats2half2_rn(v[2 * e], v[2 * e + 1]);
            w[e] = *reinterpret_cast<const uint32_t*>(&t);
        }
    }
#pragma unroll
    for (int k = 0; k < N / 8; ++k)
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

template <int MODE, int HT, int CG>
__device__ void ffn_epilogue(const FfnGemmArgs& a, const FfnSmem& S, uint32_t tmem, int rank) {
    using C = FfnCfg<MODE, HT, CG>;
    const int first = blockIdx.x / CG, step = gridDim.x / CG;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int q = warp & 3, half = ((warp - 4) >> 2) & 1, group = (warp - 4) >> 3;
    const int m = q * 32 + lane;
    const uint32_t lane_addr = static_cast<uint32_t>(q * 32) << 16;
    constexpr bool SHARED = C::UNITS == 1 || MODE == FFN_HBACK;  // both halves fill the same unit
    const int bar_id = SHARED ? 1 + group : 1 + half;
    const int bar_threads = SHARED ? 256 : 128;
    const bool issuer = lane == 0 && q == 0 && (!SHARED || half == 0);
    bool ok = true;
    int it = 0;
    for (int tile = first; tile < a.tiles * a.splits; tile += step, ++it) {
        const FfnTile t = ffn_tile(a, tile);
        const int slot = it & 1;
        const int m0 = (t.mt * CG + rank) * 128, n0 = t.nt * HT;
        const int rows = a.rows[t.prob], cols = a.cols[t.prob];
        ok = ok && wait_or_abort(&S.acc_full[slot], static_cast<uint32_t>(it >> 1) & 1, S.abort, a.status);
        ok = __all_sync(0xffffffffu, ok);
        tc_fence_after();
        const uint32_t acc = tmem + lane_addr + static_cast<uint32_t>(C::column(it, 1));
        // the accumulators have been read (the pair's issuer is the first CTA's)
        auto release = [&]() {
            tc_fence_before();
            uint64_t* bar = &S.acc_empty[C::BANKS ? 0 : slot];
            if constexpr (CG == 2) {
                __syncwarp();
                if (lane == 0) mbar_arrive_cluster(map_rank(smem_u32(bar), 0));
            } else {
                warp_arrive(bar);
            }
        };
        if constexpr (MODE == FFN_HBACK) {
            uint8_t* units = S.out + group * 3 * C::UNIT_BYTES;
            if (issuer) bulk_wait_read();
            named_bar(bar_id, bar_threads);
            if (ok) {
#pragma unroll
                for (int cc = 0; cc < 2; ++cc) {
                    const int cu = half * 32 + cc * 16, c0 = group * 64 + cu;  // column of the unit, of the tile
                    uint32_t rg[16], ru[16], rd[16];
                    tmem_ld16(acc + c0, rg);
                    tmem_ld16(acc + HT + c0, ru);
                    tmem_ld16(tmem + lane_addr + static_cast<uint32_t>(C::column(it, 0)) + c0, rd);
                    tmem_wait_ld_regs(rg);
                    tmem_wait_ld_regs(ru);
                    tmem_wait_ld_regs(rd);
                    if (cc == 1) release();
                    float g[16], u[16], d[16];
                    to_floats(rg, g);
                    to_floats(ru, u);
                    to_floats(rd, d);
                    add_bias(a.bias0, n0 + c0, cols, g);
                    add_bias(a.bias1, n0 + c0, cols, u);
                    gate_back_chunk(a.act, g, u, d);
                    put_unit(units, m, cu / 8, g, a.bf16);
                    put_unit(units + C::UNIT_BYTES, m, cu / 8, u, a.bf16);
                    put_unit(units + 2 * C::UNIT_BYTES, m, cu / 8, d, a.bf16);
                    if (a.bias_part) {
                        const bool live = m0 + m < rows;
#pragma unroll
                        for (int e = 0; e < 16; ++e) {
                            g[e] = live ? g[e] : 0.f;
                            u[e] = live ? u[e] : 0.f;
                        }
                        const float sg = column_sums16(g, lane), su = column_sums16(u, lane);
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
                for (int o = 0; o < 3; ++o)
                    if (n0 + group * 64 < cols && m0 < rows)
                        tma_store_2d(&a.mo[o], smem_u32(units + o * C::UNIT_BYTES), n0 + group * 64, m0);
                bulk_commit();
            }
            if (ok && a.bias_part) {
                const int e = static_cast<int>(threadIdx.x) - 128 - group * 256;  // this group's 64 columns of both sums
                if (e < 128) {
                    const int which = e / 64, col = group * 64 + e % 64;
                    if (n0 + col < cols && m0 < rows) {
                        float s = 0.f;
#pragma unroll
                        for (int w = 0; w < 4; ++w) s += S.red[(w * 2 + which) * HT + col];
                        a.bias_part[(static_cast<int64_t>(t.mt * CG + rank) * 2 + which) * cols + n0 + col] = s;
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
                        float v[32];
                        if constexpr (MODE == FFN_HIDDEN) {
                            uint32_t rg[32], ru[32];
                            tmem_ld32(acc + u0 + cc, rg);
                            tmem_ld32(acc + HT + u0 + cc, ru);
                            tmem_wait_ld_regs(rg);
                            tmem_wait_ld_regs(ru);
                            if (last && cc + 32 == NC) release();
                            float u[32];
                            to_floats(rg, v);
                            to_floats(ru, u);
                            add_bias(a.bias0, n0 + u0 + cc, cols, v);
                            add_bias(a.bias1, n0 + u0 + cc, cols, u);
                            gate_chunk(a.act, v, u);
                        } else {
                            uint32_t r[32];
                            tmem_ld32(acc + u0 + cc, r);
                            tmem_wait_ld_regs(r);
                            if (last && cc + 32 == NC) release();
                            to_floats(r, v);
                            if (direct) {
                                if (m0 + m < rows) {
                                    float* p = a.partial + t.split * a.partial_split + a.partial_prob[t.prob] +
                                               static_cast<int64_t>(m0 + m) * cols + n0 + u0 + cc;
#pragma unroll
                                    for (int e = 0; e < 32; e += 4)
                                        if (n0 + u0 + cc + e < cols)
                                            *reinterpret_cast<float4*>(p + e) = make_float4(v[e], v[e + 1], v[e + 2], v[e + 3]);
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
                        if (col < cols && m0 < rows) tma_store_2d(&a.mo[t.prob], smem_u32(unit), col, m0);
                        bulk_commit();
                    }
                }
            }
        }
    }
    if (issuer) bulk_wait();
}

template <int MODE, int HT, int CG>
__global__ void __launch_bounds__(FfnCfg<MODE, HT, CG>::THREADS, 1) ffn_gemm_kernel(const __grid_constant__ FfnGemmArgs a) {
    using C = FfnCfg<MODE, HT, CG>;
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

    // the next kernel of the pass may set itself up on SMs that fall idle
    launch_dependents();
    const int warp = threadIdx.x >> 5;
    if (threadIdx.x == 0) {
        for (int s = 0; s < C::STAGES; ++s) {
            mbar_init(&S.full[s], 1);
            mbar_init(&S.empty[s], 1);
        }
        for (int s = 0; s < 2; ++s) {
            mbar_init(&S.acc_full[s], 1);
            mbar_init(&S.acc_empty[s], CG * C::EPI_WARPS);
        }
        mbar_init(S.drained, 1);
        *S.abort = 0;
        fence_mbar_init();
    }
    const int rank = CG == 2 ? static_cast<int>(cluster_rank()) : 0;
    if (warp == 2) {
        if constexpr (CG == 2) {
            tmem_alloc_pair(S.tmem, C::TMEM_COLS);
        } else {
            tmem_alloc(S.tmem, C::TMEM_COLS);
            tmem_relinquish();
        }
    }
    __syncwarp();
    tc_fence_before();
    if constexpr (CG == 2)
        cluster_sync();  // the other CTA's barriers are initialised
    else
        __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *S.tmem;
    // nothing of the kernels before is read, and nothing they read is
    // written, until they are done
    wait_dependency();

    if (warp == 0) {
        if ((threadIdx.x & 31) == 0) ffn_producer<MODE, HT, CG>(a, S, rank);
        __syncwarp();
    } else if (warp == 1) {
        if ((threadIdx.x & 31) == 0 && rank == 0) ffn_issuer<MODE, HT, CG>(a, S, tmem);
        __syncwarp();
    } else if (warp >= 4) {
        ffn_epilogue<MODE, HT, CG>(a, S, tmem, rank);
    }
    tc_fence_before();
    __syncthreads();
    if (*reinterpret_cast<volatile int*>(S.abort) && rank == 0) {
        // MMAs sent before the abort may still write TMEM: a commit tracks
        // them all; wait (bounded) before the columns go
        if (threadIdx.x == 32) {
            if constexpr (CG == 2)
                umma_commit_pair(S.drained);
            else
                umma_commit(S.drained);
            (void)mbar_wait(S.drained, 0);
        }
        __syncthreads();
    }
    // neither CTA leaves while the other may still reach its shared memory
    if constexpr (CG == 2) {
        __syncwarp();
        cluster_sync();
    }
    if (warp == 2) {
        tc_fence_after();
        if constexpr (CG == 2)
            tmem_dealloc_pair(tmem, C::TMEM_COLS);
        else
            tmem_dealloc(tmem, C::TMEM_COLS);
    }
}

}  // namespace msc
