// Gated feed-forward block of many rows and few channels (c <= 128) in one
// kernel: the hidden values never leave the SM.
//
// With c channels a hidden value costs 6 c flops but, written out and read
// back, 4 bytes of HBM traffic: at c = 128 that traffic (and the store path)
// takes longer than the products.  Here a CTA keeps two 128-row subtiles of x
// in shared memory and walks the hidden units in chunks of 64:
//   D = x [Wg chunk | Wu chunk]^T   (TMEM, 128 rows x 128 columns, K = c)
//   h = act(D_g + bg) * (D_u + bu)  (epilogue warps -> shared memory, 16 bits)
//   Y += h Wd[:, chunk]^T           (TMEM, 128 rows x c columns, K = 64)
// The weights stream through shared memory once per 256 rows (they stay in
// L2).  The epilogue is the long pole (a gated activation an element: issue
// slots 57 % busy and the special-function unit 48 % at 128 channels, 60 and 30 %
// at 64, the rest is its hand-overs), so that its warps take D
// into registers and release it before they are done computing, and the next
// chunk's D is there when they come back.  The two products have an issuing
// warp each, so that neither waits for the other's operands.
//
// Up to 64 channels three groups of 8 warps take the (chunk, subtile) items in
// turn, and a warp of its own stores; at 128, where the products take longer
// and the registers of a third group would cost more than it brings (177 us
// against 170 at 402,131 x 128 -> 512, bf16), each subtile has a group.
//
// Y's chain in its accumulator is the whole hidden size, at most 65,536: not
// cut at 32,768 as the products of ffn.cu are (it would have to leave the SM):
// what the longest drifts by for terms of one sign, 4.4e-4 there, stays below
// fp16's own rounding.
//
// TMEM: Y 2 x 128 columns, D 2 x 128 columns.  Warps: 0 TMA producer, 1 and 2
// MMA issuers (D, Y), 3 TMEM allocation (and stores), 4 on epilogue (8 per
// group: lane quarter x half of the chunk).  Every wait is bounded, as in
// ffn_gemm.cuh.
//
// Measured: 402,131 x 128 -> 512 bf16 172 us (0.92 PFLOP/s; two kernels with
// h in memory: 291 us); without the activations the products and copies alone
// take 120 us, bound by shared-memory operand reads of 128-column products
// and the weights' way from L2 (24 KB per item and SM).  101,117 x 64 -> 256
// fp16 38 us (two kernels: 67 us).
#include "ffn_fused.h"

#include "common.cuh"
#include "conv.h"
#include "conv_common.cuh"
#include "ffn_act.cuh"
#include "ffn_gemm.cuh"
#include "tma.cuh"

#include <algorithm>
#include <mutex>

namespace msc {
namespace {

constexpr int kGroupWarps = 8;

// KC: 64-channel blocks of a row (c padded with zeros by the copies).
template <int KC>
struct FusedCfg {
    static constexpr int GROUPS = KC == 1 ? 3 : 2;  // epilogue groups
    static constexpr int THREADS = 32 * (4 + GROUPS * kGroupWarps);
    static constexpr int XR = KC == 1 ? 4 : 2;   // x subtile slots
    static constexpr int W1R = KC == 1 ? 4 : 3;  // gate and up weight stages
    static constexpr int W2R = KC == 1 ? 4 : 2;  // down weight stages
    static constexpr int X_BYTES = KC * 128 * 128;
    static constexpr int W1_BYTES = KC * 128 * 128;  // per 64-channel block: 64 gate rows, then 64 up rows
    static constexpr int W2_BYTES = KC * 64 * 128;   // c rows of 64 hidden units
    static constexpr int H_BYTES = 128 * 128;
    static constexpr int CP = KC * 64;  // padded channels
    // (a subtile's h unit also takes its y out, 64 columns at a time)
    static constexpr int SMEM = 1024 + XR * X_BYTES + W1R * W1_BYTES + W2R * W2_BYTES + 2 * H_BYTES + 512;
    static_assert(SMEM <= kFfnSmemMax, "shared memory budget");
};

struct alignas(64) FusedArgs {
    CUtensorMap mx, mg, mu, md, my;
    int tiles, chunks;  // 256-row tiles, 64-unit hidden chunks
    int rows, c, hidden;
    const float* b_gate;
    const float* b_up;
    const float* b_down;
    int act, bf16;
    uint32_t* status;
};

struct FusedSmem {
    uint8_t *x, *w1, *w2, *h;
    uint64_t *x_full, *x_empty, *w1_full, *w1_empty, *w2_full, *w2_empty;
    // per subtile; d_full, h_free and y_full one for even and one for odd
    // chunks (tiles): a group may come to a chunk while another still waits
    // for the one before, and a parity tells only two phases apart
    uint64_t *d_full, *d_free, *h_ready, *h_free, *y_full, *y_empty, *out_ready, *out_free;
    uint64_t* drained;  // per issuer
    uint32_t* tmem;
    int* abort;
};

__device__ __forceinline__ void tma_prefetch_2d(const CUtensorMap* map, int x, int y) {
    asm volatile("cp.async.bulk.prefetch.tensor.2d.L2.global.tile [%0, {%1, %2}];" ::"l"(map), "r"(x), "r"(y) : "memory");
}

template <int KC>
__device__ void fused_producer(const FusedArgs& a, const FusedSmem& S) {
    using C = FusedCfg<KC>;
    int ix = 0, i1 = 0, i2 = 0;
    // waits until `slot` of a ring is free for its i-th use
    auto free_slot = [&](uint64_t* empty, int i, int ring) {
        return i < ring ||
               wait_briefly(&empty[i % ring], static_cast<uint32_t>(i / ring - 1) & 1, S.abort, a.status);
    };
    auto load_w1 = [&](int j) {
        if (!free_slot(S.w1_empty, i1, C::W1R)) return false;
        const int s = i1++ % C::W1R;
        const uint32_t dst = smem_u32(S.w1 + s * C::W1_BYTES);
        mbar_arrive_expect_tx(&S.w1_full[s], C::W1_BYTES);
#pragma unroll
        for (int kb = 0; kb < KC; ++kb) {
            tma_load_2d(dst + kb * 16384, &a.mg, kb * 64, j * 64, &S.w1_full[s]);
            tma_load_2d(dst + kb * 16384 + 8192, &a.mu, kb * 64, j * 64, &S.w1_full[s]);
        }
        return true;
    };
    auto run = [&]() {
        for (int tile = blockIdx.x; tile < a.tiles; tile += gridDim.x) {
            if (!load_w1(0)) return false;
#pragma unroll
            for (int sub = 0; sub < 2; ++sub, ++ix) {
                if (!free_slot(S.x_empty, ix, C::XR)) return false;
                const int s = ix % C::XR;
                mbar_arrive_expect_tx(&S.x_full[s], C::X_BYTES);
#pragma unroll
                for (int kb = 0; kb < KC; ++kb)
                    tma_load_2d(smem_u32(S.x + s * C::X_BYTES + kb * 16384), &a.mx, kb * 64, tile * 256 + sub * 128,
                                &S.x_full[s]);
            }
            // the next tile's rows on their way to L2
            if (tile + static_cast<int>(gridDim.x) < a.tiles)
#pragma unroll
                for (int kb = 0; kb < 2 * KC; ++kb)
                    tma_prefetch_2d(&a.mx, (kb % KC) * 64, (tile + static_cast<int>(gridDim.x)) * 256 + kb / KC * 128);
            for (int j = 0; j < a.chunks; ++j) {
                if (!free_slot(S.w2_empty, i2, C::W2R)) return false;
                const int s = i2++ % C::W2R;
                mbar_arrive_expect_tx(&S.w2_full[s], C::W2_BYTES);
                tma_load_2d(smem_u32(S.w2 + s * C::W2_BYTES), &a.md, j * 64, 0, &S.w2_full[s]);
                if (j + 1 < a.chunks && !load_w1(j + 1)) return false;
            }
        }
        return true;
    };
    if (!run()) {
        // aborted: copies in flight land within microseconds; wait 100 us
        // before the CTA's shared memory can go away
        const uint64_t t_end = global_timer_ns() + 100000ull;
        while (global_timer_ns() < t_end) __nanosleep(1000);
    }
}

// D = x [Wg | Wu]^T of every chunk, subtiles in turn.
template <int KC>
__device__ void fused_issue_d(const FusedArgs& a, const FusedSmem& S, uint32_t tmem) {
    using C = FusedCfg<KC>;
    const uint32_t idesc = idesc_f16(128, 128, a.bf16 ? 1u : 0u);
    int ix = 0, c = 0;  // x slots, chunks so far
    auto wait = [&](uint64_t* bar, int n) { return wait_briefly(bar, static_cast<uint32_t>(n) & 1, S.abort, a.status); };
    for (int tile = blockIdx.x; tile < a.tiles; tile += gridDim.x, ix += 2) {
        for (int j = 0; j < a.chunks; ++j, ++c) {
            const int s = c % C::W1R;
            if (!wait(&S.w1_full[s], c / C::W1R)) return;
#pragma unroll
            for (int sub = 0; sub < 2; ++sub) {
                const int xs = (ix + sub) % C::XR;
                if (j == 0 && !wait(&S.x_full[xs], (ix + sub) / C::XR)) return;
                if (c > 0 && !wait(&S.d_free[sub], c - 1)) return;
                tc_fence_after();
                const uint32_t sx = smem_u32(S.x + xs * C::X_BYTES);
                const uint32_t sw = smem_u32(S.w1 + s * C::W1_BYTES);
#pragma unroll
                for (int ks = 0; ks < KC * 4; ++ks) {
                    const uint32_t off = (ks / 4) * 16384 + (ks % 4) * 32;
                    umma_f16(tmem + 256 + sub * 128, sdesc_k_sw128(sx + off), sdesc_k_sw128(sw + off), idesc, ks > 0 ? 1u : 0u);
                }
                umma_commit(&S.d_full[sub * 2 + (c & 1)]);
                if (j + 1 == a.chunks) umma_commit(&S.x_empty[xs]);
            }
            umma_commit(&S.w1_empty[s]);
        }
    }
}

// Y += h Wd^T of every chunk, subtiles in turn.
template <int KC>
__device__ void fused_issue_y(const FusedArgs& a, const FusedSmem& S, uint32_t tmem) {
    using C = FusedCfg<KC>;
    const uint32_t idesc = idesc_f16(128, C::CP, a.bf16 ? 1u : 0u);
    int c = 0, k = 0;  // chunks, tiles so far
    auto wait = [&](uint64_t* bar, int n) { return wait_briefly(bar, static_cast<uint32_t>(n) & 1, S.abort, a.status); };
    for (int tile = blockIdx.x; tile < a.tiles; tile += gridDim.x, ++k) {
        for (int j = 0; j < a.chunks; ++j, ++c) {
            const int s = c % C::W2R;
            if (!wait(&S.w2_full[s], c / C::W2R)) return;
#pragma unroll
            for (int sub = 0; sub < 2; ++sub) {
                if (!wait(&S.h_ready[sub], c)) return;
                if (j == 0 && k > 0 && !wait(&S.y_empty[sub], k - 1)) return;
                tc_fence_after();
                const uint32_t sh = smem_u32(S.h + sub * C::H_BYTES);
                const uint32_t sw = smem_u32(S.w2 + s * C::W2_BYTES);
#pragma unroll
                for (int ks = 0; ks < 4; ++ks)
                    umma_f16(tmem + sub * 128, sdesc_k_sw128(sh + ks * 32), sdesc_k_sw128(sw + ks * 32), idesc,
                             (j > 0 || ks > 0) ? 1u : 0u);
                umma_commit(&S.h_free[sub * 2 + (c & 1)]);
                if (j + 1 == a.chunks) umma_commit(&S.y_full[sub * 2 + (k & 1)]);
            }
            umma_commit(&S.w2_empty[s]);
        }
    }
}

// The epilogue up to 64 channels: three groups in turn.
template <int KC>
__device__ void fused_epilogue(const FusedArgs& a, const FusedSmem& S, uint32_t tmem) {
    using C = FusedCfg<KC>;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int q = warp & 3, half = ((warp - 4) >> 2) & 1;
    const int m = q * 32 + lane;
    const uint32_t lanes = static_cast<uint32_t>(q * 32) << 16;
    auto wait = [&](uint64_t* bar, int n) {
        return __all_sync(0xffffffffu, wait_briefly(bar, static_cast<uint32_t>(n) & 1, S.abort, a.status));
    };
    const int mine = (a.tiles - static_cast<int>(blockIdx.x) + static_cast<int>(gridDim.x) - 1) / static_cast<int>(gridDim.x);
    const int items = mine * a.chunks * 2;
    for (int i = (warp - 4) / kGroupWarps; i < items; i += C::GROUPS) {
        const int sub = i & 1, c = i >> 1;      // subtile, its chunk count so far
        const int k = c / a.chunks, j = c % a.chunks;  // this CTA's tile, chunk
        const uint32_t d = tmem + lanes + 256 + sub * 128;
        uint8_t* unit = S.h + sub * C::H_BYTES;
        if (!wait(&S.d_full[sub * 2 + (c & 1)], c >> 1)) return;
        tc_fence_after();
        constexpr int N = 16;
#pragma unroll
        for (int cc = 0; cc < 32; cc += N) {
            const int col = half * 32 + cc;
            float g[N], u[N];
            {
                uint32_t rg[N], ru[N];
                tmem_ld<N>(d + col, rg);
                tmem_ld<N>(d + 64 + col, ru);
                tmem_wait_ld_regs(rg);
                tmem_wait_ld_regs(ru);
                if (cc + N == 32) {
                    tc_fence_before();
                    warp_arrive(&S.d_free[sub]);
                }
                to_floats(rg, g);
                to_floats(ru, u);
            }
            add_bias(a.b_gate, j * 64 + col, a.hidden, g);
            add_bias(a.b_up, j * 64 + col, a.hidden, u);
            gate_chunk(a.act, g, u);
            if (cc == 0) {
                // the product of the chunk before, and the store of the tile
                // before, have read the unit
                if (c > 0 && !wait(&S.h_free[sub * 2 + ((c - 1) & 1)], (c - 1) >> 1)) return;
                if (j == 0 && k > 0 && !wait(&S.out_free[sub], k * KC - 1)) return;
            }
            put_unit(unit, m, col / 8, g, a.bf16);
        }
        fence_proxy_async();
        warp_arrive(&S.h_ready[sub]);
        if (j + 1 < a.chunks) continue;
        // the subtile's last chunk: its rows out through the unit, 64 columns at a time
        if (!wait(&S.y_full[sub * 2 + (k & 1)], k >> 1)) return;
        tc_fence_after();
        const uint32_t y = tmem + lanes + sub * 128;
#pragma unroll
        for (int u0 = 0; u0 < C::CP; u0 += 64) {
            if (u0 > 0 && !wait(&S.out_free[sub], k * KC + u0 / 64 - 1)) return;
#pragma unroll
            for (int cc = 0; cc < 32; cc += 16) {
                const int col = half * 32 + cc;
                uint32_t r[16];
                tmem_ld16(y + u0 + col, r);
                tmem_wait_ld_regs(r);
                if (u0 + 64 == C::CP && cc == 16) {
                    tc_fence_before();
                    warp_arrive(&S.y_empty[sub]);
                }
                float v[16];
                to_floats(r, v);
                add_bias(a.b_down, u0 + col, a.c, v);
                put_unit(unit, m, col / 8, v, a.bf16);
            }
            fence_proxy_async();
            warp_arrive(&S.out_ready[sub]);
        }
    }
}

// The epilogue at 128 channels: a group for each subtile, which also stores
// its rows.
template <int KC>
__device__ void fused_epilogue_pair(const FusedArgs& a, const FusedSmem& S, uint32_t tmem) {
    using C = FusedCfg<KC>;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int q = warp & 3, sub = (warp - 4) >> 3, half = ((warp - 4) >> 2) & 1;
    const int m = q * 32 + lane;
    const uint32_t lanes = static_cast<uint32_t>(q * 32) << 16;
    const uint32_t d = tmem + lanes + 256 + sub * 128, y = tmem + lanes + sub * 128;
    uint8_t* unit = S.h + sub * C::H_BYTES;
    const bool issuer = lane == 0 && half == 0 && q == 0;
    auto wait = [&](uint64_t* bar, int n) { return wait_briefly(bar, static_cast<uint32_t>(n) & 1, S.abort, a.status); };
    bool ok = true;
    int c = 0, k = 0;
    for (int tile = blockIdx.x; tile < a.tiles; tile += gridDim.x, ++k) {
        for (int j = 0; j < a.chunks; ++j, ++c) {
            ok = ok && wait(&S.d_full[sub * 2 + (c & 1)], c >> 1);
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) continue;
            tc_fence_after();
            const int col = half * 32;
            float g[32], u[32];
            {
                uint32_t rg[32], ru[32];
                tmem_ld32(d + col, rg);
                tmem_ld32(d + 64 + col, ru);
                tmem_wait_ld_regs(rg);
                tmem_wait_ld_regs(ru);
                tc_fence_before();
                warp_arrive(&S.d_free[sub]);
                to_floats(rg, g);
                to_floats(ru, u);
            }
            add_bias(a.b_gate, j * 64 + col, a.hidden, g);
            add_bias(a.b_up, j * 64 + col, a.hidden, u);
            gate_chunk(a.act, g, u);
            // the product of the chunk before has read the unit
            if (c > 0) ok = wait(&S.h_free[sub * 2 + ((c - 1) & 1)], (c - 1) >> 1);
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) continue;
            put_unit(unit, m, col / 8, g, a.bf16);
            fence_proxy_async();
            warp_arrive(&S.h_ready[sub]);
        }
        // the subtile's rows out through the unit, 64 columns at a time
        ok = ok && wait(&S.y_full[sub * 2 + (k & 1)], k >> 1);
        ok = __all_sync(0xffffffffu, ok);
        tc_fence_after();
#pragma unroll
        for (int u0 = 0; u0 < C::CP; u0 += 64) {
            if (u0 > 0) {
                if (issuer) bulk_wait_read();
                named_bar(1 + sub, 32 * kGroupWarps);
            }
            if (ok) {
#pragma unroll
                for (int cc = 0; cc < 2; ++cc) {
                    const int col = half * 32 + cc * 16;
                    uint32_t r[16];
                    tmem_ld16(y + u0 + col, r);
                    tmem_wait_ld_regs(r);
                    if (u0 + 64 == C::CP && cc == 1) {
                        tc_fence_before();
                        warp_arrive(&S.y_empty[sub]);
                    }
                    float v[16];
                    to_floats(r, v);
                    add_bias(a.b_down, u0 + col, a.c, v);
                    put_unit(unit, m, col / 8, v, a.bf16);
                }
                fence_proxy_async();
            }
            named_bar(1 + sub, 32 * kGroupWarps);
            if (ok && issuer) {
                const int row0 = tile * 256 + sub * 128;
                if (u0 < a.c && row0 < a.rows) tma_store_2d(&a.my, smem_u32(unit), u0, row0);
                bulk_commit();
            }
        }
        // the next tile's first h waits for the store to have read the unit
        if (issuer) bulk_wait_read();
        named_bar(1 + sub, 32 * kGroupWarps);
    }
    if (issuer) bulk_wait();
}

// Stores a subtile's finished rows (one thread each).
template <int KC>
__device__ void fused_store(const FusedArgs& a, const FusedSmem& S, int sub) {
    using C = FusedCfg<KC>;
    int i = 0;  // units stored so far
    for (int tile = blockIdx.x; tile < a.tiles; tile += gridDim.x) {
        const int row0 = tile * 256 + sub * 128;
#pragma unroll
        for (int u = 0; u < KC; ++u, ++i) {
            if (!wait_briefly(&S.out_ready[sub], static_cast<uint32_t>(i) & 1, S.abort, a.status)) {
                bulk_wait();
                return;
            }
            if (row0 < a.rows && u * 64 < a.c) tma_store_2d(&a.my, smem_u32(S.h + sub * C::H_BYTES), u * 64, row0);
            bulk_commit();
            bulk_wait_read();
            mbar_arrive(&S.out_free[sub]);
        }
    }
    bulk_wait();
}

template <int KC>
__global__ void __launch_bounds__(FusedCfg<KC>::THREADS, 1) ffn_fused_kernel(const __grid_constant__ FusedArgs a) {
    using C = FusedCfg<KC>;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* p = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    FusedSmem S;
    S.x = p;
    p += C::XR * C::X_BYTES;
    S.w1 = p;
    p += C::W1R * C::W1_BYTES;
    S.w2 = p;
    p += C::W2R * C::W2_BYTES;
    S.h = p;
    p += 2 * C::H_BYTES;
    S.x_full = reinterpret_cast<uint64_t*>(p);
    S.x_empty = S.x_full + C::XR;
    S.w1_full = S.x_empty + C::XR;
    S.w1_empty = S.w1_full + C::W1R;
    S.w2_full = S.w1_empty + C::W1R;
    S.w2_empty = S.w2_full + C::W2R;
    S.d_full = S.w2_empty + C::W2R;
    S.h_free = S.d_full + 4;
    S.y_full = S.h_free + 4;
    S.d_free = S.y_full + 4;
    S.h_ready = S.d_free + 2;
    S.y_empty = S.h_ready + 2;
    S.out_ready = S.y_empty + 2;
    S.out_free = S.out_ready + 2;
    S.drained = S.out_free + 2;
    S.tmem = reinterpret_cast<uint32_t*>(S.drained + 2);
    S.abort = reinterpret_cast<int*>(S.tmem + 1);
    static_assert((2 * (C::XR + C::W1R + C::W2R) + 24) * 8 + 8 <= 512, "barriers fit");

    const int warp = threadIdx.x >> 5;
    if (threadIdx.x == 0) {
        for (int s = 0; s < 2 * (C::XR + C::W1R + C::W2R); ++s) mbar_init(&S.x_full[s], 1);
        for (int s = 0; s < 4; ++s) {
            mbar_init(&S.d_full[s], 1);
            mbar_init(&S.h_free[s], 1);
            mbar_init(&S.y_full[s], 1);
        }
        for (int s = 0; s < 2; ++s) {
            mbar_init(&S.d_free[s], kGroupWarps);
            mbar_init(&S.h_ready[s], kGroupWarps);
            mbar_init(&S.y_empty[s], kGroupWarps);
            mbar_init(&S.out_ready[s], kGroupWarps);
            mbar_init(&S.out_free[s], 1);
            mbar_init(&S.drained[s], 1);
        }
        *S.abort = 0;
        fence_mbar_init();
    }
    if (warp == 3) {
        tmem_alloc(S.tmem, 512);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *S.tmem;

    if (warp == 0) {
        if ((threadIdx.x & 31) == 0) fused_producer<KC>(a, S);
        __syncwarp();
    } else if (warp <= 2) {
        if ((threadIdx.x & 31) == 0) {
            if (warp == 1)
                fused_issue_d<KC>(a, S, tmem);
            else
                fused_issue_y<KC>(a, S, tmem);
        }
        __syncwarp();
    } else if (warp == 3) {
        if (KC == 1 && (threadIdx.x & 31) < 2) fused_store<KC>(a, S, threadIdx.x & 31);
        __syncwarp();
    } else {
        if constexpr (KC == 1)
            fused_epilogue<KC>(a, S, tmem);
        else
            fused_epilogue_pair<KC>(a, S, tmem);
    }
    tc_fence_before();
    __syncthreads();
    if (*reinterpret_cast<volatile int*>(S.abort)) {
        // MMAs sent before the abort may still write TMEM: a commit tracks an
        // issuer's; wait (bounded) before the columns go
        if ((warp == 1 || warp == 2) && (threadIdx.x & 31) == 0) {
            umma_commit(&S.drained[warp - 1]);
            (void)mbar_wait(&S.drained[warp - 1], 0);
        }
        __syncthreads();
    }
    if (warp == 3) {
        tc_fence_after();
        tmem_dealloc(tmem, 512);
    }
}

template <int KC>
cudaError_t launch_t(const FusedArgs& a, cudaStream_t st) {
    using C = FusedCfg<KC>;
    static std::mutex mu;
    static int num_sms[64] = {0};
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (dev < 0 || dev >= 64) return cudaErrorInvalidDevice;
    int sms = 0;
    {
        std::lock_guard<std::mutex> lk(mu);
        if (!num_sms[dev]) {
            e = cudaFuncSetAttribute(ffn_fused_kernel<KC>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM);
            if (e != cudaSuccess) return e;
            int count = 0;
            e = cudaDeviceGetAttribute(&count, cudaDevAttrMultiProcessorCount, dev);
            if (e != cudaSuccess) return e;
            num_sms[dev] = count;
        }
        sms = num_sms[dev];
    }
    ffn_fused_kernel<KC><<<std::min(a.tiles, sms), C::THREADS, C::SMEM, st>>>(a);
    return cudaGetLastError();
}

}  // namespace

cudaError_t launch_ffn_fused(const FfnShape& s, const void* x, const FfnWeights& w, void* y, uint32_t* status,
                             cudaStream_t st) {
    const bool bf = s.dtype == DT_BF16;
    FusedArgs a{};
    const int kc = s.c > 64 ? 2 : 1;
    cudaError_t e = make_map_16bit(&a.mx, x, bf, s.n, s.c, 128);
    if (e == cudaSuccess) e = make_map_16bit(&a.mg, w.w_gate, bf, s.hidden, s.c, 64);
    if (e == cudaSuccess) e = make_map_16bit(&a.mu, w.w_up, bf, s.hidden, s.c, 64);
    if (e == cudaSuccess) e = make_map_16bit(&a.md, w.w_down, bf, s.c, s.hidden, 64 * kc);
    if (e == cudaSuccess) e = make_map_16bit(&a.my, y, bf, s.n, s.c, 128);
    if (e != cudaSuccess) return e;
    a.tiles = static_cast<int>((s.n + 255) / 256);
    a.chunks = (s.hidden + 63) / 64;
    a.rows = static_cast<int>(s.n);
    a.c = s.c;
    a.hidden = s.hidden;
    a.b_gate = w.b_gate, a.b_up = w.b_up, a.b_down = w.b_down;
    a.act = s.act;
    a.bf16 = bf;
    a.status = status;
    return kc == 2 ? launch_t<2>(a, st) : launch_t<1>(a, st);
}

}  // namespace msc
