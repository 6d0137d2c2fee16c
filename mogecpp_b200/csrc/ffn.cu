// Gated feed-forward block over the channels of each row, [n][c] rows of fp16
// or bf16:
//   g = x Wg^T + bg;  u = x Wu^T + bu;  h = act(g) * u;  y = h Wd^T + bd
// (SwiGLU / GeGLU), and its backward pass, which computes g and u again:
//   dh = dy Wd;  dg = dh u act'(g);  du = dh act(g)
//   dx = dg Wg + du Wu;  dWg = dg^T x;  dWu = du^T x;  dWd = dy^T h
//   dbg, dbu, dbd = column sums of dg, du, dy
//
// Every product runs on tcgen05 (ffn_gemm.cuh) with fp32 accumulators; the
// activation, its derivative and the gating product are fp32 in the epilogue.
// h, dg and du are rounded once to the features' type, because the tensor
// cores take them as 16-bit operands of the next product; the bias sums are
// taken from the unrounded fp32 values.
#include "ffn.h"

#include "conv.h"
#include "ffn_fused.h"
#include "ffn_gemm.cuh"
#include "ffn_rows.h"

#include <algorithm>
#include <cstring>
#include <mutex>

namespace msc {
namespace {

using EncodeTiled = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                 const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                 CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeTiled encode_tiled() {
    static std::mutex mu;
    static EncodeTiled fn = nullptr;
    std::lock_guard<std::mutex> lk(mu);
    if (!fn) {
        void* p = nullptr;
        cudaDriverEntryPointQueryResult found;
        if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &p, 12000, cudaEnableDefault, &found) == cudaSuccess &&
            found == cudaDriverEntryPointSuccess)
            fn = reinterpret_cast<EncodeTiled>(p);
    }
    return fn;
}

constexpr int kSms = 148;  // B200; fixed, so that the split of a sum and the workspace do not depend on the device

int64_t cdiv(int64_t a, int64_t b) { return (a + b - 1) / b; }
size_t align256(size_t v) { return (v + 255) / 256 * 256; }

// Tile of a product with `cols` output columns: pairs of CTAs on 256 rows
// where every pair of SMs gets one, else the widest column tile that gives
// half the SMs one (wider tiles read less shared memory per product; narrower
// ones spread few rows over more SMs).  Measured with half / all of the SMs as
// the rule (us, whole block): 1,237 rows of 1024 -> 1376 23.0 / 27.8, 3,000 of
// 512 -> 2048 33.7 / 41.2; backward 1,237 of 1024 -> 1376 60.2 / 69.2.
struct TilePlan {
    int ht, cg;
};
TilePlan tile_plan(int64_t rows, int cols) {
    const int64_t m = cdiv(rows, 128), pairs = cdiv(rows, 256);
    for (int ht = 256; ht > 64; ht /= 2) {
        if (cols <= ht / 2) continue;
        if (pairs * cdiv(cols, ht) >= kSms / 2) return {ht, 2};
        if (m * cdiv(cols, ht) >= kSms / 2) return {ht, 1};
    }
    return {64, 1};
}

// Splits of a K of `ksteps` steps when `tiles` output tiles leave SMs idle, of
// at least kMinSteps steps each.  The splits of equal length that K is then cut
// into may be fewer (24 steps: 6 of 4; 25: 5 of 5); the most there may be grows
// with K.
constexpr int kMinSteps = 4;
int most_splits(int64_t tiles, int ksteps) {
    const int64_t s = tiles > 0 && tiles * 2 <= kSms ? kSms / tiles : 1;
    return static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(s, ksteps / kMinSteps)));
}
int k_splits(int64_t tiles, int ksteps, int* ksplit) {
    const int s = most_splits(tiles, ksteps);
    ksteps = std::max(ksteps, 1);
    *ksplit = static_cast<int>(cdiv(ksteps, s));
    return static_cast<int>(cdiv(ksteps, *ksplit));
}

// No sum in one accumulator runs over more than 32768 elements: the tensor
// core's fp32 accumulator truncates, so that a sum of one sign drifts towards
// zero with the length of its chain.  Measured on dx (fp16, positive terms of
// like size): 2.6e-5 of the sum over 4,096 elements, 1.2e-4 over 16,384, 2.2e-4
// over 32,768 and 4.4e-4 over 65,536, where the output's own rounding is 4.9e-4
// at most; a truncation of half 2^-23 per 8 elements fits them all.
constexpr int kChainSteps = 512;
void limit_chain(int ksteps, int* splits, int* ksplit) {
    if (*ksplit <= kChainSteps) return;
    *ksplit = kChainSteps;
    *splits = static_cast<int>(cdiv(ksteps, kChainSteps));
}

struct ProjPlan {
    int ht, cg, splits, ksplit;
};
ProjPlan proj_plan(int64_t n, int cols, int ksteps) {
    const TilePlan t = tile_plan(n, cols);
    ProjPlan p{t.ht, t.cg, 1, ksteps};
    if (t.cg == 1) p.splits = k_splits(cdiv(n, 128) * cdiv(cols, p.ht), ksteps, &p.ksplit);
    limit_chain(ksteps, &p.splits, &p.ksplit);
    return p;
}

struct DwPlan {
    int ht, cg, splits, ksplit, tiles;
};
DwPlan dw_plan(int64_t n, int c, int hidden) {
    DwPlan p{};
    p.ht = c > 128 ? 256 : (c > 64 ? 128 : 64);
    p.cg = 1;
    auto tiles = [&](int cg) {
        return static_cast<int>(2 * cdiv(hidden, 128 * cg) * cdiv(c, p.ht) + cdiv(c, 128 * cg) * cdiv(hidden, p.ht));
    };
    if (p.ht == 256 && tiles(2) >= kSms / 2) p.cg = 2;
    p.tiles = tiles(p.cg);
    const int ksteps = static_cast<int>(cdiv(n, 64));
    p.splits = 1;
    p.ksplit = std::max(ksteps, 1);
    if (p.cg == 1) p.splits = k_splits(p.tiles, ksteps, &p.ksplit);
    limit_chain(ksteps, &p.splits, &p.ksplit);
    return p;
}

// Lets a kernel of a pass start while the one before it drains (it waits for
// it before it touches memory): 1,237 x 512 -> 1376 takes 19.1 us for 20.7.  A
// pass's first kernel is launched without it, after all earlier work.
cudaLaunchAttribute overlap_attribute() {
    cudaLaunchAttribute at{};
    at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at.val.programmaticStreamSerializationAllowed = 1;
    return at;
}

template <int MODE, int HT, int CG>
cudaError_t launch_gemm_t(const FfnGemmArgs& a, bool first, cudaStream_t st) {
    using C = FfnCfg<MODE, HT, CG>;
    auto kern = ffn_gemm_kernel<MODE, HT, CG>;
    cudaLaunchConfig_t cfg{};
    cfg.blockDim = dim3(C::THREADS);
    cfg.dynamicSmemBytes = C::SMEM;
    cfg.stream = st;
    cudaLaunchAttribute at[2]{};
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = CG;
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    at[1] = overlap_attribute();
    cfg.attrs = at;
    cfg.numAttrs = 1;
    // per device and instantiation: the shared-memory opt-in and the CTAs
    // (pairs) that run at once, set up once under a lock
    static std::mutex mu;
    static int at_once[64] = {0};
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (dev < 0 || dev >= 64) return cudaErrorInvalidDevice;
    int running = 0;
    {
        std::lock_guard<std::mutex> lk(mu);
        if (!at_once[dev]) {
            e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM);
            if (e != cudaSuccess) return e;
            int count = 0;
            if constexpr (CG == 2) {
                cfg.gridDim = dim3(CG);
                e = cudaOccupancyMaxActiveClusters(&count, kern, &cfg);
            } else {
                e = cudaDeviceGetAttribute(&count, cudaDevAttrMultiProcessorCount, dev);
            }
            if (e != cudaSuccess) return e;
            if (count < 1) return cudaErrorInvalidConfiguration;
            at_once[dev] = count;
        }
        running = at_once[dev];
    }
    cfg.gridDim = dim3(static_cast<unsigned>(CG * std::min(a.tiles * a.splits, running)));
    cfg.numAttrs = first ? 1 : 2;
    return cudaLaunchKernelEx(&cfg, kern, a);
}

template <int MODE>
cudaError_t launch_gemm(const FfnGemmArgs& a, int ht, int cg, bool first, cudaStream_t st) {
    if constexpr (MODE == FFN_HBACK) {
        return cg == 2 ? launch_gemm_t<MODE, 128, 2>(a, first, st) : launch_gemm_t<MODE, 64, 1>(a, first, st);
    } else if constexpr (MODE == FFN_HIDDEN) {
        if (cg == 2) return launch_gemm_t<MODE, 128, 2>(a, first, st);
        return ht == 128 ? launch_gemm_t<MODE, 128, 1>(a, first, st) : launch_gemm_t<MODE, 64, 1>(a, first, st);
    } else {
        if constexpr (MODE != FFN_DW)  // (its pairs have 256 columns, dw_plan)
            if (cg == 2 && ht == 128) return launch_gemm_t<MODE, 128, 2>(a, first, st);
        if (cg == 2) return launch_gemm_t<MODE, 256, 2>(a, first, st);
        if (ht == 256) return launch_gemm_t<MODE, 256, 1>(a, first, st);
        return ht == 128 ? launch_gemm_t<MODE, 128, 1>(a, first, st) : launch_gemm_t<MODE, 64, 1>(a, first, st);
    }
}

void one_problem(FfnGemmArgs& a, int64_t rows, int cols, int ht, int cg) {
    a.nprob = 1;
    a.m_tiles[0] = static_cast<int>(cdiv(rows, 128 * cg));
    a.n_tiles[0] = static_cast<int>(cdiv(cols, ht));
    a.rows[0] = static_cast<int>(rows);
    a.cols[0] = cols;
    a.tiles = a.m_tiles[0] * a.n_tiles[0];
    a.splits = 1;
    a.ksplit = a.ksteps[0] + a.ksteps[1];
}

// Column sums of a 16-bit [n][c] matrix over a run of rows per block, fp32.
// Rows of a run: few where the rows are few, so that more SMs have loads in
// flight (1,237 x 256: 3.4 us with 64, 8.2 with 256); more runs cost their
// totals (101,117 x 128: 13.1 + 6.5 us with 256, 10.9 + 10.0 with 64).
int colsum_rows(int64_t n) { return n <= 16384 ? 64 : 256; }
__global__ void __launch_bounds__(256) colsum_kernel(const void* y, int64_t n, int c, int bf16, int lanes, int run, float* part) {
    // `lanes` threads (8, 16 or 32) x 8 columns a row, 256 / lanes rows at once
    launch_dependents();
    __shared__ float red[256][9];
    const int tx = threadIdx.x & (lanes - 1), ty = threadIdx.x / lanes, ry = 256 / lanes;
    const int col = (blockIdx.y * lanes + tx) * 8;
    const int64_t r0 = static_cast<int64_t>(blockIdx.x) * run;
    const int64_t r1 = min(r0 + run, n);
    float s[8] = {};
    if (col < c) {
#pragma unroll 4
        for (int64_t r = r0 + ty; r < r1; r += ry) {
            const uint4 w4 = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(y) + r * c + col);
            const uint32_t w[4] = {w4.x, w4.y, w4.z, w4.w};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float2 t = bf16 ? __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&w[e]))
                                      : __half22float2(*reinterpret_cast<const __half2*>(&w[e]));
                s[2 * e] += t.x, s[2 * e + 1] += t.y;
            }
        }
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) red[threadIdx.x][e] = s[e];
    __syncthreads();
    for (int o = threadIdx.x; o < lanes * 8; o += 256) {
        const int t = o >> 3, e = o & 7;
        const int cc = (blockIdx.y * lanes + t) * 8 + e;
        if (cc >= c) continue;
        float q = 0.f;
        for (int w = 0; w < ry; ++w) q += red[w * lanes + t][e];
        part[static_cast<int64_t>(blockIdx.x) * c + cc] = q;
    }
}

// out[i] = sum over the splits of part[s][i] (+ bias of column i % cols), in
// split order; four elements a thread.
struct SplitSum {
    const float* part;
    int64_t stride;      // floats per split
    int splits;
    void* out[3];
    int64_t begin[4];    // first element of each output, and the end (0: nothing to do)
    const float* bias;
    int cols;
};
__device__ void split_sum(const SplitSum& a, int64_t block, int bf16) {
    const int64_t i = (block * 256 + threadIdx.x) * 4;
    if (i >= a.begin[3]) return;
    float4 s = *reinterpret_cast<const float4*>(a.part + i);
    for (int k = 1; k < a.splits; ++k) {
        const float4 t = *reinterpret_cast<const float4*>(a.part + k * a.stride + i);
        s.x += t.x, s.y += t.y, s.z += t.z, s.w += t.w;
    }
    if (a.bias) {
        const float4 b = __ldg(reinterpret_cast<const float4*>(a.bias + i % a.cols));
        s.x += b.x, s.y += b.y, s.z += b.z, s.w += b.w;
    }
    const int p = i >= a.begin[2] ? 2 : (i >= a.begin[1] ? 1 : 0);
    uint2 w;
    if (bf16) {
        const __nv_bfloat162 lo = __floats2bfloat162_rn(s.x, s.y), hi = __floats2bfloat162_rn(s.z, s.w);
        w = make_uint2(*reinterpret_cast<const uint32_t*>(&lo), *reinterpret_cast<const uint32_t*>(&hi));
    } else {
        const __half2 lo = __floats2half2_rn(s.x, s.y), hi = __floats2half2_rn(s.z, s.w);
        w = make_uint2(*reinterpret_cast<const uint32_t*>(&lo), *reinterpret_cast<const uint32_t*>(&hi));
    }
    uint16_t* out = static_cast<uint16_t*>(p == 2 ? a.out[2] : (p == 1 ? a.out[1] : a.out[0]));
    *reinterpret_cast<uint2*>(out + (i - (p == 2 ? a.begin[2] : (p == 1 ? a.begin[1] : a.begin[0])))) = w;
}

// Totals over the units of part [units][cols] in double and in a fixed order,
// 8 columns a block; the first n0 columns go to out[0], the others to out[1]
// (either may be NULL).
struct ColumnTotal {
    const float* part;
    int64_t units;
    int cols, n0;  // cols 0: nothing to do
    float* out[2];
};
__device__ void column_total(const ColumnTotal& a, int block) {
    __shared__ double red[32][9];
    const int tx = threadIdx.x & 7, ty = threadIdx.x >> 3;
    const int col = block * 8 + tx;
    double s = 0.0;
    if (col < a.cols) {
#pragma unroll 8
        for (int64_t u = ty; u < a.units; u += 32) s += a.part[u * a.cols + col];
    }
    red[ty][tx] = s;
    __syncthreads();
    for (int o = 16; o >= 1; o >>= 1) {
        if (ty < o) red[ty][tx] += red[ty + o][tx];
        __syncthreads();
    }
    if (ty == 0 && col < a.cols) {
        float* o = col < a.n0 ? a.out[0] : a.out[1];
        if (o) o[col < a.n0 ? col : col - a.n0] = static_cast<float>(red[0][tx]);
    }
}

// What is left of a pass after its products, in one launch: the K splits'
// sums and the bias gradients' column totals.
struct FinishArgs {
    SplitSum split[2];
    ColumnTotal total[2];
    int end[4];  // last block (exclusive) of split[0], split[1], total[0], total[1]
    int bf16;
};
__global__ void __launch_bounds__(256) finish_kernel(const __grid_constant__ FinishArgs a) {
    wait_dependency();
    const int b = blockIdx.x;
    if (b < a.end[0]) split_sum(a.split[0], b, a.bf16);
    else if (b < a.end[1]) split_sum(a.split[1], b - a.end[0], a.bf16);
    else if (b < a.end[2]) column_total(a.total[0], b - a.end[1]);
    else column_total(a.total[1], b - a.end[2]);
}

cudaError_t launch_finish(FinishArgs& a, cudaStream_t st) {
    int64_t end = 0;
    for (int i = 0; i < 2; ++i) a.end[i] = static_cast<int>(end += cdiv(a.split[i].begin[3], 1024));
    for (int i = 0; i < 2; ++i) a.end[2 + i] = static_cast<int>(end += cdiv(a.total[i].cols, 8));
    if (end == 0) return cudaSuccess;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(static_cast<unsigned>(end));
    cfg.blockDim = dim3(256);
    cfg.stream = st;
    cudaLaunchAttribute at = overlap_attribute();
    cfg.attrs = &at;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, finish_kernel, a);
}

#define MSC_TRY(expr)                        \
    do {                                     \
        const cudaError_t e_ = (expr);       \
        if (e_ != cudaSuccess) return e_;    \
    } while (0)

// One kernel for the whole block where the channels fit its accumulators and
// the rows fill the SMs with 256-row tiles.
bool use_fused(int64_t n, int c) { return c <= kFfnFusedMaxC && n >= kFfnFusedMinRows; }

struct FwdWs {
    size_t hidden, part, total;
};
FwdWs fwd_ws(int64_t n, int c, int hidden) {
    FwdWs w{};
    if (use_fused(n, c)) return w;
    if (ffn_few_rows(n, c, hidden)) {
        w.total = align256(static_cast<size_t>(n) * hidden * 4);
        return w;
    }
    const ProjPlan p = proj_plan(n, c, static_cast<int>(cdiv(hidden, 64)));
    w.hidden = 0;
    w.part = align256(static_cast<size_t>(n) * hidden * 2);
    w.total = w.part + (p.splits > 1 ? align256(static_cast<size_t>(p.splits) * n * c * 4) : 0);
    return w;
}

struct BwdWs {
    size_t dg, du, h, bias, dbd, part_x, part_w, total;
};
BwdWs bwd_ws(int64_t n, int c, int hidden) {
    BwdWs w{};
    const size_t nh = align256(static_cast<size_t>(n) * hidden * 2);
    w.dg = 0;
    w.du = nh;
    w.h = 2 * nh;
    w.bias = 3 * nh;
    w.dbd = w.bias + align256(static_cast<size_t>(cdiv(n, 128)) * 2 * hidden * 4);
    w.part_x = w.dbd + align256(static_cast<size_t>(cdiv(n, colsum_rows(n))) * c * 4);
    const ProjPlan px = proj_plan(n, c, static_cast<int>(2 * cdiv(hidden, 64)));
    const DwPlan pw = dw_plan(n, c, hidden);
    w.part_w = w.part_x + (px.splits > 1 ? align256(static_cast<size_t>(px.splits) * n * c * 4) : 0);
    w.total = w.part_w + (pw.splits > 1 ? align256(static_cast<size_t>(pw.splits) * 3 * c * hidden * 4) : 0);
    return w;
}

}  // namespace

cudaError_t make_map_16bit(CUtensorMap* map, const void* base, bool bf16, int64_t rows, int64_t cols, int box_rows) {
    const EncodeTiled enc = encode_tiled();
    if (!enc) return cudaErrorNotSupported;
    const cuuint64_t dims[2] = {static_cast<cuuint64_t>(cols), static_cast<cuuint64_t>(rows)};
    const cuuint64_t strides[1] = {static_cast<cuuint64_t>(cols) * 2};
    const cuuint32_t box[2] = {64, static_cast<cuuint32_t>(box_rows)};
    const cuuint32_t es[2] = {1, 1};
    const CUresult r = enc(map, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2,
                           const_cast<void*>(base), dims, strides, box, es, CU_TENSOR_MAP_INTERLEAVE_NONE,
                           CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                           CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return r == CUDA_SUCCESS ? cudaSuccess : cudaErrorInvalidValue;
}

size_t ffn_workspace_bytes(int64_t n, int c, int hidden) { return fwd_ws(n, c, hidden).total; }

size_t ffn_workspace_bound(int64_t n, int c, int hidden) {
    if (use_fused(n, c)) return 0;
    // the dot products' fp32 hidden values end at a size (ffn_few_rows)
    int few = hidden / 8 * 8;
    if (!ffn_few_rows(n, c, few)) few = ffn_few_rows(n, c, 8) ? static_cast<int>(kFewRowsWork / (n * c) / 8 * 8) : 0;
    const size_t rows = align256(static_cast<size_t>(n) * few * 4);
    if (few >= hidden) return rows;
    const TilePlan t = tile_plan(n, c);
    const int ksteps = static_cast<int>(cdiv(hidden, 64));
    const int splits = std::max(t.cg == 1 ? most_splits(cdiv(n, 128) * cdiv(c, t.ht), ksteps) : 1,
                                static_cast<int>(cdiv(ksteps, kChainSteps)));
    const size_t part = splits > 1 ? align256(static_cast<size_t>(splits) * n * c * 4) : 0;
    return std::max(rows, align256(static_cast<size_t>(n) * hidden * 2) + part);
}
size_t ffn_backward_workspace_bytes(int64_t n, int c, int hidden) { return bwd_ws(n, c, hidden).total; }

cudaError_t launch_ffn(const FfnShape& s, const void* x, const FfnWeights& w, void* y, void* ws, uint32_t* status,
                       cudaStream_t st) {
    if (s.n == 0) return cudaSuccess;
    if (use_fused(s.n, s.c)) return launch_ffn_fused(s, x, w, y, status, st);
    if (ffn_few_rows(s.n, s.c, s.hidden)) return launch_ffn_rows(s, x, w, y, static_cast<float*>(ws), st);
    const bool bf = s.dtype == DT_BF16;
    const FwdWs o = fwd_ws(s.n, s.c, s.hidden);
    char* base = static_cast<char*>(ws);
    void* h = base + o.hidden;
    const int64_t m = cdiv(s.n, 128);
    {
        FfnGemmArgs a{};
        // pairs on 256 rows x 128 hidden units, as tile_plan; below, the wide
        // tile while half the SMs get one (us, 128 / 64 columns: 300 rows of
        // 1024 -> 4096 24.4 / 26.8, 1,237 of 1024 -> 1376 27.6 / 29.5)
        const int cg = cdiv(s.n, 256) * cdiv(s.hidden, 128) >= kSms / 2 ? 2 : 1;
        const int ht = cg == 2 || m * cdiv(s.hidden, 128) >= kSms / 2 ? 128 : 64;
        MSC_TRY(make_map_16bit(&a.ma[0], x, bf, s.n, s.c, 128));
        MSC_TRY(make_map_16bit(&a.mb[0], w.w_gate, bf, s.hidden, s.c, ht));
        MSC_TRY(make_map_16bit(&a.mb[1], w.w_up, bf, s.hidden, s.c, ht));
        MSC_TRY(make_map_16bit(&a.mo[0], h, bf, s.n, s.hidden, 128));
        a.ksteps[0] = static_cast<int>(cdiv(s.c, 64));
        one_problem(a, s.n, s.hidden, ht, cg);
        a.bias0 = w.b_gate, a.bias1 = w.b_up;
        a.act = s.act, a.bf16 = bf, a.status = status;
        MSC_TRY(launch_gemm<FFN_HIDDEN>(a, ht, cg, true, st));
    }
    FfnGemmArgs a{};
    a.ksteps[0] = static_cast<int>(cdiv(s.hidden, 64));
    const ProjPlan p = proj_plan(s.n, s.c, a.ksteps[0]);
    MSC_TRY(make_map_16bit(&a.ma[0], h, bf, s.n, s.hidden, 128));
    MSC_TRY(make_map_16bit(&a.mb[0], w.w_down, bf, s.c, s.hidden, p.ht / p.cg));
    MSC_TRY(make_map_16bit(&a.mo[0], y, bf, s.n, s.c, 128));
    one_problem(a, s.n, s.c, p.ht, p.cg);
    a.splits = p.splits, a.ksplit = p.ksplit;
    a.bias0 = w.b_down;
    a.bf16 = bf, a.status = status;
    if (p.splits > 1) {
        a.partial = reinterpret_cast<float*>(base + o.part);
        a.partial_split = s.n * s.c;
    }
    MSC_TRY(launch_gemm<FFN_PROJ>(a, p.ht, p.cg, false, st));
    if (p.splits > 1) {
        const int64_t e = s.n * s.c;
        FinishArgs f{};
        f.split[0] = SplitSum{a.partial, e, p.splits, {y, nullptr, nullptr}, {0, e, e, e}, w.b_down, s.c};
        f.bf16 = bf;
        MSC_TRY(launch_finish(f, st));
    }
    return cudaSuccess;
}

cudaError_t launch_ffn_backward(const FfnShape& s, const void* x, const void* dy, const FfnWeights& w,
                                const FfnGrads& g, void* ws, uint32_t* status, cudaStream_t st) {
    const bool bf = s.dtype == DT_BF16;
    const int64_t ch = static_cast<int64_t>(s.c) * s.hidden;
    if (s.n == 0) {
        if (g.w_gate) {
            MSC_TRY(cudaMemsetAsync(g.w_gate, 0, ch * 2, st));
            MSC_TRY(cudaMemsetAsync(g.w_up, 0, ch * 2, st));
            MSC_TRY(cudaMemsetAsync(g.w_down, 0, ch * 2, st));
        }
        if (g.b_gate) MSC_TRY(cudaMemsetAsync(g.b_gate, 0, s.hidden * sizeof(float), st));
        if (g.b_up) MSC_TRY(cudaMemsetAsync(g.b_up, 0, s.hidden * sizeof(float), st));
        if (g.b_down) MSC_TRY(cudaMemsetAsync(g.b_down, 0, s.c * sizeof(float), st));
        return cudaSuccess;
    }
    const BwdWs o = bwd_ws(s.n, s.c, s.hidden);
    char* base = static_cast<char*>(ws);
    void* dg = base + o.dg;
    void* du = base + o.du;
    void* h = base + o.h;
    FinishArgs fin{};
    fin.bf16 = bf;
    const int kc = static_cast<int>(cdiv(s.c, 64)), kh = static_cast<int>(cdiv(s.hidden, 64));
    const int64_t m = cdiv(s.n, 128);
    if (g.b_down) {
        float* cp = reinterpret_cast<float*>(base + o.dbd);
        const int64_t units = cdiv(s.n, colsum_rows(s.n));
        const int lanes = s.c <= 64 ? 8 : (s.c <= 128 ? 16 : 32);
        colsum_kernel<<<dim3(static_cast<unsigned>(units), static_cast<unsigned>(cdiv(s.c, 8 * lanes))), 256, 0, st>>>(
            dy, s.n, s.c, bf, lanes, colsum_rows(s.n), cp);
        MSC_TRY(cudaGetLastError());
        fin.total[1] = ColumnTotal{cp, units, s.c, s.c, {g.b_down, nullptr}};
    }
    {
        FfnGemmArgs a{};
        const int cg = cdiv(s.n, 256) * cdiv(s.hidden, 128) >= kSms / 2 ? 2 : 1;
        const int ht = 64 * cg;
        MSC_TRY(make_map_16bit(&a.ma[0], dy, bf, s.n, s.c, 128));
        MSC_TRY(make_map_16bit(&a.ma[1], x, bf, s.n, s.c, 128));
        MSC_TRY(make_map_16bit(&a.mb[0], w.w_gate, bf, s.hidden, s.c, ht));
        MSC_TRY(make_map_16bit(&a.mb[1], w.w_up, bf, s.hidden, s.c, ht));
        MSC_TRY(make_map_16bit(&a.mb[2], w.w_down, bf, s.c, s.hidden, 64));
        MSC_TRY(make_map_16bit(&a.mo[0], dg, bf, s.n, s.hidden, 128));
        MSC_TRY(make_map_16bit(&a.mo[1], du, bf, s.n, s.hidden, 128));
        MSC_TRY(make_map_16bit(&a.mo[2], h, bf, s.n, s.hidden, 128));
        a.ksteps[0] = a.ksteps[1] = kc;
        one_problem(a, s.n, s.hidden, ht, cg);
        a.bias0 = w.b_gate, a.bias1 = w.b_up;
        if (g.b_gate || g.b_up) a.bias_part = reinterpret_cast<float*>(base + o.bias);
        a.act = s.act, a.bf16 = bf, a.status = status;
        MSC_TRY(launch_gemm<FFN_HBACK>(a, ht, cg, !g.b_down, st));
        if (a.bias_part) fin.total[0] = ColumnTotal{a.bias_part, m, 2 * s.hidden, s.hidden, {g.b_gate, g.b_up}};
    }
    if (g.dx) {
        FfnGemmArgs a{};
        const ProjPlan p = proj_plan(s.n, s.c, 2 * kh);
        MSC_TRY(make_map_16bit(&a.ma[0], dg, bf, s.n, s.hidden, 128));
        MSC_TRY(make_map_16bit(&a.ma[1], du, bf, s.n, s.hidden, 128));
        MSC_TRY(make_map_16bit(&a.mb[0], w.w_gate, bf, s.hidden, s.c, 64));
        MSC_TRY(make_map_16bit(&a.mb[1], w.w_up, bf, s.hidden, s.c, 64));
        MSC_TRY(make_map_16bit(&a.mo[0], g.dx, bf, s.n, s.c, 128));
        a.ksteps[0] = a.ksteps[1] = kh;
        one_problem(a, s.n, s.c, p.ht, p.cg);
        a.splits = p.splits, a.ksplit = p.ksplit;
        a.bf16 = bf, a.status = status;
        if (p.splits > 1) {
            const int64_t e = s.n * s.c;
            a.partial = reinterpret_cast<float*>(base + o.part_x);
            a.partial_split = e;
            fin.split[0] = SplitSum{a.partial, e, p.splits, {g.dx, nullptr, nullptr}, {0, e, e, e}, nullptr, s.c};
        }
        MSC_TRY(launch_gemm<FFN_DX>(a, p.ht, p.cg, false, st));
    }
    if (g.w_gate) {
        FfnGemmArgs a{};
        const DwPlan p = dw_plan(s.n, s.c, s.hidden);
        const void* am[3] = {dg, du, dy};
        const void* bm[3] = {x, x, h};
        void* om[3] = {g.w_gate, g.w_up, g.w_down};
        a.nprob = 3;
        for (int i = 0; i < 3; ++i) {
            const int rows = i < 2 ? s.hidden : s.c, cols = i < 2 ? s.c : s.hidden;
            MSC_TRY(make_map_16bit(&a.ma[i], am[i], bf, s.n, rows, 64));
            MSC_TRY(make_map_16bit(&a.mb[i], bm[i], bf, s.n, cols, 64));
            MSC_TRY(make_map_16bit(&a.mo[i], om[i], bf, rows, cols, 128));
            a.m_tiles[i] = static_cast<int>(cdiv(rows, 128 * p.cg));
            a.n_tiles[i] = static_cast<int>(cdiv(cols, p.ht));
            a.rows[i] = rows, a.cols[i] = cols;
            a.partial_prob[i] = i * ch;
        }
        a.tiles = p.tiles;
        a.ksteps[0] = static_cast<int>(cdiv(s.n, 64));
        a.splits = p.splits, a.ksplit = p.ksplit;
        a.bf16 = bf, a.status = status;
        if (p.splits > 1) {
            a.partial = reinterpret_cast<float*>(base + o.part_w);
            a.partial_split = 3 * ch;
            fin.split[1] = SplitSum{a.partial, 3 * ch, p.splits, {om[0], om[1], om[2]}, {0, ch, 2 * ch, 3 * ch}, nullptr, s.c};
        }
        MSC_TRY(launch_gemm<FFN_DW>(a, p.ht, p.cg, false, st));
    }
    return launch_finish(fin, st);
}

}  // namespace msc
