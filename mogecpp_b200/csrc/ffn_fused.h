// Gated feed-forward block of many rows and few channels in one kernel
// (ffn_fused.cu).
#pragma once

#include "ffn.h"

namespace msc {

constexpr int kFfnFusedMaxC = 128;
// From this many rows on (half the SMs have a 256-row tile).  Measured (bf16,
// us, one kernel / two): 128 -> 512, 9,472 rows 27.3 / 20.5, 18,944 rows 27.7 /
// 30.6, 37,888 rows 28.5 / 45.7; 64 -> 256, 9,472 rows 14.3 / 14.2, 18,944 rows
// 14.4 / 19.2.
constexpr int64_t kFfnFusedMinRows = 256 * 74;

cudaError_t launch_ffn_fused(const FfnShape& s, const void* x, const FfnWeights& w, void* y, uint32_t* status,
                             cudaStream_t st);

}  // namespace msc
