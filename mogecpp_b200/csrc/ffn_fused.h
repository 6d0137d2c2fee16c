// Gated feed-forward block of many rows and few channels in one kernel
// (ffn_fused.cu).
#pragma once

#include "ffn.h"

namespace msc {

constexpr int kFfnFusedMaxC = 128;
// From this many rows on (half the SMs have a 256-row tile).
constexpr int64_t kFfnFusedMinRows = 256 * 74;

cudaError_t launch_ffn_fused(const FfnShape& s, const void* x, const FfnWeights& w, void* y, uint32_t* status,
                             cudaStream_t st);

}  // namespace msc
