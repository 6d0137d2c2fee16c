// Gated feed-forward block of a few rows (ffn_rows.cu).
#pragma once

#include "ffn.h"

namespace msc {

// At most this many rows run as dot products over the weights.
constexpr int kFfnFewRows = 8;

// h: fp32 scratch [n][hidden].
cudaError_t launch_ffn_rows(const FfnShape& s, const void* x, const FfnWeights& w, void* y, float* h, cudaStream_t st);

}  // namespace msc
