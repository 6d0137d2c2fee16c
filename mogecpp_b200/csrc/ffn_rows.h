// Gated feed-forward block of a few rows (ffn_rows.cu).
#pragma once

#include "ffn.h"

namespace msc {

// A few rows run as dot products over the weights: up to 4, and up to 8 where
// the weights are small.  A row more costs the CUDA cores its products, the
// tensor-core path nothing, but that takes longer to start.  Measured (bf16,
// us, dot products / tensor cores): 1024 -> 4096, 4 rows 15.6 / 19.1, 8 rows
// 24.4 / 18.8; 128 -> 512, 8 rows 6.6 / 11.5.
constexpr int64_t kFewRowsWork = int64_t(1) << 24;
inline bool ffn_few_rows(int64_t n, int c, int hidden) {
    return n <= 4 || (n <= 8 && n * c * hidden <= kFewRowsWork);
}

// h: fp32 scratch [n][hidden].
cudaError_t launch_ffn_rows(const FfnShape& s, const void* x, const FfnWeights& w, void* y, float* h, cudaStream_t st);

}  // namespace msc
