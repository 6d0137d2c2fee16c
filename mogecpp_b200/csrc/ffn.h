// Gated feed-forward block over the channels of each row (ffn.cu):
//   g = x Wg^T + bg;  u = x Wu^T + bu;  y = (act(g) * u) Wd^T + bd
// and its backward pass.
#pragma once

#include <cstddef>
#include <cstdint>
#include <cuda_runtime.h>

namespace msc {

enum FfnAct : int { ACT_SILU = 0, ACT_GELU = 1, ACT_GELU_ERF = 2 };

struct FfnWeights {
    const void* w_gate;  // [hidden][c]
    const void* w_up;    // [hidden][c]
    const void* w_down;  // [c][hidden]
    const float* b_gate;  // [hidden] or NULL
    const float* b_up;
    const float* b_down;  // [c] or NULL
};

struct FfnShape {
    int64_t n;
    int c, hidden;
    int dtype;  // DT_F16 or DT_BF16: x, weights, y and their gradients
    int act;
};

struct FfnGrads {
    void* dx;      // [n][c] or NULL
    void* w_gate;  // as the weights, or NULL (all three together)
    void* w_up;
    void* w_down;
    float* b_gate;
    float* b_up;
    float* b_down;
};

size_t ffn_workspace_bytes(int64_t n, int c, int hidden);
// Enough for every block of at most `hidden` hidden units (the size itself
// shrinks here and there as hidden grows: fewer K splits, or another path).
size_t ffn_workspace_bound(int64_t n, int c, int hidden);
cudaError_t launch_ffn(const FfnShape& s, const void* x, const FfnWeights& w, void* y, void* ws, uint32_t* status,
                       cudaStream_t st);
size_t ffn_backward_workspace_bytes(int64_t n, int c, int hidden);
cudaError_t launch_ffn_backward(const FfnShape& s, const void* x, const void* dy, const FfnWeights& w,
                                const FfnGrads& g, void* ws, uint32_t* status, cudaStream_t st);

}  // namespace msc
