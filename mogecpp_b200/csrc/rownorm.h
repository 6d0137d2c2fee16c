// Fused residual norms over the channels of each row (rownorm.cu):
//   t = Norm_post(f);  r = s x + gate * t;  h = Norm_pre(r)
// and their backward pass.
#pragma once

#include <cstdint>
#include <cuda_runtime.h>

namespace msc {

enum NormKind : int { NORM_NONE = 0, NORM_LAYER = 1, NORM_RMS = 2 };

struct NormParams {
    int kind;
    const float* w;  // [c] or NULL (ones)
    const float* b;  // [c] or NULL (zeros)
    float eps;
};

struct RowNormArgs {
    int64_t n;
    int c;
    int x_dtype, f_dtype;  // residual stream (x, r, dr, dx), branch (f, h, dh, df)
    NormParams post, pre;
    const float* gate;     // NULL: ones
    int nsamples;          // 0: gate [c]; else gate [nsamples][c], sample = coords[row][3]
    const int32_t* coords;
    float res_scale;
    uint32_t* status;
    // forward
    const void* x;
    const void* f;
    void* r;
    void* h;
    // backward (x is r)
    const void* dr;
    const void* dh;
    void* dx;
    void* df;
    float* partial;  // [units][4 + gate rows][c]
    int64_t units, rows_per_unit;
    int slab_clear;  // slab rows that start at zero (the others go on)
};

struct RowNormGrads {
    float* gate;
    float* post_w;
    float* post_b;
    float* pre_w;
    float* pre_b;
};

constexpr int kRowNormMaxC = 8192;
constexpr int kRowNormMaxSamples = 1 << 15;

bool rownorm_dtypes_supported(int x_dtype, int f_dtype);
cudaError_t launch_rownorm(const RowNormArgs& a, cudaStream_t st);
size_t rownorm_backward_workspace_bytes(int64_t n, int c, int nsamples);
cudaError_t launch_rownorm_backward(RowNormArgs a, const RowNormGrads& g, void* ws, cudaStream_t st);

}  // namespace msc
