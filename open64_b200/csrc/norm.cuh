// Host-side interface of the RMS-norm kernels (norm.cu).
#pragma once
#include <cstddef>
#include <cstdint>
#include <cuda_runtime.h>

#include "../../include/o64gemm.h"

namespace o64 {

constexpr int64_t kNormMaxCols = 32768;  // one row lives in the registers of at most 512 threads

struct NormCall {
    int64_t T, N;
    const void *X;
    int64_t ldx;
    const void *R;  // NULL: no residual
    int64_t ldr;
    void *S;  // x + r as bf16; NULL: not wanted
    int64_t lds;
    const void *W;
    bool w_f32;
    float eps;
    int out_kind;
    bool row_scale;  // e4m3: one scale per row instead of one per 128 columns
    void *Y;
    int64_t ldy;
    float *scales;
    int64_t ldscales;
    float *rstd;  // may be NULL
    int *status;
    unsigned long long wait_ns;
    cudaStream_t stream;
};
int norm_forward(const NormCall &c, int num_sms);

struct NormBackwardCall {
    int64_t T, N;
    const void *dY;
    int64_t lddy;
    const void *S;
    int64_t lds;
    const void *W;
    bool w_f32;
    const float *rstd;
    const void *dR;  // NULL: nothing arrives on the residual
    int64_t lddr;
    void *dX;
    int64_t lddx;
    float *dW;  // NULL: not wanted
    float *workspace;
    int *status;
    unsigned long long wait_ns;
    cudaStream_t stream;
};
// Rows of partial sums of dW (each N floats) that norm_backward leaves in the workspace.
int64_t norm_backward_partials(int64_t T, int64_t N);
int norm_backward(const NormBackwardCall &c, int num_sms);

}  // namespace o64
