// head_i8.cuh -- launcher interface of the 8-bit head (head_i8.cu).
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

namespace z2 {

struct HeadI8Args {
    const int8_t *W;        // [n_cb*rows_per_cb][dim]
    const float *w_scale;   // [n_cb*rows_per_cb]
    int rows_per_cb, n_cb, vocab, dim;
    const void *hidden;     // [batch][dim]
    int batch;
    float softcap;          // <= 0: no cap
    void *work;             // head_i8_work_bytes
    float *out;             // [batch][n_cb][vocab]
};

// The rounded hidden rows, and their scales behind them, in whole steps of the epilogue's 16.
inline long long head_i8_work_bytes(int batch, int dim)
{
    return (((long long)batch * dim + 15) & ~15ll) + 4ll * ((batch + 15ll) & ~15ll);
}

cudaError_t launch_quantize_rows(const void *x, bool bf16, int rows, int dim, long long stride,
                                 int8_t *q, float *scale, cudaStream_t stream);
cudaError_t launch_head_i8(const HeadI8Args &a, bool bf16, cudaStream_t stream);

// Reads and clears the device error word of the tensor-core kernel's bounded waits.
int read_and_clear_head_i8_error(int *value);

}  // namespace z2
