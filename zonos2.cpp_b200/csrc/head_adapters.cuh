// head_adapters.cuh -- launcher interface of the output head with low-rank
// adapters (head_adapters.cu).
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

#include "head.cuh"

namespace z2 {

struct AdapterArgs {
    const void *A;         // [n_adapters][rank][dim]
    const void *B;         // [n_adapters][n_cb * rows_per_cb][rank]
    const float *scale;    // [n_adapters] or nullptr (1)
    int n_adapters, rank;
    const int32_t *which;  // hidden row b's adapter is which[b / rows_per_id]; outside
                           // [0, n_adapters): none
    int rows_per_id;       // 1, or 2 for guidance pairs
    void *work;            // adapter_work_bytes() bytes, 16-byte aligned
    float *delta = nullptr;  // [batch][n_cb * vocab] scratch of a bf16 head with guidance; else
                             // the logits' buffer serves
};

// Bytes of AdapterArgs::work: scale * A h per hidden row, f64 for an f32 head, f32 for
// a bf16 one, and an order of the rows.
size_t adapter_work_bytes(bool bf16, int batch, int rank);

// The tcgen05 kernel (head_adapters_tc.cu), for bf16; cudaErrorNotSupported for the
// sizes and alignments it does not take.
cudaError_t launch_head_adapters_tc(const HeadArgs &h, const AdapterArgs &ad, cudaStream_t stream);

// Reads and clears the device error word of its bounded waits.
int read_and_clear_adapter_error(int *value);

// HeadArgs with adapters: everything of `dtype` bf16 or f32.
cudaError_t launch_head_adapters(const HeadArgs &h, const AdapterArgs &ad, bool bf16,
                                 cudaStream_t stream);

}  // namespace z2
