// verify.cuh -- launcher interface of the draft verification (verify.cu).
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

namespace z2 {

struct VerifyArgs {
    const float *logits;      // row (s, d, c) at ((s * (n_draft + 1) + d) * n_cb + c) * row_stride
    long long row_stride;
    int n_streams, n_draft, n_cb, vocab;
    float temperature, top_p, min_p, rho, inv_rho;
    double inv_temp;
    float log2_scale;         // log2(e) / temperature
    int top_k, pad_id;
    const int32_t *drafts;    // [n_streams][n_draft][n_cb]
    const float *probs;       // [n_streams][n_draft][n_cb][vocab] or nullptr: drafts are certain
    const int32_t *n_drafts;  // [n_streams] or nullptr: n_draft everywhere
    const float *uniforms;    // [n_streams][n_draft + 1][n_cb][2]: test, draw
    int32_t *hist;            // [n_streams][n_cb][hist_len] or nullptr
    int hist_len;
    int32_t *hist_pos;        // [n_streams]
    const uint32_t *allow;    // [n_streams][ceil(vocab / 32)] or nullptr
    int delay_step;
    int32_t *codes;           // [n_streams][n_draft + 1][n_cb]
    int32_t *n_accepted;      // [n_streams]
    int32_t *flags;           // as codes, or nullptr
    int vec_logits;           // rows 16-byte aligned and vocab % 4 == 0
};

cudaError_t launch_verify(const VerifyArgs &a, cudaStream_t stream);

}  // namespace z2
