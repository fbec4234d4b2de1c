// block_norm.cuh -- launcher interface of the block-tail norm (block_norm.cu).
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

namespace z2 {

struct BlockNormArgs {
    const void *resid;        // [rows] of resid_stride elements
    const void *block;        // [rows] of block_stride elements
    long long resid_stride, block_stride;
    int rows, dim;
    float rcp_dim;            // 1 / dim
    int post_norm;            // normalise the block's output first
    const float *post_weight; // [dim] or nullptr
    float post_eps;
    const void *gate;         // element (r, d) at r * gate_row_stride + d * gate_col_stride, or nullptr
    long long gate_row_stride;
    int gate_col_stride;      // 0 or 1
    int gate_sigmoid;
    float scale;
    const float *norm_weight; // [dim] or nullptr
    float norm_eps;
    void *resid_out;          // [rows] of out_stride elements, or nullptr
    void *normed_out;         // the same, or nullptr
    long long out_stride;
};

// Elements are bf16 when `bf16`, else f32.
cudaError_t launch_block_norm(const BlockNormArgs &a, bool bf16, cudaStream_t stream);

}  // namespace z2
