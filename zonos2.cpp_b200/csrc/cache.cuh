// cache.cuh -- launcher interface of the paged cache's kernels (cache_append.cu,
// cache_attend.cu, cache_attend_tc.cu), and what they share on the device.
#pragma once

#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "common.cuh"

namespace z2 {

struct CacheArgs {
    void *k, *v;            // pages of [n_kv][page][dim], page_stride elements apart
    int n_pages, page_shift, n_kv, dim;   // a page holds 1 << page_shift tokens
    long long page_stride;
    const int32_t *table;   // [n_streams][max_pages]
    int n_streams, max_pages;
    const int32_t *kv_len;  // [n_streams]
    const int32_t *q_start; // [n_streams + 1]
    int rows;               // token rows of the call's buffers
};

struct AppendArgs {
    const void *q, *k, *v;  // q may be nullptr
    long long q_stride, k_stride, v_stride;
    int n_heads;
    const float *q_weight, *k_weight;   // [dim] or nullptr
    int norm;
    float eps;
    const float *freq;      // [rot / 2]
    int rot, halves;
    void *q_out;
    long long q_out_stride;
};

struct AttendArgs {
    const void *q;
    long long q_stride;
    int n_heads, group;     // query heads, and those of one key head
    float scale;
    int window;             // <= 0: none
    const void *gate;       // element (row, head) at row * gate_stride + head, or nullptr
    long long gate_stride;
    int max_new;            // a hint (<= 0: none)
    void *out;
    long long out_stride;
};

cudaError_t launch_cache_append(const CacheArgs &c, const AppendArgs &a, bool bf16, cudaStream_t stream);
cudaError_t launch_cache_attend(const CacheArgs &c, const AttendArgs &a, bool bf16, cudaStream_t stream);

namespace {

// (The device arrays are read by plain loads: under programmatic dependent launch a kernel may have
// started while the one before it still wrote them, which read-only loads do not allow for.)

// One stream's part of a call: its token rows and where they stand.  Whatever the device
// arrays hold, rows stay inside the call's buffers and len is not negative.
struct Chunk {
    int first, n;    // token rows [first, first + n)
    int len;         // tokens of the stream
    int stream;
};

__device__ __forceinline__ Chunk chunk_of(const CacheArgs &c, int s)
{
    Chunk k;
    k.stream = s;
    k.first = min(max(c.q_start[s], 0), c.rows);
    k.n = min(max(c.q_start[s + 1], k.first), c.rows) - k.first;
    k.len = max(c.kv_len[s], 0);
    return k;
}

// Tokens of a stream that its table has room for (and positions, to a step past the last, room in
// 32 bits).
constexpr int kMostTokens = 0x7fffff00;

__device__ __forceinline__ int room_of(const CacheArgs &c)
{
    const long long room = (long long)c.max_pages << c.page_shift;
    return room > kMostTokens ? kMostTokens : (int)room;
}

// The page of a stream's token j (0 <= j < room), or -1 where there is none.
__device__ __forceinline__ int page_of(const CacheArgs &c, int s, int j)
{
    const int p = c.table[(long long)s * c.max_pages + (j >> c.page_shift)];
    return p >= 0 && p < c.n_pages ? p : -1;
}

// Element offset of token j's row for key head h on page p.
__device__ __forceinline__ long long row_on_page(const CacheArgs &c, int p, int h, int j)
{
    const int slot = j & ((1 << c.page_shift) - 1);
    return (long long)p * c.page_stride + (((long long)h << c.page_shift) + slot) * c.dim;
}

__device__ __forceinline__ float as_f(float v) { return v; }
__device__ __forceinline__ float as_f(__nv_bfloat16 v) { return __bfloat162float(v); }

}  // namespace

}  // namespace z2
