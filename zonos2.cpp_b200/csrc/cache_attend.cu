// cache_attend.cu -- attention of new tokens over a paged cache (sm_100a).
//
// One warp per (token row, query head): a pass over the keys it sees with the softmax's running
// maximum and sum.
#include <math.h>

#include "cache.cuh"

namespace z2 {

namespace {

template <typename T>
__global__ void __launch_bounds__(128) attend_any_kernel(const CacheArgs c, const AttendArgs a)
{
    const int lane = threadIdx.x & 31;
    const long long item = ((long long)blockIdx.x * 128 + threadIdx.x) >> 5;
    const int row = (int)(item / a.n_heads), h = (int)(item % a.n_heads);
    if (item / a.n_heads >= c.rows) return;
    int s = -1;
    for (int i = 0; i < c.n_streams; i++)
        if (__ldg(c.q_start + i) <= row) s = i;
    if (s < 0) return;
    const Chunk ch = chunk_of(c, s);
    if (row < ch.first || row >= ch.first + ch.n) return;
    const int pos = ch.len - ch.n + (row - ch.first);
    float q[8], o[8], m = -INFINITY, l = 0.0f;
    for (int i = 0; i < 8; i++) {
        const int e = lane + 32 * i;
        q[i] = e < c.dim ? as_f(((const T *)a.q)[row * a.q_stride + (long long)h * c.dim + e]) : 0.0f;
        o[i] = 0.0f;
    }
    const int end = min(pos + 1, room_of(c));
    for (int j = a.window > 0 ? max(0, pos - a.window + 1) : 0; j < end; j++) {
        const int p = page_of(c, s, j);
        if (p < 0) continue;
        const long long at = row_on_page(c, p, h / a.group, j);
        float x = 0.0f;
        for (int i = 0; i < 8; i++)
            if (lane + 32 * i < c.dim) x += q[i] * as_f(((const T *)c.k)[at + lane + 32 * i]);
        for (int d = 16; d >= 1; d >>= 1) x += __shfl_xor_sync(kFull, x, d);
        x *= a.scale;
        const float top = fmaxf(m, x), keep = m == -INFINITY ? 0.0f : expf(m - top), w = expf(x - top);
        m = top;
        l = l * keep + w;
        for (int i = 0; i < 8; i++)
            if (lane + 32 * i < c.dim)
                o[i] = o[i] * keep + w * as_f(((const T *)c.v)[at + lane + 32 * i]);
    }
    float g = 1.0f;
    if (a.gate) g = 1.0f / (1.0f + expf(-as_f(((const T *)a.gate)[row * a.gate_stride + h])));
    for (int i = 0; i < 8; i++) {
        const int e = lane + 32 * i;
        if (e < c.dim)
            ((T *)a.out)[row * a.out_stride + (long long)h * c.dim + e] = (T)(l == 0.0f ? 0.0f : g * o[i] / l);
    }
}

}  // namespace

cudaError_t launch_cache_attend(const CacheArgs &c, const AttendArgs &a, bool bf16, cudaStream_t stream)
{
    const long long blocks = ((long long)c.rows * a.n_heads + 3) / 4;
    if (bf16)
        attend_any_kernel<__nv_bfloat16><<<(unsigned)blocks, 128, 0, stream>>>(c, a);
    else
        attend_any_kernel<float><<<(unsigned)blocks, 128, 0, stream>>>(c, a);
    return cudaGetLastError();
}

}  // namespace z2
