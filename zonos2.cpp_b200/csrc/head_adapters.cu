// head_adapters.cu -- the output head beside low-rank adapters of many requests
// (sm_100a):
//
//     t[b]         = s_a * (A_a h[b])                       a = the row's adapter
//     logits[b, n] = softcap(W[n] . h[b] + B_a[n] . t[b])   n = (codebook, token)
//
// for hidden rows that each name one of n_adapters adapters, or none.  t is kept
// in f32 (f64 beside an f32 head): rounding it to bf16 would put 2^-9 of the
// adapter's contribution into f32 logits.
//
// A bf16 head runs on the tensor cores (head_adapters_tc.cu) where its sizes and
// alignment allow.  Here: adapter_down_kernel makes t, and adapter_any_kernel, one
// warp per weight row, takes every size and type.
#include <cuda_bf16.h>
#include <math.h>

#include "common.cuh"
#include "head_adapters.cuh"

namespace z2 {

namespace {

constexpr int kWarps = 8;

__device__ __forceinline__ float load_f(const float *p) { return __ldg(p); }
__device__ __forceinline__ float load_f(const __nv_bfloat16 *p) { return __bfloat162float(*p); }

template <typename T>
struct Acc {   // the accumulator beside an operand type
    using type = float;
};
template <>
struct Acc<float> {
    using type = double;
};

// t[b][r], one warp per element.
template <typename T>
__global__ void __launch_bounds__(32 * kWarps)
    adapter_down_kernel(const HeadArgs h, const AdapterArgs ad)
{
    using S = typename Acc<T>::type;
    const int lane = threadIdx.x & 31;
    const long long i = (long long)blockIdx.x * kWarps + (threadIdx.x >> 5);
    if (i >= (long long)h.batch * ad.rank) return;
    const int b = (int)(i / ad.rank), r = (int)(i % ad.rank);
    const int a = ad.which[b / ad.rows_per_id];
    if ((unsigned)a >= (unsigned)ad.n_adapters) return;
    const T *x = static_cast<const T *>(h.hidden) + (size_t)b * h.dim;
    const T *w = static_cast<const T *>(ad.A) + ((size_t)a * ad.rank + r) * h.dim;
    S acc = 0;
    for (int d = lane; d < h.dim; d += 32) acc += (S)load_f(x + d) * (S)load_f(w + d);
#pragma unroll
    for (int o = 16; o; o >>= 1) acc += __shfl_xor_sync(kFull, acc, o);
    if (lane == 0) static_cast<S *>(ad.work)[i] = acc * (S)(ad.scale ? __ldg(ad.scale + a) : 1.0f);
}

// The logits, one warp per weight row.
template <typename T>
__global__ void __launch_bounds__(32 * kWarps)
    adapter_any_kernel(const HeadArgs h, const AdapterArgs ad)
{
    using S = typename Acc<T>::type;
    const int lane = threadIdx.x & 31;
    const int o = blockIdx.x * kWarps + (threadIdx.x >> 5);
    if (o >= h.n_cb * h.vocab) return;
    const int c = o / h.vocab, v = o - c * h.vocab;
    const size_t n = (size_t)c * h.rows_per_cb + v;
    const T *w = static_cast<const T *>(h.W) + n * h.dim;
    float cond = 0.0f;   // with guidance: the logit of the pair's conditional row
    for (int b = 0; b < h.batch; b++) {
        const T *x = static_cast<const T *>(h.hidden) + (size_t)b * h.dim;
        S acc = 0;
        for (int d = lane; d < h.dim; d += 32) acc += (S)load_f(w + d) * (S)load_f(x + d);
        const int a = ad.which[b / ad.rows_per_id];
        if ((unsigned)a < (unsigned)ad.n_adapters) {
            const T *up = static_cast<const T *>(ad.B) +
                          ((size_t)a * h.n_cb * h.rows_per_cb + n) * ad.rank;
            const S *t = static_cast<const S *>(ad.work) + (size_t)b * ad.rank;
            for (int r = lane; r < ad.rank; r += 32) acc += (S)load_f(up + r) * t[r];
        }
#pragma unroll
        for (int s = 16; s; s >>= 1) acc += __shfl_xor_sync(kFull, acc, s);
        if (lane == 0) {
            float l = (float)acc;
            if (h.row_scale) l *= __ldg(h.row_scale + b);
            if (h.softcap > 0.0f) l = h.softcap * tanhf(l / h.softcap);
            if (!h.cfg) {
                h.out[((size_t)b * h.n_cb + c) * h.vocab + v] = l;
            } else if ((b & 1) == 0) {
                cond = l;
            } else {
                h.out[((size_t)(b >> 1) * h.n_cb + c) * h.vocab + v] =
                    __fadd_rn(l, __fmul_rn(h.cfg_scale, __fsub_rn(cond, l)));
            }
        }
    }
}

template <typename T>
cudaError_t launch_any(const HeadArgs &h, const AdapterArgs &ad, cudaStream_t stream)
{
    const long long down = (long long)h.batch * ad.rank;
    adapter_down_kernel<T><<<(unsigned)((down + kWarps - 1) / kWarps), 32 * kWarps, 0, stream>>>(h, ad);
    cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) return e;
    const int rows = h.n_cb * h.vocab;
    adapter_any_kernel<T><<<(unsigned)((rows + kWarps - 1) / kWarps), 32 * kWarps, 0, stream>>>(h, ad);
    return cudaGetLastError();
}

}  // namespace

size_t adapter_work_bytes(bool bf16, int batch, int rank)
{
    const size_t t = (size_t)batch * (size_t)rank;
    // beside t (a multiple of 8 ranks), the tensor-core path keeps the rows' order and its
    // items: batch + 3 words, and two for each of at most batch / 8 + batch items
    const size_t b = (size_t)batch;
    return !bf16 ? 8 * t : rank % 8 == 0 ? 4 * (t + b + 3 + 2 * (b / 8 + b)) : 4 * t;
}

cudaError_t launch_head_adapters(const HeadArgs &h, const AdapterArgs &ad, bool bf16,
                                 cudaStream_t stream)
{
    if (h.batch == 0) return cudaSuccess;
    if (!bf16) return launch_any<float>(h, ad, stream);
    const cudaError_t e = launch_head_adapters_tc(h, ad, stream);
    return e == cudaErrorNotSupported ? launch_any<__nv_bfloat16>(h, ad, stream) : e;
}

}  // namespace z2
