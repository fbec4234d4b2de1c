// head_i8.cu -- the output head in 8-bit integers (sm_100a).
#include <cuda_bf16.h>
#include <math.h>

#include "common.cuh"
#include "head_i8.cuh"
#include "tc.cuh"

namespace z2 {

int read_and_clear_head_i8_error(int *value) { return take_device_error(value); }

namespace {

__device__ __forceinline__ float value_of(float v) { return v; }
__device__ __forceinline__ float value_of(__nv_bfloat16 v) { return __bfloat162float(v); }

template <typename T>
__global__ void __launch_bounds__(256)
    quantize_kernel(const T *x, int dim, long long stride, int8_t *q, float *scale)
{
    __shared__ float s_part[8];
    const T *row = x + blockIdx.x * stride;
    float most = 0.0f;
    bool odd = false;
    for (int i = threadIdx.x; i < dim; i += 256) {
        const float v = fabsf(value_of(row[i]));
        odd |= !(v <= 3.402823466e38f);
        most = fmaxf(most, v);
    }
    for (int d = 16; d >= 1; d >>= 1) most = fmaxf(most, __shfl_xor_sync(kFull, most, d));
    if ((threadIdx.x & 31) == 0) s_part[threadIdx.x >> 5] = most;
    odd = __syncthreads_or(odd);
    for (int i = 0; i < 8; i++) most = fmaxf(most, s_part[i]);
    if (threadIdx.x == 0) scale[blockIdx.x] = odd ? __int_as_float(0x7fc00000) : most / 127.0f;
    for (int i = threadIdx.x; i < dim; i += 256)
        q[(long long)blockIdx.x * dim + i] =
            odd || most == 0.0f ? 0 : (int8_t)(int)rint(127.0 * (double)value_of(row[i]) / (double)most);
}

__global__ void __launch_bounds__(128) head_i8_any_kernel(const HeadI8Args a, const int8_t *q, const float *scale)
{
    const int lane = threadIdx.x & 31, wide = a.n_cb * a.vocab;
    const long long item = ((long long)blockIdx.x * 128 + threadIdx.x) >> 5;
    const int b = (int)(item / wide), n = (int)(item % wide);
    if (item / wide >= a.batch) return;
    const long long w = (long long)(n / a.vocab) * a.rows_per_cb + n % a.vocab;
    int sum = 0;
    for (int i = lane * 4; i < a.dim; i += 128)
        sum = __dp4a(*(const int *)(a.W + w * a.dim + i), *(const int *)(q + (long long)b * a.dim + i), sum);
    for (int d = 16; d >= 1; d >>= 1) sum += __shfl_xor_sync(kFull, sum, d);
    const float y = (float)sum * scale[b] * a.w_scale[w];
    if (lane == 0) a.out[(long long)b * wide + n] = a.softcap > 0.0f ? a.softcap * tanhf(y / a.softcap) : y;
}

}  // namespace

cudaError_t launch_quantize_rows(const void *x, bool bf16, int rows, int dim, long long stride,
                                 int8_t *q, float *scale, cudaStream_t stream)
{
    if (bf16)
        quantize_kernel<<<rows, 256, 0, stream>>>((const __nv_bfloat16 *)x, dim, stride, q, scale);
    else
        quantize_kernel<<<rows, 256, 0, stream>>>((const float *)x, dim, stride, q, scale);
    return cudaGetLastError();
}

cudaError_t launch_head_i8(const HeadI8Args &a, bool bf16, cudaStream_t stream)
{
    int8_t *q = (int8_t *)a.work;
    float *scale = (float *)((char *)a.work + (((long long)a.batch * a.dim + 15) & ~15ll));
    const cudaError_t e = launch_quantize_rows(a.hidden, bf16, a.batch, a.dim, a.dim, q, scale, stream);
    if (e != cudaSuccess) return e;
    const long long items = (long long)a.batch * a.n_cb * a.vocab;
    head_i8_any_kernel<<<(unsigned)((items + 3) / 4), 128, 0, stream>>>(a, q, scale);
    return cudaGetLastError();
}

}  // namespace z2
