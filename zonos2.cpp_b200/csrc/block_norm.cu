// block_norm.cu -- the tail of a decoder block (sm_100a): the norm of the
// block's output, its gate, the scaled residual sum and the RMSNorm that
// follows it (the next block's, or the output norm ahead of the head), in one
// pass over the row:
//
//     y = block * w_post / rms(block)          (post_norm; else y = block)
//     r = resid + scale * g * y                (g = gate, or sigmoid(gate), or 1)
//     n = r * w_norm / rms(r),   rms(x) = sqrt(mean(x^2) + eps)
//
// r and n are computed in f32 and rounded once, each on its own store: n is
// taken from the unrounded r, so a bf16 residual stream costs n no second
// rounding.  The sums of squares are f32: every thread's partial sum has at most
// 32 terms and the rest is a tree, so their error is a few ulp.
//
// Bound: memory.  A row is read once (residual, block output, gate) and written
// twice; it stays in registers between its two reductions.
#include <cuda_bf16.h>
#include <math.h>

#include "block_norm.cuh"
#include "common.cuh"

namespace z2 {

namespace {

template <typename T>
__device__ __forceinline__ float to_f(T v);
template <>
__device__ __forceinline__ float to_f<float>(float v) { return v; }
template <>
__device__ __forceinline__ float to_f<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T>
__device__ __forceinline__ T from_f(float v);
template <>
__device__ __forceinline__ float from_f<float>(float v) { return v; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

__device__ __forceinline__ float sigmoid(float g) { return __frcp_rn(1.0f + expf(-g)); }

// The sum over the block's threads, in every thread.  `part` holds one float per warp.
__device__ __forceinline__ float block_sum(float v, float *part)
{
#pragma unroll
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(kFull, v, o);
    const int warps = blockDim.x >> 5;
    if (warps == 1) return v;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    if (lane == 0) part[warp] = v;
    __syncthreads();
    v = lane < warps ? part[lane] : 0.0f;
#pragma unroll
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(kFull, v, o);
    return v;
}

__device__ __forceinline__ float rcp_rms(float ss, int dim, float eps)
{
    return __fdiv_rn(1.0f, sqrtf(__fdiv_rn(ss, (float)dim) + eps));
}

// One block per row, elements one by one, the row re-read (from L1 or L2) by
// each of its reductions: any size, stride and alignment.
template <typename T>
__global__ void __launch_bounds__(1024) block_norm_any_kernel(const BlockNormArgs a)
{
    __shared__ float part[2][32];
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const size_t row = blockIdx.x;
    const T *x = static_cast<const T *>(a.resid) + row * a.resid_stride;
    const T *y = static_cast<const T *>(a.block) + row * a.block_stride;
    const T *g = a.gate ? static_cast<const T *>(a.gate) + row * a.gate_row_stride : nullptr;
    float rcp = 1.0f;
    if (a.post_norm) {
        float ss = 0.0f;
        for (int d = threadIdx.x; d < a.dim; d += blockDim.x) {
            const float v = to_f<T>(y[d]);
            ss = fmaf(v, v, ss);
        }
        rcp = rcp_rms(block_sum(ss, part[0]), a.dim, a.post_eps);
    }
    auto sum_at = [&](int d) {
        float v = to_f<T>(y[d]);
        if (a.post_norm) v = v * rcp * (a.post_weight ? a.post_weight[d] : 1.0f);
        if (g) {
            const float t = to_f<T>(g[(size_t)d * a.gate_col_stride]);
            v *= a.gate_sigmoid ? sigmoid(t) : t;
        }
        return fmaf(a.scale, v, to_f<T>(x[d]));
    };
    float rcp2 = 1.0f;
    if (a.normed_out) {
        float ss = 0.0f;
        for (int d = threadIdx.x; d < a.dim; d += blockDim.x) {
            const float v = sum_at(d);
            ss = fmaf(v, v, ss);
        }
        rcp2 = rcp_rms(block_sum(ss, part[1]), a.dim, a.norm_eps);
    }
    T *ro = a.resid_out ? static_cast<T *>(a.resid_out) + row * a.out_stride : nullptr;
    T *no = a.normed_out ? static_cast<T *>(a.normed_out) + row * a.out_stride : nullptr;
    for (int d = threadIdx.x; d < a.dim; d += blockDim.x) {
        const float v = sum_at(d);
        if (no) no[d] = from_f<T>(v * rcp2 * (a.norm_weight ? a.norm_weight[d] : 1.0f));
        if (ro) ro[d] = from_f<T>(v);
    }
}

template <class Kernel>
cudaError_t launch(Kernel kernel, int grid, int threads, const BlockNormArgs &a, cudaStream_t stream)
{
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)grid);
    cfg.blockDim = dim3((unsigned)threads);
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kernel, a);
}

}  // namespace

cudaError_t launch_block_norm(const BlockNormArgs &a, bool bf16, cudaStream_t stream)
{
    if (a.rows == 0) return cudaSuccess;
    int threads = 32;
    while (threads < 1024 && threads * 4 < a.dim) threads *= 2;
    return bf16 ? launch(block_norm_any_kernel<__nv_bfloat16>, a.rows, threads, a, stream)
                : launch(block_norm_any_kernel<float>, a.rows, threads, a, stream);
}

}  // namespace z2
