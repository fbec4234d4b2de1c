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
// rounding.  The sums of squares are f32: 8 terms in a thread of block_norm_kernel,
// the rest a tree, so their error is a few ulp.
//
// Bound: memory.  A row is read once (residual, block output, gate) and written
// twice; it stays in registers between its two reductions.  16384 bf16 rows of 2048 with a
// full sigmoid gate (336 MB): 59 us, 5.7 TB/s; 297 us by block_norm_any_kernel, which
// re-reads the row and works element by element (now rows past 8192).  The issue slots come next: with
// full-precision divisions and exponentials everywhere the same bytes took 83 us, so the
// reciprocal root, the sigmoid and the join of a row's partial sums are kept short.
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

// 1 / (1 + exp(-g)), 1 + exp(-g) being 1 at least and perhaps infinite.  A bf16 gate takes the
// exponential as a power of two: rounding g log2(e) costs |g| 2^-24 of it, less than
// a hundredth of a bf16 step for any g whose sigmoid is not lost in the sum.
template <typename T>
__device__ __forceinline__ float sigmoid(float g)
{
    float e, r;
    if (sizeof(T) == 2)
        asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(g * -1.44269504f));
    else
        e = expf(-g);
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.0f + e));
    return r;
}

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

// rsqrtf is off by 2 ulp at most.
__device__ __forceinline__ float rcp_rms(float ss, const BlockNormArgs &a, float eps)
{
    return rsqrtf(fmaf(ss, a.rcp_dim, eps));
}

// 16 bytes of a row.  Not the read-only path: the sums may go back to where the row was.
__device__ __forceinline__ uint4 load16(const void *p)
{
    uint4 u;
    asm volatile("ld.global.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];"
                 : "=r"(u.x), "=r"(u.y), "=r"(u.z), "=r"(u.w) : "l"(p) : "memory");
    return u;
}

template <typename T>
constexpr int kVec = 16 / (int)sizeof(T);   // elements of a 16-byte vector

__device__ __forceinline__ void widen(const uint4 &u, float (&f)[4])
{
    f[0] = __uint_as_float(u.x), f[1] = __uint_as_float(u.y), f[2] = __uint_as_float(u.z), f[3] = __uint_as_float(u.w);
}
__device__ __forceinline__ void widen(const uint4 &u, float (&f)[8])
{
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; i++) f[2 * i] = __uint_as_float(w[i] << 16), f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
}
__device__ __forceinline__ uint4 narrow(const float (&f)[4])
{
    return make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
}
__device__ __forceinline__ uint4 narrow(const float (&f)[8])
{
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; i++)
        asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(w[i]) : "f"(f[2 * i + 1]), "f"(f[2 * i]));
    return make_uint4(w[0], w[1], w[2], w[3]);
}

// The sum over a row's threads, in each of them; blockDim.x / 32 warps make a row, and
// threadIdx.y is the row within the block.  One barrier, the block's: the partial sums
// alternate between two buffers.
struct RowSum {
    float4 (*part)[8];
    int warps, first, warp, lane, buf;

    __device__ __forceinline__ RowSum(float4 (*p)[8]) : part(p), buf(0)
    {
        warps = blockDim.x >> 5;
        lane = threadIdx.x & 31;
        first = threadIdx.y * ((warps + 3) >> 2);
        warp = 4 * first + (threadIdx.x >> 5);
        if (threadIdx.y == 0 && threadIdx.x < 32) reinterpret_cast<float2 *>(part)[lane] = make_float2(0.0f, 0.0f);
        __syncthreads();   // places past a row's warps stay zero
    }
    __device__ __forceinline__ float operator()(float v)
    {
#pragma unroll
        for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(kFull, v, o);
        if (warps == 1) return v;
        if (lane == 0) reinterpret_cast<float *>(part[buf])[warp] = v;
        __syncthreads();
        v = 0.0f;
        for (int i = 0; i < warps; i += 4) {
            const float4 p = part[buf][first + (i >> 2)];
            v += (p.x + p.y) + (p.z + p.w);
        }
        buf ^= 1;
        return v;
    }
};

// A vector of 16 bytes per thread.  A block walks over rows a grid apart, so that its weights
// are loaded once, into registers, and the next row's loads are under way while this one is
// reduced.
template <typename T>
__global__ void __launch_bounds__(1024) block_norm_kernel(const BlockNormArgs a)
{
    constexpr int V = kVec<T>;
    __shared__ float4 part[2][8];
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    RowSum row_sum(part);
    const int d = threadIdx.x * V;
    const bool in_row = d < a.dim;
    const bool by_row = a.gate && !a.gate_col_stride, by_elem = a.gate && a.gate_col_stride;
    const uint32_t step = gridDim.x * blockDim.y, rows = a.rows;   // the sums below stay under 2^32
    const uint32_t rs = a.resid_stride, bs = a.block_stride, gs = a.gate_row_stride, os = a.out_stride;
    uint32_t row = blockIdx.x * blockDim.y + threadIdx.y;
    uint4 x, y, g;
    float g_row = 1.0f;
    auto fetch = [&](uint32_t r) {
        x = y = g = make_uint4(0, 0, 0, 0);
        if (r >= rows) return;
        if (in_row) {
            y = load16(static_cast<const T *>(a.block) + (size_t)r * bs + d);
            if (by_elem) g = load16(static_cast<const T *>(a.gate) + (size_t)r * gs + d);
            x = load16(static_cast<const T *>(a.resid) + (size_t)r * rs + d);
        }
        if (by_row) g_row = to_f<T>(static_cast<const T *>(a.gate)[(size_t)r * gs]);
    };
    fetch(row);
    float wp[V], wn[V];
#pragma unroll
    for (int j = 0; j < V; j += 4) {
        float4 p = make_float4(1.0f, 1.0f, 1.0f, 1.0f), n = p;
        if (a.post_weight && in_row) p = __ldg(reinterpret_cast<const float4 *>(a.post_weight + d + j));
        if (a.norm_weight && in_row) n = __ldg(reinterpret_cast<const float4 *>(a.norm_weight + d + j));
        wp[j] = p.x, wp[j + 1] = p.y, wp[j + 2] = p.z, wp[j + 3] = p.w;
        wn[j] = n.x, wn[j + 1] = n.y, wn[j + 2] = n.z, wn[j + 3] = n.w;
    }
    // By the block's first row: all its threads take the same number of turns and barriers.
    for (uint32_t r0 = blockIdx.x * blockDim.y; r0 < rows; r0 += step, row += step) {
        float s[V];
        widen(y, s);
        const uint4 x0 = x, g0 = g;
        const float gate_row = a.gate_sigmoid && by_row ? sigmoid<T>(g_row) : g_row;
        fetch(row + step);
        if (a.post_norm) {
            float ss = 0.0f;
#pragma unroll
            for (int j = 0; j < V; j++) ss = fmaf(s[j], s[j], ss);
            const float rcp = rcp_rms(row_sum(ss), a, a.post_eps);
#pragma unroll
            for (int j = 0; j < V; j++) s[j] = s[j] * rcp * wp[j];
        }
        if (by_elem) {
            float t[V];
            widen(g0, t);
            if (a.gate_sigmoid) {
#pragma unroll
                for (int j = 0; j < V; j++) t[j] = sigmoid<T>(t[j]);
            }
#pragma unroll
            for (int j = 0; j < V; j++) s[j] *= t[j];
        } else if (by_row) {
#pragma unroll
            for (int j = 0; j < V; j++) s[j] *= gate_row;
        }
        float f[V];
        widen(x0, f);
#pragma unroll
        for (int j = 0; j < V; j++) s[j] = fmaf(a.scale, s[j], f[j]);
        const bool store = in_row && row < rows;
        if (a.resid_out && store)
            *reinterpret_cast<uint4 *>(static_cast<T *>(a.resid_out) + (size_t)row * os + d) = narrow(s);
        if (a.normed_out) {
            float ss = 0.0f;
            if (in_row) {
#pragma unroll
                for (int j = 0; j < V; j++) ss = fmaf(s[j], s[j], ss);
            }
            const float rcp = rcp_rms(row_sum(ss), a, a.norm_eps);
#pragma unroll
            for (int j = 0; j < V; j++) s[j] = s[j] * rcp * wn[j];
            if (store) *reinterpret_cast<uint4 *>(static_cast<T *>(a.normed_out) + (size_t)row * os + d) = narrow(s);
        }
    }
}

// E elements per thread, blockDim.x apart: any stride and alignment, rows up to 8192.  The loads
// in flight are those of an SM's other rows.  16384 rows of 1023: bf16 61 us (issue slots: a
// load and a store per element), f32 61 us, 5.5 TB/s; block_norm_any_kernel 110 and 122 us.
template <typename T, int E>
__global__ void __launch_bounds__(1024) block_norm_odd_kernel(const BlockNormArgs a)
{
    __shared__ float4 part[2][8];
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    RowSum row_sum(part);
    const uint32_t step = gridDim.x * blockDim.y, rows = a.rows;
    uint32_t row = blockIdx.x * blockDim.y + threadIdx.y;
    const int dim = a.dim, d0 = threadIdx.x, stride = blockDim.x;
    float wp[E], wn[E];
#pragma unroll
    for (int j = 0; j < E; j++) {
        const int d = d0 + j * stride;
        wp[j] = a.post_weight && d < dim ? __ldg(a.post_weight + d) : 1.0f;
        wn[j] = a.norm_weight && d < dim ? __ldg(a.norm_weight + d) : 1.0f;
    }
    for (uint32_t r0 = blockIdx.x * blockDim.y; r0 < rows; r0 += step, row += step) {
        const int end = row < rows ? dim : 0;
        const T *yp = static_cast<const T *>(a.block) + (size_t)row * a.block_stride + d0;
        const T *xp = static_cast<const T *>(a.resid) + (size_t)row * a.resid_stride + d0;
        const T *gp = static_cast<const T *>(a.gate) + (size_t)row * a.gate_row_stride + (size_t)d0 * a.gate_col_stride;
        T y[E], x[E], g[E];
#pragma unroll
        for (int j = 0; j < E; j++) {
            const bool in = d0 + j * stride < end;
            y[j] = x[j] = g[j] = from_f<T>(0.0f);
            if (in) y[j] = yp[j * stride];
            if (in && a.gate) g[j] = gp[j * stride * a.gate_col_stride];
            if (in) x[j] = xp[j * stride];
        }
        float s[E], ss = 0.0f;
#pragma unroll
        for (int j = 0; j < E; j++) {
            s[j] = to_f<T>(y[j]);
            ss = fmaf(s[j], s[j], ss);
        }
        if (a.post_norm) {
            const float rcp = rcp_rms(row_sum(ss), a, a.post_eps);
#pragma unroll
            for (int j = 0; j < E; j++) s[j] = s[j] * rcp * wp[j];
        }
        if (a.gate) {
#pragma unroll
            for (int j = 0; j < E; j++) s[j] *= a.gate_sigmoid ? sigmoid<T>(to_f<T>(g[j])) : to_f<T>(g[j]);
        }
        T *ro = static_cast<T *>(a.resid_out) + (size_t)row * a.out_stride + d0;
        T *no = static_cast<T *>(a.normed_out) + (size_t)row * a.out_stride + d0;
        ss = 0.0f;
#pragma unroll
        for (int j = 0; j < E; j++) {
            const bool in = d0 + j * stride < end;
            s[j] = fmaf(a.scale, s[j], to_f<T>(x[j]));
            if (in) ss = fmaf(s[j], s[j], ss);
            if (in && a.resid_out) ro[j * stride] = from_f<T>(s[j]);
        }
        if (a.normed_out) {
            const float rcp = rcp_rms(row_sum(ss), a, a.norm_eps);
#pragma unroll
            for (int j = 0; j < E; j++)
                if (d0 + j * stride < end) no[j * stride] = from_f<T>(s[j] * rcp * wn[j]);
        }
    }
}

// Longer rows still: one block per row, elements one by one, the row re-read (from L1 or L2) by
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
        rcp = rcp_rms(block_sum(ss, part[0]), a, a.post_eps);
    }
    auto sum_at = [&](int d) {
        float v = to_f<T>(y[d]);
        if (a.post_norm) v = v * rcp * (a.post_weight ? a.post_weight[d] : 1.0f);
        if (g) {
            const float t = to_f<T>(g[(size_t)d * a.gate_col_stride]);
            v *= a.gate_sigmoid ? sigmoid<T>(t) : t;
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
        rcp2 = rcp_rms(block_sum(ss, part[1]), a, a.norm_eps);
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
cudaError_t launch(Kernel kernel, unsigned grid, dim3 block, const BlockNormArgs &a, cudaStream_t stream)
{
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(grid);
    cfg.blockDim = block;
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kernel, a);
}

// Rows of `x` threads each, on all SMs; short rows share a block of up to 256 threads, unless
// there are too few of them for that.
template <class Kernel>
cudaError_t launch_rows(Kernel kernel, int x, const BlockNormArgs &a, cudaStream_t stream)
{
    int dev = 0, sms = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e == cudaSuccess) e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
    if (e != cudaSuccess) return e;
    x = (x + 31) & ~31;
    int y = x < 256 ? 256 / x : 1;
    while (y > 1 && a.rows < (long long)sms * y) y--;
    const int blocks = (a.rows - 1) / y + 1;
    const int most = sms * max(1, 1024 / (x * y));   // at a time: 1024 threads of 64 registers an SM
    return launch(kernel, (unsigned)min(blocks, most), dim3(x, y), a, stream);
}

template <typename T>
cudaError_t launch_type(const BlockNormArgs &a, cudaStream_t stream)
{
    auto fits = [&](const void *p, long long stride) {   // absent, or whole vectors
        return !p || ((uintptr_t)p % 16 == 0 && stride % kVec<T> == 0 && stride <= INT32_MAX);
    };
    const bool vec = a.dim % kVec<T> == 0 && fits(a.resid, a.resid_stride) && fits(a.block, a.block_stride) &&
                     (a.gate_col_stride ? fits(a.gate, a.gate_row_stride) : a.gate_row_stride <= INT32_MAX) && fits(a.resid_out, a.out_stride) &&
                     fits(a.normed_out, a.out_stride) && fits(a.post_weight, 0) && fits(a.norm_weight, 0);
    if (vec && a.dim <= 1024 * kVec<T>) return launch_rows(block_norm_kernel<T>, a.dim / kVec<T>, a, stream);
    // One warp a row up to 256 elements.
    if (a.dim <= 32) return launch_rows(block_norm_odd_kernel<T, 1>, a.dim, a, stream);
    if (a.dim <= 64) return launch_rows(block_norm_odd_kernel<T, 2>, (a.dim + 1) / 2, a, stream);
    if (a.dim <= 8192) return launch_rows(block_norm_odd_kernel<T, 8>, (a.dim + 7) / 8, a, stream);
    int threads = 32;
    while (threads < 1024 && threads * 4 < a.dim) threads *= 2;
    return launch(block_norm_any_kernel<T>, (unsigned)a.rows, dim3(threads), a, stream);
}

}  // namespace

cudaError_t launch_block_norm(const BlockNormArgs &a, bool bf16, cudaStream_t stream)
{
    if (a.rows == 0) return cudaSuccess;
    return bf16 ? launch_type<__nv_bfloat16>(a, stream) : launch_type<float>(a, stream);
}

}  // namespace z2
