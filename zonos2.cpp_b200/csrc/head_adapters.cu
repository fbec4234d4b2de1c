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

// Four neighbouring elements.
__device__ __forceinline__ float4 load4(const float *p) { return __ldg(reinterpret_cast<const float4 *>(p)); }
__device__ __forceinline__ float4 load4(const __nv_bfloat16 *p)
{
    const uint2 u = __ldg(reinterpret_cast<const uint2 *>(p));
    return make_float4(__uint_as_float(u.x << 16), __uint_as_float(u.x & 0xffff0000u), __uint_as_float(u.y << 16),
                       __uint_as_float(u.y & 0xffff0000u));
}

__device__ __forceinline__ float dot4(const float4 &a, const float4 &b)
{
    return fmaf(a.w, b.w, fmaf(a.z, b.z, fmaf(a.y, b.y, a.x * b.x)));
}

// t[b][r], one warp per element.  VEC: as below.
template <typename T, bool VEC>
__global__ void __launch_bounds__(32 * kWarps)
    adapter_down_kernel(const HeadArgs h, const AdapterArgs ad)
{
    using S = typename Acc<T>::type;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const int lane = threadIdx.x & 31;
    const long long i = (long long)blockIdx.x * kWarps + (threadIdx.x >> 5);
    if (i >= (long long)h.batch * ad.rank) return;
    const int b = (int)(i / ad.rank), r = (int)(i % ad.rank);
    const int a = ad.which[b / ad.rows_per_id];
    if ((unsigned)a >= (unsigned)ad.n_adapters) return;
    const T *x = static_cast<const T *>(h.hidden) + (size_t)b * h.dim;
    const T *w = static_cast<const T *>(ad.A) + ((size_t)a * ad.rank + r) * h.dim;
    S acc = 0;
    if (VEC) {
#pragma unroll 8
        for (int d = 4 * lane; d < h.dim; d += 128) acc += (S)dot4(load4(x + d), load4(w + d));
    } else {
#pragma unroll 8
        for (int d = lane; d < h.dim; d += 32) acc += (S)load_f(x + d) * (S)load_f(w + d);
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) acc += __shfl_xor_sync(kFull, acc, o);
    if (lane == 0) static_cast<S *>(ad.work)[i] = acc * (S)(ad.scale ? __ldg(ad.scale + a) : 1.0f);
}

constexpr int kRows = 2;    // weight rows per warp
constexpr int kBatch = 4;   // hidden rows at a time: a weight is read and widened once for four

// The logits, one warp per kRows weight rows of one codebook.  VEC: rows 16-byte aligned
// (f32) or 8-byte aligned (bf16) and dim a multiple of 4.  An f32 head's sums are f64, of
// single products or (VEC) of four in f32: their roundings, half a step of the products each,
// average out over dim / 4 terms, and the conversions, of which an SM makes 16 a cycle,
// are few: widening both operands takes six times as many.  Four blocks an SM (64 registers, at
// the price of 100 bytes of spills with VEC f32) hold all of a head's 4608 warps at once, and W's
// part runs beside adapter_down_kernel.
// 4 rows by 9216 x 2048 f32 with rank 12: 23.5 us, 3.3 TB/s; 52 us with widened operands,
// two blocks an SM and the kernels one after the other, 104 us with a row and a warp each.  W is
// read again, mostly from L2, for every four hidden rows: 20 f32 rows of rank 16 take 97 us, 64
// rows 259 us, 333 rows 1.30 ms, 64 bf16 rows of rank 12 212 us and 4096 of them 12.5 ms.
template <typename T, bool VEC>
__global__ void __launch_bounds__(32 * kWarps, 4)
    adapter_any_kernel(const HeadArgs h, const AdapterArgs ad)
{
    using S = typename Acc<T>::type;
    const int lane = threadIdx.x & 31, per_cb = (h.vocab + kRows - 1) / kRows;
    const int o = blockIdx.x * kWarps + (threadIdx.x >> 5);
    if (o >= h.n_cb * per_cb) return;
    const int c = o / per_cb, v = (o - c * per_cb) * kRows, rows = min(kRows, h.vocab - v);
    const size_t n = (size_t)c * h.rows_per_cb + v;
    const T *w = static_cast<const T *>(h.W) + n * h.dim;
    const int second = rows > 1 ? h.dim : 0;   // offset of the second row
    for (int b0 = 0; b0 < h.batch; b0 += kBatch) {
        const T *x[kBatch];
        int id[kBatch];
#pragma unroll
        for (int i = 0; i < kBatch; i++) {
            const int b = min(b0 + i, h.batch - 1);
            x[i] = static_cast<const T *>(h.hidden) + (size_t)b * h.dim;
            id[i] = ad.which[b / ad.rows_per_id];
        }
        S acc[kRows][kBatch] = {};
        if (VEC) {
#pragma unroll 4
            for (int d = 4 * lane; d < h.dim; d += 128) {
                const float4 w0 = load4(w + d), w1 = load4(w + second + d);
#pragma unroll
                for (int i = 0; i < kBatch; i++) {
                    const float4 f = load4(x[i] + d);
                    acc[0][i] += (S)dot4(w0, f);
                    acc[1][i] += (S)dot4(w1, f);
                }
            }
        } else {
            for (int d = lane; d < h.dim; d += 32) {
                const S u0 = (S)load_f(w + d), u1 = (S)load_f(w + second + d);
#pragma unroll
                for (int i = 0; i < kBatch; i++) {
                    const S y = (S)load_f(x[i] + d);
                    acc[0][i] += u0 * y;
                    acc[1][i] += u1 * y;
                }
            }
        }
        // W's part needed nothing of adapter_down_kernel's, which ran beside it.
        asm volatile("griddepcontrol.wait;" ::: "memory");
        for (int r = lane; r < ad.rank; r += 32) {
#pragma unroll
            for (int i = 0; i < kBatch; i++) {
                if (b0 + i >= h.batch || (unsigned)id[i] >= (unsigned)ad.n_adapters) continue;
                const T *up = static_cast<const T *>(ad.B) + ((size_t)id[i] * h.n_cb * h.rows_per_cb + n) * ad.rank + r;
                const S t = static_cast<const S *>(ad.work)[(size_t)(b0 + i) * ad.rank + r];
                acc[0][i] += (S)load_f(up) * t;
                if (rows > 1) acc[1][i] += (S)load_f(up + ad.rank) * t;
            }
        }
        float l[kRows][kBatch];
#pragma unroll
        for (int i = 0; i < kBatch; i++) {
#pragma unroll
            for (int m = 0; m < kRows; m++) {
                S sum = acc[m][i];
#pragma unroll
                for (int s = 16; s; s >>= 1) sum += __shfl_xor_sync(kFull, sum, s);
                float f = (float)sum;
                if (h.row_scale) f *= __ldg(h.row_scale + min(b0 + i, h.batch - 1));
                l[m][i] = h.softcap > 0.0f ? h.softcap * tanhf(f / h.softcap) : f;
            }
        }
        if (lane < rows) {   // lane m stores row m (every lane has the sums)
#pragma unroll
            for (int i = 0; i < kBatch; i++) {
                const int b = b0 + i;
                if (b >= h.batch) break;
                const float f = lane ? l[1][i] : l[0][i];
                if (!h.cfg) {
                    h.out[((size_t)b * h.n_cb + c) * h.vocab + v + lane] = f;
                } else if (i & 1) {   // the pair's blend; its conditional row came before
                    const float cond = lane ? l[1][i - 1] : l[0][i - 1];
                    h.out[((size_t)(b >> 1) * h.n_cb + c) * h.vocab + v + lane] =
                        __fadd_rn(f, __fmul_rn(h.cfg_scale, __fsub_rn(cond, f)));
                }
            }
        }
    }
}

template <class Kernel>
cudaError_t launch(Kernel kernel, long long warps, const HeadArgs &h, const AdapterArgs &ad, cudaStream_t stream)
{
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)((warps + kWarps - 1) / kWarps));
    cfg.blockDim = dim3(32 * kWarps);
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kernel, h, ad);
}

template <typename T>
cudaError_t launch_any(const HeadArgs &h, const AdapterArgs &ad, cudaStream_t stream)
{
    const auto fits = [&](const void *p) { return h.dim % 4 == 0 && (uintptr_t)p % (4 * sizeof(T)) == 0; };
    const long long down = (long long)h.batch * ad.rank, warps = (long long)h.n_cb * ((h.vocab + kRows - 1) / kRows);
    const cudaError_t e = fits(ad.A) && fits(h.hidden) ? launch(adapter_down_kernel<T, true>, down, h, ad, stream)
                                                       : launch(adapter_down_kernel<T, false>, down, h, ad, stream);
    if (e != cudaSuccess) return e;
    return fits(h.W) && fits(h.hidden) ? launch(adapter_any_kernel<T, true>, warps, h, ad, stream)
                                       : launch(adapter_any_kernel<T, false>, warps, h, ad, stream);
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
