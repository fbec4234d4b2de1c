// head_i8.cu -- the output head in 8-bit integers (sm_100a): hidden rows rounded to 8 bits with
// a scale each, their product with 8-bit weight rows on the tcgen05 tensor cores, scales and
// softcap in the epilogue:
//
//     s_b = max |h_b| / 127,  q_b = round(127 h_b / max |h_b|)
//     logits[b, n] = softcap(s_b w_scale[n] (q_b . W[n]))
//
// The products are summed exactly, in 32-bit integers, so that nothing is rounded but the rows
// themselves and, at the end, the logits.
// 9 x 1024 x 2048, with the rounding: 1 row 9.3 us, 64 rows 10.8 us, 333 rows 14.8 us, 4096 rows 78 us (92 us for
// seconds on end, at the power limit; 1.98 POP/s; the product alone 73 us with the tensor pipe 58 % active, the rounding 14 us of
// which the product's start hides part).
#include <cuda_bf16.h>
#include <math.h>

#include <mutex>

#include "common.cuh"
#include "head_i8.cuh"
#include "tc.cuh"

namespace z2 {

int read_and_clear_head_i8_error(int *value) { return take_device_error(value); }

namespace {

// ---- rounding rows -----------------------------------------------------------
// A block to a row; its elements stay in registers between the maximum and the rounding (up to
// kKeep pieces of eight a thread, past that they are read again).  127 x / most is tried with one
// f32 division a row: where the product comes within 1e-4 of a half, more than f32 can move it
// (127 * 3 * 2^-24 = 2.3e-5), the quotient is taken in f64, which is exact enough to tell every
// side and tie (127 x is exact there, and a quotient of two f32 values that is not a tie is
// 2^-33 from one at least).
// Bound: memory; latency for a few rows.
constexpr int kQuantThreads = 128, kKeep = 4;

__device__ __forceinline__ float value_of(float v) { return v; }
__device__ __forceinline__ float value_of(__nv_bfloat16 v) { return __bfloat162float(v); }

__device__ __forceinline__ void load8(const float *p, float (&x)[8])
{
    const float4 a = *reinterpret_cast<const float4 *>(p), b = *reinterpret_cast<const float4 *>(p + 4);
    x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w;
    x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
}
__device__ __forceinline__ void load8(const __nv_bfloat16 *p, float (&x)[8])
{
    const uint4 v = *reinterpret_cast<const uint4 *>(p);
    const uint32_t u[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; i++) {
        x[2 * i] = __uint_as_float(u[i] << 16);
        x[2 * i + 1] = __uint_as_float(u[i] & 0xffff0000u);
    }
}

__device__ __forceinline__ int round_to_8(float x, float rate, float most, bool careful)
{
    const float p = x * rate, n = rintf(p);
    if (careful || fabsf(p - n) > 0.5f - 1e-4f) return (int)rint(127.0 * (double)x / (double)most);
    return (int)n;
}

// The row's scale, and the factors of its rounding (odd: a NaN or an infinity among it).
struct Rounding {
    float most, rate;
    bool odd, zero, careful;
};
__device__ __forceinline__ Rounding rounding_of(float most, bool odd)
{
    Rounding r;
    r.odd = odd;
    r.zero = odd || most == 0.0f;
    r.most = most;
    r.careful = most < 1e-30f;   // 127 / most may not be finite
    r.rate = r.zero || r.careful ? 0.0f : 127.0f / most;
    return r;
}

// The block's largest magnitude, and whether some thread saw a value that is not finite.
__device__ __forceinline__ Rounding block_rounding(float most, bool odd)
{
    __shared__ float s_part[kQuantThreads / 32];
#pragma unroll
    for (int d = 16; d >= 1; d >>= 1) most = fmaxf(most, __shfl_xor_sync(kFull, most, d));
    if ((threadIdx.x & 31) == 0) s_part[threadIdx.x >> 5] = most;
    odd = __syncthreads_or(odd);
#pragma unroll
    for (int i = 0; i < kQuantThreads / 32; i++) most = fmaxf(most, s_part[i]);
    return rounding_of(most, odd);
}

__device__ __forceinline__ void store_scale(const Rounding &r, float *scale)
{
    if (threadIdx.x == 0) *scale = r.odd ? __int_as_float(0x7fc00000) : r.most / 127.0f;
}

// Rows of whole 16-byte pieces, dim a multiple of 8.
template <typename T>
__global__ void __launch_bounds__(kQuantThreads)
    quantize_kernel(const T *x, int dim, long long stride, int8_t *q, float *scale)
{
    // after the wait: what a dependent kernel reads ahead of its own wait is then complete
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const T *row = x + blockIdx.x * stride;
    int8_t *to = q + (long long)blockIdx.x * dim;
    const int pieces = dim / 8;
    float v[kKeep][8];
    float most = 0.0f;
    bool odd = false;
    auto look = [&](const float (&e)[8]) {
#pragma unroll
        for (int i = 0; i < 8; i++) {
            most = fmaxf(most, fabsf(e[i]));
            odd |= !(fabsf(e[i]) <= 3.402823466e38f);
        }
    };
#pragma unroll
    for (int i = 0; i < kKeep; i++) {
        const int p = threadIdx.x + i * kQuantThreads;
        if (p < pieces) load8(row + 8 * p, v[i]);
    }
#pragma unroll
    for (int i = 0; i < kKeep; i++)
        if (threadIdx.x + i * kQuantThreads < pieces) look(v[i]);
    for (int p = threadIdx.x + kKeep * kQuantThreads; p < pieces; p += kQuantThreads) {
        float e[8];
        load8(row + 8 * p, e);
        look(e);
    }
    const Rounding r = block_rounding(most, odd);
    store_scale(r, scale + blockIdx.x);
    auto put = [&](int p, const float (&e)[8]) {
        uint32_t w[2] = {0, 0};
        if (!r.zero) {
#pragma unroll
            for (int i = 0; i < 8; i++)
                w[i >> 2] |= ((uint32_t)round_to_8(e[i], r.rate, r.most, r.careful) & 0xffu) << (8 * (i & 3));
        }
        *reinterpret_cast<uint2 *>(to + 8 * p) = make_uint2(w[0], w[1]);
    };
#pragma unroll
    for (int i = 0; i < kKeep; i++) {
        const int p = threadIdx.x + i * kQuantThreads;
        if (p < pieces) put(p, v[i]);
    }
    for (int p = threadIdx.x + kKeep * kQuantThreads; p < pieces; p += kQuantThreads) {
        float e[8];
        load8(row + 8 * p, e);
        put(p, e);
    }
}

// Any rows, element by element.
template <typename T>
__global__ void __launch_bounds__(kQuantThreads)
    quantize_any_kernel(const T *x, int dim, long long stride, int8_t *q, float *scale)
{
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const T *row = x + blockIdx.x * stride;
    int8_t *to = q + (long long)blockIdx.x * dim;
    float most = 0.0f;
    bool odd = false;
    for (int i = threadIdx.x; i < dim; i += kQuantThreads) {
        const float v = fabsf(value_of(row[i]));
        odd |= !(v <= 3.402823466e38f);
        most = fmaxf(most, v);
    }
    const Rounding r = block_rounding(most, odd);
    store_scale(r, scale + blockIdx.x);
    for (int i = threadIdx.x; i < dim; i += kQuantThreads)
        to[i] = r.zero ? 0 : (int8_t)round_to_8(value_of(row[i]), r.rate, r.most, r.careful);
}

template <typename Kernel, typename... Args>
cudaError_t launch_pdl(Kernel kernel, int grid, int threads, size_t smem, cudaStream_t stream, Args... args)
{
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)grid);
    cfg.blockDim = dim3((unsigned)threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kernel, args...);
}

template <typename T>
cudaError_t launch_quantize(const void *x, int rows, int dim, long long stride, int8_t *q, float *scale,
                            cudaStream_t stream)
{
    const bool whole = dim % 8 == 0 && (uintptr_t)x % 16 == 0 && stride * (long long)sizeof(T) % 16 == 0 &&
                       (uintptr_t)q % 8 == 0;
    return launch_pdl(whole ? quantize_kernel<T> : quantize_any_kernel<T>, rows, kQuantThreads, 0, stream,
                      (const T *)x, dim, stride, q, scale);
}

// ---- the product ---------------------------------------------------------------
// Weight rows are the MMA's M (TMEM lanes), hidden rows its N (columns): few hidden rows then
// leave no part of a tile empty, and a warp's logits of one hidden row are 128 consecutive
// bytes.  Persistent, one block per SM (or pair of blocks, CTAS = 2: M = 256, each half of
// the weight rows and of the hidden rows):
//   warp 0       TMA producer: 128 x 128 bytes of weights and the hidden rows' 128 bytes, 128-byte
//                swizzled, into a ring of stages; the first stages' weights are asked for
//                before the rounding kernel ahead has ended (it started after all else had);
//   warp 1       TMEM allocation, tcgen05.mma kind::i8 (K = 32), two accumulators in turn;
//   warps 2..17  epilogue, four to a TMEM lane quarter, each a quarter of the hidden rows.
// Every wait is bounded, as in head_tc.cu.  No load uses cluster multicast.
constexpr int kEpi = 16;             // epilogue warps
constexpr int kI8Threads = 64 + 32 * kEpi;
constexpr int kI8MaxStages = 16;
constexpr int kI8Rows = 128;         // weight rows per block
constexpr int kI8SmemMax = 232448 - 1024;   // dynamic; the static part takes 1 KB

struct I8Args {
    int batch, n_cb, vocab, rows_per_cb, dim;
    int nb;                    // hidden rows per tile: a multiple of 16, of 32 for pairs
    int tiles_b, per_cb, n_tiles, stages, tmem_cols;
    float softcap;
    const float *w_scale, *scale;
    float *out;
};

__device__ __forceinline__ void mma_i8(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate)
{
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
        : "memory");
}
__device__ __forceinline__ void mma_i8_pair(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate)
{
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
        : "memory");
}
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t (&r)[16])
{
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
          "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr));
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
    for (int i = 0; i < 16; i++) asm volatile("" : "+r"(r[i]));   // no use moves ahead of the wait
}

// cap * tanh(l / cap) of 16 values, two to an instruction: y (1 + z q(z)), z = y^2, below |y| =
// 0.9, q of degree 5 with the least relative error (1.4e-8); past it, where a warp has such a value at
// all, cap - 2 cap / (exp(2 y) + 1), whose rounding (a few 2^-24 of cap) is small against it.
__device__ __forceinline__ void softcap16(float (&l)[16], float cap, float inv_cap)
{
    auto two = [](float x) { return make_float2(x, x); };
    float most = 0.0f;
#pragma unroll
    for (int i = 0; i < 16; i += 2) most = fmaxf(most, fmaxf(fabsf(l[i]), fabsf(l[i + 1])));
    const bool small = __all_sync(kFull, most * inv_cap < 0.9f);
    const float2 inv = two(inv_cap);
    const float k2 = 2.0f * 1.4426950408889634f * inv_cap;
#pragma unroll
    for (int i = 0; i < 16; i += 2) {
        const float2 x = make_float2(l[i], l[i + 1]), y = __fmul2_rn(x, inv), z = __fmul2_rn(y, y);
        float2 p = __ffma2_rn(z, two(0.00128645188f), two(-0.00681405789f));
        p = __ffma2_rn(z, p, two(0.0208577033f));
        p = __ffma2_rn(z, p, two(-0.0536990522f));
        p = __ffma2_rn(z, p, two(0.133298353f));
        p = __ffma2_rn(z, p, two(-0.333331602f));
        p = __ffma2_rn(__fmul2_rn(x, z), p, x);
        l[i] = p.x;
        l[i + 1] = p.y;
        if (!small) {
            float e0, e1, r0, r1;
            asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e0) : "f"(x.x * k2));
            asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e1) : "f"(x.y * k2));
            asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r0) : "f"(e0 + 1.0f));
            asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r1) : "f"(e1 + 1.0f));
            if (!(fabsf(y.x) < 0.9f)) l[i] = fmaf(-2.0f * cap, r0, cap);
            if (!(fabsf(y.y) < 0.9f)) l[i + 1] = fmaf(-2.0f * cap, r1, cap);
        }
    }
}

template <int CTAS>
__global__ void __launch_bounds__(kI8Threads, 1)
    head_i8_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_h,
                   const __grid_constant__ I8Args args)
{
    constexpr bool PAIR = CTAS == 2;
    constexpr int BM = kI8Rows;
    constexpr uint32_t kWBytes = BM * 128;
    extern __shared__ __align__(1024) unsigned char smem_raw[];
    const uint32_t smem0 = (smem_u32(smem_raw) + 1023) & ~1023u;
    const int nb_own = args.nb / CTAS, stages = args.stages;
    const uint32_t stage_bytes = kWBytes + (uint32_t)nb_own * 128;
    const uint32_t bar0 = smem0 + (uint32_t)stages * stage_bytes;
    auto full = [&](int s) { return bar0 + 8u * (uint32_t)s; };
    auto empty = [&](int s) { return bar0 + 8u * (uint32_t)(kI8MaxStages + s); };
    auto done = [&](int b) { return bar0 + 8u * (uint32_t)(2 * kI8MaxStages + b); };       // MMA -> epilogue
    auto open = [&](int b) { return bar0 + 8u * (uint32_t)(2 * kI8MaxStages + 2 + b); };   // epilogue -> MMA
    __shared__ uint32_t s_tmem;
    __shared__ int s_abort;
    auto aborted = [&]() { return *(volatile int *)&s_abort != 0; };

    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = PAIR ? cluster_rank() : 0u;
    const int KB = (args.dim + 127) / 128;
    if (threadIdx.x == 0) {
        s_abort = 0;
        for (int s = 0; s < stages; s++) {
            mbar_init(full(s), 1);
            mbar_init(empty(s), 1);
        }
        for (int b = 0; b < 2; b++) {
            mbar_init(done(b), 1);
            mbar_init(open(b), kEpi * CTAS);   // the epilogue warps
        }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        prefetch_map(&map_w);
        prefetch_map(&map_h);
    }
    if (warp == 1) {
        if (PAIR) {
            asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&s_tmem)), "r"(args.tmem_cols) : "memory");
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
        } else {
            asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&s_tmem)), "r"(args.tmem_cols) : "memory");
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
        }
    }
    tc_fence_before();
    __syncthreads();
    if (PAIR) cluster_sync();
    tc_fence_after();
    const uint32_t tmem = s_tmem;
    const int unit0 = (int)blockIdx.x / CTAS, units = (int)gridDim.x / CTAS;
    // the tile's first hidden row, its codebook and this block's first weight row there
    auto tile_at = [&](int tile, int &b0, int &c, int &v0) {
        const int nt = tile / args.tiles_b;
        b0 = (tile - nt * args.tiles_b) * args.nb;
        c = nt / args.per_cb;
        v0 = (nt - c * args.per_cb) * (BM * CTAS) + (int)rank * BM;
    };

    if (warp == 0) {
        if (lane == 0) {
            const uint32_t full0 = PAIR ? peer_addr(full(0), 0) : full(0);
            auto load_w = [&](int s, int kb, int w_row) {
                const uint32_t d = smem0 + (uint32_t)s * stage_bytes, fb = full0 + 8u * (uint32_t)s;
                if (rank == 0) mbar_expect_tx(full(s), (uint32_t)CTAS * stage_bytes);
                if (PAIR)
                    tma_load_2d_pair(d, &map_w, kb * 128, w_row, fb);
                else
                    tma_load_2d(d, &map_w, kb * 128, w_row, fb);
            };
            auto load_h = [&](int s, int kb, int h_row) {
                const uint32_t d = smem0 + (uint32_t)s * stage_bytes + kWBytes, fb = full0 + 8u * (uint32_t)s;
                if (PAIR)
                    tma_load_2d_pair(d, &map_h, kb * 128, h_row, fb);
                else
                    tma_load_2d(d, &map_h, kb * 128, h_row, fb);
            };
            // the first stages' weights, ahead of the rounded rows
            int ahead = 0;
            if (unit0 < args.n_tiles) {
                int b0, c, v0;
                tile_at(unit0, b0, c, v0);
                for (; ahead < KB && ahead < stages; ahead++)
                    load_w(ahead, ahead, c * args.rows_per_cb + v0);
            }
            asm volatile("griddepcontrol.wait;" ::: "memory");
            // (a stage and its phase are counted up: a division by their number would cost a slice
            // more than its MMAs)
            int it = 0, s = 0;
            uint32_t ph = 1;
            bool ok = true;
            for (int tile = unit0; tile < args.n_tiles && ok; tile += units) {
                int b0, c, v0;
                tile_at(tile, b0, c, v0);
                const int w_row = c * args.rows_per_cb + v0, h_row = b0 + (int)rank * nb_own;
                for (int kb = 0; kb < KB; kb++, it++) {
                    if (it >= ahead) {
                        if (!mbar_wait(empty(s), ph) || aborted()) {
                            ok = false;
                            break;
                        }
                        load_w(s, kb, w_row);
                    }
                    load_h(s, kb, h_row);
                    if (++s == stages) {
                        s = 0;
                        ph ^= 1u;
                    }
                }
            }
            if (!ok) {
                s_abort = 1;
                if (rank == 0)   // copies still in flight land first
                    for (int k = 0; k < stages && k < it; k++) {
                        const int j = it - 1 - k;
                        mbar_wait(full(j % stages), (uint32_t)(j / stages) & 1u);
                    }
            }
        }
    } else if (warp == 1) {
        if (lane == 0 && rank == 0) {
            // kind::i8: D s32, A and B s8, both K-major
            const uint32_t idesc = (2u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(args.nb >> 3) << 17) |
                                   ((uint32_t)((CTAS * BM) >> 4) << 24);
            int s = 0, local = 0;
            uint32_t ph = 0;
            bool ok = true;
            for (int tile = unit0; tile < args.n_tiles && ok && !aborted(); tile += units, local++) {
                const int buf = local & 1;
                const uint32_t bph = ((uint32_t)(local >> 1) & 1u) ^ 1u;
                if (!(PAIR ? mbar_wait_cl(open(buf), bph) : mbar_wait(open(buf), bph))) {
                    ok = false;
                    break;
                }
                tc_fence_after();
                const uint32_t d = tmem + (uint32_t)(buf * args.nb);
                for (int kb = 0; kb < KB; kb++) {
                    if (!(PAIR ? mbar_wait_cl(full(s), ph) : mbar_wait(full(s), ph))) {
                        ok = false;
                        break;
                    }
                    const uint32_t sa = smem0 + (uint32_t)s * stage_bytes;
                    const uint64_t ad = sw128_desc(sa), bd = sw128_desc(sa + kWBytes);
#pragma unroll
                    for (int k = 0; k < 4; k++) {   // 32 bytes of K each
                        if (PAIR)
                            mma_i8_pair(d, ad + (uint64_t)(2 * k), bd + (uint64_t)(2 * k), idesc, (kb | k) != 0);
                        else
                            mma_i8(d, ad + (uint64_t)(2 * k), bd + (uint64_t)(2 * k), idesc, (kb | k) != 0);
                    }
                    if (PAIR) {
                        mma_commit_pair(empty(s));
                        mma_commit_pair(peer_addr(empty(s), 1));
                    } else {
                        mma_commit(empty(s));
                    }
                    if (++s == stages) {
                        s = 0;
                        ph ^= 1u;
                    }
                }
                if (ok) {
                    if (PAIR) {
                        mma_commit_pair(done(buf));
                        mma_commit_pair(peer_addr(done(buf), 1));
                    } else {
                        mma_commit(done(buf));
                    }
                }
            }
            if (!ok) s_abort = 1;
        }
    } else {
        const int q = warp & 3, part = (warp - 2) >> 2;
        const int row = 32 * q + lane;   // of the block's weight rows
        const uint32_t open0 = PAIR ? peer_addr(open(0), 0) : open(0);
        const long long wide = (long long)args.n_cb * args.vocab;
        const float inv_cap = 1.0f / args.softcap;
        asm volatile("griddepcontrol.wait;" ::: "memory");   // the hidden rows' scales
        int local = 0;
        for (int tile = unit0; tile < args.n_tiles; tile += units, local++) {
            const int buf = local & 1;
            int b0, c, v0;
            tile_at(tile, b0, c, v0);
            const int v = v0 + row;
            const bool live = v < args.vocab;
            const float ws = live ? args.w_scale[(long long)c * args.rows_per_cb + v] : 0.0f;
            const int cols = min(args.nb, args.batch - b0);   // hidden rows of the tile
            // columns [from, to) in steps of 16
            const int each = (args.nb / 16 + kEpi / 4 - 1) / (kEpi / 4) * 16;
            const int from = part * each, to = min(from + each, cols);
            const bool got = mbar_wait(done(buf), (uint32_t)(local >> 1) & 1u) && !aborted();
            if (!__all_sync(kFull, got)) {
                s_abort = 1;
                break;
            }
            tc_fence_after();
            float *out = args.out + (long long)b0 * wide + (long long)c * args.vocab + v;
            for (int j0 = from; j0 < to; j0 += 16) {
                uint32_t r[16];
                __syncwarp();
                tmem_ld16(tmem + ((uint32_t)(32 * q) << 16) + (uint32_t)(buf * args.nb + j0), r);
                const float4 *scale = reinterpret_cast<const float4 *>(args.scale + b0 + j0);   // (16 of them lie there)
                float l[16];
#pragma unroll
                for (int j = 0; j < 16; j += 4) {
                    const float4 s = scale[j / 4];
                    l[j] = (float)(int)r[j] * s.x * ws;
                    l[j + 1] = (float)(int)r[j + 1] * s.y * ws;
                    l[j + 2] = (float)(int)r[j + 2] * s.z * ws;
                    l[j + 3] = (float)(int)r[j + 3] * s.w * ws;
                }
                if (args.softcap > 0.0f) softcap16(l, args.softcap, inv_cap);
                if (live) {
                    float *to = out + j0 * wide;
                    if (j0 + 16 <= cols) {
#pragma unroll
                        for (int j = 0; j < 16; j++, to += wide) *to = l[j];
                    } else {
#pragma unroll
                        for (int j = 0; j < 16; j++, to += wide)
                            if (j0 + j < cols) *to = l[j];
                    }
                }
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) {
                if (PAIR)
                    mbar_arrive_cluster_relaxed(open0 + 8u * (uint32_t)buf);
                else
                    mbar_arrive(open(buf));
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    if (PAIR) cluster_sync();
    tc_fence_after();
    if (warp == 1) {
        if (PAIR)
            asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(args.tmem_cols) : "memory");
        else
            asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(args.tmem_cols) : "memory");
    }
}

// Rows of dim bytes, box 128 bytes x box_rows.
bool make_map_i8(CUtensorMap *m, const void *base, long long rows, int dim, int box_rows)
{
    EncodeTiledFn enc = encode_fn();
    if (!enc) return false;
    const cuuint64_t dims[2] = {(cuuint64_t)dim, (cuuint64_t)rows};
    const cuuint64_t strides[1] = {(cuuint64_t)dim};
    const cuuint32_t box[2] = {128, (cuuint32_t)box_rows};
    const cuuint32_t estr[2] = {1, 1};
    return enc(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void *>(base), dims, strides, box, estr,
               CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
               CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

struct Plan {
    int ctas, nb, tiles_b;
};

template <int CTAS>
cudaError_t launch_product(const HeadI8Args &a, const Plan &p, int dev, int sms, const int8_t *q, const float *scale,
                           cudaStream_t stream)
{
    static std::mutex mu;
    static int units_at_once[64] = {0};
    int units = 0;
    {
        std::lock_guard<std::mutex> lk(mu);
        if (units_at_once[dev] == 0) {
            cudaError_t e = cudaFuncSetAttribute(head_i8_kernel<CTAS>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                                 kI8SmemMax);
            if (e != cudaSuccess) return e;
            int n = sms;
            if (CTAS == 2) {
                cudaLaunchConfig_t cfg = {};
                cfg.gridDim = dim3((unsigned)(2 * (sms / 2)));
                cfg.blockDim = dim3(kI8Threads);
                cfg.dynamicSmemBytes = kI8SmemMax;
                cudaLaunchAttribute attr[1];
                attr[0].id = cudaLaunchAttributeClusterDimension;
                attr[0].val.clusterDim.x = 2;
                attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
                cfg.attrs = attr;
                cfg.numAttrs = 1;
                e = cudaOccupancyMaxActiveClusters(&n, head_i8_kernel<CTAS>, &cfg);
                if (e != cudaSuccess) return e;
            }
            units_at_once[dev] = n > 0 ? n : 1;
        }
        units = units_at_once[dev];
    }
    CUtensorMap mw, mh;
    if (!make_map_i8(&mw, a.W, (long long)a.n_cb * a.rows_per_cb, a.dim, kI8Rows) ||
        !make_map_i8(&mh, q, a.batch, a.dim, p.nb / CTAS))
        return cudaErrorInvalidValue;
    I8Args t;
    t.batch = a.batch;
    t.n_cb = a.n_cb;
    t.vocab = a.vocab;
    t.rows_per_cb = a.rows_per_cb;
    t.dim = a.dim;
    t.nb = p.nb;
    t.tiles_b = p.tiles_b;
    t.per_cb = (a.vocab + kI8Rows * CTAS - 1) / (kI8Rows * CTAS);
    const long long tiles = (long long)p.tiles_b * t.per_cb * a.n_cb;
    if (tiles > 0x7fffffffll) return cudaErrorInvalidConfiguration;
    t.n_tiles = (int)tiles;
    t.softcap = a.softcap;
    t.w_scale = a.w_scale;
    t.scale = scale;
    t.out = a.out;
    t.tmem_cols = 32;
    while (t.tmem_cols < 2 * p.nb) t.tmem_cols *= 2;
    const int stage = (kI8Rows + p.nb / CTAS) * 128, bars = 8 * (2 * kI8MaxStages + 4);
    t.stages = (kI8SmemMax - 1024 - bars) / stage;
    if (t.stages > kI8MaxStages) t.stages = kI8MaxStages;
    const size_t smem = (size_t)t.stages * stage + bars + 1024;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(CTAS * (t.n_tiles < units ? t.n_tiles : units)));
    cfg.blockDim = dim3(kI8Threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = CTAS;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = CTAS == 2 ? 2 : 1;
    return cudaLaunchKernelEx(&cfg, head_i8_kernel<CTAS>, mw, mh, t);
}

// The tiles, by a model of the time fitted to a B200: for each kind of block (alone or in pairs) and
// the counts of hidden tiles that its accumulators allow, the waves times a tile's hidden rows and a
// fixed part.  Measured there, 9 x 1024 x 2048, us with the rounding (tiles of hidden rows):
//   rows      64        128       256       333       512       700       1024      2048      4096
//   alone   10.6 (1)  11.9 (2)  13.6 (2)  15.2 (2)  18.0 (2)  21.6 (4)  26.1 (4)  44.6 (8)  84.5 (16)
//   pairs   11.4 (1)  13.1 (1)  14.8 (2)  15.9 (2)  17.3 (2)  23.4 (4)  25.6 (4)  41.6 (8)  77.8 (16)
// Blocks of 64 weight rows were slower than of 128 from 16 hidden rows on, and no faster below.
Plan plan_tiles(const HeadI8Args &a, int sms)
{
    Plan best{0, 0, 0};
    long long best_cost = -1;
    for (int ctas = 1; ctas <= 2; ctas++) {
        const int unit = 16 * ctas;
        const long long n = (long long)a.n_cb * ((a.vocab + kI8Rows * ctas - 1) / (kI8Rows * ctas));
        const int least = (a.batch + 255) / 256;
        for (int tb = least; tb < least + 4; tb++) {
            const int nb = ((a.batch + tb - 1) / tb + unit - 1) / unit * unit, wide = nb < 64 ? 64 : nb;
            const long long waves = (n * tb + sms / ctas - 1) / (sms / ctas);
            const long long cost = ctas == 1 ? 300 + waves * (5 * wide + 200) : 500 + waves * (4 * wide + 250);
            if (best_cost < 0 || cost < best_cost) {
                best_cost = cost;
                best = Plan{ctas, nb, (a.batch + nb - 1) / nb};
            }
        }
    }
    return best;
}

}  // namespace

cudaError_t launch_quantize_rows(const void *x, bool bf16, int rows, int dim, long long stride,
                                 int8_t *q, float *scale, cudaStream_t stream)
{
    return bf16 ? launch_quantize<__nv_bfloat16>(x, rows, dim, stride, q, scale, stream)
                : launch_quantize<float>(x, rows, dim, stride, q, scale, stream);
}

cudaError_t launch_head_i8(const HeadI8Args &a, bool bf16, cudaStream_t stream)
{
    int8_t *q = (int8_t *)a.work;
    float *scale = (float *)((char *)a.work + (((long long)a.batch * a.dim + 15) & ~15ll));
    int dev = 0, sms = 148;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (dev < 0 || dev >= 64) return cudaErrorInvalidDevice;
    cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
    e = launch_quantize_rows(a.hidden, bf16, a.batch, a.dim, a.dim, q, scale, stream);
    if (e != cudaSuccess) return e;
    const Plan p = plan_tiles(a, sms);
    return p.ctas == 2 ? launch_product<2>(a, p, dev, sms, q, scale, stream) : launch_product<1>(a, p, dev, sms, q, scale, stream);
}

}  // namespace z2
