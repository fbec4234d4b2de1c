// head_adapters_tc.cu -- the bf16 output head beside low-rank adapters on the tensor
// cores (sm_100a):
//
//     t[b]         = s_a * (A_a h[b])                     adapter_down_*_kernel
//     delta[b, n]  = B_a[n] . t[b]
//     logits[b, n] = softcap(W[n] . h[b] + delta[b, n])   adapter_head_kernel
//
// Up to 64 hidden rows, delta is made inside the GEMM: eight warps of its own put it into
// the accumulator that the last part of the tile's depth adds to, while W streams in.
// Beyond, adapter_up_kernel writes it to the logits' own buffer, and the GEMM reads an
// element, adds it and stores the logit in its place.  The kernels are chained by
// programmatic dependent launch, and only the steps that need t or delta wait for it, so
// the GEMM's main loop covers the small kernels of a batch that fills the SMs once.
//
// Everything is as good as f32: t enters its MMA as three bf16 parts, which hold all
// of its 24 bits, and the GEMM's depth is summed in parts (kPartSteps).
//
// Measured (9 x 1024 x 2048, 32 adapters, rank 16, in a graph): 14.8 us at 1 row (38 MB of
// weights, 2.6 TB/s), 19.7 at 64, 33 at 333, 57 at 1024, 188 at 4096 (155 GFLOP, 0.82
// PFLOP/s; 145 where no row has an adapter).  4096 rows at a time for seconds on end take 216 us:
// at the power limit the SMs' clock falls from 1.97 to 1.55 GHz.
// Up to 64 rows the GEMM's stream of W bounds it, beyond a few hundred the MMAs, and
// between them the chain of three kernels.  Delta in the GEMM against the separate kernel
// measured 16 / 26 us at 1 row, 27 / 34 at 64, 284 / 224 at 4096, when both were first built
// (nothing between, and not since):
// with more than a few rows per SM, the warps' latency per adapter exceeds the tile's MMAs.
// Slower still at 4096 rows: added in the epilogue on the FMA pipe, t broadcast from shared
// memory (16 B per 512 B of register writes), 370-540 us; hidden rows gathered by adapter
// with TMA gather4 (a quarter of the plain copies' rate), 540 us.
#include <cuda_bf16.h>
#include <limits.h>
#include <math.h>

#include "common.cuh"
#include "head_adapters.cuh"
#include "tc.cuh"

namespace z2 {

int read_and_clear_adapter_error(int *value) { return take_device_error(value); }

namespace {

constexpr int kMaxAdapters = 4096;   // below kNone
constexpr int kItem = 8;   // hidden rows per item at most: rows of one adapter

// ---- the rows' order ---------------------------------------------------------

// Scratch, after t: the rows by (adapter, row), those without an adapter last; and the
// items, of the adapters and then of the rows without one.
struct Order {
    int32_t *rows;      // [batch]
    int32_t *n_items;   // [2]: of the adapters, of all rows
    int2 *items;        // x: adapter (kNone: none) | rows << 16, y: the first row's place
};
constexpr int kNone = 0xffff;

// At most this many items.
__host__ __device__ constexpr int max_items(int batch, int n_adapters)
{
    return batch / kItem + (batch <= n_adapters ? batch : n_adapters + 1);
}

constexpr int kOrderRows = 128;   // rows per CTA
constexpr size_t order_bytes(int n_adapters) { return 2 * sizeof(int) * (size_t)(n_adapters + 1); }

// CTA `block` of those that order the rows (of at most 256 threads): it counts all rows
// and ranks its own kOrderRows by counting.  `s_count`: order_bytes() of shared memory.
__device__ __forceinline__ void order_rows(const int32_t *which, int batch, int rows_per_id, int n, const Order &o,
                                           int block, int *s_count)
{
    __shared__ int s_part[2][8];
    __shared__ __align__(16) int s_key[kOrderRows];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, threads = blockDim.x;
    const int b0 = block * kOrderRows, rows = min(kOrderRows, batch - b0);
    int *s_before = s_count + n + 1;   // rows of each key (n: none) before this CTA's
    auto key_of = [&](int b) {
        const int a = __ldg(which + b / rows_per_id);
        return (unsigned)a < (unsigned)n ? a : n;
    };
    for (int i = tid; i < 2 * (n + 1); i += threads) s_count[i] = 0;
    for (int i = tid; i < kOrderRows; i += threads) s_key[i] = i < rows ? key_of(b0 + i) : -1;
    __syncthreads();
#pragma unroll 4
    for (int i = tid; i < batch; i += threads) {
        const int k = batch <= kOrderRows ? s_key[i] : key_of(i);
        atomicAdd(&s_count[k], 1);
        if (i < b0) atomicAdd(&s_before[k], 1);
    }
    __syncthreads();
    // the first place and the first item of each key
    const int per = (n + threads) / threads;
    const int a0 = min(tid * per, n + 1), a1 = min(a0 + per, n + 1);
    int own = 0, own_items = 0;
    for (int a = a0; a < a1; a++) {
        own += s_count[a];
        own_items += (s_count[a] + kItem - 1) / kItem;
    }
    int sum = own, sum_items = own_items;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const int t = __shfl_up_sync(kFull, sum, d), u = __shfl_up_sync(kFull, sum_items, d);
        if (lane >= d) {
            sum += t;
            sum_items += u;
        }
    }
    if (lane == 31) {
        s_part[0][warp] = sum;
        s_part[1][warp] = sum_items;
    }
    __syncthreads();
    int base = sum - own, item = sum_items - own_items;
    for (int w = 0; w < warp; w++) {
        base += s_part[0][w];
        item += s_part[1][w];
    }
    for (int a = a0; a < a1; a++) {
        const int c = s_count[a], k = (c + kItem - 1) / kItem;
        if (block == 0) {
            for (int i = 0; i < k; i++)
                o.items[item + i] = make_int2((a < n ? a : kNone) | min(kItem, c - i * kItem) << 16, base + i * kItem);
            if (a == n) {
                o.n_items[0] = item;
                o.n_items[1] = item + k;
            }
        }
        s_count[a] = base;
        base += c;
        item += k;
    }
    __syncthreads();
    for (int i = tid; i < rows; i += threads) {   // after the rows with this key before this one
        const int mine = s_key[i];
        int same = 0;
#pragma unroll 4
        for (int j = 0; j < i; j += 4) {
            const int4 k = *reinterpret_cast<const int4 *>(&s_key[j]);
            same += (k.x == mine) + (k.y == mine && j + 1 < i) + (k.z == mine && j + 2 < i) + (k.w == mine && j + 3 < i);
        }
        o.rows[s_count[mine] + s_before[mine] + same] = b0 + i;
    }
}

__global__ void __launch_bounds__(256)
    order_rows_kernel(const int32_t *__restrict__ which, int batch, int rows_per_id, int n_adapters, Order o)
{
    extern __shared__ int s_count[];
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    order_rows(which, batch, rows_per_id, n_adapters, o, (int)blockIdx.x, s_count);
}

// ---- t = s_a A_a h ---------------------------------------------------------

struct DownArgs {
    const __nv_bfloat16 *hidden, *A;
    const float *scale;
    const int32_t *which;
    int batch, dim, n_adapters, rank, rows_per_id;
    float *t;                       // [batch][rank]
    Order order;
    int order_blocks;               // few rows: the first blocks order the rows
};

// Few rows: a CTA per row and four ranks, which share the row's loads, a quarter of the
// depth per warp, so that all loads are in flight at once and ahead of those of the GEMM,
// which may start after them and whose copies of W fill the memory's queues.  64 rows of
// 2048, rank 16: t is there after 2.2 us; with a warp per CTA's work, its loads behind W's,
// after 11.5 us, and the whole call took 25.7 us instead of 19.7.
// The first blocks order the rows.
// Up to kFewMost rows x ranks the loads of A by every row (from L2) cost less than the
// ordering as a step of its own: 1024 x 16 57 us against 70 by adapter_down_mma_kernel,
// 2048 x 16 102 / 105, 4096 x 16 196 / 189.
constexpr int kFewWarps = 4;
constexpr long long kFewMost = 32768;   // rows x ranks

__global__ void __launch_bounds__(32 * kFewWarps) adapter_down_few_kernel(const DownArgs g)
{
    __shared__ float s_sum[kFewWarps][4];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, quads = g.rank / 4;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    if ((int)blockIdx.x < g.order_blocks) {
        asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
        extern __shared__ int s_count[];
        order_rows(g.which, g.batch, g.rows_per_id, g.n_adapters, g.order, (int)blockIdx.x, s_count);
        return;
    }
    const int block = (int)blockIdx.x - g.order_blocks, b = block / quads, r0 = 4 * (block % quads);
    const int a = __ldg(g.which + b / g.rows_per_id);
    if ((unsigned)a >= (unsigned)g.n_adapters) return;
    const float s = g.scale ? __ldg(g.scale + a) : 1.0f;
    const uint4 *x = reinterpret_cast<const uint4 *>(g.hidden + (size_t)b * g.dim);
    const uint4 *w = reinterpret_cast<const uint4 *>(g.A + ((size_t)a * g.rank + r0) * g.dim);
    const int n = g.dim / 8;
    float acc[4] = {};
    auto add = [&](const uint4 &xv, const uint4 (&wv)[4]) {
        const uint32_t xs[4] = {xv.x, xv.y, xv.z, xv.w};
#pragma unroll
        for (int r = 0; r < 4; r++) {
            const uint32_t ws[4] = {wv[r].x, wv[r].y, wv[r].z, wv[r].w};
#pragma unroll
            for (int j = 0; j < 4; j++) {
                acc[r] = fmaf(__uint_as_float(xs[j] << 16), __uint_as_float(ws[j] << 16), acc[r]);
                acc[r] = fmaf(__uint_as_float(xs[j] & 0xffff0000u), __uint_as_float(ws[j] & 0xffff0000u), acc[r]);
            }
        }
    };
    constexpr int kAhead = 2, kStep = 32 * kFewWarps;   // 2048 deep: all of a lane's loads
    uint4 xv[kAhead] = {}, wv[kAhead][4] = {};
#pragma unroll
    for (int i = 0; i < kAhead; i++) {
        const int k = threadIdx.x + i * kStep;
        if (k >= n) continue;
        xv[i] = __ldg(x + k);
#pragma unroll
        for (int r = 0; r < 4; r++) wv[i][r] = __ldg(w + (size_t)r * n + k);
    }
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
#pragma unroll
    for (int i = 0; i < kAhead; i++) add(xv[i], wv[i]);
    for (int k = threadIdx.x + kAhead * kStep; k < n; k += kStep) {
        const uint4 xk = __ldg(x + k);
        uint4 wk[4];
#pragma unroll
        for (int r = 0; r < 4; r++) wk[r] = __ldg(w + (size_t)r * n + k);
        add(xk, wk);
    }
#pragma unroll
    for (int r = 0; r < 4; r++)
#pragma unroll
        for (int o = 16; o; o >>= 1) acc[r] += __shfl_xor_sync(kFull, acc[r], o);
    if (lane == 0)
#pragma unroll
        for (int r = 0; r < 4; r++) s_sum[warp][r] = acc[r];
    __syncthreads();
    if (threadIdx.x < 4) {
        float sum = 0.0f;
#pragma unroll
        for (int v = 0; v < kFewWarps; v++) sum += s_sum[v][threadIdx.x];
        g.t[(size_t)b * g.rank + r0 + threadIdx.x] = s * sum;
    }
}

constexpr int kDownRows = 32;    // rows per CTA
constexpr int kDownRank = 16;    // ranks per CTA
constexpr int kDownWarps = 8;    // each takes every eighth 32-deep slice of dim

__device__ __forceinline__ void mma_16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                          uint32_t a3, uint32_t b0, uint32_t b1)
{
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, "
        "{%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// Many rows, in the order of their adapters: CTA (i, j) takes places 32 i .. 32 i + 31 and ranks
// 16 j .. 16 j + 15, once for each adapter among them (mostly one).
// The depth is permuted alike for both operands, so that every thread loads 16
// consecutive bytes: of a 32-deep slice, thread q of a quad holds elements 8q ..
// 8q+7 of its rows, two of them per register of two 16-deep MMAs.
__global__ void __launch_bounds__(32 * kDownWarps, 1) adapter_down_mma_kernel(const DownArgs g)
{
    __shared__ int s_row[kDownRows], s_key[kDownRows];
    __shared__ float s_sum[kDownWarps][kDownRows][kDownRank + 1];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int p0 = (int)blockIdx.x * kDownRows, r0 = (int)blockIdx.y * kDownRank;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    if (tid < kDownRows) {
        int row = -1, key = -1;
        if (p0 + tid < g.batch) {
            row = g.order.rows[p0 + tid];
            key = __ldg(g.which + row / g.rows_per_id);
            if ((unsigned)key >= (unsigned)g.n_adapters) key = -1;
        }
        s_row[tid] = row;
        s_key[tid] = key;
    }
    __syncthreads();
    const int quad = lane >> 2, q = lane & 3;
    const uint4 zero = make_uint4(0, 0, 0, 0);
    const __nv_bfloat16 *x[4];
#pragma unroll
    for (int i = 0; i < 4; i++) x[i] = g.hidden + (size_t)max(s_row[quad + 8 * i], 0) * g.dim + 8 * q;
    for (int first = 0; first < kDownRows;) {
        const int a = s_key[first];
        int end = first + 1;
        while (end < kDownRows && s_key[end] == a) end++;
        if (a >= 0) {
            const __nv_bfloat16 *w[2];
#pragma unroll
            for (int i = 0; i < 2; i++)
                w[i] = g.A + ((size_t)a * g.rank + min(r0 + 8 * i + quad, g.rank - 1)) * g.dim + 8 * q;
            float d[2][2][4] = {};
#pragma unroll 4
            for (int k = 32 * warp; k < g.dim; k += 32 * kDownWarps) {
                const bool in = k + 8 * q < g.dim;
                uint4 xv[4], wv[2];
#pragma unroll
                for (int i = 0; i < 2; i++) wv[i] = in ? __ldg(reinterpret_cast<const uint4 *>(w[i] + k)) : zero;
#pragma unroll
                for (int i = 0; i < 4; i++) xv[i] = in ? __ldg(reinterpret_cast<const uint4 *>(x[i] + k)) : zero;
#pragma unroll
                for (int m = 0; m < 2; m++)
#pragma unroll
                    for (int n = 0; n < 2; n++) {
                        mma_16816(d[m][n], xv[2 * m].x, xv[2 * m + 1].x, xv[2 * m].y, xv[2 * m + 1].y, wv[n].x, wv[n].y);
                        mma_16816(d[m][n], xv[2 * m].z, xv[2 * m + 1].z, xv[2 * m].w, xv[2 * m + 1].w, wv[n].z, wv[n].w);
                    }
            }
#pragma unroll
            for (int m = 0; m < 2; m++)
#pragma unroll
                for (int n = 0; n < 2; n++)
#pragma unroll
                    for (int i = 0; i < 4; i++)
                        s_sum[warp][16 * m + quad + 8 * (i >> 1)][8 * n + 2 * q + (i & 1)] = d[m][n][i];
            __syncthreads();
            const float s = g.scale ? __ldg(g.scale + a) : 1.0f;
            for (int i = tid; i < (end - first) * kDownRank; i += 32 * kDownWarps) {
                const int row = first + i / kDownRank, r = i % kDownRank;
                if (r0 + r >= g.rank) continue;
                float sum = 0.0f;
#pragma unroll
                for (int v = 0; v < kDownWarps; v++) sum += s_sum[v][row][r];
                g.t[(size_t)s_row[row] * g.rank + r0 + r] = sum * s;
            }
            __syncthreads();
        }
        first = end;
    }
}

// ---- delta = B_a t ----------------------------------------------------------

// x = hi + mid + lo in bf16, two values to a register, the first in the low half.  Each part is the
// leading 8 bits of what is left, cut off: exact for the 24 bits of x, and no x rounds up
// to infinity.  An infinite x is its first part alone (what is left would be a NaN).
__device__ __forceinline__ float cut_bf16(float x) { return __uint_as_float(__float_as_uint(x) & 0xffff0000u); }
__device__ __forceinline__ uint32_t pack_high(float x, float y)
{
    return __byte_perm(__float_as_uint(x), __float_as_uint(y), 0x7632);
}
__device__ __forceinline__ void split3(float x, float y, uint32_t &hi, uint32_t &mid, uint32_t &lo)
{
    hi = pack_high(x, y);
    x = x == cut_bf16(x) ? 0.0f : x - cut_bf16(x);
    y = y == cut_bf16(y) ? 0.0f : y - cut_bf16(y);
    mid = pack_high(x, y);
    lo = pack_high(x - cut_bf16(x), y - cut_bf16(y));
}

struct UpArgs {
    const __nv_bfloat16 *B;
    const float *t;                // [batch][rank]
    Order order;
    int n_cb, vocab, rows_per_cb, rank;
    float *delta;                  // [batch][n_cb * vocab]
};

constexpr int kUpWarps = 4;
constexpr int kUpRows = 64;        // weight rows per step of a warp: four 16-row tiles
constexpr int kUpTiles = kUpRows / 16;
constexpr int kUpSteps = 4;        // steps per warp
constexpr int kUpSpan = kUpWarps * kUpRows * kUpSteps;   // weight rows per CTA

// CTA (i, j): item i and kUpSpan weight rows of one codebook.  mma.sync with the weight
// rows as M and the item's rows as N; ranks are permuted alike for both operands, so
// that a lane loads four neighbours (4 k4 .. 4 k4 + 3 of 16) of its rows of B and of the
// t of row g.  The result goes through shared memory, so that 128 neighbouring bytes of
// a row are stored at once.  KT: with at most 16 KT ranks, t's parts stay in registers and
// the next step's rows of B are on their way; 0: any number.
// Bound: the store of delta (with 32 adapters, 151 MB for 4096 rows of 9 x 1024).
template <int KT>
__global__ void __launch_bounds__(32 * kUpWarps) adapter_up_kernel(const UpArgs a)
{
    __shared__ float s_turn[kUpWarps][kItem][kUpRows + 4];   // rows 4 banks apart: no conflicts
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, k4 = lane & 3;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const int me = (int)blockIdx.x, items = *a.order.n_items;
    const int2 item = a.order.items[me];   // (the buffer holds gridDim.x of them)
    if (me >= items) return;
    const int per_cb = (a.vocab + kUpSpan - 1) / kUpSpan;
    const int c = (int)blockIdx.y / per_cb, first = ((int)blockIdx.y % per_cb) * kUpSpan + warp * kUpRows;
    const int adapter = item.x & 0xffff, len = item.x >> 16;
    const int row = a.order.rows[item.y + min(lane, len - 1)];
    const float *t_row = a.t + (size_t)__shfl_sync(kFull, row, g) * a.rank + 4 * k4;
    const __nv_bfloat16 *base = a.B + ((size_t)adapter * a.n_cb * a.rows_per_cb + (size_t)c * a.rows_per_cb) * a.rank + 4 * k4;
    const uint32_t ldo = (uint32_t)(a.n_cb * a.vocab);
    uint32_t to_row[kItem];
#pragma unroll
    for (int j = 0; j < kItem; j++) to_row[j] = (uint32_t)__shfl_sync(kFull, row, j);

    struct Parts {   // t's parts of 16 ranks, as the MMA's B
        uint32_t h[2], m[2], l[2];
    };
    auto parts = [&](int k, Parts &p) {
        const float4 t = k + 4 * k4 < a.rank ? *reinterpret_cast<const float4 *>(t_row + k) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        split3(t.x, t.y, p.h[0], p.m[0], p.l[0]);
        split3(t.z, t.w, p.h[1], p.m[1], p.l[1]);
    };
    auto rows_of_b = [&](int v0, int k, uint2 (&w)[kUpTiles][2]) {
        const bool in = k + 4 * k4 < a.rank && v0 < a.vocab;
        const __nv_bfloat16 *from = base + (uint32_t)((v0 + g) * a.rank + k);
#pragma unroll
        for (int i = 0; i < 2 * kUpTiles; i++, from += 8 * a.rank)
            w[i >> 1][i & 1] = in && v0 + 8 * i + g < a.vocab ? __ldg(reinterpret_cast<const uint2 *>(from)) : make_uint2(0u, 0u);
    };
    auto multiply = [&](const uint2 (&w)[kUpTiles][2], const Parts &p, float (&d)[kUpTiles][4], bool add) {
#pragma unroll
        for (int m = 0; m < kUpTiles; m++) {
            float e[4] = {};   // the tensor cores add by truncation: 16 ranks at a time, then rounded
            mma_16816(e, w[m][0].x, w[m][1].x, w[m][0].y, w[m][1].y, p.l[0], p.l[1]);
            mma_16816(e, w[m][0].x, w[m][1].x, w[m][0].y, w[m][1].y, p.m[0], p.m[1]);
            mma_16816(e, w[m][0].x, w[m][1].x, w[m][0].y, w[m][1].y, p.h[0], p.h[1]);
#pragma unroll
            for (int i = 0; i < 4; i++) d[m][i] = add ? d[m][i] + e[i] : e[i];
        }
    };
    Parts kept[KT ? KT : 1];
    uint2 w[KT ? KT : 1][kUpTiles][2];
#pragma unroll
    for (int k = 0; k < KT; k++) {
        rows_of_b(first, 16 * k, w[k]);
        parts(16 * k, kept[k]);
    }
    for (int step = 0; step < kUpSteps; step++) {
        const int v0 = first + step * kUpWarps * kUpRows;
        if (v0 >= a.vocab) break;
        float d[kUpTiles][4];
        if (KT) {
#pragma unroll
            for (int k = 0; k < KT; k++) {
                multiply(w[k], kept[k], d, k > 0);
                if (step + 1 < kUpSteps) rows_of_b(v0 + kUpWarps * kUpRows, 16 * k, w[k]);
            }
        } else {
            for (int k = 0; k < a.rank; k += 16) {
                rows_of_b(v0, k, w[0]);
                parts(k, kept[0]);
                multiply(w[0], kept[0], d, k > 0);
            }
        }
#pragma unroll
        for (int m = 0; m < kUpTiles; m++)
#pragma unroll
            for (int i = 0; i < 4; i++) s_turn[warp][2 * k4 + (i & 1)][16 * m + 8 * (i >> 1) + g] = d[m][i];
        __syncwarp();
        float *to = a.delta + (size_t)c * a.vocab + v0 + lane;
        const bool in0 = v0 + lane < a.vocab, in1 = v0 + 32 + lane < a.vocab;
#pragma unroll
        for (int j = 0; j < kItem; j++) {
            if (j >= len) continue;
            float *at = to + (size_t)to_row[j] * ldo;
            const float x = s_turn[warp][j][lane], y = s_turn[warp][j][32 + lane];
            if (in0) at[0] = x;
            if (in1) at[32] = y;
        }
        __syncwarp();
    }
}

// ---- the GEMM --------------------------------------------------------------
//
// Its operands trade places against the plain head's: the weight rows are the M of its
// tiles (TMEM lanes), the hidden rows the N (TMEM columns).  Few streams then fill the
// tile (N = 16 is enough) instead of leaving most of an M = 128 tile empty, and a warp's
// logits of one hidden row are 128 consecutive bytes.
//   warp 0       TMA producer of the weight and hidden tiles (128-byte swizzle);
//   warp 1       TMEM allocation, tcgen05.mma (M = 64, or 256 over a two-SM pair);
//   warp 2       (UNITS) brings the items to shared memory;
//   UNITS warps  delta, two items at a time, into the accumulator that the last part adds
//                to (two warps per TMEM lane quarter);
//   SUMS warps   the sums of the parts of the depth, delta (no UNITS), softcap, stores (two
//                or four warps per TMEM lane quarter, each its share of the columns).
// Every wait is bounded, as in head_tc.cu: a warp whose wait expires sets the error
// word, stops waiting and copying, and the CTA winds down (copies in flight waited
// for, TMEM freed).  No TMA load here uses cluster multicast.

constexpr int kBK = 64;             // bf16 elements per 128-byte swizzled row
constexpr int kSmallN = 64, kPairN = 256;   // hidden rows per tile (TMEM columns) at most
constexpr int kUnits = 8, kSmallSums = 8, kPairSums = 16;
// The pair kernel's five warp groups (roles, four of sums) split the launch's 5 * 96
// registers a thread as 32 + 4 * 112 = 480.  Spills are dear here, since shared memory leaves
// the L1 so little that a spilled value costs a trip to L2; 24 bytes of stores are left.
constexpr int kRoleRegs = 32, kSumRegs = 112;
constexpr int kGroup = 2;           // items that a unit warp works on at once
constexpr int kPitch = 36;          // floats per column of a warp's transposition (conflict-free)
constexpr int threads_of(int units, int sums) { return 32 * (4 + units + sums); }
constexpr int kKsub = 2;            // 64-deep slices per stage
constexpr int kMaxStages = 12;
constexpr int kMaxBufs = 4;
constexpr int kBars = 2 * kMaxStages + 3 * kMaxBufs + 1;
constexpr int kSmemMax = 232448;
// The tensor cores add to an f32 accumulator by truncation, which costs about
// depth * 2^-30 of the logits' size: 2e-6 over 2048.  The depth is therefore cut into
// parts of about this many 16-deep steps, summed in registers with rounding to
// nearest (0.7e-6 with three parts).
constexpr int kPartSteps = 48;

struct GemmArgs {
    int batch, n_cb, vocab, rows_per_cb, dim;
    int tiles_b, per_cb, n_tiles;
    int nb;                     // hidden rows per tile, a multiple of 16 (32 for a pair)
    int stages, parts, bufs, buf_cols, tmem_cols;
    float softcap;
    float *out;
    int cfg;
    float cfg_scale;
    const float *row_scale;
    const int32_t *which;
    int rows_per_id, n_adapters;
    const float *delta;         // (no UNITS) rows that name an adapter; may be out
    int rank;                   // (UNITS)
    uint32_t b_stride;          // elements of one adapter's B
    const __nv_bfloat16 *B;
    const float *t;             // [batch][rank]
    Order order;
};

// cap * tanh(l / cap) of N values: an odd polynomial (Taylor to y^11) below |y| = 0.35,
// where its remainder is under 2e-8 of the value, and cap - 2 cap / (exp(2 y) + 1) above,
// whose rounding (a few 2^-24 of cap) is small against the value there.  Where all of the
// warp's values are small, as an output head's mostly are, only the polynomial is
// computed, two values to an instruction.
template <int N>
__device__ __forceinline__ void softcap_exact(float (&l)[N], float cap)
{
    const float inv_cap = 1.0f / cap;
    float most = fabsf(l[0]);
#pragma unroll
    for (int i = 1; i < N; i++) most = fmaxf(most, fabsf(l[i]));
    const bool tiny = __all_sync(kFull, most * inv_cap < 0.35f);
    const float k2 = 2.0f * 1.4426950408889634f * inv_cap;
    auto both = [](float x) { return make_float2(x, x); };
#pragma unroll
    for (int i = 0; i < N; i += 2) {
        const float2 x = make_float2(l[i], l[i + 1]), y = __fmul2_rn(x, both(inv_cap)), z = __fmul2_rn(y, y);
        float2 p = __ffma2_rn(z, both(-1382.0f / 155925.0f), both(62.0f / 2835.0f));
        p = __ffma2_rn(z, p, both(-17.0f / 315.0f));
        p = __ffma2_rn(z, p, both(2.0f / 15.0f));
        p = __ffma2_rn(z, p, both(-1.0f / 3.0f));
        p = __ffma2_rn(__fmul2_rn(x, z), p, x);
        if (!tiny) {
            float e0, e1, r0, r1;
            asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e0) : "f"(x.x * k2));
            asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e1) : "f"(x.y * k2));
            asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r0) : "f"(e0 + 1.0f));
            asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r1) : "f"(e1 + 1.0f));
            if (!(fabsf(y.x) < 0.35f)) p.x = fmaf(-2.0f * cap, r0, cap);
            if (!(fabsf(y.y) < 0.35f)) p.y = fmaf(-2.0f * cap, r1, cap);
        }
        l[i] = p.x;
        l[i + 1] = p.y;
    }
}

__device__ __forceinline__ void tmem_ld8(uint32_t taddr, uint32_t *r)
{
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
                 : "r"(taddr));
}

__device__ __forceinline__ void tmem_st1(uint32_t taddr, float v)
{
    asm volatile("tcgen05.st.sync.aligned.32x32b.x1.b32 [%0], {%1};" ::"r"(taddr), "r"(__float_as_uint(v)) : "memory");
}

__device__ __forceinline__ uint4 lds_u4(uint32_t a)
{
    uint4 v;
    asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a));
    return v;
}
// Waits for the loads issued so far; their values pass through, so that no use of
// them moves ahead of the wait.
template <int N>
__device__ __forceinline__ void tmem_wait(uint32_t (&r)[N])
{
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
    for (int i = 0; i < N; i++) asm volatile("" : "+r"(r[i]));
}

__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// *p, or 0 without the load; a predicate, not a branch, so that a run of these is in
// flight together.
__device__ __forceinline__ float load_if(const float *p, bool yes)
{
    float v;
    asm volatile("{\n\t.reg .pred q;\n\tsetp.ne.u32 q, %2, 0;\n\tmov.f32 %0, 0f00000000;\n\t@q ld.global.f32 %0, [%1];\n\t}"
                 : "=f"(v) : "l"(p), "r"((uint32_t)yes) : "memory");
    return v;
}

// CTAS: 2 for a two-SM pair; BM: weight rows per CTA (TMEM lanes; 64 of them lie in the
// first 16 lanes of each quarter); NB: hidden rows per tile at most; UNITS: unit warps (a
// kernel with one tile of hidden rows), or 0; SUMS: sum warps.
template <int CTAS, int BM, int NB, int UNITS, int SUMS>
__global__ void __launch_bounds__(threads_of(UNITS, SUMS), 1)
    adapter_head_kernel(const __grid_constant__ CUtensorMap map_w,
                        const __grid_constant__ CUtensorMap map_h, const __grid_constant__ GemmArgs args)
{
    constexpr bool PAIR = CTAS == 2;
    constexpr uint32_t kWBytes = BM * kBK * 2;
    extern __shared__ __align__(1024) unsigned char smem_raw[];
    unsigned char *smem = reinterpret_cast<unsigned char *>(
        (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    const int nb_own = args.nb / CTAS;                  // hidden rows this CTA loads
    const uint32_t sub_bytes = kWBytes + (uint32_t)nb_own * kBK * 2;   // one slice of both operands
    const uint32_t stage_bytes = kKsub * sub_bytes;
    const int stages = args.stages, bufs = args.bufs;
    const uint32_t smem0 = smem_u32(smem);
    // after the stages: (UNITS) the items (16 bytes each) and their number, the unit warps'
    // transpositions
    unsigned char *tail = smem + (size_t)stages * stage_bytes;
    const uint32_t item0 = smem_u32(tail);
    int *s_items = reinterpret_cast<int *>(tail + 16 * max_items(NB, NB));
    float *s_turn = reinterpret_cast<float *>(s_items + 4);   // [UNITS][kGroup * kItem][kPitch]
    uint64_t *bars = UNITS ? reinterpret_cast<uint64_t *>(s_turn + UNITS * kGroup * kItem * kPitch)
                           : reinterpret_cast<uint64_t *>(tail);
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(bars + kBars);
    __shared__ int s_abort;

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = PAIR ? cluster_rank() : 0u;
    const int KB = (args.dim + kBK * kKsub - 1) / (kBK * kKsub);
    const int parts = args.parts, per_part = (KB + parts - 1) / parts;
    const uint32_t bar0 = smem_u32(bars);
    auto full = [&](int s) { return bar0 + 8u * (uint32_t)s; };
    auto empty = [&](int s) { return bar0 + 8u * (uint32_t)(kMaxStages + s); };
    auto done = [&](int b) { return bar0 + 8u * (uint32_t)(2 * kMaxStages + b); };                  // MMA -> sums
    auto open = [&](int b) { return bar0 + 8u * (uint32_t)(2 * kMaxStages + kMaxBufs + b); };   // -> MMA
    auto cleared = [&](int b) { return bar0 + 8u * (uint32_t)(2 * kMaxStages + 2 * kMaxBufs + b); };   // (UNITS) sums -> units
    const uint32_t ifull = bar0 + 8u * (uint32_t)(2 * kMaxStages + 3 * kMaxBufs);
    auto aborted = [&]() { return *(volatile int *)&s_abort != 0; };

    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    if (threadIdx.x == 0) {
        s_abort = 0;
        for (int s = 0; s < stages; s++) {
            mbar_init(full(s), 1);
            mbar_init(empty(s), 1);
        }
        for (int b = 0; b < bufs; b++) {
            mbar_init(done(b), 1);
            mbar_init(open(b), UNITS ? UNITS : CTAS * SUMS);
            mbar_init(cleared(b), SUMS);
        }
        mbar_init(ifull, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        prefetch_map(&map_w);
        prefetch_map(&map_h);
    }
    if (warp == 1) {
        if (PAIR) {
            asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(args.tmem_cols) : "memory");
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
        } else {
            asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(args.tmem_cols) : "memory");
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
        }
    }
    tc_fence_before();
    __syncthreads();
    if (PAIR) cluster_sync();
    tc_fence_after();
    const uint32_t tmem_base = *tmem_slot;
    const int unit0 = (int)blockIdx.x / CTAS, units = (int)gridDim.x / CTAS;
    // the tile's first hidden row, its codebook and this CTA's first weight row there
    auto tile_at = [&](int tile, int &b0, int &c, int &v0) {
        const int nt = tile / args.tiles_b;
        b0 = (tile - nt * args.tiles_b) * args.nb;
        c = nt / args.per_cb;
        v0 = (nt - c * args.per_cb) * (BM * CTAS) + (int)rank * BM;
    };

    // The hidden states and W were complete before the kernels that make delta started
    // (they wait for all work before them), so they are loaded at once; only the sum or the
    // unit warps wait for delta or t.
    //
    // A tile's depth is computed in `parts`, each in the next of `bufs` accumulators.  The sum
    // warps open an accumulator again once they have read it; with UNITS they only clear it,
    // and the unit warps open it, after storing delta there before a tile's last part.
    if constexpr (PAIR) {
        if (warp < 4) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRoleRegs));
    }
    if (warp == 0) {
        if (lane == 0) {
            int s = 0, used = 0;
            uint32_t ph = 0;
            bool ok = true;
            const uint32_t full0 = PAIR ? peer_addr(full(0), 0) : full(0);
            for (int tile = unit0; tile < args.n_tiles && ok; tile += units) {
                int b0, c, v0;
                tile_at(tile, b0, c, v0);
                const int w_row = c * args.rows_per_cb + v0, h_row = b0 + (int)rank * nb_own;
                for (int kb = 0; kb < KB; kb++) {
                    if (!mbar_wait(empty(s), ph ^ 1u) || aborted()) {
                        ok = false;
                        break;
                    }
                    const uint32_t sa = smem0 + (uint32_t)s * stage_bytes, fb = full0 + 8u * (uint32_t)s;
                    if (rank == 0) mbar_expect_tx(full(s), (uint32_t)CTAS * stage_bytes);
#pragma unroll
                    for (int j = 0; j < kKsub; j++) {
                        const int kx = (kb * kKsub + j) * kBK;
                        const uint32_t d = sa + (uint32_t)j * sub_bytes;
                        if (PAIR) {
                            tma_load_2d_pair(d, &map_w, kx, w_row, fb);
                            tma_load_2d_pair(d + kWBytes, &map_h, kx, h_row, fb);
                        } else {
                            tma_load_2d(d, &map_w, kx, w_row, fb);
                            tma_load_2d(d + kWBytes, &map_h, kx, h_row, fb);
                        }
                    }
                    used = min(used + 1, stages);
                    if (++s == stages) {
                        s = 0;
                        ph ^= 1u;
                    }
                }
            }
            if (!ok) {
                s_abort = 1;
                if (rank == 0)   // copies still in flight land first
                    for (int k = 0; k < used; k++) {
                        if (s == 0) {
                            s = stages;
                            ph ^= 1u;
                        }
                        s--;
                        mbar_wait(full(s), ph);
                    }
            }
        }
    } else if (warp == 1) {
        if (lane == 0 && rank == 0) {
            const uint32_t idesc = (1u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(args.nb >> 3) << 17) |
                                   ((uint32_t)((CTAS * BM) >> 4) << 24);
            int s = 0, buf = 0;
            uint32_t ph = 0, bph = 0;
            bool ok = true;
            const uint32_t empty1 = PAIR ? peer_addr(empty(0), 1) : 0u, done1 = PAIR ? peer_addr(done(0), 1) : 0u;
            for (int tile = unit0; tile < args.n_tiles && ok; tile += units) {
                for (int k0 = 0; k0 < KB && ok; k0 += per_part) {   // one part of the depth
                    const int k1 = min(k0 + per_part, KB);
                    if (!(PAIR ? mbar_wait_cl(open(buf), bph ^ 1u) : mbar_wait(open(buf), UNITS ? bph : bph ^ 1u))) {
                        ok = false;
                        break;
                    }
                    tc_fence_after();
                    const uint32_t d_tmem = tmem_base + (uint32_t)(buf * args.buf_cols);
                    const bool onto = UNITS && k1 == KB;   // the last part adds to delta
                    for (int kb = k0; kb < k1; kb++) {
                        if (!(PAIR ? mbar_wait_cl(full(s), ph) : mbar_wait(full(s), ph)) || aborted()) {
                            ok = false;
                            break;
                        }
                        tc_fence_after();
                        const uint32_t sa = smem0 + (uint32_t)s * stage_bytes;
#pragma unroll
                        for (int j = 0; j < kKsub; j++) {
                            const uint64_t wd = sw128_desc(sa + (uint32_t)j * sub_bytes);
                            const uint64_t hd = sw128_desc(sa + (uint32_t)j * sub_bytes + kWBytes);
#pragma unroll
                            for (int k = 0; k < kBK / 16; k++) {
                                const uint32_t more = onto || kb != k0 || (j | k) != 0;
                                if (PAIR)
                                    mma_bf16_pair(d_tmem, wd + (uint64_t)(2 * k), hd + (uint64_t)(2 * k), idesc, more);
                                else
                                    mma_bf16(d_tmem, wd + (uint64_t)(2 * k), hd + (uint64_t)(2 * k), idesc, more);
                            }
                        }
                        if (PAIR) {
                            mma_commit_pair(empty(s));
                            mma_commit_pair(empty1 + 8u * (uint32_t)s);
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
                            mma_commit_pair(done1 + 8u * (uint32_t)buf);
                        } else {
                            mma_commit(done(buf));
                        }
                    }
                    if (++buf == bufs) {
                        buf = 0;
                        bph ^= 1u;
                    }
                }
            }
            if (!ok) s_abort = 1;
        }
    } else if (UNITS && warp == 2) {
        // ---- items, 16 bytes each: the adapter, -, eight columns (the last one repeated)
        asm volatile("griddepcontrol.wait;" ::: "memory");   // t and the order are complete
        const int items = args.order.n_items[1];
        for (int i = lane; i < items; i += 32) {
            const int2 item = args.order.items[i];
            const int len = item.x >> 16;
            uint32_t col[2] = {0, 0};
#pragma unroll
            for (int j = 0; j < kItem; j++)
                col[j >> 2] |= (uint32_t)args.order.rows[item.y + min(j, len - 1)] << (8 * (j & 3));
            asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(item0 + 16u * (uint32_t)i), "r"(item.x & 0xffff), "r"(0),
                         "r"(col[0]), "r"(col[1])
                         : "memory");
        }
        if (lane == 0) *s_items = items;
        __syncwarp();
        if (lane == 0) mbar_arrive(ifull);
    } else if (UNITS && warp >= 4 && warp < 4 + UNITS) {
        // ---- units: opens the turns' accumulators
        const int q = warp & 3;             // the TMEM lane quarter this warp may access
        const int g = lane >> 2, k4 = lane & 3;
        constexpr int kTiles = BM / 64;     // 16-row tiles of the quarter
        constexpr int kStride = UNITS / 4 * kGroup;   // items until this warp's next group
        float *turn_mem = s_turn + (warp - 4) * kGroup * kItem * kPitch;
        int buf = 0, turn = 0;
        uint32_t bph = 0;
        bool ok = true;
        for (int tile = unit0; tile < args.n_tiles && ok; tile += units) {
            int b0, c, v0;
            tile_at(tile, b0, c, v0);
            // this lane's rows of each adapter's B: mma.sync's rows g and g + 8 of one or two
            // 16-row tiles; past the codebook any row will do
            int b_row[kTiles][2];
#pragma unroll
            for (int m = 0; m < kTiles; m++)
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    const int row = v0 + (BM / 4) * q + 16 * m + 8 * h + g;
                    b_row[m][h] = (c * args.rows_per_cb + (row < args.vocab ? row : 0)) * args.rank + 4 * k4;
                }
            for (int part = 0; part < parts; part++, turn++) {
                if (turn >= bufs) {   // its sums have been read
                    ok = mbar_wait(cleared(buf), bph ^ 1u) && !aborted();
                    ok = __all_sync(kFull, ok);
                    if (!ok) break;
                }
                tc_fence_after();
                const uint32_t tm = tmem_base + ((uint32_t)(32 * q) << 16) + (uint32_t)(buf * args.buf_cols);
                if (part == parts - 1) {
                    ok = mbar_wait(ifull, 0) && !aborted();   // once: every tile has the same rows
                    ok = __all_sync(kFull, ok);
                    if (!ok) break;
                    const int items = *(volatile int *)s_items;
                    // A step is 16 ranks of a group of items; two steps are in flight.  The ranks are
                    // permuted alike for both operands, so that a lane loads four neighbours: ranks
                    // 4 k4 .. 4 k4 + 3 of its rows of B, and of the t of each item's row g.
                    struct Step {
                        uint2 w[kGroup][kTiles][2];
                        float4 t[kGroup];
                    } step[2];
                    const int item1 = ((warp - 4) >> 2) * kGroup;   // this warp's first group
                    int fi = item1, fk = 0, left = 0;               // the next step to fetch; steps fetched, not used
                    auto fetch = [&](Step &s) {
                        if (fi >= items) return;
                        left++;
#pragma unroll
                        for (int n = 0; n < kGroup; n++) {
                            // past the last item: the last one again, with the same result
                            const uint4 item = lds_u4(item0 + 16u * (uint32_t)min(fi + n, items - 1));
                            const bool in = item.x != (uint32_t)kNone && fk + 4 * k4 < args.rank;
                            const uint32_t col = (g < 4 ? item.z : item.w) >> (8 * (g & 3)) & 255u;
                            const __nv_bfloat16 *from = args.B + (size_t)item.x * args.b_stride + fk;
#pragma unroll
                            for (int m = 0; m < kTiles; m++)
#pragma unroll
                                for (int h = 0; h < 2; h++)
                                    s.w[n][m][h] = in ? __ldg(reinterpret_cast<const uint2 *>(from + b_row[m][h])) : make_uint2(0u, 0u);
                            s.t[n] = in ? *reinterpret_cast<const float4 *>(args.t + (size_t)(b0 + (int)col) * args.rank + fk + 4 * k4)
                                        : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                        }
                        fk += 16;
                        if (fk >= args.rank) {
                            fk = 0;
                            fi += kStride;
                        }
                    };
                    int it = item1, k = 0;    // the step to use
                    float d[kGroup][kTiles][4] = {};
                    auto use = [&](const Step &s) {
                        left--;
#pragma unroll
                        for (int n = 0; n < kGroup; n++) {
                            uint32_t h0, h1, m0, m1, l0, l1;
                            split3(s.t[n].x, s.t[n].y, h0, m0, l0);
                            split3(s.t[n].z, s.t[n].w, h1, m1, l1);
#pragma unroll
                            for (int m = 0; m < kTiles; m++) {
                                const uint2 a = s.w[n][m][0], b = s.w[n][m][1];
                                float e[4] = {};   // steps are summed with rounding to nearest
                                mma_16816(e, a.x, b.x, a.y, b.y, l0, l1);
                                mma_16816(e, a.x, b.x, a.y, b.y, m0, m1);
                                mma_16816(e, a.x, b.x, a.y, b.y, h0, h1);
#pragma unroll
                                for (int i = 0; i < 4; i++) d[n][m][i] += e[i];
                            }
                        }
                        k += 16;
                    };
                    auto finish = [&]() {   // rows of the tile to lanes, through this warp's shared memory
#pragma unroll
                        for (int n = 0; n < kGroup; n++)
#pragma unroll
                            for (int m = 0; m < kTiles; m++)
#pragma unroll
                                for (int i = 0; i < 4; i++) {
                                    turn_mem[(n * kItem + 2 * k4 + (i & 1)) * kPitch + 16 * m + 8 * (i >> 1) + g] = d[n][m][i];
                                    d[n][m][i] = 0.0f;
                                }
                        uint4 item[kGroup];
#pragma unroll
                        for (int n = 0; n < kGroup; n++) item[n] = lds_u4(item0 + 16u * (uint32_t)min(it + n, items - 1));
                        __syncwarp();
                        float v[kGroup][kItem];
#pragma unroll
                        for (int n = 0; n < kGroup; n++)
#pragma unroll
                            for (int j = 0; j < kItem; j++) v[n][j] = turn_mem[(n * kItem + j) * kPitch + (BM == 64 ? lane & 15 : lane)];
#pragma unroll
                        for (int n = 0; n < kGroup; n++)
#pragma unroll
                            for (int j = 0; j < kItem; j++)
                                tmem_st1(tm + ((j < 4 ? item[n].z : item[n].w) >> (8 * (j & 3)) & 255u), v[n][j]);
                        __syncwarp();
                        k = 0;
                        it += kStride;
                    };
                    fetch(step[0]);
                    fetch(step[1]);
                    while (left) {
#pragma unroll
                        for (int n = 0; n < 2; n++) {
                            if (!left) break;
                            use(step[n]);
                            fetch(step[n]);
                            if (k >= args.rank) finish();
                        }
                    }
                }
                if (!ok) break;
                tmem_wait_st();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(open(buf));
                if (++buf == bufs) {
                    buf = 0;
                    bph ^= 1u;
                }
            }
        }
        if (!ok) s_abort = 1;
    } else if (warp >= 4 + UNITS) {
        if constexpr (PAIR) asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kSumRegs));
        // ---- sums, softcap, stores
        const int q = warp & 3;             // the TMEM lane quarter this warp may access
        const int share = (warp - 4 - UNITS) >> 2;   // its share of the tile's columns
        constexpr int kShares = SUMS / 4, kCols = NB / kShares;
        const int row = BM == 64 ? 16 * q + (lane & 15) : 32 * q + lane;
        const uint32_t open0 = PAIR ? peer_addr(open(0), 0) : open(0);
        const float cap = args.softcap;
        const size_t ldo = (size_t)args.n_cb * args.vocab;
        const int cols = args.nb / kShares;          // a multiple of 8
        int buf = 0;
        uint32_t bph = 0;
        bool ok = true, waited = false;
        for (int tile = unit0; tile < args.n_tiles && ok; tile += units) {
            int b0, c, v0;
            tile_at(tile, b0, c, v0);
            const bool valid = v0 + row < args.vocab && (BM == 128 || lane < 16);
            const size_t at_n = (size_t)c * args.vocab + v0 + row;
            const int first = b0 + share * cols, end = min(args.batch, first + cols);
            auto names = [&](int b) {   // whether hidden row b names an adapter
                if (b >= end) return false;
                const int a = __ldg(args.which + b / args.rows_per_id);
                return (unsigned)a < (unsigned)args.n_adapters;
            };
            float sum[kCols];
#pragma unroll
            for (int i = 0; i < kCols; i++) sum[i] = 0.0f;   // not live from tile to tile
            for (int part = 0; part < parts; part++) {
                if (!UNITS && part == parts - 1) {   // delta is complete; this warp's part of it goes towards L2
                    if (!waited) asm volatile("griddepcontrol.wait;" ::: "memory");
                    waited = true;
                    if (v0 + BM / 4 * q < args.vocab)
                        for (int i = lane; i < cols; i += 32)
                            if (names(first + i))
                                asm volatile("prefetch.global.L2 [%0];" ::"l"(args.delta + (size_t)(first + i) * ldo +
                                                                              (size_t)c * args.vocab + v0 + BM / 4 * q));
                }
                ok = mbar_wait(done(buf), bph) && !aborted();
                ok = __all_sync(kFull, ok);
                if (!ok) break;
                tc_fence_after();
                const uint32_t at = tmem_base + ((uint32_t)(32 * q) << 16) + (uint32_t)(buf * args.buf_cols + share * cols);
#pragma unroll
                for (int g = 0; g < kCols; g += 16) {
                    if (g >= cols) continue;
                    uint32_t v[16];
                    tmem_ld8(at + (uint32_t)g, v);
                    if (g + 8 < cols) tmem_ld8(at + (uint32_t)(g + 8), v + 8);
                    tmem_wait(v);
#pragma unroll
                    for (int j = 0; j < 16 && g + j < kCols; j++) sum[g + j] += __uint_as_float(v[j]);
                }
                // the accumulator has been read: it goes on before the stores below, which wait
                // for memory
                tc_fence_before();
                __syncwarp();
                if (lane == 0) {
                    if (UNITS)
                        mbar_arrive(cleared(buf));
                    else if (PAIR)
                        mbar_arrive_cluster_relaxed(open0 + 8u * (uint32_t)buf);
                    else
                        mbar_arrive(open(buf));
                }
                if (++buf == bufs) {
                    buf = 0;
                    bph ^= 1u;
                }
            }
            if (!ok) break;
            // kStep hidden rows at a time
            constexpr int kStep = 16;
#pragma unroll
            for (int g = 0; g < kCols; g += kStep) {
                const int b = first + g;
                if (g >= cols || b >= end) continue;
                float l[kStep];
                if (!UNITS) {
                    const uint32_t named = __ballot_sync(kFull, lane < kStep && g + lane < cols && names(b + lane));
                    const float *from = args.delta + (size_t)b * ldo + at_n;
#pragma unroll
                    for (int j = 0; j < kStep; j++, from += ldo) l[j] = load_if(from, (named >> j) & 1u && valid);
                }
#pragma unroll
                for (int j = 0; j < kStep; j++) l[j] = UNITS ? sum[g + j] : sum[g + j] + l[j];
                if (args.row_scale) {
#pragma unroll
                    for (int j = 0; j < kStep; j++) l[j] *= __ldg(args.row_scale + min(b + j, args.batch - 1));
                }
                if (cap > 0.0f) softcap_exact(l, cap);
                if (!valid) continue;
                const int n = min(min(kStep, cols - g), end - b);
                float *to = args.out + (args.cfg ? (size_t)(b >> 1) : (size_t)b) * ldo + at_n;
                if (args.cfg) {   // rows 2s, 2s + 1 (conditional, unconditional) are neighbours
#pragma unroll
                    for (int j = 0; j < kStep; j += 2, to += ldo)
                        if (j < n) *to = __fadd_rn(l[j + 1], __fmul_rn(args.cfg_scale, __fsub_rn(l[j], l[j + 1])));
                } else if (n == kStep) {
#pragma unroll
                    for (int j = 0; j < kStep; j++, to += ldo) *to = l[j];
                } else {
#pragma unroll
                    for (int j = 0; j < kStep; j++, to += ldo)
                        if (j < n) *to = l[j];
                }
            }
        }
        if (!UNITS && !waited) asm volatile("griddepcontrol.wait;" ::: "memory");
        if (!ok) s_abort = 1;
    }

    tc_fence_before();
    __syncthreads();
    if (PAIR) cluster_sync();
    tc_fence_after();
    if (warp == 1) {
        if (PAIR)
            asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(args.tmem_cols) : "memory");
        else
            asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(args.tmem_cols) : "memory");
    }
}

typedef void (*HeadKernel)(CUtensorMap, CUtensorMap, GemmArgs);

HeadKernel head_kernel(bool pair)
{
    return pair ? adapter_head_kernel<2, 128, kPairN, 0, kPairSums> : adapter_head_kernel<1, 64, kSmallN, kUnits, kSmallSums>;
}

// 2-D bf16 tensor map over rows x cols (cols contiguous), box box_cols x box_rows.
bool map_2d(CUtensorMap *m, const void *base, uint64_t rows, uint64_t cols, uint32_t box_rows,
            uint32_t box_cols, CUtensorMapSwizzle swizzle)
{
    EncodeTiledFn enc = encode_fn();
    if (!enc) return false;
    const cuuint64_t dims[2] = {cols, rows};
    const cuuint64_t strides[1] = {cols * 2};
    const cuuint32_t box[2] = {box_cols, box_rows};
    const cuuint32_t estr[2] = {1, 1};
    return enc(m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, const_cast<void *>(base), dims, strides, box,
               estr, CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
               CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

struct DeviceInfo {   // filled on a device's first launch
    bool ready = false;
    int sms = 0, pairs = 0;
};

cudaError_t device_info(DeviceInfo *out)
{
    static std::mutex mu;
    static DeviceInfo info[64];
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (dev < 0 || dev >= 64) return cudaErrorInvalidDevice;
    std::lock_guard<std::mutex> lk(mu);
    DeviceInfo &d = info[dev];
    if (!d.ready) {
        e = cudaDeviceGetAttribute(&d.sms, cudaDevAttrMultiProcessorCount, dev);
        for (int i = 0; i < 2 && e == cudaSuccess; i++)
            e = cudaFuncSetAttribute(head_kernel(i), cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemMax - 1024);
        if (e != cudaSuccess) return e;
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3((unsigned)(2 * (d.sms / 2)));
        cfg.blockDim = dim3(threads_of(0, kPairSums));
        cfg.dynamicSmemBytes = kSmemMax - 1024;
        cudaLaunchAttribute attr[1];
        attr[0].id = cudaLaunchAttributeClusterDimension;
        attr[0].val.clusterDim.x = 2;
        attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
        cfg.attrs = attr;
        cfg.numAttrs = 1;
        e = cudaOccupancyMaxActiveClusters(&d.pairs, head_kernel(true), &cfg);
        if (e != cudaSuccess) return e;
        if (d.pairs < 1) d.pairs = 1;
        d.ready = true;
    }
    *out = d;
    return cudaSuccess;
}

}  // namespace

cudaError_t launch_head_adapters_tc(const HeadArgs &h, const AdapterArgs &ad, cudaStream_t stream)
{
    const long long wide = (long long)h.n_cb * h.rows_per_cb;
    if (h.dim % 8 != 0 || ad.rank % 8 != 0 || ad.n_adapters > kMaxAdapters ||
        (uintptr_t)h.W % 16 || (uintptr_t)h.hidden % 16 || (uintptr_t)ad.A % 16 ||
        (uintptr_t)ad.B % 16 || wide * ad.rank > INT_MAX / 2)
        return cudaErrorNotSupported;
    const bool pair = h.batch > kSmallN;
    const long long up_blocks = h.n_cb * (((long long)h.vocab + kUpSpan - 1) / kUpSpan);   // a grid's y
    if (pair && up_blocks > 65535) return cudaErrorNotSupported;
    DeviceInfo dev;
    cudaError_t e = device_info(&dev);
    if (e != cudaSuccess) return e;

    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.stream = stream;
    cfg.attrs = attr;
    cfg.numAttrs = 1;

    // ---- t and the rows' order; delta
    float *t = static_cast<float *>(ad.work);
    Order order;
    order.rows = reinterpret_cast<int32_t *>(t + (size_t)h.batch * ad.rank);
    order.n_items = order.rows + (h.batch + 1) / 2 * 2;
    order.items = reinterpret_cast<int2 *>(order.n_items + 2);
    DownArgs d{static_cast<const __nv_bfloat16 *>(h.hidden), static_cast<const __nv_bfloat16 *>(ad.A),
               ad.scale, ad.which, h.batch, h.dim, ad.n_adapters, ad.rank, ad.rows_per_id, t, order, 0};
    const unsigned order_blocks = (unsigned)((h.batch + kOrderRows - 1) / kOrderRows);
    cfg.dynamicSmemBytes = order_bytes(ad.n_adapters);
    if ((long long)h.batch * ad.rank <= kFewMost) {
        d.order_blocks = (int)order_blocks;
        cfg.gridDim = dim3(order_blocks + (unsigned)(h.batch * (ad.rank / 4)));
        cfg.blockDim = dim3(32 * kFewWarps);
        e = cudaLaunchKernelEx(&cfg, adapter_down_few_kernel, d);
    } else {
        cfg.gridDim = dim3(order_blocks);
        cfg.blockDim = dim3(256);
        e = cudaLaunchKernelEx(&cfg, order_rows_kernel, ad.which, h.batch, ad.rows_per_id, ad.n_adapters, order);
        if (e != cudaSuccess) return e;
        cfg.gridDim = dim3((unsigned)((h.batch + kDownRows - 1) / kDownRows), (unsigned)((ad.rank + kDownRank - 1) / kDownRank));
        cfg.blockDim = dim3(32 * kDownWarps);
        cfg.dynamicSmemBytes = 0;
        e = cudaLaunchKernelEx(&cfg, adapter_down_mma_kernel, d);
    }
    if (e != cudaSuccess) return e;
    float *delta = ad.delta ? ad.delta : h.out;
    if (pair) {
        const UpArgs u{static_cast<const __nv_bfloat16 *>(ad.B), t, order, h.n_cb, h.vocab, h.rows_per_cb, ad.rank, delta};
        cfg.gridDim = dim3((unsigned)max_items(h.batch, ad.n_adapters), (unsigned)up_blocks);
        cfg.blockDim = dim3(32 * kUpWarps);
        cfg.dynamicSmemBytes = 0;
        e = ad.rank <= 16   ? cudaLaunchKernelEx(&cfg, adapter_up_kernel<1>, u)
            : ad.rank <= 32 ? cudaLaunchKernelEx(&cfg, adapter_up_kernel<2>, u)
                            : cudaLaunchKernelEx(&cfg, adapter_up_kernel<0>, u);
        if (e != cudaSuccess) return e;
    }

    // ---- the GEMM: 64 weight rows per CTA up to 64 hidden rows; pairs of CTAs beyond, in
    // two tiles or more (the model's 36 x 256 weight rows then give nearly every SM one)
    const int bm = pair ? 128 : 64;         // weight rows per CTA
    const int m = pair ? 2 * bm : bm;
    const int n_max = pair ? kPairN : kSmallN;
    GemmArgs g{};
    g.tiles_b = (h.batch + n_max - 1) / n_max;
    if (pair && g.tiles_b < 2) g.tiles_b = 2;
    const int even = (h.batch + g.tiles_b - 1) / g.tiles_b, step = pair ? 32 : 16;
    g.nb = (even + step - 1) / step * step;
    g.tiles_b = (h.batch + g.nb - 1) / g.nb;
    g.batch = h.batch;
    // codebooks whose rows follow each other without a gap are one run of rows
    const bool joined = h.rows_per_cb == h.vocab;
    g.n_cb = joined ? 1 : h.n_cb;
    g.vocab = joined ? (int)wide : h.vocab;
    g.rows_per_cb = joined ? (int)wide : h.rows_per_cb;
    g.dim = h.dim;
    g.per_cb = (g.vocab + m - 1) / m;
    g.n_tiles = g.tiles_b * g.n_cb * g.per_cb;
    g.softcap = h.softcap;
    g.out = h.out;
    g.cfg = h.cfg;
    g.cfg_scale = h.cfg_scale;
    g.row_scale = h.row_scale;
    g.which = ad.which;
    g.rows_per_id = ad.rows_per_id;
    g.n_adapters = ad.n_adapters;
    g.delta = delta;
    g.rank = ad.rank;
    g.b_stride = (uint32_t)(wide * ad.rank);
    g.B = static_cast<const __nv_bfloat16 *>(ad.B);
    g.t = t;
    g.order = order;
    const int nb_own = pair ? g.nb / 2 : g.nb;
    const int stage = kKsub * (bm + nb_own) * kBK * 2;
    const int kb = (h.dim + kKsub * kBK - 1) / (kKsub * kBK);
    g.parts = (h.dim / 16 + kPartSteps - 1) / kPartSteps;
    if (g.parts < 1) g.parts = 1;
    g.parts = (kb + (kb + g.parts - 1) / g.parts - 1) / ((kb + g.parts - 1) / g.parts);   // none empty
    g.buf_cols = (g.nb + 31) / 32 * 32;
    g.bufs = 512 / g.buf_cols < kMaxBufs ? 512 / g.buf_cols : kMaxBufs;
    if (g.bufs > g.parts + 1) g.bufs = g.parts + 1;
    g.tmem_cols = 32;
    while (g.tmem_cols < g.bufs * g.buf_cols) g.tmem_cols *= 2;
    // beside the stages: alignment, barriers, the TMEM slot, what the unit warps keep
    const int fixed = 1024 + 8 * kBars + 64 +
                      (pair ? 0 : 16 * max_items(kSmallN, kSmallN) + 16 + 4 * kUnits * kGroup * kItem * kPitch);
    g.stages = (kSmemMax - 1024 - fixed) / stage;
    if (g.stages > kMaxStages) g.stages = kMaxStages;

    CUtensorMap mw, mh;
    if (!map_2d(&mw, h.W, (uint64_t)wide, (uint64_t)h.dim, (uint32_t)bm, kBK, CU_TENSOR_MAP_SWIZZLE_128B) ||
        !map_2d(&mh, h.hidden, (uint64_t)h.batch, (uint64_t)h.dim, (uint32_t)nb_own, kBK, CU_TENSOR_MAP_SWIZZLE_128B))
        return cudaErrorInvalidValue;
    cfg.blockDim = dim3((unsigned)(pair ? threads_of(0, kPairSums) : threads_of(kUnits, kSmallSums)));
    cfg.dynamicSmemBytes = (size_t)(g.stages * stage + fixed);
    if (!pair) {
        cfg.gridDim = dim3((unsigned)(g.n_tiles < dev.sms ? g.n_tiles : dev.sms));
    } else {
        attr[1].id = cudaLaunchAttributeClusterDimension;
        attr[1].val.clusterDim.x = 2;
        attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
        cfg.numAttrs = 2;
        cfg.gridDim = dim3((unsigned)(2 * (g.n_tiles < dev.pairs ? g.n_tiles : dev.pairs)));
    }
    return cudaLaunchKernelEx(&cfg, head_kernel(pair), mw, mh, g);
}

}  // namespace z2
