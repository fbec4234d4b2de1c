// head_adapters_tc.cu -- the bf16 output head beside low-rank adapters on the
// tcgen05 tensor cores (sm_100a).
//
//     t[b]         = s_a * (A_a h[b])
//     logits[b, n] = softcap(W[n] . h[b] + B_a[n] . t[b])
//
// A small kernel (two for a large batch) makes t (f32) and orders each tile's hidden
// rows by adapter; adapter_head_kernel is the GEMM, whose accumulators start from B_a t.
//
// The GEMM's operands trade places against the plain head's: the weight rows are
// the M of its tiles (TMEM lanes), the hidden rows the N (TMEM columns).  Few
// streams then fill the tile (N = 16 is enough) instead of leaving most of an
// M = 128 tile empty, and a warp's logits of one hidden row are 128 consecutive
// bytes.
//
// The low-rank product is made beside the main loop by four warps of their own, with
// mma.sync on at most eight hidden rows of one adapter at a time, and stored in the
// accumulator that the last part of the tile's depth adds to.  t enters it as three
// bf16 parts, which hold all of its 24 bits: B t is as good as in f32.  As extra depth
// of the main MMAs every adapter of a tile would cost a full-size step (and an
// infinity in one adapter would reach the other rows' logits as inf * 0); on the FMA
// pipe, t's values would have to be broadcast from shared memory (16 B per 512 B of
// register writes), which took longer than the main loop itself.
//
// Warp roles (16 warps):
//   warp 0       TMA producer of the weight and hidden tiles (128-byte swizzle);
//   warp 1       TMEM allocation, tcgen05.mma (M = 64 or 128, or 256 over a two-SM pair);
//   warp 2       cuts the tile's ordered rows into items (up to eight rows of one
//                adapter).  It alone waits for the kernel that makes t and the order
//                (griddepcontrol.wait): the GEMM's main loop overlaps that kernel;
//   warps 4..7   B t into TMEM, an item at a time (one warp per lane quarter);
//   warps 8..15  the sums of the parts of the depth, softcap, stores.
// Every wait is bounded, as in head_tc.cu: a warp whose wait expires sets the error
// word, stops waiting and copying, and the CTA winds down (copies in flight waited
// for, TMEM freed).
// No TMA load here uses cluster multicast.
#include <cuda_bf16.h>
#include <limits.h>
#include <math.h>

#include "common.cuh"
#include "head_adapters.cuh"
#include "tc.cuh"

namespace z2 {

int read_and_clear_adapter_error(int *value) { return take_device_error(value); }

namespace {

// ---- the rows' order ---------------------------------------------------------

constexpr int kMaxN = 256;          // hidden rows per tile (TMEM columns) at most
constexpr int kMaxAdapters = 4096;
constexpr uint32_t kNone = 0xffffffu;   // the key of a row without an adapter: last

// The entries (key << 8) | column of a tile's rows, ascending: thread i ranks its rows
// by counting.  *place and *group: the row's place, and the place of its key's first row.
__device__ __forceinline__ uint32_t row_entry(const int32_t *which, int rows_per_id, int n_adapters,
                                              int b0, int col)
{
    const int a = __ldg(which + (b0 + col) / rows_per_id);
    return ((unsigned)a < (unsigned)n_adapters ? (uint32_t)a << 8 : kNone << 8) | (uint32_t)col;
}

__device__ __forceinline__ void rank_entry(const uint32_t *s_entry, int rows, uint32_t mine, int *place,
                                           int *group)
{
    int n = 0, m = 0;
    const uint32_t key = mine & ~255u;
    for (int i = 0; i < rows; i += 4) {   // entries past the rows are all ones: none is smaller
        const uint4 e = *reinterpret_cast<const uint4 *>(s_entry + i);
        n += (e.x < mine) + (e.y < mine) + (e.z < mine) + (e.w < mine);
        m += (e.x < key) + (e.y < key) + (e.z < key) + (e.w < key);
    }
    *place = n;
    *group = m;
}

// One CTA per tile: list[b0 ..] = the tile's entries in order, and the rows' places in
// the order of the whole batch by (adapter, row): order[place] = row.
constexpr int kOrderThreads = 256;

__global__ void __launch_bounds__(kOrderThreads)
    order_rows_kernel(const int32_t *__restrict__ which, int batch, int nb, int rows_per_id,
                      int n_adapters, uint32_t *__restrict__ list, int32_t *__restrict__ order)
{
    extern __shared__ int s_count[];   // [n + 1] rows of each key (n: none), then [n + 1] before this tile
    __shared__ int s_part[kOrderThreads / 32];
    __shared__ __align__(16) uint32_t s_entry[kMaxN];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, n = n_adapters;
    const int b0 = (int)blockIdx.x * nb, rows = min(nb, batch - b0);
    int *before = s_count + n + 1;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    for (int i = tid; i < 2 * (n + 1); i += kOrderThreads) s_count[i] = 0;
    s_entry[tid] = tid < rows ? row_entry(which, rows_per_id, n, b0, tid) : ~0u;
    __syncthreads();
#pragma unroll 4
    for (int i = tid; i < batch; i += kOrderThreads) {
        const int a = __ldg(which + i / rows_per_id), k = (unsigned)a < (unsigned)n ? a : n;
        atomicAdd(&s_count[k], 1);
        if (i < b0) atomicAdd(&before[k], 1);
    }
    __syncthreads();
    // the first place of each key in the whole order
    const int per = (n + kOrderThreads) / kOrderThreads;
    const int a0 = min(tid * per, n + 1), a1 = min(a0 + per, n + 1);
    int own = 0;
    for (int a = a0; a < a1; a++) own += s_count[a];
    int sum = own;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int t = __shfl_up_sync(kFull, sum, o);
        if (lane >= o) sum += t;
    }
    if (lane == 31) s_part[warp] = sum;
    __syncthreads();
    int base = sum - own;
    for (int w = 0; w < warp; w++) base += s_part[w];
    for (int a = a0; a < a1; a++) {
        const int c = s_count[a];
        s_count[a] = base;
        base += c;
    }
    __syncthreads();
    if (tid < rows) {
        const uint32_t mine = s_entry[tid];
        int place, group;
        rank_entry(s_entry, rows, mine, &place, &group);
        list[b0 + place] = mine;
        const int k = (mine >> 8) == kNone ? n : (int)(mine >> 8);
        order[s_count[k] + before[k] + place - group] = b0 + tid;
    }
}

// ---- t = s_a A_a h ---------------------------------------------------------

struct DownArgs {
    const __nv_bfloat16 *hidden, *A;
    const float *scale;
    const int32_t *which, *order;   // order: the rows by adapter (many rows only)
    int batch, dim, n_adapters, rank, rows_per_id;
    float *t;                       // [batch][rank]
    uint32_t *list;                 // [batch] the tiles' entries (few rows only)
    int nb, down_blocks;            // rows per tile; blocks before those that order the tiles
};

// Few rows: one warp per row and four ranks, which share the row's loads; the last
// blocks order one tile's rows each.
constexpr int kFewWarps = 4;
constexpr long long kFewMost = 8192;   // rows x ranks

__global__ void __launch_bounds__(32 * kFewWarps) adapter_down_few_kernel(const DownArgs g)
{
    const int lane = threadIdx.x & 31, quads = (g.rank + 3) / 4;
    const long long i = (long long)blockIdx.x * kFewWarps + (threadIdx.x >> 5);
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    if ((int)blockIdx.x >= g.down_blocks) {
        __shared__ __align__(16) uint32_t s_entry[kMaxN];
        const int b0 = ((int)blockIdx.x - g.down_blocks) * g.nb, rows = min(g.nb, g.batch - b0);
        for (int j = threadIdx.x; j < kMaxN; j += 32 * kFewWarps)
            s_entry[j] = j < rows ? row_entry(g.which, g.rows_per_id, g.n_adapters, b0, j) : ~0u;
        __syncthreads();
        for (int j = threadIdx.x; j < rows; j += 32 * kFewWarps) {
            int place, group;
            rank_entry(s_entry, rows, s_entry[j], &place, &group);
            g.list[b0 + place] = s_entry[j];
        }
        return;
    }
    if (i >= (long long)g.batch * quads) return;
    const int b = (int)(i / quads), r0 = 4 * (int)(i % quads);
    const int a = __ldg(g.which + b / g.rows_per_id);
    if ((unsigned)a >= (unsigned)g.n_adapters) return;
    const uint4 *x = reinterpret_cast<const uint4 *>(g.hidden + (size_t)b * g.dim);
    const uint4 *w = reinterpret_cast<const uint4 *>(g.A + ((size_t)a * g.rank + r0) * g.dim);
    const int n = g.dim / 8;   // rank is a multiple of 8: the four ranks exist
    float acc[4] = {};
#pragma unroll 2
    for (int k = lane; k < n; k += 32) {
        const uint4 xv = __ldg(x + k);
        const uint32_t xs[4] = {xv.x, xv.y, xv.z, xv.w};
#pragma unroll
        for (int r = 0; r < 4; r++) {
            const uint4 wv = __ldg(w + (size_t)r * n + k);
            const uint32_t ws[4] = {wv.x, wv.y, wv.z, wv.w};
#pragma unroll
            for (int j = 0; j < 4; j++) {
                acc[r] = fmaf(__uint_as_float(xs[j] << 16), __uint_as_float(ws[j] << 16), acc[r]);
                acc[r] = fmaf(__uint_as_float(xs[j] & 0xffff0000u), __uint_as_float(ws[j] & 0xffff0000u), acc[r]);
            }
        }
    }
#pragma unroll
    for (int r = 0; r < 4; r++)
#pragma unroll
        for (int o = 16; o; o >>= 1) acc[r] += __shfl_xor_sync(kFull, acc[r], o);
    const float s = g.scale ? __ldg(g.scale + a) : 1.0f;
    if (lane == 0)
        *reinterpret_cast<float4 *>(g.t + (size_t)b * g.rank + r0) = make_float4(s * acc[0], s * acc[1], s * acc[2], s * acc[3]);
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
__global__ void __launch_bounds__(32 * kDownWarps, 2) adapter_down_mma_kernel(const DownArgs g)
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
            row = __ldg(g.order + p0 + tid);
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
#pragma unroll 2
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

// ---- the GEMM --------------------------------------------------------------

constexpr int kBK = 64;             // bf16 elements per 128-byte swizzled row
constexpr int kSumWarps = 8;
// With 256 hidden rows per tile a sum warp holds 128 sums per thread.  The four warp
// groups (roles, units, sums, sums) then split the launch's 4 * 128 registers a thread as
// 80 + 128 + 2 * 152 = 512.
constexpr int kRoleRegs = 80, kSumRegs = 152;
constexpr int kItem = 8;            // hidden rows per item at most
constexpr int kGroup = 2;           // items that a unit warp works on at once
constexpr int kPitch = 36;          // floats per column of a warp's transposition (conflict-free)
constexpr int kMaxStages = 12;
constexpr int kMaxBufs = 4;
constexpr int kBars = 2 * kMaxStages + 3 * kMaxBufs + 2;
constexpr int kSmemMax = 232448;
// The tensor cores add to an f32 accumulator by truncation, which costs about
// depth * 2^-30 of the logits' size: 2e-6 over 2048.  The depth is therefore cut into
// parts of about this many 16-deep steps, summed in registers with rounding to
// nearest (0.7e-6 with three parts).
constexpr int kPartSteps = 48;

struct GemmArgs {
    int batch, n_cb, vocab, rows_per_cb, dim, wide;   // wide: n_cb * rows_per_cb of the caller
    int tiles_b, per_cb, n_tiles;
    int nb;                     // hidden rows per tile, a multiple of 16 (32 for a pair)
    int stages, parts, bufs, buf_cols, tmem_cols;
    float softcap;
    float *out;
    int cfg;
    float cfg_scale;
    const float *row_scale;
    int rank;
    const __nv_bfloat16 *B;
    const float *t;             // [batch][rank]
    const uint32_t *list;       // [batch] the tiles' rows in order: (adapter << 8) | column
};

// cap * tanh(l / cap): an odd polynomial (Taylor to y^11) below |y| = 0.35, where its
// remainder is under 2e-8 of the value, and cap - 2 cap / (exp(2 y) + 1) above, whose
// rounding (a few 2^-24 of cap) is small against the value there.
__device__ __forceinline__ float softcap_exact(float l, float cap, float inv_cap, float k2)
{
    const float y = l * inv_cap, z = y * y;
    float p = fmaf(z, -1382.0f / 155925.0f, 62.0f / 2835.0f);
    p = fmaf(z, p, -17.0f / 315.0f);
    p = fmaf(z, p, 2.0f / 15.0f);
    p = fmaf(z, p, -1.0f / 3.0f);
    const float small = fmaf(l * z, p, l);
    float e, r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(l * k2));
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(e + 1.0f));
    const float large = fmaf(-2.0f * cap, r, cap);
    return fabsf(y) < 0.35f ? small : large;
}

__device__ __forceinline__ void tmem_st1(uint32_t taddr, float v)
{
    asm volatile("tcgen05.st.sync.aligned.32x32b.x1.b32 [%0], {%1};" ::"r"(taddr), "r"(__float_as_uint(v)) : "memory");
}

__device__ __forceinline__ void tmem_ld8(uint32_t taddr, uint32_t *r)
{
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
                 : "r"(taddr));
}

__device__ __forceinline__ void tmem_st8(uint32_t taddr, const float *v)
{
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"r"(taddr),
                 "r"(__float_as_uint(v[0])), "r"(__float_as_uint(v[1])), "r"(__float_as_uint(v[2])),
                 "r"(__float_as_uint(v[3])), "r"(__float_as_uint(v[4])), "r"(__float_as_uint(v[5])),
                 "r"(__float_as_uint(v[6])), "r"(__float_as_uint(v[7]))
                 : "memory");
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

// x = hi + mid + lo in bf16, exactly but for bits below 2^-25 of x; two values to a
// register, the first in the low half.
__device__ __forceinline__ uint32_t pack_bf16(float x, float y)
{
    uint32_t r;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(y), "f"(x));
    return r;
}
__device__ __forceinline__ uint4 lds_u4(uint32_t a)
{
    uint4 v;
    asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a));
    return v;
}
__device__ __forceinline__ void split3(float x, float y, uint32_t &hi, uint32_t &mid, uint32_t &lo)
{
    hi = pack_bf16(x, y);
    x -= __uint_as_float(hi << 16);
    y -= __uint_as_float(hi & 0xffff0000u);
    mid = pack_bf16(x, y);
    x -= __uint_as_float(mid << 16);
    y -= __uint_as_float(mid & 0xffff0000u);
    lo = pack_bf16(x, y);
}

// Threads: four role warps, UNITS unit warps, the sum warps.
constexpr int threads_of(int units) { return 32 * (4 + units + kSumWarps); }

// CTAS: 2 for a two-SM pair; BM: weight rows per CTA (TMEM lanes; 64 of them lie in the
// first 16 lanes of each quarter); NB: hidden rows per tile at most; UNITS: unit warps
// (4 or 8: one or two per lane quarter).
// A sum warp holds NB / 2 sums per thread.  Nothing may spill: shared memory leaves the
// L1 so little that a spilled value costs a trip to L2.
template <int CTAS, int BM, int NB, int UNITS>
__global__ void __launch_bounds__(threads_of(UNITS), 1)
    adapter_head_kernel(const __grid_constant__ CUtensorMap map_w,
                        const __grid_constant__ CUtensorMap map_h, const __grid_constant__ GemmArgs args)
{
    constexpr bool PAIR = CTAS == 2;
    constexpr uint32_t kWBytes = BM * kBK * 2;
    constexpr int kKsub = PAIR ? 1 : 2;                 // 64-deep slices per stage
    extern __shared__ __align__(1024) unsigned char smem_raw[];
    unsigned char *smem = reinterpret_cast<unsigned char *>(
        (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    const int nb_own = args.nb / CTAS;                  // hidden rows this CTA loads
    const uint32_t sub_bytes = kWBytes + (uint32_t)nb_own * kBK * 2;   // one slice of both operands
    const uint32_t stage_bytes = kKsub * sub_bytes;
    const int stages = args.stages, bufs = args.bufs;
    const uint32_t smem0 = smem_u32(smem);
    // after the stages: the tile's items (16 bytes each) and their number, the unit warps'
    // transpositions
    unsigned char *tail = smem + (size_t)stages * stage_bytes;
    const uint32_t item0 = smem_u32(tail);
    uint32_t *s_items = reinterpret_cast<uint32_t *>(tail + 16 * NB);
    float *s_turn = reinterpret_cast<float *>(s_items + 4);   // [UNITS][kGroup * kItem][kPitch]
    uint64_t *bars = reinterpret_cast<uint64_t *>(s_turn + UNITS * kGroup * kItem * kPitch);
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
    auto open = [&](int b) { return bar0 + 8u * (uint32_t)(2 * kMaxStages + kMaxBufs + b); };       // -> MMA
    auto cleared = [&](int b) { return bar0 + 8u * (uint32_t)(2 * kMaxStages + 2 * kMaxBufs + b); };   // sums -> units
    const uint32_t ifull = bar0 + 8u * (uint32_t)(2 * kMaxStages + 3 * kMaxBufs), iempty = ifull + 8u;
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
            mbar_init(open(b), CTAS * UNITS);
            mbar_init(cleared(b), kSumWarps);
        }
        mbar_init(ifull, 1);
        mbar_init(iempty, UNITS);
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

    // The hidden states and W were complete before the kernel that makes t started (it
    // waits for all work before it), so the roles below use them at once; only the adapter
    // producer waits for t and the rows' order.
    //
    // A tile's depth is computed in `parts`, each in the next of `bufs` accumulators.  A
    // turn (part) may start in an accumulator when the unit warps open it: the sum warps
    // clear it first, and before a tile's last part the unit warps store B t there.
    if (warp < 4) {
        if constexpr (NB == kMaxN) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRoleRegs));
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
                        if (!(PAIR ? mbar_wait_cl(open(buf), bph) : mbar_wait(open(buf), bph))) {
                            ok = false;
                            break;
                        }
                        tc_fence_after();
                        const uint32_t d_tmem = tmem_base + (uint32_t)(buf * args.buf_cols);
                        const bool onto = k1 == KB;   // the last part adds to the low-rank product
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
        } else if (warp == 2) {
            // ---- items, 16 bytes each: adapter, rows, their columns in a byte each
            asm volatile("griddepcontrol.wait;" ::: "memory");   // t and the order are complete
            bool ok = true;
            uint32_t ph = 0;
            for (int tile = unit0; tile < args.n_tiles && ok; tile += units, ph ^= 1u) {
                int b0, c, v0;
                tile_at(tile, b0, c, v0);
                const int rows = min(args.nb, args.batch - b0);
                if (lane == 0) ok = mbar_wait(iempty, ph ^ 1u) && !aborted();
                __syncwarp();
                ok = __shfl_sync(kFull, ok, 0);
                if (!ok) break;
                int items = 0;
                for (int p0 = 0; p0 < rows; p0 += 32) {
                    const int p = p0 + lane, count = min(32, rows - p0);
                    const uint32_t entry = lane < count ? args.list[b0 + p] : ~0u, key = entry >> 8;
                    const uint32_t before = __shfl_up_sync(kFull, key, 1);
                    const bool start = lane < count && (lane % kItem == 0 || key != before);
                    const uint32_t starts = __ballot_sync(kFull, start);
                    const uint32_t upto = starts & (0xffffffffu >> (31 - lane));   // starts at or before this lane
                    const int first = 31 - __clz(upto);
                    const uint32_t at = item0 + 16u * (uint32_t)(items + __popc(upto) - 1);
                    if (lane < count)
                        asm volatile("st.shared.b8 [%0], %1;" ::"r"(at + 8u + (uint32_t)(lane - first)), "r"(entry & 255u) : "memory");
                    if (start) {
                        const uint32_t rest = starts >> lane >> 1;
                        const int len = rest ? __ffs(rest) : count - lane;
                        asm volatile("st.shared.v2.b32 [%0], {%1, %2};" ::"r"(at), "r"(key), "r"(len) : "memory");
                    }
                    items += __popc(starts);
                }
                if (lane == 0) *s_items = (uint32_t)items;
                __syncwarp();
                if (lane == 0) mbar_arrive(ifull);
            }
            if (!ok && lane == 0) s_abort = 1;
            __syncwarp();
        }
    } else if (warp < 4 + UNITS) {
        // ---- units: opens the turns' accumulators
        const int q = warp & 3;             // the TMEM lane quarter this warp may access
        const int g = lane >> 2, k4 = lane & 3;
        constexpr int kTiles = BM / 64;     // 16-row tiles of the quarter
        constexpr int kStride = UNITS / 4 * kGroup;   // items until this warp's next group
        float *turn_mem = s_turn + (warp - 4) * kGroup * kItem * kPitch;
        const uint32_t open0 = PAIR ? peer_addr(open(0), 0) : open(0);
        int buf = 0, turn = 0;
        uint32_t bph = 0, iph = 0;
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
                    ok = mbar_wait(ifull, iph) && !aborted();
                    ok = __all_sync(kFull, ok);
                    if (!ok) break;
                    iph ^= 1u;
                    const int items = (int)*(volatile uint32_t *)s_items;
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
                            const uint4 item = lds_u4(item0 + 16u * (uint32_t)min(fi + n, items - 1));
                            const bool in = item.x != kNone && fi + n < items && fk + 4 * k4 < args.rank;
                            const int r = min(g, (int)item.y - 1);
                            const uint32_t col = (r < 4 ? item.z : item.w) >> (8 * (r & 3)) & 255u;
                            const __nv_bfloat16 *from = args.B + (size_t)item.x * args.wide * args.rank + fk;
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
                                if (it + n < items && j < (int)item[n].y)
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
                    __syncwarp();
                    if (lane == 0) mbar_arrive(iempty);
                }
                if (!ok) break;
                tmem_wait_st();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) {
                    if (PAIR)
                        mbar_arrive_cluster(open0 + 8u * (uint32_t)buf);
                    else
                        mbar_arrive(open(buf));
                }
                if (++buf == bufs) {
                    buf = 0;
                    bph ^= 1u;
                }
            }
        }
        if (!ok) s_abort = 1;
    } else {
        if constexpr (NB == kMaxN) asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kSumRegs));
        // ---- sums, softcap, stores
        const int q = warp & 3;             // the TMEM lane quarter this warp may access
        const int half = (warp - 4 - UNITS) >> 2;   // its half of the tile's columns
        const int row = BM == 64 ? 16 * q + (lane & 15) : 32 * q + lane;
        const float cap = args.softcap, inv_cap = 1.0f / cap, k2 = 2.0f * 1.4426950408889634f / cap;
        const long long ldo = (long long)args.n_cb * args.vocab;
        const int cols = args.nb / 2;       // a multiple of 8
        int buf = 0;
        uint32_t bph = 0;
        bool ok = true;
        for (int tile = unit0; tile < args.n_tiles && ok; tile += units) {
            int b0, c, v0;
            tile_at(tile, b0, c, v0);
            const uint32_t lanes = tmem_base + ((uint32_t)(32 * q) << 16) + (uint32_t)(half * cols);
            auto clear = [&]() {   // the accumulator has been read: hand it on, go to the next
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(cleared(buf));
                if (++buf == bufs) {
                    buf = 0;
                    bph ^= 1u;
                }
            };
            {
                float sum[NB / 2];
#pragma unroll
                for (int i = 0; i < NB / 2; i++) sum[i] = 0.0f;   // not live from tile to tile
                for (int part = 0; part < parts; part++) {
                    ok = mbar_wait(done(buf), bph) && !aborted();
                    ok = __all_sync(kFull, ok);
                    if (!ok) break;
                    tc_fence_after();
                    if (parts == 1) break;
                    const uint32_t at = lanes + (uint32_t)(buf * args.buf_cols);
                    const bool last = part == parts - 1;
#pragma unroll
                    for (int g = 0; g < NB / 2; g += 8) {
                        if (g >= cols) continue;
                        uint32_t v[8];
                        tmem_ld8(at + (uint32_t)g, v);
                        tmem_wait(v);
#pragma unroll
                        for (int j = 0; j < 8; j++) sum[g + j] += __uint_as_float(v[j]);
                        if (last) tmem_st8(at + (uint32_t)g, sum + g);
                    }
                    if (!last) clear();
                }
                tmem_wait_st();
            }
            if (!ok) break;
            const bool valid = v0 + row < args.vocab && (BM == 128 || lane < 16);
            float *out = args.out + (size_t)c * args.vocab + v0 + row;
            const uint32_t at = lanes + (uint32_t)(buf * args.buf_cols);
            const int first = b0 + half * cols, end = min(args.batch, first + cols);
            // eight hidden rows at a time, the next eight on their way
            uint32_t v[8], ahead[8];
            if (first < end) tmem_ld8(at, ahead);
            for (int b = first; b < end; b += 8) {
                tmem_wait(ahead);
#pragma unroll
                for (int j = 0; j < 8; j++) v[j] = ahead[j];
                if (b + 8 < end) tmem_ld8(at + (uint32_t)(b + 8 - first), ahead);
                float l[8];
#pragma unroll
                for (int j = 0; j < 8; j++) l[j] = __uint_as_float(v[j]);
                if (args.row_scale) {
#pragma unroll
                    for (int j = 0; j < 8; j++) l[j] *= __ldg(args.row_scale + min(b + j, args.batch - 1));
                }
                if (cap > 0.0f) {   // (no branch per column: the eight chains overlap)
#pragma unroll
                    for (int j = 0; j < 8; j++) l[j] = softcap_exact(l[j], cap, inv_cap, k2);
                }
                if (!valid) continue;
                if (!args.cfg && b + 8 <= end) {
                    float *to = out + (long long)b * ldo;
#pragma unroll
                    for (int j = 0; j < 8; j++, to += ldo) *to = l[j];
                } else if (!args.cfg) {
#pragma unroll
                    for (int j = 0; j < 8; j++)
                        if (b + j < end) out[(long long)(b + j) * ldo] = l[j];
                } else {   // rows 2s, 2s + 1 (conditional, unconditional) are neighbours
#pragma unroll
                    for (int j = 0; j < 8; j += 2)
                        if (b + j < end)
                            out[(long long)((b + j) >> 1) * ldo] =
                                __fadd_rn(l[j + 1], __fmul_rn(args.cfg_scale, __fsub_rn(l[j], l[j + 1])));
                }
            }
            clear();
        }
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

enum : int { kSmall = 0, kMedium = 1, kLarge = 2, kShapes = 3 };

HeadKernel head_kernel(int shape)
{
    return shape == kSmall    ? adapter_head_kernel<1, 64, 64, 8>
           : shape == kMedium ? adapter_head_kernel<2, 128, 128, 4>
                              : adapter_head_kernel<2, 128, kMaxN, 4>;
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
        for (int i = 0; i < kShapes && e == cudaSuccess; i++)
            e = cudaFuncSetAttribute(head_kernel(i), cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemMax - 1024);
        if (e != cudaSuccess) return e;
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3((unsigned)(2 * (d.sms / 2)));
        cfg.blockDim = dim3((unsigned)threads_of(4));
        cfg.dynamicSmemBytes = kSmemMax - 1024;
        cudaLaunchAttribute attr[1];
        attr[0].id = cudaLaunchAttributeClusterDimension;
        attr[0].val.clusterDim.x = 2;
        attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
        cfg.attrs = attr;
        cfg.numAttrs = 1;
        e = cudaOccupancyMaxActiveClusters(&d.pairs, head_kernel(kLarge), &cfg);
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
        (uintptr_t)ad.B % 16 || wide * ad.n_adapters > INT_MAX - 1024)
        return cudaErrorNotSupported;
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

    // 64 weight rows per CTA up to 64 hidden rows; then pairs of CTAs, with up to 512 rows
    // in two tiles (every SM gets one) and 256 a tile beyond.
    const int shape = h.batch <= 64 ? kSmall : h.batch <= 256 ? kMedium : kLarge;
    const bool pair = shape != kSmall;
    const int bm = pair ? 128 : 64;         // weight rows per CTA
    const int m = pair ? 2 * bm : bm;
    const int n_max = shape == kSmall ? 64 : shape == kMedium ? 128 : kMaxN;
    int tiles_b = (h.batch + n_max - 1) / n_max;
    if (pair && tiles_b < 2) tiles_b = 2;
    const int even = (h.batch + tiles_b - 1) / tiles_b, step = pair ? 32 : 16;
    const int nb = (even + step - 1) / step * step;
    tiles_b = (h.batch + nb - 1) / nb;

    const bool many = (long long)h.batch * ad.rank > kFewMost;
    float *t = static_cast<float *>(ad.work);
    uint32_t *list = reinterpret_cast<uint32_t *>(t + (size_t)h.batch * ad.rank);
    int32_t *order = reinterpret_cast<int32_t *>(list + h.batch);
    DownArgs d{static_cast<const __nv_bfloat16 *>(h.hidden), static_cast<const __nv_bfloat16 *>(ad.A),
               ad.scale, ad.which, order, h.batch, h.dim, ad.n_adapters, ad.rank, ad.rows_per_id, t, list, nb, 0};
    if (many) {
        cfg.gridDim = dim3((unsigned)tiles_b);
        cfg.blockDim = dim3(kOrderThreads);
        cfg.dynamicSmemBytes = 2 * sizeof(int) * (size_t)(ad.n_adapters + 1);
        e = cudaLaunchKernelEx(&cfg, order_rows_kernel, ad.which, h.batch, nb, ad.rows_per_id,
                               ad.n_adapters, list, order);
        if (e != cudaSuccess) return e;
        cfg.gridDim = dim3((unsigned)((h.batch + kDownRows - 1) / kDownRows), (unsigned)((ad.rank + kDownRank - 1) / kDownRank));
        cfg.blockDim = dim3(32 * kDownWarps);
        cfg.dynamicSmemBytes = 0;
        e = cudaLaunchKernelEx(&cfg, adapter_down_mma_kernel, d);
    } else {
        d.down_blocks = (h.batch * ((ad.rank + 3) / 4) + kFewWarps - 1) / kFewWarps;
        cfg.gridDim = dim3((unsigned)(d.down_blocks + tiles_b));
        cfg.blockDim = dim3(32 * kFewWarps);
        e = cudaLaunchKernelEx(&cfg, adapter_down_few_kernel, d);
    }
    if (e != cudaSuccess) return e;

    GemmArgs g{};
    g.batch = h.batch;
    g.wide = (int)wide;
    // codebooks whose rows follow each other without a gap are one run of rows
    const bool joined = h.rows_per_cb == h.vocab && wide <= INT_MAX / 2;
    g.n_cb = joined ? 1 : h.n_cb;
    g.vocab = joined ? (int)wide : h.vocab;
    g.rows_per_cb = joined ? (int)wide : h.rows_per_cb;
    g.dim = h.dim;
    g.tiles_b = tiles_b;
    g.nb = nb;
    g.per_cb = (g.vocab + m - 1) / m;
    g.n_tiles = g.tiles_b * g.n_cb * g.per_cb;
    g.softcap = h.softcap;
    g.out = h.out;
    g.cfg = h.cfg;
    g.cfg_scale = h.cfg_scale;
    g.row_scale = h.row_scale;
    g.rank = ad.rank;
    g.B = static_cast<const __nv_bfloat16 *>(ad.B);
    g.t = t;
    g.list = list;
    const int nb_own = pair ? g.nb / 2 : g.nb;
    const int ksub = pair ? 1 : 2;
    const int stage = ksub * (bm + nb_own) * kBK * 2;
    const int kb = (h.dim + ksub * kBK - 1) / (ksub * kBK);
    g.parts = (h.dim / 16 + kPartSteps - 1) / kPartSteps;
    if (g.parts < 1) g.parts = 1;
    g.parts = (kb + (kb + g.parts - 1) / g.parts - 1) / ((kb + g.parts - 1) / g.parts);   // none empty
    g.buf_cols = (g.nb + 31) / 32 * 32;
    g.bufs = 512 / g.buf_cols < kMaxBufs ? 512 / g.buf_cols : kMaxBufs;
    if (g.bufs > g.parts + 1) g.bufs = g.parts + 1;
    g.tmem_cols = 32;
    while (g.tmem_cols < g.bufs * g.buf_cols) g.tmem_cols *= 2;
    // the kernel's shared memory after the stages: items, transpositions, barriers
    const int unit_warps = shape == kSmall ? 8 : 4;
    const int fixed = 1024 + 16 * n_max + 16 + 4 * unit_warps * kGroup * kItem * kPitch + 8 * kBars + 64;
    g.stages = (kSmemMax - 1024 - fixed) / stage;
    if (g.stages > kMaxStages) g.stages = kMaxStages;
    const size_t smem = (size_t)(g.stages * stage + fixed);

    CUtensorMap mw, mh;
    if (!map_2d(&mw, h.W, (uint64_t)wide, (uint64_t)h.dim, (uint32_t)bm, kBK, CU_TENSOR_MAP_SWIZZLE_128B) ||
        !map_2d(&mh, h.hidden, (uint64_t)h.batch, (uint64_t)h.dim, (uint32_t)nb_own, kBK, CU_TENSOR_MAP_SWIZZLE_128B))
        return cudaErrorInvalidValue;
    cfg.blockDim = dim3((unsigned)threads_of(unit_warps));
    cfg.dynamicSmemBytes = smem;
    if (!pair) {
        cfg.gridDim = dim3((unsigned)(g.n_tiles < dev.sms ? g.n_tiles : dev.sms));
    } else {
        attr[1].id = cudaLaunchAttributeClusterDimension;
        attr[1].val.clusterDim.x = 2;
        attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
        cfg.numAttrs = 2;
        cfg.gridDim = dim3((unsigned)(2 * (g.n_tiles < dev.pairs ? g.n_tiles : dev.pairs)));
    }
    return cudaLaunchKernelEx(&cfg, head_kernel(shape), mw, mh, g);
}

}  // namespace z2
