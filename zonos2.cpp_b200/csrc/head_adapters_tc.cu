// head_adapters_tc.cu -- the bf16 output head beside low-rank adapters on the
// tcgen05 tensor cores (sm_100a).
//
//     t[b]         = s_a * (A_a h[b])
//     logits[b, n] = softcap(W[n] . h[b] + B_a[n] . t[b])
//
// adapter_down_mma_kernel makes t (f32) with mma.sync on the rows of one adapter
// at a time; adapter_head_kernel is the GEMM, and adds B_a t in its epilogue.
//
// The GEMM's operands trade places against the plain head's: the weight rows are
// the M of its tiles (TMEM lanes), the hidden rows the N (TMEM columns).  Few
// streams then fill the tile (N = 16 is enough) instead of leaving most of an
// M = 128 tile empty, a lane's logits of one hidden row are 128 consecutive bytes
// per warp, and a lane keeps its row of B_a in registers for all the hidden rows
// that share the adapter.
//
// The low-rank product stays on the FMA pipe, in f32: as extra MMA depth it would
// need one 16-deep step per adapter of the tile and t split into three bf16 parts
// to keep f32 accuracy, while the epilogue's FMAs (rank per logit) hide under the
// next tile's MMAs.  The tile's hidden rows are ordered by adapter first, so that
// B is read once per adapter and tile.
//
// Warp roles (11 warps):
//   warp 0      TMA producer of the weight and hidden tiles (128-byte swizzle);
//   warp 1      TMEM allocation, tcgen05.mma (M = 128, or 256 over a two-SM pair);
//   warps 2..9  order the tile's rows by adapter, then the epilogue (two warps per
//               TMEM lane quarter, alternating pairs of columns);
//   warp 10     adapter producer: per run of at most 16 ordered rows of one
//               adapter (and 32 ranks), B's tile and the rows' t into a ring of
//               slots.  It alone waits for the kernel that makes t
//               (griddepcontrol.wait): the GEMM's main loop overlaps that kernel.
// Every wait is bounded, as in head_tc.cu: a warp whose wait expires sets the
// error word and goes on without waiting or copying, so that the CTA's barriers
// are still met; copies in flight are waited for (bounded) before the CTA ends.
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

// ---- t = s_a A_a h ---------------------------------------------------------

constexpr int kDownRows = 32;    // hidden rows per CTA, all of one adapter
constexpr int kDownRank = 16;    // ranks per CTA
constexpr int kDownWarps = 8;    // each takes every eighth 32-deep slice of dim
constexpr int kDownMaxAdapters = 4096;

__device__ __forceinline__ void mma_16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                          uint32_t a3, uint32_t b0, uint32_t b1)
{
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, "
        "{%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// Exclusive prefix sum over the block's kDownWarps * 32 threads; *total the sum.
__device__ __forceinline__ int block_before(int v, int *part, int *total)
{
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int s = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int t = __shfl_up_sync(kFull, s, o);
        if (lane >= o) s += t;
    }
    if (lane == 31) part[warp] = s;
    __syncthreads();
    int before = 0, all = 0;
#pragma unroll
    for (int w = 0; w < kDownWarps; w++) {
        before += w < warp ? part[w] : 0;
        all += part[w];
    }
    __syncthreads();
    *total = all;
    return before + s - v;
}

// CTA (i, j): the i-th group of up to 32 rows that share an adapter (adapters in
// order, a row's place within its adapter by its index), ranks 16 j .. 16 j + 15.
// The depth is permuted alike for both operands, so that every thread loads 16
// consecutive bytes: of a 32-deep slice, thread q of a quad holds elements 8q ..
// 8q+7 of its rows, two of them per register of two 16-deep MMAs.
__global__ void __launch_bounds__(32 * kDownWarps)
    adapter_down_mma_kernel(const __nv_bfloat16 *__restrict__ hidden, int batch, int dim,
                            const __nv_bfloat16 *__restrict__ A, const float *__restrict__ scale,
                            int n_adapters, int rank, const int32_t *__restrict__ which,
                            int rows_per_id, float *__restrict__ t)
{
    extern __shared__ int s_count[];   // [n_adapters] rows of each adapter
    __shared__ int s_part[kDownWarps], s_pick[2], s_row[kDownRows];
    __shared__ float s_sum[kDownWarps][kDownRows][kDownRank + 1];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    constexpr int kThreads = 32 * kDownWarps;

    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    // ---- which adapter, which of its groups, which rows
    for (int i = tid; i < n_adapters; i += kThreads) s_count[i] = 0;
    if (tid < kDownRows) s_row[tid] = -1;
    if (tid == 0) s_pick[0] = -1;
    __syncthreads();
    for (int b = tid; b < batch; b += kThreads) {
        const int a = which[b / rows_per_id];
        if ((unsigned)a < (unsigned)n_adapters) atomicAdd(&s_count[a], 1);
    }
    __syncthreads();
    const int per = (n_adapters + kThreads - 1) / kThreads;
    int groups = 0;
    for (int a = tid * per; a < min((tid + 1) * per, n_adapters); a++)
        groups += (s_count[a] + kDownRows - 1) / kDownRows;
    int all;
    int first = block_before(groups, s_part, &all);
    const int me = (int)blockIdx.x;
    if (me >= all) return;
    for (int a = tid * per; a < min((tid + 1) * per, n_adapters); a++) {
        const int g = (s_count[a] + kDownRows - 1) / kDownRows;
        if (me >= first && me < first + g) {
            s_pick[0] = a;
            s_pick[1] = me - first;
        }
        first += g;
    }
    __syncthreads();
    const int a = s_pick[0], group = s_pick[1];
    const int chunk = (batch + kThreads - 1) / kThreads;
    const int b0 = min(tid * chunk, batch), b1 = min(b0 + chunk, batch);
    int mine = 0;
    for (int b = b0; b < b1; b++) mine += which[b / rows_per_id] == a;
    int place = block_before(mine, s_part, &all) - group * kDownRows;
    for (int b = b0; b < b1; b++)
        if (which[b / rows_per_id] == a) {
            if (place >= 0 && place < kDownRows) s_row[place] = b;
            place++;
        }
    __syncthreads();

    // ---- the product: rows x ranks, this warp's slices of dim
    const int g = lane >> 2, q = lane & 3;
    const int r0 = (int)blockIdx.y * kDownRank;
    const bool wide = s_row[16] >= 0;   // more than 16 rows
    const __nv_bfloat16 *x[4], *w[2];
    bool live[4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const int b = s_row[g + 8 * i];
        live[i] = b >= 0;
        x[i] = hidden + (size_t)max(b, 0) * dim + 8 * q;
    }
#pragma unroll
    for (int i = 0; i < 2; i++)
        w[i] = A + ((size_t)a * rank + min(r0 + 8 * i + g, rank - 1)) * dim + 8 * q;
    float d[2][2][4] = {};
    const uint4 zero = make_uint4(0, 0, 0, 0);
#pragma unroll 4
    for (int k = 32 * warp; k < dim; k += 32 * kDownWarps) {
        const bool in = k + 8 * q < dim;
        uint4 xv[4], wv[2];
#pragma unroll
        for (int i = 0; i < 2; i++) wv[i] = in ? __ldg(reinterpret_cast<const uint4 *>(w[i] + k)) : zero;
#pragma unroll
        for (int i = 0; i < 4; i++)
            xv[i] = in && live[i] ? __ldg(reinterpret_cast<const uint4 *>(x[i] + k)) : zero;
#pragma unroll
        for (int m = 0; m < 2; m++) {
            if (m && !wide) break;
#pragma unroll
            for (int n = 0; n < 2; n++) {
                mma_16816(d[m][n], xv[2 * m].x, xv[2 * m + 1].x, xv[2 * m].y, xv[2 * m + 1].y, wv[n].x, wv[n].y);
                mma_16816(d[m][n], xv[2 * m].z, xv[2 * m + 1].z, xv[2 * m].w, xv[2 * m + 1].w, wv[n].z, wv[n].w);
            }
        }
    }
#pragma unroll
    for (int m = 0; m < 2; m++)
#pragma unroll
        for (int n = 0; n < 2; n++)
#pragma unroll
            for (int i = 0; i < 4; i++)
                s_sum[warp][16 * m + g + 8 * (i >> 1)][8 * n + 2 * q + (i & 1)] = d[m][n][i];
    __syncthreads();
    const float s = scale ? __ldg(scale + a) : 1.0f;
    for (int i = tid; i < kDownRows * kDownRank; i += kThreads) {
        const int row = i / kDownRank, r = i % kDownRank;
        if (s_row[row] < 0 || r0 + r >= rank) continue;
        float sum = 0.0f;
#pragma unroll
        for (int v = 0; v < kDownWarps; v++) sum += s_sum[v][row][r];
        t[(size_t)s_row[row] * rank + r0 + r] = sum * s;
    }
}

// ---- the GEMM --------------------------------------------------------------

constexpr int kBM = 128;            // weight rows per CTA (TMEM lanes)
constexpr int kBK = 64;             // bf16 elements per 128-byte swizzled row
constexpr int kMaxN = 256;          // hidden rows per tile (TMEM columns)
constexpr int kKsub = 2;            // 64-deep slices per stage
constexpr int kThreads = 352;
constexpr int kEpi = 256;           // epilogue threads (warps 2..9)
constexpr int kRun = 16;            // ordered rows per run at most
constexpr int kChunk = 32;          // ranks per slot at most
constexpr int kMaxStages = 12;
constexpr int kMaxSlots = 8;
constexpr int kSmemMax = 232448;

struct GemmArgs {
    int batch, n_cb, vocab, rows_per_cb, dim, wide;   // wide: n_cb * rows_per_cb of the caller
    int tiles_b, per_cb, n_tiles;
    int nb;                     // hidden rows per tile, a multiple of 16 (32 for a pair)
    int stages, slots, slot_bytes;
    float softcap;
    float *out;
    int cfg;
    float cfg_scale;
    const float *row_scale;
    const int32_t *which;
    int rows_per_id, n_adapters, rank, rank_pad, chunks;
    const float *t;
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

__device__ __forceinline__ uint32_t tmem_ld1(uint32_t taddr)
{
    uint32_t r;
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x1.b32 {%0}, [%1];" : "=r"(r) : "r"(taddr));
    return r;
}

// Waits for the loads above; the values pass through, so that no use moves ahead of it.
__device__ __forceinline__ void tmem_wait(uint32_t (&r)[8])
{
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7])
                 :
                 : "memory");
}

__device__ __forceinline__ void bulk_load(uint32_t dst, const void *src, uint32_t bytes, uint32_t bar)
{
    asm volatile(
        "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst),
        "l"(reinterpret_cast<uint64_t>(src)), "r"(bytes), "r"(bar)
        : "memory");
}

__device__ __forceinline__ float4 lds4(uint32_t a)
{
    float4 v;
    asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(a));
    return v;
}

// The 16 bytes at element 8 c of row `lane` of a B slot, as TMA lays a row of
// 8, 16 or 32 bf16 out: no swizzle, 32-byte or 64-byte.
__device__ __forceinline__ uint32_t slot_at(uint32_t base, int row, int c, int rank_pad)
{
    const uint32_t x = rank_pad == 32 ? (uint32_t)(row >> 1) & 3u : rank_pad == 16 ? (uint32_t)(row >> 2) & 1u : 0u;
    return base + (uint32_t)row * 2u * (uint32_t)rank_pad + (((uint32_t)c ^ x) << 4);
}

template <bool PAIR>
__global__ void __launch_bounds__(kThreads, 1)
    adapter_head_kernel(const __grid_constant__ CUtensorMap map_w,
                        const __grid_constant__ CUtensorMap map_h,
                        const __grid_constant__ CUtensorMap map_b, const __grid_constant__ GemmArgs args)
{
    constexpr uint32_t kWBytes = kBM * kBK * 2;
    constexpr int kCtas = PAIR ? 2 : 1;
    extern __shared__ __align__(1024) unsigned char smem_raw[];
    unsigned char *smem = reinterpret_cast<unsigned char *>(
        (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    const int nb_own = args.nb / kCtas;                 // hidden rows this CTA loads
    const uint32_t h_bytes = (uint32_t)nb_own * kBK * 2;
    const uint32_t sub_bytes = kWBytes + h_bytes;       // one 64-deep slice of both operands
    const uint32_t stage_bytes = kKsub * sub_bytes;
    const int stages = args.stages, slots = args.slots;
    unsigned char *slot_mem = smem + (size_t)stages * stage_bytes;
    int *s_key = reinterpret_cast<int *>(slot_mem + (size_t)slots * args.slot_bytes);
    int *s_okey = s_key + kMaxN;                                     // [2][kMaxN]
    uint16_t *s_order = reinterpret_cast<uint16_t *>(s_okey + 2 * kMaxN);   // [2][kMaxN]
    uint64_t *bars = reinterpret_cast<uint64_t *>(s_order + 2 * kMaxN);
    // full[12], empty[12], tfull[2], tempty[2], sfull[8], sempty[8]; the TMEM slot
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(bars + 2 * kMaxStages + 4 + 2 * kMaxSlots);
    __shared__ int s_abort;

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = PAIR ? cluster_rank() : 0u;
    const int KB = (args.dim + kBK * kKsub - 1) / (kBK * kKsub);
    auto full = [&](int s) { return smem_u32(bars + s); };
    auto empty = [&](int s) { return smem_u32(bars + kMaxStages + s); };
    auto tfull = [&](int a) { return smem_u32(bars + 2 * kMaxStages + a); };
    auto tempty = [&](int a) { return smem_u32(bars + 2 * kMaxStages + 2 + a); };
    auto sfull = [&](int s) { return smem_u32(bars + 2 * kMaxStages + 4 + s); };
    auto sempty = [&](int s) { return smem_u32(bars + 2 * kMaxStages + 4 + kMaxSlots + s); };
    auto aborted = [&]() { return *(volatile int *)&s_abort != 0; };
    const uint32_t tmem_cols = 2u * (args.nb <= 16 ? 16u : args.nb <= 32 ? 32u : args.nb <= 64 ? 64u : args.nb <= 128 ? 128u : 256u);
    const uint32_t acc_cols = tmem_cols / 2;

    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    if (threadIdx.x == 0) {
        s_abort = 0;
        for (int s = 0; s < stages; s++) {
            mbar_init(full(s), 1);
            mbar_init(empty(s), 1);
        }
        for (int a = 0; a < 2; a++) {
            mbar_init(tfull(a), 1);
            mbar_init(tempty(a), kCtas * kEpi / 32);
        }
        for (int s = 0; s < slots; s++) {
            mbar_init(sfull(s), 1);
            mbar_init(sempty(s), kEpi / 32);
        }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        prefetch_map(&map_w);
        prefetch_map(&map_h);
        prefetch_map(&map_b);
    }
    if (warp == 1) {
        if (PAIR) {
            asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(tmem_cols) : "memory");
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
        } else {
            asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(tmem_cols) : "memory");
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
        }
    }
    tc_fence_before();
    __syncthreads();
    if (PAIR) cluster_sync();
    tc_fence_after();
    const uint32_t tmem_base = *tmem_slot;
    const int unit = (int)blockIdx.x / kCtas, units = (int)gridDim.x / kCtas;
    // the tile's first hidden row, and this CTA's first weight row within its codebook
    auto tile_at = [&](int tile, int &b0, int &c, int &v0) {
        const int nt = tile / args.tiles_b;
        b0 = (tile - nt * args.tiles_b) * args.nb;
        c = nt / args.per_cb;
        v0 = (nt - c * args.per_cb) * (kBM * kCtas) + (int)rank * kBM;
    };

    // The hidden states, W and the adapter ids were complete before the kernel that
    // makes t started (it waits for all work before it), so the roles below use them
    // at once; only the adapter producer waits for t.
    if (warp == 0) {
        if (lane == 0) {
            int s = 0, used = 0;
            uint32_t ph = 0;
            bool ok = true;
            const uint32_t full0 = PAIR ? peer_addr(full(0), 0) : full(0);
            for (int tile = unit; tile < args.n_tiles && ok; tile += units) {
                int b0, c, v0;
                tile_at(tile, b0, c, v0);
                const int w_row = c * args.rows_per_cb + v0, h_row = b0 + (int)rank * nb_own;
                for (int kb = 0; kb < KB; kb++) {
                    if (!mbar_wait(empty(s), ph ^ 1u) || aborted()) {
                        ok = false;
                        break;
                    }
                    const uint32_t sa = smem_u32(smem + (size_t)s * stage_bytes);
                    if (rank == 0) mbar_expect_tx(full(s), (uint32_t)kCtas * stage_bytes);
#pragma unroll
                    for (int j = 0; j < kKsub; j++) {
                        const int kx = (kb * kKsub + j) * kBK;
                        const uint32_t d = sa + (uint32_t)j * sub_bytes;
                        if (PAIR) {
                            tma_load_2d_pair(d, &map_w, kx, w_row, full0 + 8u * (uint32_t)s);
                            tma_load_2d_pair(d + kWBytes, &map_h, kx, h_row, full0 + 8u * (uint32_t)s);
                        } else {
                            tma_load_2d(d, &map_w, kx, w_row, full(s));
                            tma_load_2d(d + kWBytes, &map_h, kx, h_row, full(s));
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
                                   ((uint32_t)((kCtas * kBM) >> 4) << 24);
            int s = 0, local = 0;
            uint32_t ph = 0;
            bool ok = true;
            const uint32_t empty1 = PAIR ? peer_addr(empty(0), 1) : 0u, tfull1 = PAIR ? peer_addr(tfull(0), 1) : 0u;
            for (int tile = unit; tile < args.n_tiles && ok; tile += units, local++) {
                const int acc = local & 1;
                const uint32_t aph = (uint32_t)(local >> 1) & 1u;
                if (!(PAIR ? mbar_wait_cl(tempty(acc), aph ^ 1u) : mbar_wait(tempty(acc), aph ^ 1u))) {
                    ok = false;
                    break;
                }
                tc_fence_after();
                const uint32_t d_tmem = tmem_base + (uint32_t)acc * acc_cols;
                for (int kb = 0; kb < KB; kb++) {
                    if (!(PAIR ? mbar_wait_cl(full(s), ph) : mbar_wait(full(s), ph)) || aborted()) {
                        ok = false;
                        break;
                    }
                    tc_fence_after();
                    const uint32_t sa = smem_u32(smem + (size_t)s * stage_bytes);
#pragma unroll
                    for (int j = 0; j < kKsub; j++) {
                        const uint64_t wd = sw128_desc(sa + (uint32_t)j * sub_bytes);
                        const uint64_t hd = sw128_desc(sa + (uint32_t)j * sub_bytes + kWBytes);
#pragma unroll
                        for (int k = 0; k < kBK / 16; k++) {
                            if (PAIR)
                                mma_bf16_pair(d_tmem, wd + (uint64_t)(2 * k), hd + (uint64_t)(2 * k), idesc, (kb | j | k) != 0);
                            else
                                mma_bf16(d_tmem, wd + (uint64_t)(2 * k), hd + (uint64_t)(2 * k), idesc, (kb | j | k) != 0);
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
                        mma_commit_pair(tfull(acc));
                        mma_commit_pair(tfull1 + 8u * (uint32_t)acc);
                    } else {
                        mma_commit(tfull(acc));
                    }
                }
            }
            if (!ok) s_abort = 1;
        }
    } else if (warp == 10) {
        // ---- adapter producer
        asm volatile("griddepcontrol.wait;" ::: "memory");   // t is complete
        int slot = 0, used = 0, local = 0;
        uint32_t ph = 0;
        bool ok = true;
        const uint32_t b_bytes = (uint32_t)kBM * 2u * (uint32_t)args.rank_pad;
        for (int tile = unit; tile < args.n_tiles; tile += units, local++) {
            int b0, c, v0;
            tile_at(tile, b0, c, v0);
            const int *okey = s_okey + (local & 1) * kMaxN;
            const uint16_t *order = s_order + (local & 1) * kMaxN;
            asm volatile("bar.sync 1, %0;" ::"n"(kEpi + 32) : "memory");   // the order is there
            const int rows = min(args.nb, args.batch - b0);
            for (int p0 = 0; p0 < rows; p0 += kRun) {
                const int key = lane < kRun && p0 + lane < rows ? okey[p0 + lane] : INT_MAX;
                const int mine = lane < kRun && p0 + lane < rows ? b0 + order[p0 + lane] : 0;
                for (int p = 0; p < kRun && p0 + p < rows;) {
                    const int a = __shfl_sync(kFull, key, p);
                    if (a == INT_MAX) break;   // rows without an adapter come last
                    const uint32_t run = __ballot_sync(kFull, key == a);
                    const int len = __popc(run);
                    for (int ch = 0; ch < args.chunks; ch++) {
                        if (ok) ok = mbar_wait(sempty(slot), ph ^ 1u) && !aborted();
                        ok = __all_sync(kFull, ok);
                        if (ok) {
                            const int rk = min(args.rank_pad, args.rank - ch * kChunk);
                            const uint32_t dst = smem_u32(slot_mem + (size_t)slot * args.slot_bytes);
                            if (lane == 0) {
                                mbar_expect_tx(sfull(slot), b_bytes + 4u * (uint32_t)(len * rk));
                                tma_load_2d(dst, &map_b, ch * kChunk, a * args.wide + c * args.rows_per_cb + v0, sfull(slot));
                            }
                            __syncwarp();
                            if (lane >= p && lane < p + len)
                                bulk_load(dst + b_bytes + (uint32_t)((lane - p) * args.rank_pad) * 4u,
                                          args.t + (size_t)mine * args.rank + ch * kChunk, 4u * (uint32_t)rk, sfull(slot));
                            used = min(used + 1, slots);
                            if (++slot == slots) {
                                slot = 0;
                                ph ^= 1u;
                            }
                        }
                    }
                    p += len;
                }
            }
        }
        if (!ok) {
            s_abort = 1;
            for (int k = 0; k < used; k++) {   // copies still in flight land first
                if (slot == 0) {
                    slot = slots;
                    ph ^= 1u;
                }
                slot--;
                mbar_wait(sfull(slot), ph);
            }
        }
    } else {
        // ---- epilogue
        const int et = (int)threadIdx.x - 64;
        const int q = warp & 3;             // the TMEM lane quarter this warp may read
        const int half = (warp - 2) >> 2;   // which of every four ordered rows: 2 half, 2 half + 1
        const int row = 32 * q + lane;      // the weight row within the CTA's 128
        const uint32_t tempty0 = PAIR ? peer_addr(tempty(0), 0) : tempty(0);
        const float cap = args.softcap, inv_cap = 1.0f / cap, k2 = 2.0f * 1.4426950408889634f / cap;
        const long long ldo = (long long)args.n_cb * args.vocab;
        int slot = 0, local = 0;
        uint32_t ph = 0;
        bool ok = true;
        for (int tile = unit; tile < args.n_tiles; tile += units, local++) {
            const int acc = local & 1;
            const uint32_t aph = (uint32_t)(local >> 1) & 1u;
            int b0, c, v0;
            tile_at(tile, b0, c, v0);
            const int rows = min(args.nb, args.batch - b0);
            // the tile's rows ordered by adapter: row i goes to the number of rows before it
            int *okey = s_okey + (local & 1) * kMaxN;
            uint16_t *order = s_order + (local & 1) * kMaxN;
            int key = INT_MAX;
            if (et < rows) {
                const int a = __ldg(args.which + (b0 + et) / args.rows_per_id);
                if ((unsigned)a < (unsigned)args.n_adapters) key = a;
            }
            s_key[et] = key;
            asm volatile("bar.sync 2, %0;" ::"n"(kEpi) : "memory");
            int place = et;
            if (et < rows) {
                place = 0;
                const int4 *k4 = reinterpret_cast<const int4 *>(s_key);
                for (int i = 0; i < rows; i += 4) {   // keys past the rows are INT_MAX, at higher places
                    const int4 k = k4[i >> 2];
                    place += (k.x < key || (k.x == key && i < et)) + (k.y < key || (k.y == key && i + 1 < et)) +
                             (k.z < key || (k.z == key && i + 2 < et)) + (k.w < key || (k.w == key && i + 3 < et));
                }
            }
            order[place] = (uint16_t)et;
            okey[place] = key;
            asm volatile("bar.sync 1, %0;" ::"n"(kEpi + 32) : "memory");

            if (ok) ok = mbar_wait(tfull(acc), aph) && !aborted();
            ok = __all_sync(kFull, ok);
            tc_fence_after();
            const uint32_t tm = tmem_base + ((uint32_t)(32 * q) << 16) + (uint32_t)acc * acc_cols;
            const bool valid = v0 + row < args.vocab;
            float *out = args.out + (size_t)c * args.vocab + v0 + row;
            for (int p0 = 0; p0 < rows && ok; p0 += kRun) {
                int col[8];
                uint32_t r[8];
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    col[i] = order[p0 + 4 * (i >> 1) + 2 * half + (i & 1)];
                    r[i] = tmem_ld1(tm + (uint32_t)col[i]);
                }
                const int kr = lane < kRun ? okey[p0 + lane] : INT_MAX;
                tmem_wait(r);
                float2 sum[8];
#pragma unroll
                for (int i = 0; i < 8; i++) sum[i] = make_float2(0.0f, 0.0f);
                for (int p = 0; p < kRun && ok;) {
                    const int a = __shfl_sync(kFull, kr, p);
                    if (a == INT_MAX) break;
                    const int len = __popc(__ballot_sync(kFull, kr == a));
                    const uint32_t live = ((1u << len) - 1u) << p;
                    for (int ch = 0; ch < args.chunks; ch++) {
                        ok = mbar_wait(sfull(slot), ph) && !aborted();
                        ok = __all_sync(kFull, ok);
                        if (!ok) break;
                        const int rk = min(args.rank_pad, args.rank - ch * kChunk);
                        const uint32_t sb = smem_u32(slot_mem + (size_t)slot * args.slot_bytes);
                        const uint32_t st = sb + (uint32_t)kBM * 2u * (uint32_t)args.rank_pad - (uint32_t)(p * args.rank_pad) * 4u;
                        for (int k = 0; k < rk; k += 8) {
                            const float4 raw = lds4(slot_at(sb, row, k >> 3, args.rank_pad));
                            const uint32_t w4[4] = {__float_as_uint(raw.x), __float_as_uint(raw.y), __float_as_uint(raw.z), __float_as_uint(raw.w)};
                            float2 w[4];
#pragma unroll
                            for (int j = 0; j < 4; j++)
                                w[j] = make_float2(__uint_as_float(w4[j] << 16), __uint_as_float(w4[j] & 0xffff0000u));
#pragma unroll
                            for (int i = 0; i < 8; i++) {
                                const int pos = 4 * (i >> 1) + 2 * half + (i & 1);
                                if ((live >> pos) & 1u) {
                                    const float4 t0 = lds4(st + (uint32_t)(pos * args.rank_pad + k) * 4u);
                                    const float4 t1 = lds4(st + (uint32_t)(pos * args.rank_pad + k) * 4u + 16u);
                                    sum[i] = __ffma2_rn(w[0], make_float2(t0.x, t0.y), sum[i]);
                                    sum[i] = __ffma2_rn(w[1], make_float2(t0.z, t0.w), sum[i]);
                                    sum[i] = __ffma2_rn(w[2], make_float2(t1.x, t1.y), sum[i]);
                                    sum[i] = __ffma2_rn(w[3], make_float2(t1.z, t1.w), sum[i]);
                                }
                            }
                        }
                        __syncwarp();
                        if (lane == 0) mbar_arrive(sempty(slot));
                        if (++slot == slots) {
                            slot = 0;
                            ph ^= 1u;
                        }
                    }
                    p += len;
                }
                if (!ok) break;
                float l[8];
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    l[i] = __uint_as_float(r[i]) + (sum[i].x + sum[i].y);
                    if (args.row_scale && p0 + 4 * (i >> 1) + 2 * half + (i & 1) < rows)
                        l[i] *= __ldg(args.row_scale + b0 + col[i]);
                    if (cap > 0.0f) l[i] = softcap_exact(l[i], cap, inv_cap, k2);
                }
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    if (p0 + 4 * (i >> 1) + 2 * half + (i & 1) >= rows || !valid) continue;
                    if (!args.cfg) {
                        out[(long long)(b0 + col[i]) * ldo] = l[i];
                    } else if ((i & 1) == 0) {   // the pair (2s, 2s + 1) stays together in the order
                        out[(long long)((b0 + col[i]) >> 1) * ldo] =
                            __fadd_rn(l[i + 1], __fmul_rn(args.cfg_scale, __fsub_rn(l[i], l[i + 1])));
                    }
                }
            }
            if (!ok) s_abort = 1;
            tc_fence_before();
            __syncwarp();
            if (lane == 0) {
                if (PAIR)
                    mbar_arrive_cluster(tempty0 + 8u * (uint32_t)acc);
                else
                    mbar_arrive(tempty(acc));
            }
        }
    }

    tc_fence_before();
    __syncthreads();
    if (PAIR) cluster_sync();
    tc_fence_after();
    if (warp == 1) {
        if (PAIR)
            asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(tmem_cols) : "memory");
        else
            asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(tmem_cols) : "memory");
    }
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
        if (e == cudaSuccess)
            e = cudaFuncSetAttribute(adapter_head_kernel<false>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemMax - 1024);
        if (e == cudaSuccess)
            e = cudaFuncSetAttribute(adapter_head_kernel<true>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemMax - 1024);
        if (e != cudaSuccess) return e;
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3((unsigned)(2 * (d.sms / 2)));
        cfg.blockDim = dim3(kThreads);
        cfg.dynamicSmemBytes = kSmemMax - 1024;
        cudaLaunchAttribute attr[1];
        attr[0].id = cudaLaunchAttributeClusterDimension;
        attr[0].val.clusterDim.x = 2;
        attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
        cfg.attrs = attr;
        cfg.numAttrs = 1;
        e = cudaOccupancyMaxActiveClusters(&d.pairs, adapter_head_kernel<true>, &cfg);
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
    if (h.dim % 8 != 0 || ad.rank % 8 != 0 || ad.n_adapters > kDownMaxAdapters ||
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
    // groups of rows: at most one short group per adapter
    const int groups = h.batch / kDownRows + (h.batch < ad.n_adapters ? h.batch : ad.n_adapters);
    cfg.gridDim = dim3((unsigned)groups, (unsigned)((ad.rank + kDownRank - 1) / kDownRank));
    cfg.blockDim = dim3(32 * kDownWarps);
    cfg.dynamicSmemBytes = sizeof(int) * (size_t)ad.n_adapters;
    e = cudaLaunchKernelEx(&cfg, adapter_down_mma_kernel, static_cast<const __nv_bfloat16 *>(h.hidden),
                           h.batch, h.dim, static_cast<const __nv_bfloat16 *>(ad.A), ad.scale,
                           ad.n_adapters, ad.rank, ad.which, ad.rows_per_id,
                           static_cast<float *>(ad.work));
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
    const bool pair = h.batch > 256;
    const int m = pair ? 2 * kBM : kBM;
    g.tiles_b = (h.batch + kMaxN - 1) / kMaxN;
    const int even = (h.batch + g.tiles_b - 1) / g.tiles_b, step = pair ? 32 : 16;
    g.nb = (even + step - 1) / step * step;
    g.tiles_b = (h.batch + g.nb - 1) / g.nb;
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
    g.rank = ad.rank;
    g.rank_pad = ad.rank <= 8 ? 8 : ad.rank <= 16 ? 16 : 32;
    g.chunks = (ad.rank + kChunk - 1) / kChunk;
    g.t = static_cast<const float *>(ad.work);
    g.slot_bytes = (kBM * 2 * g.rank_pad + kRun * 4 * g.rank_pad + 1023) / 1024 * 1024;
    const int nb_own = pair ? g.nb / 2 : g.nb;
    const int stage = kKsub * (kBM + nb_own) * kBK * 2;
    const int fixed = 1024 + kMaxN * 4 * 3 + kMaxN * 2 * 2 + (2 * kMaxStages + 4 + 2 * kMaxSlots) * 8 + 64;
    const int room = kSmemMax - 1024 - fixed;
    g.slots = 2;
    g.stages = (room - g.slots * g.slot_bytes) / stage;
    if (g.stages > kMaxStages) g.stages = kMaxStages;
    while (g.slots < kMaxSlots && g.stages * stage + (g.slots + 1) * g.slot_bytes <= room) g.slots++;
    const size_t smem = (size_t)(g.stages * stage + g.slots * g.slot_bytes + fixed);

    CUtensorMap mw, mh, mb;
    if (!map_2d(&mw, h.W, (uint64_t)wide, (uint64_t)h.dim, kBM, kBK, CU_TENSOR_MAP_SWIZZLE_128B) ||
        !map_2d(&mh, h.hidden, (uint64_t)h.batch, (uint64_t)h.dim, (uint32_t)nb_own, kBK, CU_TENSOR_MAP_SWIZZLE_128B) ||
        !map_2d(&mb, ad.B, (uint64_t)(wide * ad.n_adapters), (uint64_t)ad.rank, kBM, (uint32_t)g.rank_pad,
                g.rank_pad == 32 ? CU_TENSOR_MAP_SWIZZLE_64B
                                 : g.rank_pad == 16 ? CU_TENSOR_MAP_SWIZZLE_32B : CU_TENSOR_MAP_SWIZZLE_NONE))
        return cudaErrorInvalidValue;
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = smem;
    if (!pair) {
        cfg.gridDim = dim3((unsigned)(g.n_tiles < dev.sms ? g.n_tiles : dev.sms));
        return cudaLaunchKernelEx(&cfg, adapter_head_kernel<false>, mw, mh, mb, g);
    }
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = 2;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.numAttrs = 2;
    cfg.gridDim = dim3((unsigned)(2 * (g.n_tiles < dev.pairs ? g.n_tiles : dev.pairs)));
    return cudaLaunchKernelEx(&cfg, adapter_head_kernel<true>, mw, mh, mb, g);
}

}  // namespace z2
