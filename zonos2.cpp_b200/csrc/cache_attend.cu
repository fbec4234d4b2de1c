// cache_attend.cu -- attention of new tokens over a paged cache (sm_100a): few query rows per
// key head, and all that the tensor-core kernel of cache_attend_tc.cu does not take.
//
//     o = g * sum_j softmax_j(scale q . k_j) v_j      over the tokens j that the row sees
//
// The rows of a tile are (token, query head) pairs that share a key head, so that every key
// and value is read once for all of them.  The tokens that a tile sees are cut into groups of a
// few keys, dealt out to the warps of a block, or of a cluster of blocks where there are few
// tiles.  A warp keeps the running maximum m, sum l and output O of its groups (x = scale
// log2(e) q . k):
//     m' = max(m, x),   O' = O 2^(m - m') + sum 2^(x - m') v,   l' = l 2^(m - m') + sum 2^(x - m')
// and at the end the warps' parts are joined in the order of their numbers, over the cluster's
// shared memory: the result depends on the sizes alone, and no scratch memory is needed.
//
// Bound: memory for one token or a few per stream (keys and values are read once), so each warp
// has a ring of groups of its own in flight by asynchronous copies and no block-wide barrier
// before the join.
#include <math.h>

#include <mutex>

#include "cache.cuh"
#include "tc.cuh"

namespace z2 {

namespace {

constexpr int kWarps = 4;
constexpr int kThreadsRows = 32 * kWarps;
constexpr float kLog2e = 1.4426950408889634f;

__device__ __forceinline__ float exp2_fast(float x)
{
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

__device__ __forceinline__ void cp_async16(uint32_t dst, const void *src, bool take)
{
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src),
                 "r"(take ? 16 : 0)
                 : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait()
{
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

__device__ __forceinline__ void ldmatrix4(uint32_t addr, uint32_t (&r)[4])
{
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}
__device__ __forceinline__ void ldmatrix4_trans(uint32_t addr, uint32_t (&r)[4])
{
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}
__device__ __forceinline__ void mma_16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1)
{
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, "
        "{%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi)
{
    const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t *>(&h);
}

__device__ __forceinline__ bool odd(float v) { return (__float_as_uint(v) & 0x7f800000u) == 0x7f800000u; }
// A NaN or an infinity among the two bf16 values of a word.
__device__ __forceinline__ bool odd2(uint32_t w)
{
    return (w & 0x7f80u) == 0x7f80u || (w & 0x7f800000u) == 0x7f800000u;
}

// The tile of this block: rows [row0, row0 + rows) of stream chunk ch, counted in (token, head
// of the group) pairs.  Tile t of streams with chunks of n tokens: stream s has the numbers from
// floor(start_s * G / T) + s on, which leaves each stream enough of them (T rows to a tile), so
// that a tile's stream is found from the starts alone.
struct Tile {
    Chunk ch;
    int row0, rows;    // rows == 0: none
};

__device__ Tile find_tile(const CacheArgs &c, int group, int tile_rows, long long t, int *s_found)
{
    if (threadIdx.x == 0) *s_found = -1;
    __syncthreads();
    auto number = [&](int s) {
        const int a = min(max(__ldg(c.q_start + s), 0), c.rows);
        return (long long)a * group / tile_rows + s;
    };
    for (int s = threadIdx.x; s < c.n_streams; s += blockDim.x)
        if (number(s) <= t && t < number(s + 1)) *s_found = s;   // one stream's, as the starts rise
    __syncthreads();
    Tile tile;
    tile.rows = 0;
    const int s = *s_found;
    if (s < 0) return tile;
    tile.ch = chunk_of(c, s);
    const long long first = (t - number(s)) * tile_rows, all = (long long)tile.ch.n * group;
    if (first < all) {
        tile.row0 = (int)first;
        tile.rows = (int)(all - first < tile_rows ? all - first : tile_rows);
    }
    return tile;
}

// What a row of the tile sees: tokens [low, high).
__device__ __forceinline__ int position_of(const Chunk &ch, int group, int row)
{
    return ch.len - ch.n + row / group;
}

// KEYS keys and values of D elements (rows of `dim`) of one key head, as one stage of a warp's
// ring: the keys' rows, then the values'.  16-byte piece p of row r lies at piece p ^ (r & 7), so
// that eight rows' same piece falls on different banks.
template <typename T, int D, int KEYS>
struct Ring {
    static constexpr int kRow = D * (int)sizeof(T);      // bytes
    static constexpr int kHalf = KEYS * kRow;
    static constexpr int kStage = 2 * kHalf;
    static constexpr int kPieces = kRow / 16;

    // Loads the keys [j0, j0 + KEYS) that lie in [low, high) and on a page; zeros elsewhere.
    // Returns the bits of KEYS / 8 runs of eight that lie on a page.
    __device__ static uint32_t load(const CacheArgs &c, int s, int kvh, int j0, int low, int high, int room,
                                    uint32_t stage)
    {
        const int lane = threadIdx.x & 31;
        long long base[KEYS / 8];
        uint32_t held = 0;
#pragma unroll
        for (int e = 0; e < KEYS / 8; e++) {
            const int j = j0 + 8 * e;
            const int p = j < room ? page_of(c, s, j) : -1;
            base[e] = p >= 0 ? row_on_page(c, p, kvh, j) : 0;
            held |= p >= 0 ? 1u << e : 0u;
        }
        const int live = c.dim * (int)sizeof(T) / 16;   // pieces of a row that there are
#pragma unroll
        for (int i = 0; i < KEYS * kPieces / 32; i++) {
            const int id = i * 32 + lane, r = id / kPieces, p = id % kPieces;
            const int j = j0 + r;
            const long long at = (KEYS == 8 || r < 8 ? base[0] : base[KEYS / 8 - 1]) + (r & 7) * c.dim;
            const bool take = (held >> (r >> 3) & 1u) && j >= low && j < high;
            const uint32_t dst = stage + r * kRow + ((p ^ (r & 7)) << 4);
            if (p < live) {
                cp_async16(dst, (const T *)c.k + (take ? at : 0) + p * (16 / (int)sizeof(T)), take);
                cp_async16(dst + kHalf, (const T *)c.v + (take ? at : 0) + p * (16 / (int)sizeof(T)), take);
            }
        }
        return held;
    }
};

// Joins the parts of the block's warps (and of the cluster's blocks) and stores the rows.
// part: [kWarps][ROWS][D] f32 outputs, ml: [kWarps][ROWS] maxima and sums behind each other.
template <typename T, int D, int ROWS>
__device__ void join_and_store(const CacheArgs &c, const AttendArgs &a, const Tile &tile, int kvh,
                               float *part, float2 *ml, int ranks, int rank)
{
    constexpr int kQuads = ROWS * D / 4;
    auto weigh = [](float m, float most) { return m == -INFINITY ? 0.0f : exp2_fast(m - most); };
    __syncthreads();
    // the block's own warps, into warp 0's part
    for (int i = threadIdx.x; i < kQuads; i += kThreadsRows) {
        const int r = i / (D / 4);
        float most = -INFINITY;
#pragma unroll
        for (int w = 0; w < kWarps; w++) most = fmaxf(most, ml[w * ROWS + r].x);
        float4 sum = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
        for (int w = 0; w < kWarps; w++) {
            const float f = weigh(ml[w * ROWS + r].x, most);
            const float4 v = reinterpret_cast<const float4 *>(part)[w * kQuads + i];
            if (f != 0.0f) {
                sum.x += f * v.x;
                sum.y += f * v.y;
                sum.z += f * v.z;
                sum.w += f * v.w;
            }
        }
        reinterpret_cast<float4 *>(part)[i] = sum;
    }
    __syncthreads();
    if (threadIdx.x < ROWS) {
        const int r = threadIdx.x;
        float most = -INFINITY, l = 0.0f;
        for (int w = 0; w < kWarps; w++) most = fmaxf(most, ml[w * ROWS + r].x);
        for (int w = 0; w < kWarps; w++) {
            const float f = weigh(ml[w * ROWS + r].x, most);
            l += f != 0.0f ? f * ml[w * ROWS + r].y : 0.0f;
        }
        // a NaN among the sums stays one whatever its weight
        for (int w = 0; w < kWarps; w++)
            if (isnan(ml[w * ROWS + r].y)) l = ml[w * ROWS + r].y;
        ml[r] = make_float2(most, l);
    }
    if (ranks > 1)
        cluster_sync();
    else
        __syncthreads();
    const uint32_t part0 = smem_u32(part), ml0 = smem_u32(ml);
    // this rank's share of the rows' quads
    const int per = (kQuads + ranks - 1) / ranks;
    const int end = min(kQuads, (rank + 1) * per);
    for (int i = rank * per + threadIdx.x; i < end; i += kThreadsRows) {
        const int r = i / (D / 4), d = (i % (D / 4)) * 4;
        if (r >= tile.rows || d >= c.dim) continue;
        float4 sum = reinterpret_cast<const float4 *>(part)[i];
        float l = ml[r].y;
        if (ranks > 1) {
            float most = -INFINITY;
            for (int k = 0; k < ranks; k++) {
                float m;
                asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(m) : "r"(peer_addr(ml0 + r * 8, k)));
                most = fmaxf(most, m);
            }
            sum = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            l = 0.0f;
            for (int k = 0; k < ranks; k++) {
                float m, lk;
                float4 v;
                asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];"
                             : "=f"(m), "=f"(lk)
                             : "r"(peer_addr(ml0 + r * 8, k)));
                asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
                             : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
                             : "r"(peer_addr(part0 + i * 16, k)));
                const float f = weigh(m, most);
                if (f != 0.0f || isnan(lk)) {
                    l += f * lk;
                    sum.x += f * v.x;
                    sum.y += f * v.y;
                    sum.z += f * v.z;
                    sum.w += f * v.w;
                }
            }
        }
        const int row = tile.row0 + r, token = tile.ch.first + row / a.group;
        const int h = kvh * a.group + row % a.group;
        float f = l == 0.0f ? 0.0f : 1.0f / l;
        if (a.gate) {
            const float g = as_f(((const T *)a.gate)[token * a.gate_stride + h]);
            f *= 1.0f / (1.0f + expf(-g));
        }
        T *to = (T *)a.out + token * a.out_stride + (long long)h * c.dim + d;
        if (sizeof(T) == 2) {
            *reinterpret_cast<uint2 *>(to) = make_uint2(pack_bf16(sum.x * f, sum.y * f), pack_bf16(sum.z * f, sum.w * f));
        } else {
            *reinterpret_cast<float4 *>(to) = make_float4(sum.x * f, sum.y * f, sum.z * f, sum.w * f);
        }
    }
    if (ranks > 1) cluster_sync();   // the others have read this block's part
}

// ---- bf16, by mma.sync ------------------------------------------------------
// 16 * MB rows to a tile, groups of 16 keys: S = Q K^T by m16n8k16 (rows x 8 keys x 16
// elements), whose accumulators, rounded to bf16, are the left operand of O += P V.
template <int D, int MB, int STAGES>
__global__ void __launch_bounds__(kThreadsRows)
    attend_rows_bf16_kernel(const CacheArgs c, const AttendArgs a, int ranks)
{
    typedef Ring<__nv_bfloat16, D, 16> R;
    constexpr int ROWS = 16 * MB;
    extern __shared__ __align__(1024) unsigned char smem[];
    // the warps' rings, then the queries; at the end the parts take the rings' place
    __shared__ float2 s_ml[kWarps * ROWS];
    __shared__ int s_found;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int rank = blockIdx.x % ranks, kvh = blockIdx.y;
    const Tile tile = find_tile(c, a.group, ROWS, blockIdx.x / ranks, &s_found);
    if (tile.rows == 0) return;   // the whole cluster's tile

    const uint32_t ring = smem_u32(smem) + warp * STAGES * R::kStage;
    const uint32_t s_q = smem_u32(smem) + kWarps * STAGES * R::kStage;
    const int live = c.dim / 8;
    // queries (zeros past the rows and the head's elements), swizzled like the keys
    for (int i = threadIdx.x; i < ROWS * R::kPieces; i += kThreadsRows) {
        const int r = i / R::kPieces, p = i % R::kPieces, row = tile.row0 + r;
        uint4 v = make_uint4(0, 0, 0, 0);
        if (r < tile.rows && p < live)
            v = *reinterpret_cast<const uint4 *>((const __nv_bfloat16 *)a.q +
                                                 (tile.ch.first + row / a.group) * a.q_stride +
                                                 (long long)(kvh * a.group + row % a.group) * c.dim + p * 8);
        asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(s_q + r * R::kRow + ((p ^ (r & 7)) << 4)),
                     "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w)
                     : "memory");
    }
    if (live < R::kPieces)   // pieces that no copy fills
        for (int i = lane; i < STAGES * 32 * R::kPieces; i += 32) {
            const int r = i / R::kPieces, p = i % R::kPieces;
            if (p >= live)
                asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(ring + r * R::kRow + ((p ^ (r & 7)) << 4)),
                             "r"(0)
                             : "memory");
        }
    __syncthreads();

    // the tokens that some row of the tile sees, in groups of 16
    const int room = room_of(c);
    const int pos_first = position_of(tile.ch, a.group, tile.row0);
    const int pos_last = position_of(tile.ch, a.group, tile.row0 + tile.rows - 1);
    const int low = a.window > 0 ? max(0, pos_first - a.window + 1) : 0;
    const int high = min(pos_last + 1, room);
    const int sees_all_from = a.window > 0 ? max(0, pos_last - a.window + 1) : 0;   // .. to pos_first
    const int first_group = low >> 4, groups = high > low ? ((high + 15) >> 4) - first_group : 0;
    const int workers = ranks * kWarps, worker = rank * kWarps + warp;

    int pos[2 * MB];   // of this lane's rows (those past the tile's take the last row's)
#pragma unroll
    for (int i = 0; i < 2 * MB; i++)
        pos[i] = position_of(tile.ch, a.group, tile.row0 + min((i >> 1) * 16 + (i & 1) * 8 + (lane >> 2), tile.rows - 1));
    float m[2 * MB], l[2 * MB], o[MB][D / 8][4];
#pragma unroll
    for (int i = 0; i < 2 * MB; i++) {
        m[i] = -INFINITY;
        l[i] = 0.0f;
    }
#pragma unroll
    for (int b = 0; b < MB; b++)
#pragma unroll
        for (int n = 0; n < D / 8; n++) o[b][n][0] = o[b][n][1] = o[b][n][2] = o[b][n][3] = 0.0f;
    const float factor = a.scale * kLog2e;

    // ldmatrix: lane's row and piece of a 16 x 16 block
    const int lm_key = (lane & 7) + ((lane >> 4) << 3), lm_kp = (lane >> 3) & 1;     // keys: n blocks of 8
    const int lm_val = (lane & 7) + (((lane >> 3) & 1) << 3), lm_vp = lane >> 4;     // values, transposed
    constexpr bool kQRegs = MB * D <= 128;
    uint32_t qf[kQRegs ? MB : 1][kQRegs ? D / 16 : 1][4];
    auto load_q = [&](int b, int kk, uint32_t (&f)[4]) {
        const int r = b * 16 + (lane & 15), p = 2 * kk + (lane >> 4);
        ldmatrix4(s_q + r * R::kRow + ((p ^ (r & 7)) << 4), f);
    };
    if (kQRegs) {
#pragma unroll
        for (int b = 0; b < MB; b++)
#pragma unroll
            for (int kk = 0; kk < D / 16; kk++) load_q(b, kk, qf[b][kk]);
    }

    uint32_t held_bits = 0;   // two bits to a stage
    auto fetch = [&](int it) {
        const int g = worker + it * workers;
        if (g < groups) {
            const int st = it % STAGES;
            const uint32_t held = R::load(c, tile.ch.stream, kvh, (first_group + g) * 16, low, high, room,
                                          ring + st * R::kStage);
            held_bits = (held_bits & ~(3u << (2 * st))) | held << (2 * st);
        }
        cp_async_commit();
    };
#pragma unroll
    for (int i = 0; i < STAGES - 1; i++) fetch(i);
    for (int it = 0; worker + it * workers < groups; it++) {
        fetch(it + STAGES - 1);
        cp_async_wait<STAGES - 1>();
        __syncwarp();
        const int st = it % STAGES;
        const uint32_t keys = ring + st * R::kStage, values = keys + R::kHalf;
        const int j0 = (first_group + worker + it * workers) * 16;
        const uint32_t held = held_bits >> (2 * st) & 3u;
        float x[MB][2][4];
#pragma unroll
        for (int b = 0; b < MB; b++)
#pragma unroll
            for (int n = 0; n < 2; n++) x[b][n][0] = x[b][n][1] = x[b][n][2] = x[b][n][3] = 0.0f;
#pragma unroll
        for (int kk = 0; kk < D / 16; kk++) {
            uint32_t kf[4];
            ldmatrix4(keys + lm_key * R::kRow + (((2 * kk + lm_kp) ^ (lm_key & 7)) << 4), kf);
#pragma unroll
            for (int b = 0; b < MB; b++) {
                uint32_t f[4];
                if (!kQRegs) load_q(b, kk, f);
                mma_16816(x[b][0], kQRegs ? qf[b][kk] : f, kf[0], kf[1]);
                mma_16816(x[b][1], kQRegs ? qf[b][kk] : f, kf[2], kf[3]);
            }
        }
        // rows that do not see all of the group
        const bool partial = j0 < sees_all_from || j0 + 15 > pos_first || j0 + 15 >= high || held != 3u;
        auto sees = [&](int i, int j) {   // row slot i of this lane, token j
            return j <= pos[i] && j < high && (a.window <= 0 || j > pos[i] - a.window) && (held >> ((j - j0) >> 3) & 1u);
        };
        float keep[2 * MB];
        bool same = true;
#pragma unroll
        for (int i = 0; i < 2 * MB; i++) {
            float most = -INFINITY;
#pragma unroll
            for (int n = 0; n < 2; n++)
#pragma unroll
                for (int e = 0; e < 2; e++) {
                    float &v = x[i >> 1][n][(i & 1) * 2 + e];
                    v *= factor;
                    if (!partial || sees(i, j0 + 8 * n + 2 * (lane & 3) + e)) most = fmaxf(most, v);
                }
            most = fmaxf(most, __shfl_xor_sync(kFull, most, 1));
            most = fmaxf(most, __shfl_xor_sync(kFull, most, 2));
            most = fmaxf(most, m[i]);
            keep[i] = m[i] == -INFINITY ? 0.0f : exp2_fast(m[i] - most);
            same = same && most == m[i];
            m[i] = most;
        }
        if (!__all_sync(kFull, same)) {
#pragma unroll
            for (int i = 0; i < 2 * MB; i++) {
                l[i] *= keep[i];
#pragma unroll
                for (int n = 0; n < D / 8; n++) {
                    o[i >> 1][n][(i & 1) * 2] *= keep[i];
                    o[i >> 1][n][(i & 1) * 2 + 1] *= keep[i];
                }
            }
        }
        uint32_t pf[MB][4];
#pragma unroll
        for (int b = 0; b < MB; b++) {
#pragma unroll
            for (int n = 0; n < 2; n++)
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const int i = 2 * b + (e >> 1);
                    float w = exp2_fast(x[b][n][e] - m[i]);
                    if (partial && !sees(i, j0 + 8 * n + 2 * (lane & 3) + (e & 1))) w = 0.0f;
                    l[i] += w;
                    x[b][n][e] = w;
                }
            pf[b][0] = pack_bf16(x[b][0][0], x[b][0][1]);
            pf[b][1] = pack_bf16(x[b][0][2], x[b][0][3]);
            pf[b][2] = pack_bf16(x[b][1][0], x[b][1][1]);
            pf[b][3] = pack_bf16(x[b][1][2], x[b][1][3]);
        }
        if (partial) {
            // A value that is not finite would reach rows that do not see its token, as 0 times
            // it: it goes to the rows that do by itself, and is a zero to the product.
            bool any = false;
            for (int i = lane; i < 16 * R::kPieces; i += 32) {
                uint4 v;
                asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                             : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
                             : "r"(values + i * 16));
                any |= odd2(v.x) || odd2(v.y) || odd2(v.z) || odd2(v.w);
            }
            if (__any_sync(kFull, any)) {
                for (int k = 0; k < 16; k++)
#pragma unroll
                    for (int n = 0; n < D / 8; n++) {
                        uint32_t w;
                        asm volatile("ld.shared.b32 %0, [%1];"
                                     : "=r"(w)
                                     : "r"(values + k * R::kRow + ((n ^ (k & 7)) << 4) + 4 * (lane & 3)));
                        if (!odd2(w)) continue;
                        const float v0 = __uint_as_float(w << 16), v1 = __uint_as_float(w & 0xffff0000u);
#pragma unroll
                        for (int i = 0; i < 2 * MB; i++)
                            if (sees(i, j0 + k)) {
                                if (odd(v0)) o[i >> 1][n][(i & 1) * 2] += v0;
                                if (odd(v1)) o[i >> 1][n][(i & 1) * 2 + 1] += v1;
                            }
                    }
                __syncwarp();
                for (int i = lane; i < 64 * R::kPieces; i += 32) {
                    uint32_t w;
                    asm volatile("ld.shared.b32 %0, [%1];" : "=r"(w) : "r"(values + i * 4));
                    if ((w & 0x7f80u) == 0x7f80u) w &= 0xffff0000u;
                    if ((w & 0x7f800000u) == 0x7f800000u) w &= 0x0000ffffu;
                    asm volatile("st.shared.b32 [%0], %1;" ::"r"(values + i * 4), "r"(w) : "memory");
                }
                __syncwarp();
            }
        }
#pragma unroll
        for (int n = 0; n < D / 16; n++) {
            uint32_t vf[4];
            ldmatrix4_trans(values + lm_val * R::kRow + (((2 * n + lm_vp) ^ (lm_val & 7)) << 4), vf);
#pragma unroll
            for (int b = 0; b < MB; b++) {
                mma_16816(o[b][2 * n], pf[b], vf[0], vf[1]);
                mma_16816(o[b][2 * n + 1], pf[b], vf[2], vf[3]);
            }
        }
        __syncwarp();   // the stage is free for the copies of the next turn
    }
    cp_async_wait<0>();
    __syncthreads();   // every warp is done with its ring: the parts take their place
    float *part = reinterpret_cast<float *>(smem);
#pragma unroll
    for (int i = 0; i < 2 * MB; i++) {
        l[i] += __shfl_xor_sync(kFull, l[i], 1);
        l[i] += __shfl_xor_sync(kFull, l[i], 2);
        const int r = (i >> 1) * 16 + (i & 1) * 8 + (lane >> 2);
        if ((lane & 3) == 0) s_ml[warp * ROWS + r] = make_float2(m[i], l[i]);
#pragma unroll
        for (int n = 0; n < D / 8; n++)
            *reinterpret_cast<float2 *>(part + (warp * ROWS + r) * D + n * 8 + 2 * (lane & 3)) =
                make_float2(o[i >> 1][n][(i & 1) * 2], o[i >> 1][n][(i & 1) * 2 + 1]);
    }
    join_and_store<__nv_bfloat16, D, ROWS>(c, a, tile, kvh, part, s_ml, ranks, rank);
}

// ---- f32, on the FMA pipe ----------------------------------------------------
// ROWS rows to a tile, groups of 8 keys.  A lane takes a quarter of a key's elements for
// the scores of all rows (key lane / 4), then D / 32 of the output's columns.
template <int D, int ROWS, int STAGES>
__global__ void __launch_bounds__(kThreadsRows)
    attend_rows_f32_kernel(const CacheArgs c, const AttendArgs a, int ranks)
{
    typedef Ring<float, D, 8> R;
    extern __shared__ __align__(1024) unsigned char smem[];
    __shared__ float2 s_ml[kWarps * ROWS];
    __shared__ __align__(16) float s_w[kWarps][8][ROWS];   // a group's weights
    __shared__ int s_found;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int rank = blockIdx.x % ranks, kvh = blockIdx.y;
    const Tile tile = find_tile(c, a.group, ROWS, blockIdx.x / ranks, &s_found);
    if (tile.rows == 0) return;

    const uint32_t ring = smem_u32(smem) + warp * STAGES * R::kStage;
    float *s_q = reinterpret_cast<float *>(smem + kWarps * STAGES * R::kStage);   // [ROWS][D]
    const int live = c.dim / 4;
    for (int i = threadIdx.x; i < ROWS * R::kPieces; i += kThreadsRows) {
        const int r = i / R::kPieces, p = i % R::kPieces, row = tile.row0 + r;
        float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        if (r < tile.rows && p < live)
            v = *reinterpret_cast<const float4 *>((const float *)a.q + (tile.ch.first + row / a.group) * a.q_stride +
                                                  (long long)(kvh * a.group + row % a.group) * c.dim + p * 4);
        reinterpret_cast<float4 *>(s_q)[i] = v;
    }
    if (live < R::kPieces)
        for (int i = lane; i < STAGES * 16 * R::kPieces; i += 32) {
            const int r = i / R::kPieces, p = i % R::kPieces;
            if (p >= live)
                asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(ring + r * R::kRow + ((p ^ (r & 7)) << 4)),
                             "r"(0)
                             : "memory");
        }
    __syncthreads();

    const int room = room_of(c);
    const int pos_first = position_of(tile.ch, a.group, tile.row0);
    const int pos_last = position_of(tile.ch, a.group, tile.row0 + tile.rows - 1);
    const int low = a.window > 0 ? max(0, pos_first - a.window + 1) : 0;
    const int high = min(pos_last + 1, room);
    const int sees_all_from = a.window > 0 ? max(0, pos_last - a.window + 1) : 0;
    const int first_group = low >> 3, groups = high > low ? ((high + 7) >> 3) - first_group : 0;
    const int workers = ranks * kWarps, worker = rank * kWarps + warp;

    constexpr int kCols = D / 32;   // this lane's columns: 32 apart (piece lane / 4 + 8 i for more)
    float m[ROWS], l[ROWS], o[ROWS][kCols];
#pragma unroll
    for (int r = 0; r < ROWS; r++) {
        m[r] = -INFINITY;
        l[r] = 0.0f;
#pragma unroll
        for (int i = 0; i < kCols; i++) o[r][i] = 0.0f;
    }
    const float factor = a.scale * kLog2e;
    const int key = lane >> 2, quarter = lane & 3;

    uint32_t held_bits = 0;
    auto fetch = [&](int it) {
        const int g = worker + it * workers;
        if (g < groups) {
            const int st = it % STAGES;
            const uint32_t held = R::load(c, tile.ch.stream, kvh, (first_group + g) * 8, low, high, room,
                                          ring + st * R::kStage);
            held_bits = (held_bits & ~(1u << st)) | held << st;
        }
        cp_async_commit();
    };
#pragma unroll
    for (int i = 0; i < STAGES - 1; i++) fetch(i);
    for (int it = 0; worker + it * workers < groups; it++) {
        fetch(it + STAGES - 1);
        cp_async_wait<STAGES - 1>();
        __syncwarp();
        const int st = it % STAGES;
        const uint32_t keys = ring + st * R::kStage, values = keys + R::kHalf;
        const int j0 = (first_group + worker + it * workers) * 8;
        const bool held = held_bits >> st & 1u;
        float x[ROWS];
#pragma unroll
        for (int r = 0; r < ROWS; r++) x[r] = 0.0f;
#pragma unroll 4
        for (int i = 0; i < D / 16; i++) {
            const int p = 4 * i + quarter;
            float4 k;
            asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];"
                         : "=f"(k.x), "=f"(k.y), "=f"(k.z), "=f"(k.w)
                         : "r"(keys + key * R::kRow + ((p ^ key) << 4)));
#pragma unroll
            for (int r = 0; r < ROWS; r++) {
                const float4 q = reinterpret_cast<const float4 *>(s_q)[r * R::kPieces + p];
                x[r] = fmaf(q.x, k.x, fmaf(q.y, k.y, fmaf(q.z, k.z, fmaf(q.w, k.w, x[r]))));
            }
        }
        const bool partial = j0 < sees_all_from || j0 + 7 > pos_first || j0 + 7 >= high || !held;
        auto sees = [&](int r, int j) {
            const int pos = position_of(tile.ch, a.group, tile.row0 + min(r, tile.rows - 1));
            return held && j <= pos && j < high && (a.window <= 0 || j > pos - a.window);
        };
#pragma unroll
        for (int r = 0; r < ROWS; r++) {
            x[r] += __shfl_xor_sync(kFull, x[r], 1);
            x[r] += __shfl_xor_sync(kFull, x[r], 2);
            x[r] *= factor;
            const bool in = !partial || sees(r, j0 + key);
            float most = in ? x[r] : -INFINITY;
            most = fmaxf(most, __shfl_xor_sync(kFull, most, 4));
            most = fmaxf(most, __shfl_xor_sync(kFull, most, 8));
            most = fmaxf(most, __shfl_xor_sync(kFull, most, 16));
            if (most > m[r]) {   // the same in every lane
                const float keep = m[r] == -INFINITY ? 0.0f : exp2f(m[r] - most);
                l[r] *= keep;
#pragma unroll
                for (int i = 0; i < kCols; i++) o[r][i] *= keep;
                m[r] = most;
            }
            const float w = in ? exp2f(x[r] - m[r]) : 0.0f;
            l[r] += w;
            if (quarter == 0) s_w[warp][key][r] = w;
        }
        __syncwarp();
#pragma unroll 2
        for (int k = 0; k < 8; k++) {
            float v[kCols];
#pragma unroll
            for (int i = 0; i < kCols; i++) {
                const int col = lane + 32 * i;
                asm volatile("ld.shared.f32 %0, [%1];"
                             : "=f"(v[i])
                             : "r"(values + k * R::kRow + (((col >> 2) ^ k) << 4) + 4 * (col & 3)));
            }
#pragma unroll
            for (int r = 0; r < ROWS; r++) {
                const float w = s_w[warp][k][r];
#pragma unroll
                for (int i = 0; i < kCols; i++)
                    // a value that the row does not see has no part in it, not even as 0 times it
                    if (!partial || !odd(v[i]) || sees(r, j0 + k)) o[r][i] = fmaf(w, v[i], o[r][i]);
            }
        }
        __syncwarp();
    }
    cp_async_wait<0>();
    __syncthreads();
    float *part = reinterpret_cast<float *>(smem);
#pragma unroll
    for (int r = 0; r < ROWS; r++) {
        l[r] += __shfl_xor_sync(kFull, l[r], 4);
        l[r] += __shfl_xor_sync(kFull, l[r], 8);
        l[r] += __shfl_xor_sync(kFull, l[r], 16);
        if (lane == 0) s_ml[warp * ROWS + r] = make_float2(m[r], l[r]);
#pragma unroll
        for (int i = 0; i < kCols; i++) part[(warp * ROWS + r) * D + lane + 32 * i] = o[r][i];
    }
    join_and_store<float, D, ROWS>(c, a, tile, kvh, part, s_ml, ranks, rank);
}

template <typename Kernel>
cudaError_t launch_rows(Kernel kernel, size_t smem, int tile_rows, const CacheArgs &c, const AttendArgs &a,
                        int keys, std::mutex &mu, bool (&ready)[64], cudaStream_t stream)
{
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (dev < 0 || dev >= 64) return cudaErrorInvalidDevice;
    {
        std::lock_guard<std::mutex> lk(mu);
        if (!ready[dev]) {
            e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
            if (e == cudaSuccess) e = cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
            if (e != cudaSuccess) return e;
            ready[dev] = true;
        }
    }
    const long long tiles = (long long)c.rows * a.group / tile_rows + c.n_streams;
    // tiles that hold rows, as far as the caller says
    const int most_new = a.max_new > 0 && a.max_new < c.rows ? a.max_new : c.rows;
    const long long filled = (long long)c.n_streams * (((long long)most_new * a.group + tile_rows - 1) / tile_rows);
    const long long work = (filled < tiles ? filled : tiles) * c.n_kv;
    const long long room = ((long long)c.max_pages << c.page_shift) / (keys * kWarps);
    int ranks = 1;
    while (ranks < 16 && work * ranks < 148 * 4 && ranks < room) ranks *= 2;
#ifdef Z2_RANKS
    ranks = Z2_RANKS;
#endif
    if (tiles * ranks > 0x7fffffffll) return cudaErrorInvalidConfiguration;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(tiles * ranks), (unsigned)c.n_kv);
    cfg.blockDim = dim3(kThreadsRows);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = (unsigned)ranks;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = ranks > 1 ? 2 : 1;
    return cudaLaunchKernelEx(&cfg, kernel, c, a, ranks);
}

template <int D, int MB, int STAGES>
cudaError_t launch_bf16(const CacheArgs &c, const AttendArgs &a, cudaStream_t stream)
{
    static std::mutex mu;
    static bool ready[64] = {false};
    typedef Ring<__nv_bfloat16, D, 16> R;
    const size_t rings = kWarps * STAGES * R::kStage, parts = (size_t)kWarps * 16 * MB * D * 4;
    const size_t smem = (rings > parts ? rings : parts) + 16 * MB * R::kRow;
    return launch_rows(attend_rows_bf16_kernel<D, MB, STAGES>, smem, 16 * MB, c, a, 16, mu, ready, stream);
}

template <int D, int ROWS, int STAGES>
cudaError_t launch_f32(const CacheArgs &c, const AttendArgs &a, cudaStream_t stream)
{
    static std::mutex mu;
    static bool ready[64] = {false};
    typedef Ring<float, D, 8> R;
    const size_t rings = kWarps * STAGES * R::kStage, parts = (size_t)kWarps * ROWS * D * 4;
    const size_t smem = (rings > parts ? rings : parts) + ROWS * R::kRow;
    return launch_rows(attend_rows_f32_kernel<D, ROWS, STAGES>, smem, ROWS, c, a, 8, mu, ready, stream);
}

}  // namespace

cudaError_t launch_cache_attend(const CacheArgs &c, const AttendArgs &a, bool bf16, cudaStream_t stream)
{
    // rows of a stream that share a key head
    const int most_new = a.max_new > 0 && a.max_new < c.rows ? a.max_new : c.rows;
    const long long rows = (long long)most_new * a.group;
    if (bf16) {
        if (c.dim > 128) return launch_bf16<256, 1, 3>(c, a, stream);
        if (c.dim > 64) return rows > 16 ? launch_bf16<128, 2, 3>(c, a, stream) : launch_bf16<128, 1, 3>(c, a, stream);
        return rows > 16 ? launch_bf16<64, 2, 4>(c, a, stream) : launch_bf16<64, 1, 4>(c, a, stream);
    }
    if (c.dim > 128) return rows > 4 ? launch_f32<256, 8, 3>(c, a, stream) : launch_f32<256, 4, 3>(c, a, stream);
    if (c.dim > 64) return rows > 4 ? launch_f32<128, 16, 3>(c, a, stream) : launch_f32<128, 4, 3>(c, a, stream);
    return rows > 4 ? launch_f32<64, 16, 4>(c, a, stream) : launch_f32<64, 4, 4>(c, a, stream);
}

}  // namespace z2
