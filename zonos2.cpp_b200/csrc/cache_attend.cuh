// cache_attend.cuh -- what the paged cache's attention kernels share (cache_attend.cu,
// cache_attend_tc.cu).
#pragma once

#include <math.h>

#include "cache.cuh"
#include "tc.cuh"

namespace z2 {

namespace {

constexpr float kLog2e = 1.4426950408889634f;
// The maximum of a part whose row saw tokens with scores of -inf alone (its sum is zero): where the
// row has no other, the result is a NaN, as the definition has it.
constexpr float kLowest = -3.402823466e38f;

__device__ __forceinline__ float exp2_fast(float x)
{
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

__device__ __forceinline__ void cp_async16(uint32_t dst, const void *src)
{
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
// The same, or zeros without a read.
__device__ __forceinline__ void cp_async16_or_zero(uint32_t dst, const void *src, bool take)
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
    asm(
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

// Bits 15 and 31: an exponent of ones in the lower and the upper bf16 (one more carries out of it).
__device__ __forceinline__ uint32_t odd_bits(uint32_t w) { return (w & 0x7f807f80u) + 0x00800080u; }

__device__ __forceinline__ bool odd(float v) { return (__float_as_uint(v) & 0x7f800000u) == 0x7f800000u; }
// A NaN or an infinity among the two bf16 values of a word.
__device__ __forceinline__ bool odd2(uint32_t w)
{
    return (odd_bits(w) & 0x80008000u) != 0;
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
    if (threadIdx.x == 0) *s_found = c.n_streams;
    __syncthreads();
    auto number = [&](int s) {
        const int first = min(max(c.q_start[s], 0), c.rows);
        return (long long)first * group / tile_rows + s;
    };
    for (int s = threadIdx.x; s < c.n_streams; s += blockDim.x)
        // one stream's, as the starts rise; if they do not, the same one in every block
        if (number(s) <= t && t < number(s + 1)) atomicMin(s_found, s);
    __syncthreads();
    const int s = *s_found;
    Tile tile;
    tile.rows = 0;
    if (s >= c.n_streams) return tile;
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

// Joins the parts of the block's warps (and of the cluster's blocks) and stores the rows.
// part: [W][ROWS][D] f32 outputs, 16-byte piece p of row r at piece p ^ (2 r & 14) (rows of the
// mma.sync kernel then fall on different banks); ml: [W][ROWS] maxima and sums; weight: room
// for kMostRanks * ROWS factors, total for ROWS; gate: the rows' factors.
constexpr int kMostRanks = 16;

__device__ __forceinline__ int part_piece(int r, int p) { return p ^ ((2 * r) & 14); }

// The rows' gates, to shared memory, ahead of their use.
template <typename T>
__device__ __forceinline__ void load_gates(const AttendArgs &a, const Tile &tile, int kvh, float *gate)
{
    for (int r = threadIdx.x; r < tile.rows; r += blockDim.x) {
        const int row = tile.row0 + r;
        const T *at = (const T *)a.gate + (long long)(tile.ch.first + row / a.group) * a.gate_stride;
        gate[r] = a.gate ? 1.0f / (1.0f + expf(-as_f(at[kvh * a.group + row % a.group]))) : 1.0f;
    }
}

template <typename T, int D, int ROWS, int W, int THREADS>
__device__ void join_and_store(const CacheArgs &c, const AttendArgs &a, const Tile &tile, int kvh,
                               float *part, float2 *ml, float *weight, float *total, const float *gate,
                               int ranks, int rank)
{
    constexpr int kQuads = ROWS * D / 4;
    const int quads = tile.rows * (D / 4);   // of the tile's rows
    // A part without a visible token (m = -inf) weighs nothing; a NaN sum stays one.
    auto weigh = [](float m, float most) { return m == -INFINITY ? 0.0f : exp2_fast(m - most); };
    auto add = [](float4 &sum, float f, const float4 &v) {
        sum.x = fmaf(f, v.x, sum.x);
        sum.y = fmaf(f, v.y, sum.y);
        sum.z = fmaf(f, v.z, sum.z);
        sum.w = fmaf(f, v.w, sum.w);
    };
    __syncthreads();
    // the block's own warps, into warp 0's part
    for (int r = threadIdx.x; r < tile.rows; r += THREADS) {
        float most = -INFINITY, l = 0.0f;
#pragma unroll
        for (int w = 0; w < W; w++) most = fmaxf(most, ml[w * ROWS + r].x);
#pragma unroll
        for (int w = 0; w < W; w++) {
            const float f = weigh(ml[w * ROWS + r].x, most);
            weight[w * ROWS + r] = f;   // W <= kMostRanks
            l += f * ml[w * ROWS + r].y;
        }
        ml[r] = make_float2(most, l);
    }
    __syncthreads();
    for (int i = threadIdx.x; i < quads; i += THREADS) {
        const int r = i / (D / 4);
        float4 sum = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
        for (int w = 0; w < W; w++)
            add(sum, weight[w * ROWS + r], reinterpret_cast<const float4 *>(part)[w * kQuads + i]);
        reinterpret_cast<float4 *>(part)[i] = sum;
    }
    if (ranks > 1) {
        cluster_sync();
        // every rank's maximum and sum, all asked for at once
        for (int i = threadIdx.x; i < ranks * ROWS; i += THREADS) {
            const int k = i / ROWS, r = i % ROWS;
            float m, l;
            asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];"
                         : "=f"(m), "=f"(l)
                         : "r"(peer_addr(smem_u32(ml + r), k)));
            reinterpret_cast<float2 *>(part + ROWS * D)[i] = make_float2(m, l);   // behind the block's part
        }
        __syncthreads();
        for (int r = threadIdx.x; r < ROWS; r += THREADS) {
            const float2 *all = reinterpret_cast<const float2 *>(part + ROWS * D) + r;
            float most = -INFINITY, l = 0.0f;
            for (int k = 0; k < ranks; k++) most = fmaxf(most, all[k * ROWS].x);
            for (int k = 0; k < ranks; k++) {
                const float f = weigh(all[k * ROWS].x, most);
                weight[k * ROWS + r] = f;
                l += f * all[k * ROWS].y;
            }
            total[r] = l == 0.0f && most > -INFINITY ? NAN : l;
        }
    } else {
        for (int r = threadIdx.x; r < ROWS; r += THREADS) total[r] = ml[r].y == 0.0f && ml[r].x > -INFINITY ? NAN : ml[r].y;
    }
    __syncthreads();
    // this rank's share of the rows' quads
    const int per = (quads + ranks - 1) / ranks;
    const int end = min(quads, (rank + 1) * per);
    for (int i = rank * per + threadIdx.x; i < end; i += THREADS) {
        const int r = i / (D / 4), d = part_piece(r, i % (D / 4)) * 4;
        if (d >= c.dim) continue;
        float4 sum = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        if (ranks > 1) {
            const uint32_t at = smem_u32(part) + i * 16;
            for (int k0 = 0; k0 < ranks; k0 += 4) {   // ranks: 2, or a multiple of 4
                float4 v[4];
#pragma unroll
                for (int k = 0; k < 4; k++)
                    if (k0 + k < ranks)
                        asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
                                     : "=f"(v[k].x), "=f"(v[k].y), "=f"(v[k].z), "=f"(v[k].w)
                                     : "r"(peer_addr(at, k0 + k)));
#pragma unroll
                for (int k = 0; k < 4; k++)
                    if (k0 + k < ranks) add(sum, weight[(k0 + k) * ROWS + r], v[k]);
            }
        } else {
            sum = reinterpret_cast<const float4 *>(part)[i];
        }
        const float l = total[r];
        const int row = tile.row0 + r, token = tile.ch.first + row / a.group;
        const int h = kvh * a.group + row % a.group;
        const float f = l == 0.0f ? 0.0f : gate[r] / l;
        T *to = (T *)a.out + token * a.out_stride + (long long)h * c.dim + d;
        if (sizeof(T) == 2) {
            *reinterpret_cast<uint2 *>(to) = make_uint2(pack_bf16(sum.x * f, sum.y * f), pack_bf16(sum.z * f, sum.w * f));
        } else {
            *reinterpret_cast<float4 *>(to) = make_float4(sum.x * f, sum.y * f, sum.z * f, sum.w * f);
        }
    }
    if (ranks > 1) cluster_sync();   // the others have read this block's part
}

// Tiles that hold rows, as far as the caller says.
inline long long tiles_with_rows(const CacheArgs &c, const AttendArgs &a, int tile_rows)
{
    const long long tiles = (long long)c.rows * a.group / tile_rows + c.n_streams;
    const int most_new = a.max_new > 0 && a.max_new < c.rows ? a.max_new : c.rows;
    const long long filled = (long long)c.n_streams * (((long long)most_new * a.group + tile_rows - 1) / tile_rows);
    return filled < tiles ? filled : tiles;
}

// .. and as many as there may well be: the token rows', and half a tile more to each stream.
inline long long likely_tiles(const CacheArgs &c, const AttendArgs &a, int tile_rows)
{
    const long long most = tiles_with_rows(c, a, tile_rows), least = c.rows < c.n_streams ? c.rows : c.n_streams;
    const long long tiles = ((long long)c.rows * a.group + tile_rows - 1) / tile_rows + c.n_streams / 2;
    return tiles > most ? most : tiles < least ? least : tiles;
}

}  // namespace

// bf16, many rows to a key head (cache_attend_tc.cu).
cudaError_t launch_cache_attend_tc(const CacheArgs &c, const AttendArgs &a, cudaStream_t stream);
int read_and_clear_attend_error(int *value);

}  // namespace z2
