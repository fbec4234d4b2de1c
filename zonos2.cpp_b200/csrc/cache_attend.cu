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
// has a ring of groups of its own in flight by asynchronous copies, the pages looked up a turn
// ahead, and no block-wide barrier before the join.  16 + 4 bf16 heads of 128:
//   256 streams of 256 to 4096 tokens, one new (1.14 GB)       187 us, 6.1 TB/s
//   64 streams of 64 to 6144, up to five new (408 MB)           78 us, 5.2 TB/s
//   1 stream of 6050, one new (12.4 MB)                         10 us: a chain of latencies (1.5 the
//       tile, 2.5 its pages and queries, 3.6 the keys and the work on them, 4.5 the join)
#include <math.h>

#include <mutex>

#include "cache_attend.cuh"

namespace z2 {

namespace {

// KEYS keys and values of D elements (rows of `dim`) of one key head, as one stage of a warp's
// ring: the keys' rows, then the values'.  16-byte piece p of row r lies at piece p ^ (r & 7), so
// that eight rows' same piece falls on different banks.
template <typename T, int D, int KEYS>
struct Ring {
    static constexpr int kRow = D * (int)sizeof(T);      // bytes
    static constexpr int kHalf = KEYS * kRow;
    static constexpr int kStage = 2 * kHalf;
    static constexpr int kPieces = kRow / 16;

    // The pages of a group's runs of eight keys.  (on: the group is one; j0 of others, past the last,
    // may have left 32 bits.)
    struct Pages {
        int p[KEYS / 8];
    };
    __device__ static Pages look(const CacheArgs &c, int s, int j0, int room, bool on)
    {
        Pages pages;
#pragma unroll
        for (int e = 0; e < KEYS / 8; e++) pages.p[e] = on && j0 + 8 * e < room ? page_of(c, s, j0 + 8 * e) : -1;
        return pages;
    }

    // Loads the keys and values [j0, j0 + KEYS) that lie in [low, high) and on a page; zeros
    // elsewhere.  Returns the bits of KEYS / 8 runs of eight that lie on a page.
    __device__ static uint32_t load(const CacheArgs &c, const Pages &pages, int kvh, int j0, int low, int high,
                                    uint32_t stage)
    {
        const int lane = threadIdx.x & 31;
        const int row0 = lane / kPieces, piece = lane % kPieces;
        constexpr int kStep = 32 / kPieces > 0 ? 32 / kPieces : 1;          // rows of a warp's copy
        constexpr int kAcross = kPieces > 32 ? kPieces / 32 : 1;            // copies of a row
        // a run of eight lies on one page, and so do two unless pages hold eight
        long long base[KEYS / 8];
        uint32_t held = 0;
#pragma unroll
        for (int e = 0; e < KEYS / 8; e++) {
            base[e] = pages.p[e] >= 0 ? row_on_page(c, pages.p[e], kvh, j0 + 8 * e) : 0;
            held |= pages.p[e] >= 0 ? 1u << e : 0u;
        }
        const uint32_t to = stage + row0 * kRow;
        if (held == (1u << KEYS / 8) - 1 && j0 >= low && j0 + KEYS <= high &&
            (KEYS == 8 || c.page_shift > 3)) {   // a whole group: its rows lie behind each other
            const uint32_t bytes = (uint32_t)c.dim * sizeof(T);   // of a row
            const uint32_t from = row0 * bytes + piece * 16;
            const char *k = (const char *)((const T *)c.k + base[0]), *v = (const char *)((const T *)c.v + base[0]);
#pragma unroll
            for (int i = 0; i < KEYS / kStep; i++)
#pragma unroll
                for (int x = 0; x < kAcross; x++) {
                    const int r = i * kStep;   // row0 + r; row0 < kStep
                    if (piece * 16 + 512 * x >= (int)bytes) break;
                    const uint32_t dst = to + r * kRow + (((piece + 32 * x) ^ ((row0 + r) & 7)) << 4);
                    const uint32_t at = from + r * bytes + 512 * x;
                    cp_async16(dst, k + at);
                    cp_async16(dst + kHalf, v + at);
                }
            return held;
        }
        const int live = c.dim * (int)sizeof(T) / 16;   // pieces of a row that there are
#pragma unroll 1
        for (int i = 0; i < KEYS / kStep; i++) {
            const int r = row0 + i * kStep, j = j0 + r;
            const bool take = (held >> (r >> 3) & 1u) && j >= low && j < high;
            const long long at = take ? (KEYS == 8 || r < 8 ? base[0] : base[KEYS / 8 - 1]) + (r & 7) * c.dim : 0;
            for (int x = piece; x < live; x += 32) {
                const uint32_t dst = stage + r * kRow + ((x ^ (r & 7)) << 4);
                cp_async16_or_zero(dst, (const T *)c.k + at + x * (16 / (int)sizeof(T)), take);
                cp_async16_or_zero(dst + kHalf, (const T *)c.v + at + x * (16 / (int)sizeof(T)), take);
                if (kPieces <= 32) break;
            }
        }
        return held;
    }
};

// ---- bf16, by mma.sync ------------------------------------------------------
// 16 rows to a tile, groups of 16 keys: S = Q K^T by m16n8k16 (rows x 8 keys x 16 elements),
// whose accumulators, rounded to bf16, are the left operand of O += P V.  That rounding is chosen: both operands of an MMA are
// of one type, and the values are bf16; the weights' rest would be a second product.  It is half a step of bf16 a weight, of another sign for each
// key, so that the result's error in the 2-norm is 2.0e-3 to 2.3e-3 where its own rounding makes 1.7e-3.
// Two stages a ring, so that three blocks fit an SM: 64 streams of up to 6144 tokens and 20 rows
// took 77 us with two stages, 92 with three; by pairs of warps that shared a ring's keys between
// 32 rows 108 us, as most of the second 16 rows were none.
template <int D, int STAGES, int W>
__global__ void __launch_bounds__(32 * W, D > 128 || W > 4 ? 1 : 3)
    attend_rows_bf16_kernel(const CacheArgs c, const AttendArgs a, int ranks)
{
    typedef Ring<__nv_bfloat16, D, 16> R;
    constexpr int ROWS = 16, kThreads = 32 * W;
    extern __shared__ __align__(1024) unsigned char smem[];
    // the rings, then the queries; at the end the parts take the rings' place
    __shared__ float2 s_ml[W * ROWS];
    __shared__ float s_weight[kMostRanks * ROWS], s_total[ROWS], s_gate[ROWS];
    __shared__ int s_found;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int rank = blockIdx.x % ranks, kvh = blockIdx.y;
    const Tile tile = find_tile(c, a.group, ROWS, blockIdx.x / ranks, &s_found);
    if (tile.rows == 0) return;   // the whole cluster's tile

    // the tokens that some row of the tile sees, in groups of 16
    const int room = room_of(c);
    const int pos_first = position_of(tile.ch, a.group, tile.row0);
    const int pos_last = position_of(tile.ch, a.group, tile.row0 + tile.rows - 1);
    const int low = a.window > 0 ? max(0, pos_first - a.window + 1) : 0;
    const int high = min(pos_last + 1, room);
    const int sees_all_from = a.window > 0 ? max(0, pos_last - a.window + 1) : 0;   // .. to pos_first
    const int first_group = low >> 4, groups = high > low ? ((high + 15) >> 4) - first_group : 0;
    const int workers = ranks * W, worker = rank * W + warp;
    auto group_at = [&](int it) { return (int)((uint32_t)(first_group + worker + it * workers) * 16u); };
    auto look = [&](int it) { return R::look(c, tile.ch.stream, group_at(it), room, worker + it * workers < groups); };
    typename R::Pages pages[STAGES];   // of the first turns, then [0]: of the next one to be fetched
#pragma unroll
    for (int i = 0; i < STAGES; i++) pages[i] = look(i);

    const uint32_t ring = smem_u32(smem) + warp * STAGES * R::kStage;
    const uint32_t s_q = smem_u32(smem) + W * STAGES * R::kStage;
    const int live = c.dim / 8;
    // queries (zeros past the rows and the head's elements), swizzled like the keys
    for (int i = threadIdx.x; i < ROWS * R::kPieces; i += kThreads) {
        const int r = i / R::kPieces, p = i % R::kPieces, row = tile.row0 + r;
        const bool in = r < tile.rows && p < live;
        const long long at = in ? (tile.ch.first + row / a.group) * a.q_stride +
                                      (long long)(kvh * a.group + row % a.group) * c.dim + p * 8
                                : 0;
        cp_async16_or_zero(s_q + r * R::kRow + ((p ^ (r & 7)) << 4), (const __nv_bfloat16 *)a.q + at, in);
    }
    cp_async_commit();
    load_gates<__nv_bfloat16>(a, tile, kvh, s_gate);
    if (live < R::kPieces)   // pieces that no copy fills
        for (int i = lane; i < STAGES * 32 * R::kPieces; i += 32) {
            const int r = i / R::kPieces, p = i % R::kPieces;
            if (p >= live)
                asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(ring + r * R::kRow + ((p ^ (r & 7)) << 4)),
                             "r"(0)
                             : "memory");
        }
    uint32_t held_bits = 0;   // two bits to a stage
    auto fetch = [&](int it, const typename R::Pages &at) {
        if (worker + it * workers < groups) {
            const int st = it % STAGES;
            const uint32_t to = ring + st * R::kStage;
            const uint32_t held = R::load(c, at, kvh, group_at(it), low, high, to);
            held_bits = (held_bits & ~(3u << (2 * st))) | held << (2 * st);
        }
        cp_async_commit();
    };
#pragma unroll
    for (int i = 0; i < STAGES - 1; i++) fetch(i, pages[i]);
    pages[0] = pages[STAGES - 1];
    cp_async_wait<STAGES - 1>();   // the queries
    __syncthreads();

    int pos[2];   // of this lane's rows (those past the tile's take the last row's)
#pragma unroll
    for (int i = 0; i < 2; i++)
        pos[i] = position_of(tile.ch, a.group, tile.row0 + min(i * 8 + (lane >> 2), tile.rows - 1));
    float m[2], l[2], o[D / 8][4];
#pragma unroll
    for (int i = 0; i < 2; i++) {
        m[i] = -INFINITY;
        l[i] = 0.0f;
    }
#pragma unroll
    for (int n = 0; n < D / 8; n++) o[n][0] = o[n][1] = o[n][2] = o[n][3] = 0.0f;
    const float factor = a.scale * kLog2e;
    uint32_t saw = 0;   // bits as `seen`'s

    // ldmatrix: lane's row and piece of a 16 x 16 block
    const int lm_key = (lane & 7) + ((lane >> 4) << 3), lm_kp = (lane >> 3) & 1;     // keys: n blocks of 8
    const int lm_val = (lane & 7) + (((lane >> 3) & 1) << 3), lm_vp = lane >> 4;     // values, transposed
    constexpr bool kQRegs = D <= 128;
    uint32_t qf[kQRegs ? D / 16 : 1][4];
    auto load_q = [&](int kk, uint32_t (&f)[4]) {
        const int r = lane & 15, p = 2 * kk + (lane >> 4);
        ldmatrix4(s_q + r * R::kRow + ((p ^ (r & 7)) << 4), f);
    };
    if (kQRegs) {
#pragma unroll
        for (int kk = 0; kk < D / 16; kk++) load_q(kk, qf[kk]);
    }

    for (int it = 0; worker + it * workers < groups; it++) {
        cp_async_wait<STAGES - 2>();
        __syncwarp();   // the group has landed, and the one before it is done with
        const typename R::Pages next = look(it + STAGES);
        fetch(it + STAGES - 1, pages[0]);
        pages[0] = next;
        const int st = it % STAGES;
        const uint32_t keys = ring + st * R::kStage, values = keys + R::kHalf;
        const int j0 = group_at(it);
        const uint32_t held = held_bits >> (2 * st) & 3u;
        float x[2][4];
#pragma unroll
        for (int n = 0; n < 2; n++) x[n][0] = x[n][1] = x[n][2] = x[n][3] = 0.0f;
#pragma unroll
        for (int kk = 0; kk < D / 16; kk++) {
            uint32_t kf[4], f[4];
            ldmatrix4(keys + lm_key * R::kRow + (((2 * kk + lm_kp) ^ (lm_key & 7)) << 4), kf);
            if (!kQRegs) load_q(kk, f);
            mma_16816(x[0], kQRegs ? qf[kQRegs ? kk : 0] : f, kf[0], kf[1]);
            mma_16816(x[1], kQRegs ? qf[kQRegs ? kk : 0] : f, kf[2], kf[3]);
        }
        // scores that a row does not see: out of the maximum, and of weight zero
        const bool partial = j0 < sees_all_from || j0 + 15 > pos_first || j0 + 15 >= high || held != 3u;
        auto sees = [&](int i, int j) {   // row slot i of this lane, token j
            return j <= pos[i] && j < high && (a.window <= 0 || j > pos[i] - a.window) && (held >> ((j - j0) >> 3) & 1u);
        };
        uint32_t seen = 0xffu;   // bit 4 i + 2 n + e
        if (partial) {
            seen = 0;
#pragma unroll
            for (int b = 0; b < 8; b++) {
                const int i = b >> 2, n = (b >> 1) & 1, e = b & 1;
                if (sees(i, j0 + 8 * n + 2 * (lane & 3) + e))
                    seen |= 1u << b;
                else
                    x[n][i * 2 + e] = -INFINITY;
            }
        }
        saw |= seen;
        float top[2];
        bool same = true;
#pragma unroll
        for (int i = 0; i < 2; i++) {
            float most = fmaxf(fmaxf(x[0][2 * i], x[0][2 * i + 1]), fmaxf(x[1][2 * i], x[1][2 * i + 1]));
            most = fmaxf(most, __shfl_xor_sync(kFull, most, 1));
            most = fmaxf(most, __shfl_xor_sync(kFull, most, 2));
            top[i] = fmaxf(most * factor, m[i]);   // factor > 0
            same = same && top[i] == m[i];
        }
        if (!__all_sync(kFull, same)) {
#pragma unroll
            for (int i = 0; i < 2; i++) {
                const float keep = m[i] == -INFINITY ? 0.0f : exp2_fast(m[i] - top[i]);
                m[i] = top[i];
                l[i] *= keep;
#pragma unroll
                for (int n = 0; n < D / 8; n++) {
                    o[n][i * 2] *= keep;
                    o[n][i * 2 + 1] *= keep;
                }
            }
        }
        const float base[2] = {m[0] == -INFINITY ? 0.0f : m[0], m[1] == -INFINITY ? 0.0f : m[1]};
#pragma unroll
        for (int n = 0; n < 2; n++)
#pragma unroll
            for (int e = 0; e < 4; e++) x[n][e] = exp2_fast(fmaf(x[n][e], factor, -base[e >> 1]));
#pragma unroll
        for (int i = 0; i < 2; i++) l[i] += (x[0][2 * i] + x[0][2 * i + 1]) + (x[1][2 * i] + x[1][2 * i + 1]);
        uint32_t pf[4];
        pf[0] = pack_bf16(x[0][0], x[0][1]);
        pf[1] = pack_bf16(x[0][2], x[0][3]);
        pf[2] = pack_bf16(x[1][0], x[1][1]);
        pf[3] = pack_bf16(x[1][2], x[1][3]);
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
#pragma unroll 1
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
                        for (int i = 0; i < 2; i++)
                            if (sees(i, j0 + k)) {
                                if (odd(v0)) o[n][i * 2] += v0;
                                if (odd(v1)) o[n][i * 2 + 1] += v1;
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
            mma_16816(o[2 * n], pf, vf[0], vf[1]);
            mma_16816(o[2 * n + 1], pf, vf[2], vf[3]);
        }
    }
    cp_async_wait<0>();
    __syncthreads();   // every warp is done with its ring: the parts take their place
    float *part = reinterpret_cast<float *>(smem);
#pragma unroll
    for (int i = 0; i < 2; i++) {
        l[i] += __shfl_xor_sync(kFull, l[i], 1);
        l[i] += __shfl_xor_sync(kFull, l[i], 2);
        const int r = i * 8 + (lane >> 2);
        const bool any = __ballot_sync(kFull, (saw >> (4 * i) & 15u) != 0) >> (lane & ~3) & 15u;
        if ((lane & 3) == 0) s_ml[warp * ROWS + r] = make_float2(m[i] == -INFINITY && any ? kLowest : m[i], l[i]);
#pragma unroll
        for (int n = 0; n < D / 8; n++)
            *reinterpret_cast<float2 *>(part + (warp * ROWS + r) * D + part_piece(r, 2 * n + ((lane & 3) >> 1)) * 4 + 2 * (lane & 1)) =
                make_float2(o[n][i * 2], o[n][i * 2 + 1]);
    }
    join_and_store<__nv_bfloat16, D, ROWS, W, kThreads>(c, a, tile, kvh, part, s_ml, s_weight, s_total, s_gate, ranks, rank);
}

// ---- f32, on the FMA pipe ----------------------------------------------------
// ROWS rows to a tile, groups of 8 keys.  A lane takes a quarter of a key's elements for
// the scores of all rows (key lane / 4), then D / 32 of the output's columns.  8 + 2 heads of 128, 64
// streams of 1500 tokens, one new (197 MB): 63 us, 3.1 TB/s; 175 us with more blocks to a cluster than it takes, each group's page looked up
// in its turn and the values read four bytes at a time.
template <int D, int ROWS, int STAGES, int W>
__global__ void __launch_bounds__(32 * W)
    attend_rows_f32_kernel(const CacheArgs c, const AttendArgs a, int ranks)
{
    typedef Ring<float, D, 8> R;
    extern __shared__ __align__(1024) unsigned char smem[];
    __shared__ float2 s_ml[W * ROWS];
    __shared__ float s_weight[kMostRanks * ROWS], s_total[ROWS], s_gate[ROWS];
    __shared__ __align__(16) float s_w[W][8][ROWS];   // a group's weights
    __shared__ int s_found;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int rank = blockIdx.x % ranks, kvh = blockIdx.y;
    const Tile tile = find_tile(c, a.group, ROWS, blockIdx.x / ranks, &s_found);
    if (tile.rows == 0) return;

    const uint32_t ring = smem_u32(smem) + warp * STAGES * R::kStage;
    float *s_q = reinterpret_cast<float *>(smem + W * STAGES * R::kStage);   // [ROWS][D]
    const int live = c.dim / 4;
    for (int i = threadIdx.x; i < ROWS * R::kPieces; i += (32 * W)) {
        const int r = i / R::kPieces, p = i % R::kPieces, row = tile.row0 + r;
        float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        if (r < tile.rows && p < live)
            v = *reinterpret_cast<const float4 *>((const float *)a.q + (tile.ch.first + row / a.group) * a.q_stride +
                                                  (long long)(kvh * a.group + row % a.group) * c.dim + p * 4);
        reinterpret_cast<float4 *>(s_q)[i] = v;
    }
    load_gates<float>(a, tile, kvh, s_gate);
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
    const int workers = ranks * W, worker = rank * W + warp;

    // this lane's columns: kRun neighbours of each 32 kRun
    constexpr int kCols = D / 32, kRun = kCols < 4 ? kCols : 4;
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
    uint32_t saw = 0;   // of this lane's key, a bit to a row

    auto group_at = [&](int it) { return (int)((uint32_t)(first_group + worker + it * workers) * 8u); };
    auto look = [&](int it) { return R::look(c, tile.ch.stream, group_at(it), room, worker + it * workers < groups); };
    uint32_t held_bits = 0;
    auto fetch = [&](int it, const typename R::Pages &at) {
        if (worker + it * workers < groups) {
            const int st = it % STAGES;
            const uint32_t held = R::load(c, at, kvh, group_at(it), low, high, ring + st * R::kStage);
            held_bits = (held_bits & ~(1u << st)) | held << st;
        }
        cp_async_commit();
    };
    typename R::Pages pages[STAGES];   // of the first turns, then [0]: of the next one to be fetched
#pragma unroll
    for (int i = 0; i < STAGES; i++) pages[i] = look(i);
#pragma unroll
    for (int i = 0; i < STAGES - 1; i++) fetch(i, pages[i]);
    pages[0] = pages[STAGES - 1];
    for (int it = 0; worker + it * workers < groups; it++) {
        const typename R::Pages next = look(it + STAGES);
        fetch(it + STAGES - 1, pages[0]);
        pages[0] = next;
        cp_async_wait<STAGES - 1>();
        __syncwarp();
        const int st = it % STAGES;
        const uint32_t keys = ring + st * R::kStage, values = keys + R::kHalf;
        const int j0 = group_at(it);
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
        float top[ROWS];
        bool same = true;
#pragma unroll
        for (int r = 0; r < ROWS; r++) {
            x[r] += __shfl_xor_sync(kFull, x[r], 1);
            x[r] += __shfl_xor_sync(kFull, x[r], 2);
            x[r] *= factor;
        }
        if (partial) {
#pragma unroll
            for (int r = 0; r < ROWS; r++) {
                const bool in = sees(r, j0 + key);
                if (!in) x[r] = -INFINITY;
                saw |= in ? 1u << r : 0u;
            }
        } else {
            saw = ~0u;
        }
#pragma unroll
        for (int r = 0; r < ROWS; r++) {
            top[r] = x[r];
            top[r] = fmaxf(top[r], __shfl_xor_sync(kFull, top[r], 4));
            top[r] = fmaxf(top[r], __shfl_xor_sync(kFull, top[r], 8));
            top[r] = fmaxf(top[r], __shfl_xor_sync(kFull, top[r], 16));
            top[r] = fmaxf(top[r], m[r]);   // the same in every lane
            same = same && top[r] == m[r];
        }
        if (!__all_sync(kFull, same)) {
#pragma unroll
            for (int r = 0; r < ROWS; r++) {
                const float keep = m[r] == -INFINITY ? 0.0f : exp2_fast(m[r] - top[r]);
                l[r] *= keep;
#pragma unroll
                for (int i = 0; i < kCols; i++) o[r][i] *= keep;
                m[r] = top[r];
            }
        }
#pragma unroll
        for (int r = 0; r < ROWS; r++) {
            const float w = exp2_fast(x[r] - (m[r] == -INFINITY ? 0.0f : m[r]));   // 0 where not seen
            l[r] += w;
            if (quarter == 0) s_w[warp][key][r] = w;
        }
        __syncwarp();
#pragma unroll 2
        for (int k = 0; k < 8; k++) {
            float v[kCols];
#pragma unroll
            for (int i = 0; i < kCols; i += kRun) {
                const int col = lane * kRun + 32 * i;
                const uint32_t at = values + k * R::kRow + (((col >> 2) ^ k) << 4) + 4 * (col & 3);
                if (kRun == 4)
                    asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];"
                                 : "=f"(v[i]), "=f"(v[i + 1]), "=f"(v[(i + 2) % kCols]), "=f"(v[(i + 3) % kCols])
                                 : "r"(at));
                else
                    asm volatile("ld.shared.v2.f32 {%0, %1}, [%2];" : "=f"(v[i]), "=f"(v[i + 1]) : "r"(at));
            }
            float w[ROWS];
#pragma unroll
            for (int r = 0; r < ROWS; r += 4) {
                const float4 w4 = *reinterpret_cast<const float4 *>(&s_w[warp][k][r]);
                w[r] = w4.x;
                w[r + 1] = w4.y;
                w[r + 2] = w4.z;
                w[r + 3] = w4.w;
            }
            if (partial) {
                // a value that the row does not see has no part in it, not even as 0 times it
#pragma unroll
                for (int i = 0; i < kCols; i++) {
                    if (!odd(v[i])) continue;
#pragma unroll
                    for (int r = 0; r < ROWS; r++)
                        if (sees(r, j0 + k)) o[r][i] += v[i];
                    v[i] = 0.0f;
                }
            }
#pragma unroll
            for (int r = 0; r < ROWS; r++)
#pragma unroll
                for (int i = 0; i < kCols; i++) o[r][i] = fmaf(w[r], v[i], o[r][i]);
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
        const bool any = __any_sync(kFull, saw >> r & 1u);
        if (lane == 0) s_ml[warp * ROWS + r] = make_float2(m[r] == -INFINITY && any ? kLowest : m[r], l[r]);
#pragma unroll
        for (int i = 0; i < kCols; i++) {
            const int col = lane * kRun + 32 * (i / kRun * kRun) + i % kRun;
            part[(warp * ROWS + r) * D + part_piece(r, col >> 2) * 4 + (col & 3)] = o[r][i];
        }
    }
    join_and_store<float, D, ROWS, W, 32 * W>(c, a, tile, kvh, part, s_ml, s_weight, s_total, s_gate, ranks, rank);
}

// ---- f32, many rows ----------------------------------------------------------
// 64 rows to a tile, 16 to a warp, steps of 32 keys that the block's four warps share.  The
// products run on the tensor cores in tf32 (11 bits of a significand), each operand as the sum
// of two such parts, hi = its upper bits and lo = the rest:
//     a b = hi_a hi_b + hi_a lo_b + lo_a hi_b + (2^-22 of it)
// (6 streams, up to 333 new tokens of 16 + 4 heads of 128, a window of 512: 124 to 187 us by their lengths, 2150 us by the
// kernel above), which leaves errors of the size of f32's own in a sum of 128 products (9e-7 in the 2-norm of the result
// against 5.7e-7 by f32 products; one part alone leaves 2^-14 and more).  The tensor cores add
// to an accumulator by truncation, a bias that grows with the number of additions: the upper
// parts' products, the mixed ones (2^-11 of them, and so their bias) and each 64 elements of the
// depth or 32 keys have accumulators of their own, which are added with rounding to nearest (with
// one accumulator for all of them 2500 keys were 5.5e-6 off, now 4e-7).  On the FMA pipe
// (ROWS = 16 above) a step's operands come from shared memory four times as often for the same
// products, and that bounds it.  Where an MMA's k runs over elements or keys, any order will
// do that both operands share: a lane takes four neighbouring elements of a row in one load,
// two for each of two MMAs; and the weights of a group of 8 keys, as the scores' accumulators
// hold them, are the left operand of its values if those take their keys in the order 0, 2, 4,
// 6, 1, 3, 5, 7.  The pitches keep those loads free of bank conflicts.
__device__ __forceinline__ void mma_tf32(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1)
{
    asm(
        "mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, "
        "{%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void split_tf32(float x, uint32_t &hi, uint32_t &lo)
{
    hi = __float_as_uint(x) & 0xffffe000u;
    lo = __float_as_uint(x - __uint_as_float(hi));
}
// The product of the upper parts into d, the mixed ones into e.
__device__ __forceinline__ void mma_3tf32(float (&d)[4], float (&e)[4], const uint32_t (&ah)[4], const uint32_t (&al)[4],
                                          uint32_t bh0, uint32_t bh1, uint32_t bl0, uint32_t bl1)
{
    mma_tf32(e, al, bh0, bh1);
    mma_tf32(e, ah, bl0, bl1);
    mma_tf32(d, ah, bh0, bh1);
}

constexpr int kTileKeys = 32, kTileRows = 64;

template <int D>
struct TileF32 {
    static constexpr int kPitch = D + 16, kPitchV = D + 4;   // floats of a row of Q and K, of V
    static constexpr int kStage = kTileKeys * (kPitch + kPitchV);
    static constexpr size_t kSmem = (size_t)(kTileRows * kPitch + 2 * kStage) * 4;
};

// A score by f32 arithmetic alone.
__device__ __noinline__ float plain_score(const float *q, const float *k, int n)
{
    float sum = 0.0f;
#pragma unroll 1
    for (int i = 0; i < n; i++) sum = fmaf(q[i], k[i], sum);
    return sum;
}

template <int D>
__global__ void __launch_bounds__(128, D <= 128 ? 2 : 1)
    attend_tile_f32_kernel(const CacheArgs c, const AttendArgs a, int ranks)
{
    typedef TileF32<D> Sh;
    constexpr int ROWS = kTileRows;
    extern __shared__ __align__(1024) unsigned char smem[];
    float *s_q = reinterpret_cast<float *>(smem), *s_kv = s_q + ROWS * Sh::kPitch;   // at the end the part
    __shared__ float2 s_ml[ROWS];
    __shared__ float s_weight[kMostRanks * ROWS], s_total[ROWS], s_gate[ROWS];
    __shared__ int s_held[2][4];
    __shared__ int s_found;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
    const int rank = blockIdx.x % ranks, kvh = blockIdx.y;
    const Tile tile = find_tile(c, a.group, ROWS, (long long)(gridDim.x / ranks) - 1 - blockIdx.x / ranks, &s_found);
    if (tile.rows == 0) return;   // the whole cluster's tile

    const int room = room_of(c);
    const int pos_first = position_of(tile.ch, a.group, tile.row0);
    const int pos_last = position_of(tile.ch, a.group, tile.row0 + tile.rows - 1);
    const int low = a.window > 0 ? max(0, pos_first - a.window + 1) : 0;
    const int high = min(pos_last + 1, room);
    const int sees_all_from = a.window > 0 ? max(0, pos_last - a.window + 1) : 0;   // .. to pos_first
    const int first_step = low / kTileKeys, steps = high > low ? (high + kTileKeys - 1) / kTileKeys - first_step : 0;
    const int mine = steps > rank ? (steps - rank + ranks - 1) / ranks : 0;   // this rank's steps
    auto step_at = [&](int it) { return (int)((uint32_t)(first_step + rank + it * ranks) * kTileKeys); };
    // a warp loads the step's run of eight keys that has its number
    auto look = [&](int it) {
        const int j = step_at(it) + 8 * warp;
        return it < mine && j < room ? page_of(c, tile.ch.stream, j) : -1;
    };
    int page;
    const int live = c.dim / 4;
    for (int i = threadIdx.x; i < ROWS * (D / 4); i += 128) {
        const int r = i / (D / 4), p = i % (D / 4), row = tile.row0 + r;
        const bool in = r < tile.rows && p < live;
        const long long at = in ? (long long)(tile.ch.first + row / a.group) * a.q_stride +
                                      (long long)(kvh * a.group + row % a.group) * c.dim + p * 4
                                : 0;
        cp_async16_or_zero(smem_u32(s_q + r * Sh::kPitch + p * 4), (const float *)a.q + at, in);
    }
    load_gates<float>(a, tile, kvh, s_gate);
    if (live < D / 4)   // pieces that no copy fills
        for (int i = threadIdx.x; i < 2 * kTileKeys * (D / 4); i += 128) {
            const int r = i / (D / 4), p = i % (D / 4);
            if (p >= live) {
                float *stage = s_kv + (r / kTileKeys) * Sh::kStage;
                const float4 zero = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                *reinterpret_cast<float4 *>(stage + (r % kTileKeys) * Sh::kPitch + p * 4) = zero;
                *reinterpret_cast<float4 *>(stage + kTileKeys * Sh::kPitch + (r % kTileKeys) * Sh::kPitchV + p * 4) = zero;
            }
        }
    auto fetch = [&](int it) {
        if (it < mine) {
            float *keys = s_kv + (it & 1) * Sh::kStage + 8 * warp * Sh::kPitch;
            float *values = s_kv + (it & 1) * Sh::kStage + kTileKeys * Sh::kPitch + 8 * warp * Sh::kPitchV;
            const int j0 = step_at(it) + 8 * warp;
            if (lane == 0) s_held[it & 1][warp] = page >= 0;
            const long long base = page >= 0 ? row_on_page(c, page, kvh, j0) : 0;
            constexpr int kLanes = D / 4 < 32 ? D / 4 : 32;   // of a row's pieces
#pragma unroll 4
            for (int r = lane / kLanes; r < 8; r += 32 / kLanes) {
                const bool take = page >= 0 && j0 + r >= low && j0 + r < high;
                const long long at = take ? base + r * c.dim : 0;
                for (int p = lane % kLanes; p < live; p += kLanes) {
                    cp_async16_or_zero(smem_u32(keys + r * Sh::kPitch + p * 4), (const float *)c.k + at + p * 4, take);
                    cp_async16_or_zero(smem_u32(values + r * Sh::kPitchV + p * 4), (const float *)c.v + at + p * 4, take);
                }
            }
        }
        cp_async_commit();
        page = look(it + 1);
    };

    int pos[2];
#pragma unroll
    for (int i = 0; i < 2; i++)
        pos[i] = position_of(tile.ch, a.group, tile.row0 + min(warp * 16 + i * 8 + g, tile.rows - 1));
    float m[2], l[2], o[D / 8][4];
    const float factor = a.scale * kLog2e;
    const float *q0 = s_q + (warp * 16 + g) * Sh::kPitch + 4 * t, *q1 = q0 + 8 * Sh::kPitch;
    const bool idle = warp * 16 >= tile.rows;   // none of this warp's rows is one
    uint32_t saw;   // bits as `seen`'s

    // An infinity has no two parts: where the first pass leaves a NaN, a second one takes all that is not
    // finite by itself, as a NaN or an infinity of the result may be one of the inputs'.
    for (int careful = 0; careful < 2; careful++) {
    saw = 0;
#pragma unroll
    for (int i = 0; i < 2; i++) {
        m[i] = -INFINITY;
        l[i] = 0.0f;
    }
#pragma unroll
    for (int n = 0; n < D / 8; n++) o[n][0] = o[n][1] = o[n][2] = o[n][3] = 0.0f;
    page = look(0);
    fetch(0);
#pragma unroll 1
    for (int it = 0; it < mine; it++) {
        cp_async_wait<0>();
        __syncthreads();   // the step has landed, and the one before it is done with
        fetch(it + 1);
        const float *keys = s_kv + (it & 1) * Sh::kStage;
        float *values = s_kv + (it & 1) * Sh::kStage + kTileKeys * Sh::kPitch;
        const int j0 = step_at(it);
        uint32_t held = 0;
#pragma unroll
        for (int e = 0; e < 4; e++) held |= s_held[it & 1][e] ? 1u << e : 0u;
        const bool partial = j0 < sees_all_from || j0 + kTileKeys - 1 > pos_first || j0 + kTileKeys > high || held != 15u || careful;
        auto sees = [&](int i, int j) {   // row slot i of this lane, token j
            return j <= pos[i] && j < high && (a.window <= 0 || j > pos[i] - a.window) && (held >> ((j - j0) >> 3) & 1u);
        };
        if (partial) {
            // values that are not finite: to the rows that see them by themselves, and zeros to the
            // product, which would bring them to the others as 0 times them
            bool any = false;
            for (int i = threadIdx.x; i < kTileKeys * (D / 4); i += 128) {
                const float4 v = *reinterpret_cast<const float4 *>(values + i / (D / 4) * Sh::kPitchV + i % (D / 4) * 4);
                any |= odd(v.x) || odd(v.y) || odd(v.z) || odd(v.w);
            }
            if (__syncthreads_or(any)) {
#pragma unroll 1
                for (int k = 0; k < kTileKeys; k++)
#pragma unroll
                    for (int n = 0; n < D / 8; n++)
#pragma unroll
                        for (int e = 0; e < 2; e++) {
                            const float v = values[k * Sh::kPitchV + 32 * (n >> 2) + 8 * t + 4 * e + (n & 3)];
                            if (!odd(v)) continue;
                            if (sees(0, j0 + k)) o[n][e] += v;
                            if (sees(1, j0 + k)) o[n][2 + e] += v;
                        }
                __syncthreads();
                for (int i = threadIdx.x; i < kTileKeys * D; i += 128) {
                    float &v = values[i / D * Sh::kPitchV + i % D];
                    if (odd(v)) v = 0.0f;
                }
                __syncthreads();
            }
        }
        if (idle) continue;
        float x[4][4];
#pragma unroll
        for (int n = 0; n < 4; n++) x[n][0] = x[n][1] = x[n][2] = x[n][3] = 0.0f;
#pragma unroll 1
        for (int part = 0; part < D / 64; part++) {
        float hi[4][4], lo[4][4];
#pragma unroll
        for (int n = 0; n < 4; n++)
#pragma unroll
            for (int e = 0; e < 4; e++) hi[n][e] = lo[n][e] = 0.0f;
#pragma unroll
        for (int kd = 4 * part; kd < 4 * part + 4; kd++) {
            const float4 qa = *reinterpret_cast<const float4 *>(q0 + 16 * kd), qb = *reinterpret_cast<const float4 *>(q1 + 16 * kd);
            uint32_t h0[4], l0[4], h1[4], l1[4];
            split_tf32(qa.x, h0[0], l0[0]);
            split_tf32(qb.x, h0[1], l0[1]);
            split_tf32(qa.y, h0[2], l0[2]);
            split_tf32(qb.y, h0[3], l0[3]);
            split_tf32(qa.z, h1[0], l1[0]);
            split_tf32(qb.z, h1[1], l1[1]);
            split_tf32(qa.w, h1[2], l1[2]);
            split_tf32(qb.w, h1[3], l1[3]);
#pragma unroll
            for (int n = 0; n < 4; n++) {
                const float4 k = *reinterpret_cast<const float4 *>(keys + (8 * n + g) * Sh::kPitch + 16 * kd + 4 * t);
                uint32_t kh[4], kl[4];
                split_tf32(k.x, kh[0], kl[0]);
                split_tf32(k.y, kh[1], kl[1]);
                split_tf32(k.z, kh[2], kl[2]);
                split_tf32(k.w, kh[3], kl[3]);
                mma_3tf32(hi[n], lo[n], h0, l0, kh[0], kh[1], kl[0], kl[1]);
                mma_3tf32(hi[n], lo[n], h1, l1, kh[2], kh[3], kl[2], kl[3]);
            }
        }
#pragma unroll
        for (int n = 0; n < 4; n++)
#pragma unroll
            for (int e = 0; e < 4; e++) x[n][e] += hi[n][e] + lo[n][e];
        }
        if (careful) {
#pragma unroll
            for (int n = 0; n < 4; n++)
#pragma unroll
                for (int e = 0; e < 4; e++)
                    if (isnan(x[n][e]))
                        x[n][e] = plain_score(s_q + (warp * 16 + 8 * (e >> 1) + g) * Sh::kPitch,
                                              keys + (8 * n + 2 * t + (e & 1)) * Sh::kPitch, c.dim);
            __syncwarp();
        }
        uint32_t seen = 0xffffu;   // bit 4 n + element
        if (partial) {
            seen = 0;
#pragma unroll
            for (int b = 0; b < 16; b++) {
                if (sees((b >> 1) & 1, j0 + 8 * (b >> 2) + 2 * t + (b & 1)))
                    seen |= 1u << b;
                else
                    x[b >> 2][b & 3] = -INFINITY;
            }
        }
        saw |= seen;
#pragma unroll
        for (int i = 0; i < 2; i++) {
            float most = -INFINITY;
#pragma unroll
            for (int n = 0; n < 4; n++) most = fmaxf(most, fmaxf(x[n][2 * i], x[n][2 * i + 1]));
            most = fmaxf(most, __shfl_xor_sync(kFull, most, 1));
            most = fmaxf(most, __shfl_xor_sync(kFull, most, 2)) * factor;
            if (most > m[i]) {
                // (before the first weight O is zero, or what is not finite and added by itself)
                const float keep = m[i] == -INFINITY ? 1.0f : exp2_fast(m[i] - most);
                m[i] = most;
                l[i] *= keep;
#pragma unroll
                for (int n = 0; n < D / 8; n++) {
                    o[n][2 * i] *= keep;
                    o[n][2 * i + 1] *= keep;
                }
            }
        }
        __syncwarp();
        uint32_t ph[4][4], pl[4][4];
#pragma unroll
        for (int n = 0; n < 4; n++) {
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const float base = m[e >> 1] == -INFINITY ? 0.0f : m[e >> 1];
                const float w = exp2_fast(fmaf(x[n][e], factor, -base));   // 0 where not seen
                l[e >> 1] += w;
                x[n][e] = w;
            }
            split_tf32(x[n][0], ph[n][0], pl[n][0]);
            split_tf32(x[n][2], ph[n][1], pl[n][1]);
            split_tf32(x[n][1], ph[n][2], pl[n][2]);
            split_tf32(x[n][3], ph[n][3], pl[n][3]);
        }
        const float *v0 = values + 2 * t * Sh::kPitchV + 4 * g;
#pragma unroll
        for (int b = 0; b < D / 32; b++) {
            float hi[4][4], lo[4][4];
#pragma unroll
            for (int j = 0; j < 4; j++)
#pragma unroll
                for (int e = 0; e < 4; e++) hi[j][e] = lo[j][e] = 0.0f;
#pragma unroll
            for (int n = 0; n < 4; n++) {
                const float4 va = *reinterpret_cast<const float4 *>(v0 + 8 * n * Sh::kPitchV + 32 * b);
                const float4 vb = *reinterpret_cast<const float4 *>(v0 + (8 * n + 1) * Sh::kPitchV + 32 * b);
                const float ea[4] = {va.x, va.y, va.z, va.w}, eb[4] = {vb.x, vb.y, vb.z, vb.w};
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    uint32_t ah, al, bh, bl;
                    split_tf32(ea[j], ah, al);
                    split_tf32(eb[j], bh, bl);
                    mma_3tf32(hi[j], lo[j], ph[n], pl[n], ah, bh, al, bl);
                }
            }
#pragma unroll
            for (int j = 0; j < 4; j++)
#pragma unroll
                for (int e = 0; e < 4; e++) o[4 * b + j][e] += hi[j][e] + lo[j][e];
        }
    }
    cp_async_wait<0>();
    bool odd_result = false;
#pragma unroll
    for (int i = 0; i < 2; i++) {
        float sum = l[i];   // a NaN, if one of these is, or infinities of both signs are
#pragma unroll
        for (int n = 0; n < D / 8; n++) sum += o[n][2 * i] + o[n][2 * i + 1];
        odd_result |= isnan(sum) && warp * 16 + i * 8 + g < tile.rows;
    }
    if (!__syncthreads_or(odd_result)) break;   // (and every warp is done with the stages: the part takes their place)
    }
    float *part = s_q;
#pragma unroll
    for (int i = 0; i < 2; i++) {
        l[i] += __shfl_xor_sync(kFull, l[i], 1);
        l[i] += __shfl_xor_sync(kFull, l[i], 2);
        const int r = warp * 16 + i * 8 + g;
        const bool any = __ballot_sync(kFull, (saw & (i ? 0xccccu : 0x3333u)) != 0) >> (lane & ~3) & 15u;
        if (t == 0) s_ml[r] = make_float2(m[i] == -INFINITY && any ? kLowest : m[i], l[i]);
#pragma unroll
        for (int b = 0; b < D / 32; b++)
#pragma unroll
            for (int e = 0; e < 2; e++)
                *reinterpret_cast<float4 *>(part + r * D + part_piece(r, 8 * b + 2 * t + e) * 4) =
                    make_float4(o[4 * b][2 * i + e], o[4 * b + 1][2 * i + e], o[4 * b + 2][2 * i + e], o[4 * b + 3][2 * i + e]);
    }
    join_and_store<float, D, ROWS, 1, 128>(c, a, tile, kvh, part, s_ml, s_weight, s_total, s_gate, ranks, rank);
}

// The blocks of a tile's cluster: doubled while all blocks fit the SMs at once (`slots`: a block an SM, and then
// clusters of eight and more only until half of them are taken, as more do not fit; or several blocks), and for
// streams of unlike lengths to four while there are fewer than `few`.  16 + 4 bf16 heads of 128, one token, us:
//   16 streams of 1500 tokens   by 16, 8, 4 blocks     38.2  22.2  15.7
//   64 streams of 1500          by 4, 2, 1             47.9  49.8  37.7
//   64 streams of 64 to 6144    by 4, 2, 1             81.7  86.1  110
// heads of 256, 2 streams of 1500, by 16 and 8: 18.7 and 10.7; 16 streams, by 16 and 2: 97 and 23.7.
template <typename Kernel>
cudaError_t launch_rows(Kernel kernel, size_t smem, int tile_rows, int warps, int threads, const CacheArgs &c,
                        const AttendArgs &a, int keys, int few, int slots, std::mutex &mu, bool (&ready)[64], cudaStream_t stream)
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
    const long long work = likely_tiles(c, a, tile_rows) * c.n_kv;
    const long long room = ((long long)c.max_pages << c.page_shift) / (keys * warps);
    int ranks = 1;
    while (ranks < kMostRanks && ranks < room && (work * ranks * 2 <= (slots == 148 && ranks >= 4 ? 74 : slots) || (ranks < 4 && work * ranks < few))) ranks *= 2;
    if (tiles * ranks > 0x7fffffffll) return cudaErrorInvalidConfiguration;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(tiles * ranks), (unsigned)c.n_kv);
    cfg.blockDim = dim3((unsigned)threads);
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

template <int D, int STAGES, int W>
cudaError_t launch_bf16(const CacheArgs &c, const AttendArgs &a, cudaStream_t stream)
{
    static std::mutex mu;
    static bool ready[64] = {false};
    typedef Ring<__nv_bfloat16, D, 16> R;
    const size_t rings = W * STAGES * R::kStage, parts = (size_t)W * 16 * D * 4;
    const size_t smem = (rings > parts ? rings : parts) + 16 * R::kRow;
    return launch_rows(attend_rows_bf16_kernel<D, STAGES, W>, smem, 16, W, 32 * W, c, a, 16, D > 128 ? 0 : 592, D > 128 ? 148 : 444, mu, ready, stream);
}

// Blocks of eight rings where a cluster of the most blocks for each tile does not fill the SMs (one
// stream of 6050 tokens: 12.9 us with half as many blocks, 10.4 us; past half the SMs clusters of sixteen such
// blocks do not all fit at once: 2 streams of up to 6144 tokens 16.9 us, 10.8 by blocks of four).
template <int D, int STAGES>
cudaError_t launch_bf16(const CacheArgs &c, const AttendArgs &a, cudaStream_t stream)
{
    if (tiles_with_rows(c, a, 16) * c.n_kv * kMostRanks <= 74) return launch_bf16<D, 3, 8>(c, a, stream);
    return launch_bf16<D, STAGES, 4>(c, a, stream);
}

template <int D, int ROWS, int STAGES, int W = 4>
cudaError_t launch_f32(const CacheArgs &c, const AttendArgs &a, cudaStream_t stream)
{
    static std::mutex mu;
    static bool ready[64] = {false};
    typedef Ring<float, D, 8> R;
    const size_t rings = W * STAGES * R::kStage, parts = (size_t)W * ROWS * D * 4;
    const size_t smem = (rings > parts ? rings : parts) + ROWS * R::kRow;
    return launch_rows(attend_rows_f32_kernel<D, ROWS, STAGES, W>, smem, ROWS, W, 32 * W, c, a, 8, D > 128 ? 148 : 592, D > 128 ? 148 : D > 64 ? 296 : 444, mu, ready, stream);
}

template <int D>
cudaError_t launch_tile_f32(const CacheArgs &c, const AttendArgs &a, cudaStream_t stream)
{
    static std::mutex mu;
    static bool ready[64] = {false};
    // (a window makes the tiles of streams longer than it alike: 6 streams of up to 333 tokens on 100 to 2000, a window of 512: 136 us by two
    // blocks, 124 by one; whether they are that long is on the device, so the table's width stands for it)
    const bool even = a.window > 0 && a.window < ((long long)c.max_pages << c.page_shift) / 4;
    return launch_rows(attend_tile_f32_kernel<D>, TileF32<D>::kSmem, kTileRows, 1, 128, c, a, kTileKeys, even ? 0 : D > 128 ? 148 : 592, D > 128 ? 148 : even ? 296 : 444, mu, ready, stream);
}

}  // namespace

cudaError_t launch_cache_attend(const CacheArgs &c, const AttendArgs &a, bool bf16, cudaStream_t stream)
{
    // rows of a stream that share a key head
    const int most_new = a.max_new > 0 && a.max_new < c.rows ? a.max_new : c.rows;
    const long long rows = (long long)most_new * a.group;
    if (bf16) {
        // (20 or 32 rows on 64 streams: 90 and 94 us here, 92 there; 48 rows: 111 against 92; on 4
        // streams 21 and 22 us against 25, 48 rows 32 against 25.  Heads of 256, 32 and 64 rows on 16 streams:
        // 34 and 65 us here, 41 and 44 there; on 4 streams 18 and 23 against 25 and 26)
        if (rows > 32) return launch_cache_attend_tc(c, a, stream);
        if (c.dim > 128) return launch_bf16<256, 2, 6>(c, a, stream);
        return c.dim > 64 ? launch_bf16<128, 2>(c, a, stream) : launch_bf16<64, 4>(c, a, stream);
    }
    if (rows > 16)
        return c.dim > 128 ? launch_tile_f32<256>(c, a, stream)
                           : c.dim > 64 ? launch_tile_f32<128>(c, a, stream) : launch_tile_f32<64>(c, a, stream);
    if (c.dim > 128) return rows > 4 ? launch_f32<256, 8, 2, 6>(c, a, stream) : launch_f32<256, 4, 2, 6>(c, a, stream);
    if (c.dim > 64) return rows > 4 ? launch_f32<128, 16, 3>(c, a, stream) : launch_f32<128, 4, 3>(c, a, stream);
    return rows > 4 ? launch_f32<64, 16, 4>(c, a, stream) : launch_f32<64, 4, 4>(c, a, stream);
}

}  // namespace z2
