// cache_attend_tc.cu -- attention of chunks of new tokens over a paged cache on the tcgen05
// tensor cores (sm_100a): bf16, heads of up to 256 elements (as 64, 128 or 256, zeros past their end).
//
// A block takes 256 rows -- (token, query head) pairs that share a key head -- as two tiles of
// 128, and the tokens they see in steps of 128 keys:
//   warp 0        TMA producer: a step's keys and values (keys alone past heads of 128, where warp 2
//                 has the values), page by page (a box is a page or 128 of
//                 its tokens), 128-byte swizzled, into a ring of 128 x D tiles;
//   warp 1        allocates TMEM and issues tcgen05.mma: S = Q K^T (128 x 128, f32) and
//                 O += P V (P in TMEM as bf16 in place of S, V read as it lies, rows of D);
//   warps 4..7, 8..11  softmax of one tile each, a row to a thread: S from TMEM, its
//                 maximum, 2^(x - m), P back to TMEM, and at the end O / l to global memory.
// (P is rounded to bf16, the values' type, as cache_attend.cu says; its sum l is taken before.)
// While one tile's softmax runs, the tensor core works for the other.  A step of both tiles
// is 4 x 512 cycles of MMAs and 2 x 128 x 128 exponentials, 2048 cycles of the SM's 16 a
// cycle: neither may wait for the other.  4 chunks of 2048 tokens on 2048 to 4096 cached ones, 16 + 4
// heads of 128 (275 GFLOP): 297 to 340 us as the power limit has it, up to 0.93 PFLOP/s, the tensor pipe 48 % active; a step takes 3800
// cycles, 2300 of them a tile's softmax (1550 the exponentials) and the rest its products and
// hand-overs.  A quarter of the exponentials by a polynomial on the FMA pipe was slower (324 us),
// the tiles taking turns at them too (419 us against 394 then), and two threads to a row (475 us).
// The running maximum is raised only when a row's scores
// pass it by more than 2^8 (P is then at most 256 instead of 1, and the sum of the same scale:
// no rounding changes), so that O is seldom rescaled.  Stages hand over through mbarriers, every
// wait is bounded.
// SPLIT: where there are few rows to a key head, a block has one tile of up to 128 and its two groups
// of softmax warps take the steps in turn, each with an accumulator of its own; a cluster of
// blocks shares a tile's steps out where there are few tiles.  The parts are joined as in
// cache_attend.cu.  (Warps without rows only keep the hand-over going.)
// Heads past 128 are always SPLIT, with one group of softmax warps and one accumulator: TMEM holds that, 256
// columns, and the scores of two steps, so that the next step's scores are there when a step's softmax ends;
// shared memory holds one tile of keys and one of values beside the queries, each asked for by a warp of its own
// as soon as the one before it is done with.  The chunks above with heads of 256 (550 GFLOP): 550 us, 1.0 PFLOP/s;
// 823 us with one warp for both, whose keys wait for the values before them; 3694 us by 16 rows to a tile on mma.sync.
// Values in two halves of 64 tokens, each freed by itself, took 538 us here and 3 us more of 43 on shorter chunks.
// A value that is not finite in a step that some row does not wholly see would reach that row as
// 0 times it: such values are set to zero in shared memory before the product and added, at the
// end, to the rows that see them.
#include <math.h>

#include <mutex>

#include "cache_attend.cuh"

namespace z2 {

int read_and_clear_attend_error(int *value) { return take_device_error(value); }

namespace {

constexpr int kStep = 128;       // keys of a step
constexpr int kTcRanks = 8;      // blocks of a cluster, at most
constexpr float kSlack = 8.0f;   // how far scores may pass the running maximum, in powers of two

template <int D>
struct TcShape {
    static constexpr uint32_t kHalves = D / 64;              // 128-byte columns of a tile
    static constexpr uint32_t kTile = 128 * D * 2;           // bytes of 128 rows
    static constexpr bool kOne = D > 128;                    // one group of softmax warps
    static constexpr int kGroups = kOne ? 1 : 2, kThreads = 128 + 128 * kGroups;
    static constexpr int kSlots = kOne ? 2 : 5;              // tiles of keys or values in shared memory
    static constexpr uint32_t kQ = kOne ? kTile : 2 * kTile;
    // the parts at the end: outputs in the place of keys and values, and what lies behind them (of kOne the
    // ranks' maxima and sums first, which otherwise take the second part's place), in floats
    static constexpr uint32_t kParts = kGroups * 128 * D + (kOne ? kTcRanks * 128 * 2 : 0);
    static constexpr uint32_t kJoin = (kParts + kGroups * 128 * 2 + kMostRanks * 128 + 128) * 4;
    static constexpr uint32_t kRing = kOne ? kJoin : kSlots * kTile;
    static_assert(kJoin <= kRing && kSlots * kTile <= kRing && kRing % 8 == 0, "both fit");
    static constexpr size_t kSmem = kQ + kRing + 1024 + 256;
    // A block takes all of TMEM and, in a cluster, keeps it until the others have come as far: no two blocks of these kernels may share
    // an SM (1 KB of static shared memory, 1 KB that each block takes beside it), or two clusters could wait for each other.
    static_assert(2 * (kSmem + 2048) > 228 * 1024, "one block to an SM");
};

// Shared-memory matrix descriptor, MN-major (rows of K, the product's columns behind each
// other), 128-byte swizzle: 64 columns of 8 rows are 1024 bytes; 8 rows further on 1024 (SBO),
// 64 columns further on one 128-row half (LBO).
__device__ __forceinline__ uint64_t sw128_desc_mn(uint32_t addr)
{
    return (uint64_t)((addr & 0x3FFFFu) >> 4) | ((uint64_t)((128 * 128) >> 4) << 16) |
           ((uint64_t)(1024 >> 4) << 32) | ((uint64_t)1 << 46) | ((uint64_t)2 << 61);
}

// D += A B with A in TMEM.
__device__ __forceinline__ void mma_bf16_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t bdesc, uint32_t idesc,
                                            uint32_t accumulate)
{
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d_tmem),
        "r"(a_tmem), "l"(bdesc), "r"(idesc), "r"(accumulate)
        : "memory");
}

__device__ __forceinline__ float max3(float a, float b, float c)
{
    float r;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}
// Two f32 values at a time on the FMA pipe.
__device__ __forceinline__ uint64_t two(float a, float b)
{
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ void both(uint64_t v, float &a, float &b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v)); }
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c)
{
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b)
{
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ void tmem_ld32_start(uint32_t taddr, uint32_t *r)
{
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
          "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]),
          "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]),
          "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]),
          "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(taddr));
}
// After tcgen05.wait::ld: nothing reads these registers ahead of it.
__device__ __forceinline__ void tmem_landed(uint32_t *r)
{
    asm volatile(""
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]),
                   "+r"(r[7]), "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]),
                   "+r"(r[13]), "+r"(r[14]), "+r"(r[15]), "+r"(r[16]), "+r"(r[17]), "+r"(r[18]),
                   "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]), "+r"(r[23]), "+r"(r[24]),
                   "+r"(r[25]), "+r"(r[26]), "+r"(r[27]));
    asm volatile("" : "+r"(r[28]), "+r"(r[29]), "+r"(r[30]), "+r"(r[31]));
}
__device__ __forceinline__ void tmem_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_st32(uint32_t taddr, const uint32_t *r)
{
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
        "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, "
        "%17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};" ::"r"(taddr),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
        "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]),
        "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]),
        "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
        : "memory");
}

__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t *r)
{
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
        "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(taddr),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
        "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
        : "memory");
}

__device__ __forceinline__ void tma_load_4d(uint32_t dst, const CUtensorMap *map, int x, int y, int z, int w, uint32_t bar)
{
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes "
        "[%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(dst),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(w), "r"(bar)
        : "memory");
}

// What the rows of one 128-row tile see.
struct Span {
    int low, high;        // tokens that some row sees lie in [low, high)
    int all_from, all_to; // .. and every row sees [all_from, all_to)
};

__device__ __forceinline__ Span span_of(const CacheArgs &c, const AttendArgs &a, const Chunk &ch, int row0, int rows)
{
    Span s;
    const int first = position_of(ch, a.group, row0), last = position_of(ch, a.group, row0 + rows - 1);
    s.low = a.window > 0 ? max(0, first - a.window + 1) : 0;
    s.high = min(last + 1, room_of(c));
    s.all_from = a.window > 0 ? max(0, last - a.window + 1) : 0;
    s.all_to = min(first + 1, s.high);
    return s;
}

// Adds to a row's outputs [col, col + N) the values of step j0's tokens that are not finite, of those
// that the row sees ([from, to)); steps that every row sees wholly went through the product as they are.
template <int N>
__device__ void add_odd(const CacheArgs &c, int stream, int kvh, int j0, int all_from, int all_to, int from, int to, int col,
                        uint32_t *o)
{
    const int room = room_of(c);
    bool whole = j0 >= all_from && j0 + kStep <= all_to;
    for (int e = 0; whole && e < kStep / 8; e++) whole = j0 + 8 * e < room && page_of(c, stream, j0 + 8 * e) >= 0;
    if (whole) return;
    for (int j = max(from, j0); j < min(to, j0 + kStep); j++) {
        const int p = page_of(c, stream, j);
        if (p < 0) continue;
        const __nv_bfloat16 *v = (const __nv_bfloat16 *)c.v + row_on_page(c, p, kvh, j) + col;
#pragma unroll
        for (int k = 0; k < N; k++) {
            if (col + k >= c.dim) break;
            const float y = as_f(v[k]);
            if (odd(y)) o[k] = __float_as_uint(__uint_as_float(o[k]) + y);
        }
    }
}

template <int D, bool SPLIT>
__global__ void __launch_bounds__(TcShape<D>::kThreads, 1)
    attend_tc_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
                     const CacheArgs c, const AttendArgs a, int box_rows, int turns, int ranks)
{
    typedef TcShape<D> Sh;
    constexpr bool kOne = Sh::kOne;
    constexpr int kGroups = Sh::kGroups, kSlots = Sh::kSlots, kTcThreads = Sh::kThreads;
    static_assert(SPLIT || !kOne, "no room for two tiles");
    // kind::f16: D f32, A and B bf16; M = 128; S: N = 128, both K-major; O: N = D, B MN-major
    constexpr uint32_t kIdescS = (1u << 4) | (1u << 7) | (1u << 10) | (128u >> 3 << 17) | (128u >> 4 << 24);
    constexpr uint32_t kIdescO = (1u << 4) | (1u << 7) | (1u << 10) | (1u << 16) | ((uint32_t)D >> 3 << 17) | (128u >> 4 << 24);
    constexpr uint32_t kColS = 0, kColO = 256;   // TMEM columns: S (then P) of both tiles, O of both (kOne: of the one)

    extern __shared__ __align__(1024) unsigned char smem_raw[];
    const uint32_t smem = (smem_u32(smem_raw) + 1023) & ~1023u;
    const uint32_t s_q = smem, s_kv = smem + Sh::kQ, s_bar = s_kv + Sh::kRing;
    auto full = [&](int s) { return s_bar + 8 * s; };
    auto empty = [&](int s) { return s_bar + 8 * (kSlots + s); };
    auto s_full = [&](int q) { return s_bar + 8 * (2 * kSlots + q); };    // S, and O before it, are done
    auto p_ready = [&](int q, int h) { return s_bar + 8 * (2 * kSlots + 2 + 2 * q + h); };   // P of 64 keys
    // (kOne) a step's product, even and odd steps' apart; and odd steps' values, which share a slot with the even ones'
    auto o_done = [&](int n) { return s_bar + 8 * (2 * kSlots + 6 + (n & 1)); };
    const uint32_t odd_values_full = s_bar + 8 * (2 * kSlots + 8);
    constexpr int kTileRows = SPLIT ? 128 : 256;
    __shared__ uint32_t s_tmem;
    __shared__ int s_abort, s_odd;
    __shared__ float s_gate[SPLIT ? 128 : 1];
    // (SPLIT) the parts at the end, in the place of keys and values
    float *part = reinterpret_cast<float *>(smem_raw + (s_kv - smem_u32(smem_raw)));
    float2 *ml = reinterpret_cast<float2 *>(part + Sh::kParts);
    float *weight = reinterpret_cast<float *>(ml + kGroups * 128), *total = weight + kMostRanks * 128;

    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    // A stream's last tiles see the most tokens: every stream's come first.  (Where a stream has
    // more tiles than it was launched for, a block takes every `turns`-th.)
    const int rank = SPLIT ? blockIdx.x % ranks : 0, item = SPLIT ? blockIdx.x / ranks : blockIdx.x;
    const int kvh = item % c.n_kv, first_turn = item / c.n_kv / c.n_streams;
    const Chunk ch = chunk_of(c, item / c.n_kv % c.n_streams);
    const long long all_rows = (long long)ch.n * a.group;
    const int n_tiles = (int)((all_rows + kTileRows - 1) / kTileRows);
    if (first_turn >= n_tiles) return;
    if (threadIdx.x == 0) {
        s_abort = s_odd = 0;
        for (int s = 0; s < kSlots; s++) {
            mbar_init(full(s), 1);
            mbar_init(empty(s), 1);
        }
        for (int q = 0; q < 2; q++) {
            mbar_init(s_full(q), 1);
            mbar_init(p_ready(q, 0), 4);   // the tile's warps
            mbar_init(p_ready(q, 1), 4);
        }
        mbar_init(o_done(0), 1);
        mbar_init(o_done(1), 1);
        mbar_init(odd_values_full, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        prefetch_map(&map_k);
        prefetch_map(&map_v);
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&s_tmem)),
                     "r"(512)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    uint32_t tmem = 0;
    // phases of the barriers before this tile: tiles of keys and values, scores of either tile
    int kv0 = 0, scored0 = 0, scored1 = 0, weighed0 = 0, weighed1 = 0;
    // The barrier that step i's keys (kv = 0) or values (kv = 1) land on, and the phase's parity.
    // A wait tells a phase by its parity alone, so that whoever waits must know the phase before it to be
    // done.  Softmax warps do not wait for every step's values or products: all they know at step i is that
    // its scores are there, S(i), and what the issuer's thread had started before them.  Up to heads of 128 the slot's tile before
    // values V(i) is K(i-2), which S(i-2) has used.  Past 128 S(i) comes after PV(i-2), so that V(i-2) has landed
    // and PV(i-2) is done, but neither holds for step i - 1: a barrier for even and one for odd steps each.
    auto landing = [&](int i, int kv) {
        return kOne && kv && (i & 1) ? odd_values_full : full((kv0 + 2 * i + kv) % kSlots);
    };
    auto in_turn = [&](int i) { return (uint32_t)((i & 1 ? weighed1 : weighed0) + (i >> 1)) & 1u; };   // (kOne)
    auto landing_parity = [&](int i, int kv) { return kOne && kv ? in_turn(i) : (uint32_t)((kv0 + 2 * i + kv) / kSlots) & 1u; };
    bool dead = false;   // a wait ran out
    for (int turn = first_turn; turn < n_tiles; turn += turns) {
    const long long row_ll = (long long)(n_tiles - 1 - turn) * kTileRows;
    const int row0 = (int)row_ll;
    const int tile_rows = (int)(all_rows - row_ll < kTileRows ? all_rows - row_ll : kTileRows);
    const int rows0 = min(tile_rows, 128), rows1 = tile_rows - rows0;
    const Span span0 = span_of(c, a, ch, row0, rows0);
    const Span span1 = rows1 > 0 ? span_of(c, a, ch, row0 + 128, rows1) : span0;
    const int low = min(span0.low, span1.low), high = max(span0.high, span1.high);
    // tokens that every row of both tiles sees: the tiles share the values, and what is done to them
    const int all_from = max(span0.all_from, span1.all_from), all_to = min(span0.all_to, span1.all_to);
    const int step0 = low / kStep + rank, all_steps = high > low ? (high + kStep - 1) / kStep - low / kStep : 0;
    const int steps = all_steps > rank ? (all_steps - rank + ranks - 1) / ranks : 0;   // this rank's: step0 + i ranks
    if (SPLIT) {
        Tile tile;
        tile.ch = ch;
        tile.row0 = row0;
        tile.rows = tile_rows;
        load_gates<__nv_bfloat16>(a, tile, kvh, s_gate);
    }

    // queries, swizzled as TMA does; zeros past the rows
#pragma unroll 4
    for (int i = threadIdx.x; i < kTileRows * (D / 8); i += kTcThreads) {
        const int r = i / (D / 8), p = i % (D / 8), row = row0 + r;
        const bool in = r < tile_rows && p * 8 < c.dim;
        const long long at = in ? (long long)(ch.first + row / a.group) * a.q_stride +
                                      (long long)(kvh * a.group + row % a.group) * c.dim + p * 8
                                : 0;
        cp_async16_or_zero(s_q + (r >> 7) * Sh::kTile + (p >> 3) * (128 * 128) + (r & 127) * 128 + (((p & 7) ^ (r & 7)) << 4),
                           (const __nv_bfloat16 *)a.q + at, in);
    }
    cp_async_commit();
    cp_async_wait<0>();
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    tmem = s_tmem;

    // a row's running maximum and sum, and whether it saw a token
    float m = -INFINITY, l = 0.0f;
    bool saw = false;
    if (steps > 0 && !dead) {
        if (warp == 0 || (kOne && warp == 2)) {
            // ---- TMA producer: tile 2 i is step i's keys, 2 i + 1 its values (kOne: warp 2's, so that keys need
            // not wait for the values before them)
            const int boxes = kStep / box_rows;          // of a step, for each half
            const int room = room_of(c);
            bool ok = true;
            const int kv_first = kOne ? warp >> 1 : 0, kv_end = kOne ? kv_first + 1 : 2;   // this producer's
            int i = 0, kv = kv_first;
            for (; i < steps && ok; i++) {
                const int j0 = (step0 + i * ranks) * kStep;
                // lane's box of the step's boxes (16 at most), and of the halves every 32 / boxes-th
                const int b = lane % boxes, h0 = lane / boxes, j = j0 + b * box_rows;
                int page = -1;
                if (j < room) page = page_of(c, ch.stream, j);
                if (page < 0) page = c.n_pages;          // out of the map: zeros
                const int slot_in_page = j & ((1 << c.page_shift) - 1);
                for (kv = kv_first; kv < kv_end; kv++) {
                    const int it = kv0 + 2 * i + kv, s = it % kSlots;
                    const uint32_t bar = landing(i, kv);
                    ok = mbar_wait(empty(s), (((uint32_t)(it / kSlots)) & 1u) ^ 1u) && !*(volatile int *)&s_abort;
                    ok = __all_sync(kFull, ok);
                    if (!ok) break;
                    if (lane == 0) mbar_expect_tx(bar, Sh::kTile);
                    __syncwarp();
                    for (int h = h0; h < (int)Sh::kHalves; h += 32 / boxes)
                        tma_load_4d(s_kv + s * Sh::kTile + h * (128 * 128) + b * box_rows * 128, kv ? &map_v : &map_k,
                                    h * 64, slot_in_page, kvh, page, bar);
                }
                if (!ok) break;
            }
            if (!ok) {
                s_abort = 1;
                // copies still in flight land first (the last kSlots tiles', none of which is step i's kv-th)
                for (int t = 2 * i + kv - 1; t >= 0 && t >= 2 * i + kv - kSlots; t--)
                    if (!kOne || (t & 1) == kv) mbar_wait(landing(t >> 1, t & 1), landing_parity(t >> 1, t & 1));
            }
        } else if (warp == 1) {
            // ---- MMA issuer
            if (lane == 0) {
                bool ok = true;
                auto wait = [&](uint32_t bar, uint32_t parity) {
                    ok = ok && mbar_wait(bar, parity);
                    tc_fence_after();
                    return ok;
                };
                auto slot = [&](int t) { return s_kv + (uint32_t)((kv0 + t) % kSlots) * Sh::kTile; };
                auto landed = [&](int t) { return wait(landing(t >> 1, t & 1), landing_parity(t >> 1, t & 1)); };
                auto done = [&](int t) { mma_commit(empty((kv0 + t) % kSlots)); };
                auto scores = [&](int q, int t) {   // S of tile q by the keys in tile t
#pragma unroll
                    for (int kk = 0; kk < D / 16; kk++) {
                        const uint32_t off = (kk >> 2) * (128 * 128);
                        mma_bf16(tmem + kColS + q * 128, sw128_desc(s_q + (SPLIT ? 0 : q * Sh::kTile) + off) + 2 * (kk & 3),
                                 sw128_desc(slot(t) + off) + 2 * (kk & 3), kIdescS, kk != 0);
                    }
                    mma_commit(s_full(q));
                };
                if (SPLIT) {
                    for (int i = 0; i < 2 && i < steps; i++) {
                        if (!landed(2 * i)) break;
                        scores(i, 2 * i);
                        done(2 * i);
                    }
                    // (kOne: there is one accumulator, and S(i + 2) is issued behind PV(i); its keys have been asked for
                    // since S(i + 1) was done with the slot.)
                    for (int i = 0; i < steps && ok && !*(volatile int *)&s_abort; i++) {
                        const int q = i & 1;
                        if (!landed(2 * i + 1) || (!kOne && i + 2 < steps && !landed(2 * i + 4))) break;
#pragma unroll
                        for (int k = 0; k < kStep / 16; k++) {
                            const int kk = k ^ 4;
                            if (k % 4 == 0 && !wait(p_ready(q, kk / 4), (uint32_t)((q ? weighed1 : weighed0) + (i >> 1)) & 1u)) break;
                            mma_bf16_ts(tmem + kColO + (kOne ? 0 : q * 128), tmem + kColS + q * 128 + 32 * (kk >> 1) + 8 * (kk & 1),
                                        sw128_desc_mn(slot(2 * i + 1) + kk * 16 * 128), kIdescO, i >= kGroups || k > 0);
                        }
                        if (!ok) break;
                        done(2 * i + 1);
                        if (kOne) {
                            mma_commit(o_done(i));
                            if (i + 2 < steps) {
                                if (!landed(2 * i + 4)) break;
                                scores(q, 2 * i + 4);
                                done(2 * i + 4);
                            }
                        } else if (i + 2 < steps) {
                            scores(q, 2 * i + 4);
                            done(2 * i + 4);
                        } else {
                            mma_commit(s_full(q));   // O is whole
                        }
                    }
                }
                const int tiles = rows1 > 0 ? 2 : 1;
                if (!SPLIT && landed(0)) {
                    for (int q = 0; q < tiles; q++) scores(q, 0);
                    done(0);
                }
                for (int i = 0; !SPLIT && i < steps && ok && !*(volatile int *)&s_abort; i++) {
                    const bool more = i + 1 < steps;
                    if (!landed(2 * i + 1) || (more && !landed(2 * i + 2))) break;
                    for (int q = 0; q < tiles; q++) {
#pragma unroll
                        for (int k = 0; k < kStep / 16; k++) {
                            const int kk = k ^ 4;   // the upper 64 keys' weights come first
                            if (k % 4 == 0 && !wait(p_ready(q, kk / 4), (uint32_t)((q ? weighed1 : weighed0) + i) & 1u)) break;
                            // 32 keys' weights lie in the first 16 of their scores' columns
                            mma_bf16_ts(tmem + kColO + q * 128, tmem + kColS + q * 128 + 32 * (kk >> 1) + 8 * (kk & 1),
                                        sw128_desc_mn(slot(2 * i + 1) + kk * 16 * 128), kIdescO, (i | k) != 0);
                        }
                        if (!ok) break;
                        if (q == tiles - 1) done(2 * i + 1);
                        if (more) {
                            scores(q, 2 * i + 2);
                            if (q == tiles - 1) done(2 * i + 2);
                        } else {
                            mma_commit(s_full(q));   // O is whole
                        }
                    }
                }
                if (!ok) s_abort = 1;
            }
        } else if (warp >= 4) {
            // ---- softmax of tile q, this thread's row r of it
            const int q = (warp - 4) >> 2, r = threadIdx.x & 127;
            const int rows = SPLIT ? tile_rows : q ? rows1 : rows0;
            const int row_q = row0 + (SPLIT ? 0 : q * 128);   // the tile's first row
            // the group's n-th step is the rank's q + 2 n, or n
            const int count = SPLIT ? (steps - q + kGroups - 1) / kGroups : steps;
            // S, P and their barriers' phase of it: the group's, or (kOne) the two in turn
            auto buffer = [&](int n) { return kOne ? n & 1 : q; };
            auto turn_of = [&](int before0, int before1, int n) {
                return (uint32_t)(kOne ? (n & 1 ? before1 : before0) + (n >> 1) : (q ? before1 : before0) + n) & 1u;
            };
            const int scanners = SPLIT ? (rows + 31) & ~31 : 128;   // threads of warps with rows
            auto step_of = [&](int n) { return SPLIT ? q + kGroups * n : n; };
            if (SPLIT && 32 * (warp & 3) >= rows) {   // no row of this warp's
                for (int n = 0; n < count; n++) {
                    const bool ok = mbar_wait(s_full(buffer(n)), turn_of(scored0, scored1, n)) && !*(volatile int *)&s_abort;
                    if (!__all_sync(kFull, ok)) break;
                    if (lane == 0) {
                        mbar_arrive(p_ready(buffer(n), 0));
                        mbar_arrive(p_ready(buffer(n), 1));
                    }
                }
            } else if (rows > 0 && count > 0) {
                const uint32_t at = ((uint32_t)(warp & 3) * 32) << 16;   // this warp's TMEM lanes
                const uint32_t t_o = tmem + at + kColO + q * 128;
                const int pos = position_of(ch, a.group, row_q + min(r, rows - 1));
                const int from = a.window > 0 ? max(0, pos - a.window + 1) : 0;
                const int to = min(pos + 1, (q ? span1 : span0).high);   // this row sees [from, to)
                const float factor = a.scale * kLog2e;
                const int room = room_of(c);
                // the pages of a step's runs of eight tokens, one step ahead; bit 8 e: run e is held
                auto look = [&](int i) {
                    const int j = (int)((uint32_t)(step0 + i * ranks) * kStep) + 8 * lane;
                    return lane < 16 && (i >= steps || (j < room && page_of(c, ch.stream, j) >= 0));
                };
                bool ok = true;
                bool held_next = look(step_of(0));
                for (int n = 0; n < count; n++) {
                    const int i = step_of(n);
                    const uint32_t held = __ballot_sync(kFull, held_next) & 0xffffu;
                    held_next = look(step_of(n + 1));
                    const int j0 = (step0 + i * ranks) * kStep;
                    const bool partial = j0 < all_from || j0 + kStep > all_to || held != 0xffffu;
                    const uint32_t t_s = tmem + at + kColS + buffer(n) * 128;
                    ok = mbar_wait(s_full(buffer(n)), turn_of(scored0, scored1, n)) && !*(volatile int *)&s_abort;
                    ok = __all_sync(kFull, ok);
                    if (!ok) break;
                    tc_fence_after();
                    // S passes through registers 32 columns at a time, once for the maximum and, but for the
                    // last two pieces, which are still there, again for the weights: 128 columns at once
                    // would leave the rest of the loop's values no registers.
                    uint32_t x[2][32];
                    auto start = [&](int piece) { tmem_ld32_start(t_s + 32 * piece, x[piece & 1]); };
                    auto landed = [&](int piece) {
                        tmem_wait_ld();
                        tmem_landed(x[piece & 1]);
                    };
                    auto mask = [&](int piece) {
                        const int begin = max(0, min(32, from - j0 - 32 * piece)), end = max(0, min(32, to - j0 - 32 * piece));
                        // the runs' bits to bytes: bit e comes to 8 e
                        uint32_t in = (((held >> (4 * piece) & 15u) * 0x00204081u) & 0x01010101u) * 255u;
                        in &= (uint32_t)((1ull << end) - (1ull << min(begin, end)));
#pragma unroll
                        for (int k = 0; k < 32; k++)
                            if (!(in >> k & 1u)) x[piece & 1][k] = 0xff800000u;
                        saw |= in != 0;
                    };
                    float top[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
                    start(0);
#pragma unroll
                    for (int piece = 0; piece < 4; piece++) {
                        landed(piece);
                        if (piece < 3) start(piece + 1);
                        if (partial) mask(piece);
#pragma unroll
                        for (int k = 0; k < 32; k += 8)
#pragma unroll
                            for (int b = 0; b < 4; b++)
                                top[b] = max3(top[b], __uint_as_float(x[piece & 1][k + 2 * b]),
                                              __uint_as_float(x[piece & 1][k + 2 * b + 1]));
                    }
                    if (partial) {
                        // values that are not finite: out of the product
                        ok = __all_sync(kFull, mbar_wait(landing(i, 1), landing_parity(i, 1)));
                        if (!ok) break;
                        const uint32_t values = s_kv + (uint32_t)((kv0 + 2 * i + 1) % kSlots) * Sh::kTile;
                        uint32_t w[4], any = 0;
                        auto piece_at = [&](int k) {
                            asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                                         : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3])
                                         : "r"(values + k * 16));
                        };
#pragma unroll 4
                        for (int k = r; k < (int)Sh::kTile / 16; k += scanners) {
                            piece_at(k);
                            any |= odd_bits(w[0]) | odd_bits(w[1]) | odd_bits(w[2]) | odd_bits(w[3]);
                        }
                        if (any & 0x80008000u) {
                            s_odd = 1;   // ahead of the zeros that the other tile's threads may find
                            __threadfence_block();
#pragma unroll 1
                            for (int k = r; k < (int)Sh::kTile / 16; k += scanners) {
                                piece_at(k);
#pragma unroll
                                for (int e = 0; e < 4; e++) {
                                    if ((w[e] & 0x7f80u) == 0x7f80u) w[e] &= 0xffff0000u;
                                    if ((w[e] & 0x7f800000u) == 0x7f800000u) w[e] &= 0x0000ffffu;
                                }
                                asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(values + k * 16), "r"(w[0]),
                                             "r"(w[1]), "r"(w[2]), "r"(w[3])
                                             : "memory");
                            }
                        }
                        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                    } else {
                        saw = true;
                    }
                    const float most = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3])) * factor;
                    const bool raise = most > m + kSlack;   // (m = -inf: a first token)
                    if (__any_sync(kFull, raise)) {
                        float keep = 1.0f;
                        if (raise) {
                            keep = m == -INFINITY ? 0.0f : exp2_fast(m - most);
                            m = most;
                            l *= keep;
                        }
                        if (kOne && n > 0) ok = __all_sync(kFull, mbar_wait(o_done(n - 1), in_turn(n - 1)));
                        if (!ok) break;
                        if (n > 0) {   // O is idle: S came after its last product (kOne: that is done)
#pragma unroll 1
                            for (int b = 0; b < D / 32; b++) {
                                uint32_t o[32];
                                tmem_ld32_start(t_o + 32 * b, o);
                                tmem_wait_ld();
                                tmem_landed(o);
#pragma unroll
                                for (int k = 0; k < 32; k++) o[k] = __float_as_uint(__uint_as_float(o[k]) * keep);
                                tmem_st32(t_o + 32 * b, o);
                            }
                        }
                    }
                    const float base = m == -INFINITY ? 0.0f : -m;
                    const uint64_t factor2 = two(factor, factor), base2 = two(base, base);
                    uint64_t sum[2] = {0, 0};
#pragma unroll
                    for (int piece = 3; piece >= 0; piece--) {
                        uint32_t *y = x[piece & 1];
                        if (piece < 2) {
                            landed(piece);
                            if (partial) mask(piece);
                        }
#pragma unroll
                        for (int k = 0; k < 16; k++) {
                            float w0, w1;
                            both(fma2(two(__uint_as_float(y[2 * k]), __uint_as_float(y[2 * k + 1])), factor2, base2), w0, w1);
                            w0 = exp2_fast(w0);
                            w1 = exp2_fast(w1);
                            sum[k & 1] = add2(sum[k & 1], two(w0, w1));
                            y[k] = pack_bf16(w0, w1);   // (scores k and below have been used)
                        }
                        tmem_st16(t_s + 32 * piece, y);   // in place of its scores
                        if (piece >= 2) start(piece - 2);
                        if (piece == 2 || piece == 0) {
                            tmem_wait_st();
                            tc_fence_before();
                            __syncwarp();
                            if (lane == 0) mbar_arrive(p_ready(buffer(n), piece >> 1));
                        }
                    }
                    float s0, s1;
                    both(add2(sum[0], sum[1]), s0, s1);
                    l += s0 + s1;
                }
                // ---- O / l
                ok = ok && (kOne ? mbar_wait(o_done(count - 1), in_turn(count - 1))
                                 : mbar_wait(s_full(q), turn_of(scored0, scored1, count))) && !*(volatile int *)&s_abort;
                if (!__all_sync(kFull, ok)) {
                    s_abort = 1;
                } else if (!SPLIT) {
                    tc_fence_after();
                    const bool odd_values = *(volatile int *)&s_odd;
                    const int row = row_q + r, token = ch.first + row / a.group;
                    const int h = kvh * a.group + row % a.group;
                    const bool live = r < rows;
                    // (rows that saw nothing are zeros whatever their gate; their O is)
                    float f = l == 0.0f ? (saw ? NAN : 0.0f) : 1.0f / l;
                    if (a.gate && live && l != 0.0f) {
                        const float g = as_f(((const __nv_bfloat16 *)a.gate)[(long long)token * a.gate_stride + h]);
                        f *= 1.0f / (1.0f + expf(-g));
                    }
                    __nv_bfloat16 *out = (__nv_bfloat16 *)a.out + (long long)token * a.out_stride + (long long)h * c.dim;
#pragma unroll 1
                    for (int b = 0; b < D / 32; b++) {
                        uint32_t o[32];
                        tmem_ld32_start(t_o + 32 * b, o);
                        tmem_wait_ld();
                        tmem_landed(o);
                        for (int i = 0; odd_values && live && i < steps; i++)
                            add_odd<32>(c, ch.stream, kvh, (step0 + i) * kStep, all_from, all_to, from, to, 32 * b, o);
                        __syncwarp();
                        if (live) {
#pragma unroll
                            for (int k = 0; k < 4; k++) {
                                if (32 * b + 8 * k >= c.dim) break;
                                uint32_t w[4];
#pragma unroll
                                for (int e = 0; e < 4; e++)
                                    w[e] = pack_bf16(__uint_as_float(o[8 * k + 2 * e]) * f, __uint_as_float(o[8 * k + 2 * e + 1]) * f);
                                *reinterpret_cast<uint4 *>(out + 32 * b + 8 * k) = make_uint4(w[0], w[1], w[2], w[3]);
                            }
                        }
                        __syncwarp();
                    }
                }
            }
        }
    } else if (!SPLIT && !dead) {
        // rows that see nothing
        const int pieces = c.dim / 8;
        for (int i = threadIdx.x; i < tile_rows * pieces; i += kTcThreads) {
            const int row = row0 + i / pieces;
            *reinterpret_cast<uint4 *>((__nv_bfloat16 *)a.out + (long long)(ch.first + row / a.group) * a.out_stride +
                                       (long long)(kvh * a.group + row % a.group) * c.dim + i % pieces * 8) =
                make_uint4(0, 0, 0, 0);
        }
    }
    tc_fence_before();
    dead = __syncthreads_or(*(volatile int *)&s_abort) || dead;
    tc_fence_after();
    if (SPLIT) {
        // the groups' parts (of a block that gave up, nothing: its cluster goes on), then their join
        if (warp >= 4) {
            const int q = (warp - 4) >> 2, r = threadIdx.x & 127;
            const uint32_t t_o = tmem + (((uint32_t)(warp & 3) * 32) << 16) + kColO + q * 128;
            const bool some = !dead && steps > q;
            if (32 * (warp & 3) < tile_rows) {
                // scores of -inf alone leave a sum of zero beside a maximum that is not -inf: a NaN
                ml[q * 128 + r] = some ? make_float2(m == -INFINITY && saw ? kLowest : m, l) : make_float2(-INFINITY, 0.0f);
                const int pos = position_of(ch, a.group, row0 + min(r, tile_rows - 1));
                const int from = a.window > 0 ? max(0, pos - a.window + 1) : 0, to = min(pos + 1, span0.high);
                const bool odd_values = *(volatile int *)&s_odd;
#pragma unroll 1
                for (int b = 0; b < D / 32; b++) {
                    uint32_t o[32];
                    __syncwarp();
                    if (some) {
                        tmem_ld32_start(t_o + 32 * b, o);
                        tmem_wait_ld();
                        tmem_landed(o);
                        // (bounded by the rank's own steps of this group)
                        for (int i = q; odd_values && i < steps; i += kGroups)
                            add_odd<32>(c, ch.stream, kvh, (step0 + i * ranks) * kStep, all_from, all_to, from, to, 32 * b, o);
                    } else {
#pragma unroll
                        for (int k = 0; k < 32; k++) o[k] = 0;
                    }
#pragma unroll
                    for (int k = 0; k < 8; k++)
                        *reinterpret_cast<uint4 *>(part + (q * 128 + r) * D + part_piece(r, 8 * b + k) * 4) =
                            make_uint4(o[4 * k], o[4 * k + 1], o[4 * k + 2], o[4 * k + 3]);
                }
            }
        }
        Tile tile;
        tile.ch = ch;
        tile.row0 = row0;
        tile.rows = tile_rows;
        join_and_store<__nv_bfloat16, D, 128, kGroups, kTcThreads>(c, a, tile, kvh, part, ml, weight, total, s_gate, ranks, rank);
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncthreads();   // the next tile's keys come where the parts were
    } else if (dead) {
        break;
    }
    if (threadIdx.x == 0) s_odd = 0;   // (the next tile's barrier follows)
    if (steps > 0) {
        kv0 += 2 * steps;
        const int count0 = SPLIT ? (steps + 1) / 2 : steps, count1 = SPLIT ? steps / 2 : rows1 > 0 ? steps : 0;
        scored0 += kOne ? count0 : count0 + 1;
        weighed0 += count0;
        scored1 += kOne ? count1 : count1 > 0 ? count1 + 1 : 0;
        weighed1 += count1;
    }
    }
    if (warp == 1)
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
}

// Tiles of a stream, as far as the caller says (the mean where it says nothing).
long long turns_of(const CacheArgs &c, const AttendArgs &a, int tile_rows)
{
    const long long most_new = a.max_new > 0 && a.max_new < c.rows ? a.max_new : c.rows / c.n_streams + 1;
    return (most_new * a.group + tile_rows - 1) / tile_rows;
}

// Pages as a 4-D tensor (elements, tokens of a page, key heads, pages); a box is 64 elements of
// `box_rows` tokens.
bool make_page_map(CUtensorMap *m, const void *base, const CacheArgs &c, int box_rows)
{
    EncodeTiledFn enc = encode_fn();
    if (!enc) return false;
    const cuuint64_t page = 1ull << c.page_shift;
    const cuuint64_t dims[4] = {(cuuint64_t)c.dim, page, (cuuint64_t)c.n_kv, (cuuint64_t)c.n_pages};
    const cuuint64_t strides[3] = {(cuuint64_t)c.dim * 2, page * c.dim * 2, (cuuint64_t)c.page_stride * 2};
    const cuuint32_t box[4] = {64, (cuuint32_t)box_rows, 1, 1};
    const cuuint32_t estr[4] = {1, 1, 1, 1};
    return enc(m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, const_cast<void *>(base), dims, strides, box, estr,
               CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
               CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int D, bool SPLIT>
cudaError_t launch_tc(const CacheArgs &c, const AttendArgs &a, int ranks, cudaStream_t stream)
{
    static std::mutex mu;
    static bool ready[64] = {false};
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (dev < 0 || dev >= 64) return cudaErrorInvalidDevice;
    {
        std::lock_guard<std::mutex> lk(mu);
        if (!ready[dev]) {
            e = cudaFuncSetAttribute(attend_tc_kernel<D, SPLIT>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                     (int)TcShape<D>::kSmem);
            if (e == cudaSuccess && SPLIT)
                e = cudaFuncSetAttribute(attend_tc_kernel<D, SPLIT>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
            if (e != cudaSuccess) return e;
            ready[dev] = true;
        }
    }
    const int page = 1 << c.page_shift, box_rows = page < kStep ? page : kStep, tile = SPLIT ? 128 : 256;
    CUtensorMap mk, mv;
    if (!make_page_map(&mk, c.k, c, box_rows) || !make_page_map(&mv, c.v, c, box_rows)) return cudaErrorInvalidValue;
    const long long turns = turns_of(c, a, tile), blocks = turns * c.n_streams * c.n_kv * ranks;
    if (blocks > 0x7fffffffll) return cudaErrorInvalidConfiguration;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)blocks);
    cfg.blockDim = dim3(TcShape<D>::kThreads);
    cfg.dynamicSmemBytes = TcShape<D>::kSmem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = (unsigned)ranks;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = ranks > 1 ? 2 : 1;
    return cudaLaunchKernelEx(&cfg, attend_tc_kernel<D, SPLIT>, mk, mv, c, a, box_rows, (int)turns, ranks);
}

template <int D>
cudaError_t launch_tc_any(const CacheArgs &c, const AttendArgs &a, cudaStream_t stream)
{
    // Tiles of 128 rows while they lie on an SM each, clusters sharing a tile's steps as far as that
    // goes on (clusters of eight such blocks only until half the SMs are taken: more do not fit at
    // once); else tiles of 256.  Chunks on 1500 to 3000 cached tokens of 16 + 4 heads of 128, us, as 256 / 128
    // rows by 1, 2, 4, 8 blocks, rows being tokens x 4:
    //   1 stream,    64 rows   38.4 / 40.1  28.2  22.0  18.9      1024 rows   53.2 / 45.0  31.5  23.7  59.3
    //   4 streams,   64 rows   47.3 / 48.2  32.8  24.3  37.0      1024 rows   64.6 / 54.7  68.2  98.5  187
    //   16 streams,  64 rows   49.9 / 50.7  35.5  49.3  98.1       512 rows   64.6 / 97.6  127   192   370
    //   64 streams, 128 rows   97.2 / 103   130   193   373
    const long long tiles = turns_of(c, a, 128) * c.n_streams * c.n_kv;
    if (!TcShape<D>::kOne && tiles > 148) return launch_tc<D, TcShape<D>::kOne>(c, a, 1, stream);
    const long long room = ((long long)c.max_pages << c.page_shift) / (2 * kStep);
    int ranks = 1;
    while (ranks < kTcRanks && tiles * ranks * 2 <= (ranks < 4 ? 148 : 74) && ranks < room) ranks *= 2;
    return launch_tc<D, true>(c, a, ranks, stream);
}

}  // namespace

cudaError_t launch_cache_attend_tc(const CacheArgs &c, const AttendArgs &a, cudaStream_t stream)
{
    if (c.dim > 128) return launch_tc_any<256>(c, a, stream);
    return c.dim <= 64 ? launch_tc_any<64>(c, a, stream) : launch_tc_any<128>(c, a, stream);
}

}  // namespace z2
