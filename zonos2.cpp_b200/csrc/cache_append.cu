// cache_append.cu -- new tokens into the paged cache (sm_100a): queries and keys normalised
// per head and rotated by their positions, keys and values written to the pages.
//
//     x' = x * w / sqrt(mean(x^2) + eps)
//     (a, b) -> (a cos t - b sin t, b cos t + a sin t),   t = p f   (a pair of the head)
//
// A head's elements lie eight to a lane, so that a head of 128 is half a warp's; its sum of
// squares is a tree of f32 sums.  The angle is p f in f64, taken in turns and reduced to
// [-1/2, 1/2] there (exact to 2^-53 of the angle: a position of 2^20 keeps 2^-33 of a turn)
// and only then rounded to f32 for the sine: f32 alone would lose every digit of a far
// position's angle.  Each result is rounded once.
//
// A warp takes a token's heads one after another with the angles' sines kept, or for few tokens one
// round of them, the token's heads shared out over warps.
//
// Bound: memory for prompts (every element is read once and written once) and beside it the issue
// slots; launch latency for a few tokens.  8200 tokens of 16 + 2 x 4 bf16 heads of 128 (101 MB): 23 to 30 us,
// 3.4 to 4.4 TB/s, the issue slots 61 % taken; 34 us with one loop over all heads, which chose each head's
// address and kind again.  One token: 3.2 us in a captured stream of them, 8.8 us as called from Python.
#include <type_traits>

#include "cache.cuh"

namespace z2 {

namespace {

constexpr int kAppendThreads = 128, kAhead = 4;

template <typename T>
struct Eight;   // eight elements as they are loaded and stored
template <>
struct Eight<float> {
    float4 a, b;
    __device__ __forceinline__ void get(float (&x)[8]) const
    {
        x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w;
        x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
    }
    __device__ __forceinline__ void set(const float (&x)[8])
    {
        a = make_float4(x[0], x[1], x[2], x[3]);
        b = make_float4(x[4], x[5], x[6], x[7]);
    }
};
template <>
struct Eight<__nv_bfloat16> {
    uint4 a;
    __device__ __forceinline__ void get(float (&x)[8]) const
    {
        const uint32_t u[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
        for (int i = 0; i < 4; i++) {
            x[2 * i] = __uint_as_float(u[i] << 16);
            x[2 * i + 1] = __uint_as_float(u[i] & 0xffff0000u);
        }
    }
    __device__ __forceinline__ void set(const float (&x)[8])
    {
        uint32_t u[4];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const __nv_bfloat162 h = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
            u[i] = *reinterpret_cast<const uint32_t *>(&h);
        }
        a = make_uint4(u[0], u[1], u[2], u[3]);
    }
};

// The stream of token row `row` (the last one that starts at or before it), found 32 ways at a
// time, and its chunk: the last 32 streams' lengths come with their starts.  Every lane takes
// part; n = 0: none.
__device__ __forceinline__ Chunk chunk_with(const CacheArgs &c, int row)
{
    const int lane = threadIdx.x & 31;
    int low = 0, many = c.n_streams;   // the answer lies in [low, low + many), if it lies anywhere
    while (many > 32) {
        const int step = (many + 31) / 32;
        const bool before = lane * step < many && c.q_start[low + lane * step] <= row;
        const int last = 31 - __clz(__ballot_sync(kFull, before) | 1u);
        low += last * step;
        many = min(step, c.n_streams - low);
    }
    const bool in = lane < many;
    const int start = in ? c.q_start[low + lane] : 0, next = in ? c.q_start[low + lane + 1] : 0;
    const int len = in ? c.kv_len[low + lane] : 0;
    const unsigned votes = __ballot_sync(kFull, in && start <= row);
    const int last = 31 - __clz(votes | 1u);
    Chunk k;
    k.stream = low + last;
    k.first = min(max(__shfl_sync(kFull, start, last), 0), c.rows);
    k.n = min(max(__shfl_sync(kFull, next, last), k.first), c.rows) - k.first;
    if (votes == 0) k.n = 0;
    k.len = max(__shfl_sync(kFull, len, last), 0);
    return k;
}

// TEAM lanes to a head (eight elements each).  LANE_PAIRS: rotation by neighbours, both of a
// pair in one lane; else the other half's element is loaded as well.
template <typename T, int TEAM, bool LANE_PAIRS>
__global__ void __launch_bounds__(kAppendThreads)
    append_kernel(const CacheArgs c, const AppendArgs a, int parts)
{
    constexpr int kHeads = 32 / TEAM;   // heads of a warp's round
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int lane = threadIdx.x & 31, sub = lane % TEAM, team = lane / TEAM;
    const long long item = ((long long)blockIdx.x * kAppendThreads + threadIdx.x) >> 5;
    const long long row_ll = item / parts;
    const int part = (int)(item % parts);   // which rounds of the token's heads
    if (row_ll >= c.rows) return;
    const int row = (int)row_ll;
    const Chunk ch = chunk_with(c, row);
    if (row < ch.first || row >= ch.first + ch.n) return;
    const int pos = ch.len - ch.n + (row - ch.first);
    const int page = pos >= 0 && pos < room_of(c) ? page_of(c, ch.stream, pos) : -1;

    const int e0 = sub * 8, dim = c.dim;
    const bool active = e0 < dim;
    const int half = a.rot >> 1;
    // the angles of this lane's elements: of four pairs, or of eight elements of either half
    constexpr int kAngles = LANE_PAIRS ? 4 : 8;
    float cs[kAngles], sn[kAngles];
#pragma unroll
    for (int i = 0; i < kAngles; i++) {
        cs[i] = 1.0f;
        sn[i] = 0.0f;
        const int e = LANE_PAIRS ? e0 + 2 * i : e0 + i;
        if (active && e < a.rot) {
            const int f = LANE_PAIRS ? e >> 1 : (e < half ? e : e - half);
            const double turns = (double)pos * ((double)a.freq[f] * 0.15915494309189533577);
            sincospif(2.0f * (float)(turns - rint(turns)), &sn[i], &cs[i]);
            if (!LANE_PAIRS && e < half) sn[i] = -sn[i];   // a cos - b sin; b cos + a sin
        }
    }
    const float rcp_dim = 1.0f / (float)dim;
    // Rounds [first, end) of this part, kHeads heads each (from + h * dim to to + h * to_step, h the
    // head's number among `heads`), the loads of kAhead of them in flight together.  Values (COPY) go
    // as they are.
    auto work = [&](auto copy, int first, int end, int heads, const T *from, T *to, long long to_step, const float *weight) {
        constexpr bool COPY = decltype(copy)::value;
        int round = first + ((part - first) % parts + parts) % parts;
        if (round >= end) return;
        float w[8];
        if (!COPY) {
#pragma unroll
            for (int i = 0; i < 8; i++) w[i] = a.norm && weight && active ? weight[e0 + i] : 1.0f;
        }
        for (; round < end; round += parts * kAhead) {
            Eight<T> raws[kAhead];
#pragma unroll
            for (int u = 0; u < kAhead; u++) {
                const int h = (round + u * parts - first) * kHeads + team;
                if (active && h < heads) raws[u] = *reinterpret_cast<const Eight<T> *>(from + h * dim + e0);
            }
#pragma unroll
            for (int u = 0; u < kAhead; u++) {
                if (round + u * parts >= end) break;   // the same for the whole warp
                const int h = (round + u * parts - first) * kHeads + team;
                const bool on = active && h < heads;
                if (!COPY) {
                    float x[8], other[8];
#pragma unroll
                    for (int i = 0; i < 8; i++) x[i] = other[i] = 0.0f;
                    if (on) raws[u].get(x);
                    if (!LANE_PAIRS && on && e0 < a.rot) {
#pragma unroll
                        for (int i = 0; i < 8; i++) {
                            const int e = e0 + i;
                            if (e < a.rot) other[i] = as_f(from[h * dim + (e < half ? e + half : e - half)]);
                        }
                    }
                    if (a.norm) {
                        float sum = 0.0f;
#pragma unroll
                        for (int i = 0; i < 8; i++) sum += x[i] * x[i];
#pragma unroll
                        for (int d = TEAM / 2; d >= 1; d >>= 1) sum += __shfl_xor_sync(kFull, sum, d);
                        const float r = rsqrtf(fmaf(sum, rcp_dim, a.eps));   // 2 ulp
#pragma unroll
                        for (int i = 0; i < 8; i++) {
                            x[i] *= r * w[i];
                            if (!LANE_PAIRS) {
                                const int e = e0 + i;
                                if (on && e < a.rot)
                                    other[i] *= r * (weight ? weight[e < half ? e + half : e - half] : 1.0f);
                            }
                        }
                    }
                    float y[8];
                    if (LANE_PAIRS) {
#pragma unroll
                        for (int i = 0; i < 4; i++) {
                            // (elements past the rotated ones are no pairs: 0 times an infinite neighbour would be a NaN)
                            const bool pair = e0 + 2 * i < a.rot;
                            y[2 * i] = pair ? x[2 * i] * cs[i] - x[2 * i + 1] * sn[i] : x[2 * i];
                            y[2 * i + 1] = pair ? x[2 * i + 1] * cs[i] + x[2 * i] * sn[i] : x[2 * i + 1];
                        }
                    } else {
#pragma unroll
                        for (int i = 0; i < 8; i++) y[i] = x[i] * cs[i] + other[i] * sn[i];
                    }
                    raws[u].set(y);
                    if (!LANE_PAIRS) __syncwarp();   // q_out may be q: the other half has been read
                }
                if (on) *reinterpret_cast<Eight<T> *>(to + h * to_step + e0) = raws[u];
            }
        }
    };
    const int rounds_q = a.q ? (a.n_heads + kHeads - 1) / kHeads : 0, rounds_kv = (c.n_kv + kHeads - 1) / kHeads;
    const long long page_step = (long long)dim << c.page_shift;   // from key head to key head
    const long long at = page >= 0 ? row_on_page(c, page, 0, pos) : 0;
    if (a.q)
        work(std::false_type(), 0, rounds_q, a.n_heads, (const T *)a.q + row * a.q_stride, (T *)a.q_out + row * a.q_out_stride,
             (long long)dim, a.q_weight);
    if (page < 0) return;   // (the whole warp: a token's)
    work(std::false_type(), rounds_q, rounds_q + rounds_kv, c.n_kv, (const T *)a.k + row * a.k_stride, (T *)c.k + at, page_step,
         a.k_weight);
    work(std::true_type(), rounds_q + rounds_kv, rounds_q + 2 * rounds_kv, c.n_kv, (const T *)a.v + row * a.v_stride, (T *)c.v + at,
         page_step, nullptr);
}

template <typename T, int TEAM, bool LANE_PAIRS>
cudaError_t launch(const CacheArgs &c, const AppendArgs &a, cudaStream_t stream)
{
    const int each = 32 / TEAM, rounds = (a.q ? (a.n_heads + each - 1) / each : 0) + 2 * ((c.n_kv + each - 1) / each);
    // few tokens: their heads shared out, until every SM has a warp of each scheduler
    int parts = 1;
    while (parts < rounds && (long long)c.rows * parts < 148 * 16) parts++;
    const long long warps = (long long)c.rows * parts;
    const long long blocks = (warps * 32 + kAppendThreads - 1) / kAppendThreads;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)blocks);
    cfg.blockDim = dim3(kAppendThreads);
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, append_kernel<T, TEAM, LANE_PAIRS>, c, a, parts);
}

template <typename T, bool LANE_PAIRS>
cudaError_t launch_team(const CacheArgs &c, const AppendArgs &a, cudaStream_t stream)
{
    if (c.dim <= 64) return launch<T, 8, LANE_PAIRS>(c, a, stream);
    if (c.dim <= 128) return launch<T, 16, LANE_PAIRS>(c, a, stream);
    return launch<T, 32, LANE_PAIRS>(c, a, stream);
}

}  // namespace

cudaError_t launch_cache_append(const CacheArgs &c, const AppendArgs &a, bool bf16, cudaStream_t stream)
{
    const bool pairs = !a.halves;
    if (bf16)
        return pairs ? launch_team<__nv_bfloat16, true>(c, a, stream)
                     : launch_team<__nv_bfloat16, false>(c, a, stream);
    return pairs ? launch_team<float, true>(c, a, stream) : launch_team<float, false>(c, a, stream);
}

}  // namespace z2
