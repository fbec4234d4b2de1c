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
// Bound: memory for prompts (every element is read once and written once), launch latency for
// a few tokens.  A warp takes a token's heads one after another with the angles' sines kept, or
// for few tokens one round of them, the token's heads shared out over warps.
#include "cache.cuh"

namespace z2 {

namespace {

constexpr int kAppendThreads = 128;

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

// The stream of token row `row`: the last one that starts at or before it, 32 ways at a
// time.  Every lane takes part; -1: before the first.
__device__ __forceinline__ int stream_of(const CacheArgs &c, int row)
{
    const int lane = threadIdx.x & 31;
    int low = 0, many = c.n_streams;   // the answer lies in [low, low + many)
    if (__ldg(c.q_start) > row) return -1;
    while (many > 1) {
        const int step = (many + 31) / 32;
        const int at = low + lane * step;
        const bool before = lane * step < many && __ldg(c.q_start + at) <= row;
        const unsigned votes = __ballot_sync(kFull, before);
        const int last = 31 - __clz(votes | 1u);   // the first always is, unless the starts fall
        low += last * step;
        many = min(step, c.n_streams - low);
    }
    return low;
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
    const int s = stream_of(c, row);
    if (s < 0) return;
    const Chunk ch = chunk_of(c, s);
    if (row < ch.first || row >= ch.first + ch.n) return;
    const int pos = ch.len - ch.n + (row - ch.first);
    const int page = pos >= 0 && pos < room_of(c) ? page_of(c, s, pos) : -1;

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
            const double turns = (double)pos * ((double)__ldg(a.freq + f) * 0.15915494309189533577);
            sincospif(2.0f * (float)(turns - rint(turns)), &sn[i], &cs[i]);
            if (!LANE_PAIRS && e < half) sn[i] = -sn[i];   // a cos - b sin; b cos + a sin
        }
    }
    const int first_head = a.q ? 0 : a.n_heads;
    const int total = a.n_heads + 2 * c.n_kv;
    for (int h0 = first_head + part * kHeads; h0 < total; h0 += parts * kHeads) {
        const int h = h0 + team;
        const bool on = active && h < total;
        const bool is_q = h < a.n_heads, is_v = h >= a.n_heads + c.n_kv;
        const int kh = is_q ? 0 : is_v ? h - a.n_heads - c.n_kv : h - a.n_heads;
        const T *from = is_q ? (const T *)a.q + row * a.q_stride + (long long)h * dim
                             : is_v ? (const T *)a.v + row * a.v_stride + (long long)kh * dim
                                    : (const T *)a.k + row * a.k_stride + (long long)kh * dim;
        Eight<T> raw;
        if (on) raw = *reinterpret_cast<const Eight<T> *>(from + e0);
        float x[8], other[8];
#pragma unroll
        for (int i = 0; i < 8; i++) x[i] = other[i] = 0.0f;
        if (on) raw.get(x);
        if (!LANE_PAIRS && on && !is_v && e0 < a.rot) {
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const int e = e0 + i;
                if (e < a.rot) other[i] = as_f(from[e < half ? e + half : e - half]);
            }
        }
        float sum = 0.0f;
        if (a.norm) {   // (every lane: a warp's heads may be keys and values)
#pragma unroll
            for (int i = 0; i < 8; i++) sum += x[i] * x[i];
#pragma unroll
            for (int d = TEAM / 2; d >= 1; d >>= 1) sum += __shfl_xor_sync(kFull, sum, d);
        }
        if (!is_v) {
            if (a.norm) {
                const float r = 1.0f / sqrtf(sum / (float)dim + a.eps);
                const float *w = is_q ? a.q_weight : a.k_weight;
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    x[i] *= r * (w && on ? __ldg(w + e0 + i) : 1.0f);
                    if (!LANE_PAIRS) {
                        const int e = e0 + i;
                        if (on && e < a.rot)
                            other[i] *= r * (w ? __ldg(w + (e < half ? e + half : e - half)) : 1.0f);
                    }
                }
            }
            float y[8];
            if (LANE_PAIRS) {
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    y[2 * i] = x[2 * i] * cs[i] - x[2 * i + 1] * sn[i];
                    y[2 * i + 1] = x[2 * i + 1] * cs[i] + x[2 * i] * sn[i];
                }
            } else {
#pragma unroll
                for (int i = 0; i < 8; i++) y[i] = x[i] * cs[i] + other[i] * sn[i];
            }
            raw.set(y);
        }
        if (!LANE_PAIRS) __syncwarp();   // q_out may be q: the other half has been read
        if (on) {
            T *to = nullptr;
            if (is_q)
                to = (T *)a.q_out + row * a.q_out_stride + (long long)h * dim;
            else if (page >= 0)
                to = (T *)(is_v ? c.v : c.k) + row_on_page(c, page, kh, pos);
            if (to) *reinterpret_cast<Eight<T> *>(to + e0) = raw;
        }
    }
}

template <typename T, int TEAM, bool LANE_PAIRS>
cudaError_t launch(const CacheArgs &c, const AppendArgs &a, cudaStream_t stream)
{
    const int rounds = ((a.q ? a.n_heads : 0) + 2 * c.n_kv + 32 / TEAM - 1) / (32 / TEAM);
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
