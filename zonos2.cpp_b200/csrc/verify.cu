// verify.cu -- drafted frames checked against the sampler's distribution of the
// target's logits, from given random numbers (sm_100a).
//
// A stream has up to n_draft drafted frames of n_cb codes each, and the target's
// logits at every one of their positions and at the one after them.  At a
// (stream, position, codebook) row, p is the distribution the sampler draws from:
// penalty, masks, temperature, then top-k, top-p and min-p on the tokens ordered
// by (logit desc, token asc), renormalised; q is the draft's.  With the row's two
// uniforms u0, u1:
//   - the drafted code t stands iff u0 * q(t) < p(t);
//   - a refused code is drawn from max(p - q, 0) (from p where that is zero
//     everywhere), a code after the last draft from p: the first token in the
//     order whose cumulative weight reaches u1 of the total and has weight;
//   - the first frame that holds a refused code is the stream's last, and so is
//     the frame after its last draft.
// The codes of a frame are independent of each other given the frames before, so
// testing and correcting each codebook by itself leaves every emitted frame
// distributed as the sampler's own.
//
// Every comparison that decides a code is made in f64 on f64 exponentials and
// sums, whose differences to the mathematics are below 1e-14 relative, unless its f32 form
// has its sides further apart than f32 could have moved them (kMargin): then that one
// decides it.
//
// One warp per row, a CTA of n_cb warps per position.  Lane l holds the tokens
// 4 * (l + 32 * j) + e (j < 8, e < 4).  The row's top is found by a histogram of
// the gaps to its largest logit, and at most 128 (then 256) candidates go into
// registers.  Bounds on the kept sum, which need no order, let most drafted codes stand
// at once; otherwise the candidates are sorted, and the cuts and the draw are prefix sums
// over them.  A row whose cuts lie outside its 256 largest logits sorts all of them in
// shared memory.
// A CTA goes through its stream's positions in order and stops at the first
// refusal: later logits are not read.  With too few streams for the SMs a stream has a
// cluster of CTAs, each at a position of its own, which exchange their refusals.
//
// Bound: instruction issue and the rows' own latency, not memory.  2048 streams of 4 drafts
// with q, top-k 100 and allowed tokens (52344 rows of 1024 logits read, 214 MB): 153 us, a row
// about 1750 warp instructions (the row and its masks 520, the histogram 270, the
// candidates 400, the bounds 210, sort and decisions 700 of those that need them).  One stream of 4
// drafts: 9.4 us back to back.  All in f64 with every row sorted the first took 203 us; a
// barrier per position costs less than codebooks that run ahead of a refusal (191 / 205 us).
#include <math.h>

#include <mutex>

#include "common.cuh"
#include "sampler.cuh"
#include "verify.cuh"

namespace z2 {

namespace {

constexpr int kOpen = 127;            // the histogram's open-ended last bucket: a gap of 16 temperatures
constexpr int kMaxCand = 256;
constexpr float kMaskedAll = -1e9f;   // a row without a logit at or above this is all masked
// An f32 exponential is off by 3 g 2^-24 + 2^-22 relative at most (gap, factor and product, each
// 2^-24 of a gap of g temperatures; the power): 3.2e-6 for a candidate, whose gap is below 16.
// In a sum, all the row's too, a term's error counts by its share, and sum p g <=
// -sum p log p < 7 for 1024 tokens: 1.5e-6.  The additions, 8 of a lane and 5 levels for
// candidates and 32 and 5 for a row, bring that to 2.3e-6 and 3.7e-6 of the sum's whole.
// So a comparison of two sums is off by 7.4e-6 at most, beside three roundings of 2^-24 of the
// drafts' products or the cuts.  A code that surely_stands accepts by whole-row sums leaves
// kMargin less 7.6e-6 of the mass, 2e-6, to itself and the tokens behind it, none of them larger:
// its gap is below log(1024 / 2e-6) = 20.1, its own error below 3.9e-6, and 2 kMargin holds both.
constexpr float kMargin = 1e-5f;
// A row's answer: the code, its flags and whether the drafted code stands.
constexpr int kAllMasked = 1 << 16, kNonfinite = 2 << 16, kTaken = 1 << 30;
constexpr int kOutside = -1;          // a candidate path's answer: the cuts lie outside
constexpr int kClose = -2;            // f32 cannot decide
// Per warp: the row by token (4 pad floats after every 32), then the general
// path's token list, whose place the histogram, the candidates and the history
// bitmap take on the common path.
constexpr int kRowFloats = 1024 + 4 * 32;
constexpr int kTokWords = (1024 + 2 * 32) / 2;
constexpr int kWarpBytes = 4 * (kRowFloats + kTokWords);

__device__ __forceinline__ int row_at(int t) { return t + 4 * (t >> 5); }
__device__ __forceinline__ int tok_at(int i) { return i + 2 * (i >> 5); }

__device__ __forceinline__ float warp_max(float v)
{
    float r;
    asm("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));
    return r;
}

template <typename S>
__device__ __forceinline__ S warp_sum(S v)
{
#pragma unroll
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(kFull, v, o);
    return v;
}

// The sum of the lanes below this one, and of all of them.
template <typename S>
__device__ __forceinline__ S warp_before(S v, int lane, S *all = nullptr)
{
    S s = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const S t = __shfl_up_sync(kFull, s, o);
        if (lane >= o) s += t;
    }
    if (all) *all = __shfl_sync(kFull, s, 31);
    const S b = __shfl_up_sync(kFull, s, 1);
    return lane ? b : (S)0;
}

// kOpen for the gaps that lie past the buckets and for a scaled gap of NaN; the rounding
// only has to be the same everywhere and monotone.
__device__ __forceinline__ int gap_bucket(float top, float x, float scale)
{
    const float b = fminf(fmaf(__fsub_rn(top, x), scale, 8388608.0f), 8388608.0f + (float)kOpen);
    return (int)(__float_as_uint(b) - 0x4b000000u);
}

struct Row {
    const float *q;     // the draft's probabilities of the row (nullptr: certain of t)
    int t;              // the drafted code
    bool drafted;
    float u0, u1;
};

template <typename S>
__device__ __forceinline__ S weight(const Row &r, S e, S sum, int token)
{
    const S q = r.q ? (S)__ldg(r.q + token) : (S)(token == r.t);
    const S w = e - q * sum;   // (p - q) * sum
    return w > (S)0 ? w : (S)0;
}

// The weight of logit x in a row of largest logit `top`.
template <typename S>
__device__ __forceinline__ S power(const VerifyArgs &a, float x, float top);
template <>
__device__ __forceinline__ double power<double>(const VerifyArgs &a, float x, float top)
{
    return exp(((double)x - (double)top) * a.inv_temp);
}
template <>
__device__ __forceinline__ float power<float>(const VerifyArgs &a, float x, float top)
{
    float e;
    asm("ex2.approx.f32 %0, %1;" : "=f"(e) : "f"(__fmul_rn(__fsub_rn(x, top), a.log2_scale)));
    return e;
}

// Whether the drafted code, of weight e out of sum, stands.
__device__ __forceinline__ bool stands(const Row &r, int vocab, double e, double sum)
{
    if (!r.drafted || (unsigned)r.t >= (unsigned)vocab) return false;
    const double q = r.q ? (double)__ldg(r.q + r.t) : 1.0;
    return (double)r.u0 * q * sum < e;
}

// The general path: the whole row sorted in shared memory (x at row_at, tokens at
// tok_at), each lane owning n / 32 consecutive positions of the order.
__device__ __noinline__ int general_row(const VerifyArgs &a, const Row r, float *x, uint16_t *tok,
                                        float top, int limit)
{
    const int lane = threadIdx.x & 31;
    int n = 64;
    while (n < a.vocab) n <<= 1;
    for (int i = lane; i < n; i += 32) tok[tok_at(i)] = (uint16_t)i;
    __syncwarp();
    for (int k = 2; k <= n; k <<= 1)
        for (int j = k >> 1; j; j >>= 1) {
            for (int p = lane; p < n / 2; p += 32) {
                const int i = 2 * p - (p & (j - 1)), o = i + j;
                const float xi = x[row_at(i)], xo = x[row_at(o)];
                const int ti = tok[tok_at(i)], to = tok[tok_at(o)];
                const bool ordered = xi > xo || (xi == xo && ti < to);
                if (ordered != ((i & k) == 0)) {
                    x[row_at(i)] = xo;
                    x[row_at(o)] = xi;
                    tok[tok_at(i)] = (uint16_t)to;
                    tok[tok_at(o)] = (uint16_t)ti;
                }
            }
            __syncwarp();
        }
    const int per = n / 32, i0 = lane * per;
    auto value = [&](int i) { return power<double>(a, x[row_at(i)], top); };
    double own = 0.0, listed;
    for (int i = i0; i < i0 + per && i < limit; i++) own += value(i);
    double run = warp_before(own, lane, &listed);
    const double cut = (double)a.top_p * listed;
    double kept = 0.0;
    int count = 0;
    for (int i = i0; i < i0 + per && i < limit; i++) {
        const double e = value(i);
        if ((i == 0 || !(a.top_p < 1.0f) || run < cut) && e >= (double)a.min_p) {
            kept += e;
            count++;
        }
        run += e;
    }
    const double sum = warp_sum(kept);
    const int m = __reduce_add_sync(kFull, count);
    double et = 0.0;
    for (int i = i0; i < i0 + per && i < m; i++)
        if (tok[tok_at(i)] == r.t) et = value(i);
    et = warp_sum(et);   // one lane's, or none
    if (stands(r, a.vocab, et, sum)) return r.t | kTaken;
    bool residual = r.drafted;
    double total = 0.0;
    for (;;) {   // the residual's weights, or p's where they are all zero
        own = 0.0;
        for (int i = i0; i < i0 + per && i < m; i++) {
            const double e = value(i);
            own += residual ? weight(r, e, sum, tok[tok_at(i)]) : e;
        }
        total = warp_sum(own);
        if (!residual || total > 0.0) break;
        residual = false;
    }
    run = warp_before(own, lane);
    const double goal = (double)r.u1 * total;
    int first = n, last = -1;
    for (int i = i0; i < i0 + per && i < m; i++) {
        const double e = value(i);
        const double w = residual ? weight(r, e, sum, tok[tok_at(i)]) : e;
        run += w;
        if (w > 0.0) {
            last = i;
            if (first == n && run >= goal) first = i;
        }
    }
    first = __reduce_min_sync(kFull, first);
    last = __reduce_max_sync(kFull, last);
    return tok[tok_at(first < n ? first : last)];
}

// 32 K keys, K per lane in lane order, into ascending order.
template <int K>
__device__ __forceinline__ void sort_keys(uint32_t (&key)[K], int lane)
{
#pragma unroll
    for (int k = 2; k <= 32 * K; k <<= 1) {
#pragma unroll
        for (int j = k >> 1; j; j >>= 1) {
            const bool up = k < K || (lane & (k / K)) == 0;   // k < K: by the key's place, below
            if (j >= K) {
                const bool low = (lane & (j / K)) == 0;
#pragma unroll
                for (int i = 0; i < K; i++) {
                    const uint32_t o = __shfl_xor_sync(kFull, key[i], j / K);
                    key[i] = low == up ? min(key[i], o) : max(key[i], o);
                }
            } else {
#pragma unroll
                for (int i = 0; i < K; i++) {
                    if (i & j) continue;
                    const bool asc = k < K ? (i & k) == 0 : up;
                    const uint32_t lo = min(key[i], key[i + j]), hi = max(key[i], key[i + j]);
                    key[i] = asc ? lo : hi;
                    key[i + j] = asc ? hi : lo;
                }
            }
        }
    }
}

// What a row's candidates are: its n first tokens of the order, the top-k list covered if
// they reach its length `limit`, which is the whole row's if `whole`.
struct List {
    float top;
    int n, limit;
    bool covers, whole;
};

// The code of a row whose ordered candidates are (l, token), K per lane; kOutside where
// its cuts lie outside them, kClose where S = float cannot tell.  `all` is the sum of a row
// that is its own list without the candidates covering it.
template <typename S, int K>
__device__ __forceinline__ int decide(const VerifyArgs &a, const Row &r, const List &li, const float (&l)[K],
                                      const int (&token)[K], S all)
{
    constexpr bool kExact = sizeof(S) == 8;
    const S margin = kExact ? (S)0 : (S)kMargin;
    const int lane = threadIdx.x & 31, i0 = K * lane;
    S e[K], own = 0, listed;
#pragma unroll
    for (int j = 0; j < K; j++) {
        e[j] = i0 + j < li.n && i0 + j < li.limit ? power<S>(a, l[j], li.top) : (S)0;
        own += e[j];
    }
    S run = warp_before<S>(own, lane, &listed);
    const S least = (S)a.min_p;
    bool keep[K], close = false, cut_last = false;
#pragma unroll
    for (int j = 0; j < K; j++) {
        keep[j] = e[j] > (S)0 && e[j] >= least;
        if (!kExact) close |= i0 + j < li.n && i0 + j < li.limit && fabs(e[j] - least) <= margin * least;
        cut_last |= i0 + j == li.n - 1 && !keep[j];
    }
    // min-p cuts inside the candidates if their last one is cut
    bool inside = a.min_p > 0.0f && __any_sync(kFull, cut_last);
    if (a.top_p < 1.0f) {
        if (li.covers || li.whole) {
            if (li.covers) all = listed;
            const S cut = (S)a.top_p * all;
#pragma unroll
            for (int j = 0; j < K; j++) {
                if (!(i0 + j == 0 || run < cut)) keep[j] = false;
                if (!kExact) close |= i0 + j > 0 && e[j] > (S)0 && fabs(run - cut) <= margin * all;
                run += e[j];
            }
            inside = inside || listed >= cut;
            if (!kExact) close |= !li.covers && fabs(listed - cut) <= margin * all;
        } else {
            inside = false;   // a top-k list longer than the candidates: its sum is not known
        }
    }
    if (!kExact && __any_sync(kFull, close)) return kClose;
    if (!li.covers && !inside) return kOutside;
    S kept = 0, et = 0;
#pragma unroll
    for (int j = 0; j < K; j++) {
        kept += keep[j] ? e[j] : (S)0;
        if (keep[j] && token[j] == r.t) et = e[j];
    }
    S sum;
    const S kept_before = warp_before<S>(kept, lane, &sum);
    bool residual = false;
    if (r.drafted) {
        const unsigned holder = __ballot_sync(kFull, et > (S)0);   // at most one lane
        et = holder ? __shfl_sync(kFull, et, __ffs(holder) - 1) : (S)0;
        const bool in = (unsigned)r.t < (unsigned)a.vocab;
        const S q = !in ? (S)0 : r.q ? (S)__ldg(r.q + r.t) : (S)1, need = (S)r.u0 * q * sum;
        if (!kExact && in && fabs(need - et) <= margin * fmax(need, et)) return kClose;
        if (in && need < et) return r.t | kTaken;
        residual = true;
    }
    S w[K], total = sum;
    if (residual) {
        own = 0;
#pragma unroll
        for (int j = 0; j < K; j++) {
            w[j] = keep[j] ? weight<S>(r, e[j], sum, token[j]) : (S)0;
            own += w[j];
        }
        run = warp_before<S>(own, lane, &total);
        if (!kExact && !(total > margin * sum)) return kClose;
        residual = total > (S)0;
    }
    if (!residual) {   // after the last draft, or no weight is left: p
        run = kept_before;
        total = sum;
#pragma unroll
        for (int j = 0; j < K; j++) w[j] = keep[j] ? e[j] : (S)0;
    }
    const S goal = (S)r.u1 * total, slack = margin * (sum + total);
    int first = 32 * K, other = kExact ? -1 : 32 * K;   // other: the last with weight, or the f32 draw's latest
#pragma unroll
    for (int j = 0; j < K; j++) {
        run += w[j];
        if (kExact) {
            if (w[j] > (S)0) {
                other = i0 + j;
                if (first == 32 * K && run >= goal) first = i0 + j;
            }
        } else {
            if (first == 32 * K && run >= goal - slack) first = i0 + j;
            if (other == 32 * K && w[j] > (S)0 && run >= goal + slack) other = i0 + j;
        }
    }
    first = __reduce_min_sync(kFull, first);
    if (kExact) {
        other = __reduce_max_sync(kFull, other);
        if (first == 32 * K) first = other;
    } else {
        other = __reduce_min_sync(kFull, other);
        if (first != other || first == 32 * K) return kClose;
    }
    int hit = token[0];
#pragma unroll
    for (int j = 1; j < K; j++) hit = first % K == j ? token[j] : hit;
    return __shfl_sync(kFull, hit, first / K);
}

// Four of a lane's tokens, j of eight.
__device__ __forceinline__ float4 row_vec(const float *row, int lane, int j)
{
    return *reinterpret_cast<const float4 *>(row + row_at(4 * (lane + 32 * j)));
}

// The rare rows that f32 cannot decide: apart, so that their registers cost the others none.
template <int K>
struct Ordered {
    float l[K];
    int token[K];
};

template <int K>
__device__ __noinline__ int decide_exact(const VerifyArgs &a, const Row r, const List li, const Ordered<K> o,
                                         const float *row)
{
    double all = 0.0;
    if (a.top_p < 1.0f && !li.covers && li.whole) {
#pragma unroll 1
        for (int j = 0; j < 8; j++) {
            const float4 v = row_vec(row, threadIdx.x & 31, j);
            all += (power<double>(a, v.x, li.top) + power<double>(a, v.y, li.top)) +
                   (power<double>(a, v.z, li.top) + power<double>(a, v.w, li.top));
        }
        all = warp_sum(all);
    }
    return decide<double, K>(a, r, li, o.l, o.token, all);
}

// Whether a drafted code of weight et stands, for certain: the kept sum is at most `upper`, the
// list's sum at least `lower`, and no more than `ge` of it lies in the order up to the code.
__device__ __forceinline__ bool surely_stands(const VerifyArgs &a, const Row &r, float et, float ge, float lower,
                                              float upper)
{
    const float q = r.q ? __ldg(r.q + r.t) : 1.0f;
    return et > 0.0f && !(et < a.min_p * (1.0f + kMargin)) &&
           (!(a.top_p < 1.0f) || (ge - et) + kMargin * upper <= a.top_p * lower) &&
           r.u0 * q * upper * (1.0f + 2.0f * kMargin) < et;
}

// The candidates are the logits from here on: one comparison with the buckets' edge.  Rounding
// may put a logit at the edge on its other side, so they are counted again.
__device__ __forceinline__ float bucket_edge(float top, int last, float scale)
{
    return __fsub_rn(top, __fdividef((float)last + 0.5f, scale));
}

// The code of a row by the candidates of buckets up to `last`, at most 32 K of them; `all` is
// the row's sum where its list is the whole row and they do not cover it.
template <int K>
__device__ __forceinline__ int by_candidates(const VerifyArgs &a, const Row &r, List li, const float *row,
                                             uint32_t *cand, float scale, int last, int full, float all)
{
    const int lane = threadIdx.x & 31;
    const float top = li.top;
    const float edge = bucket_edge(top, last, scale);
    uint32_t pick = 0;
#pragma unroll
    for (int j = 0; j < 8; j++) {
        const float4 v = row_vec(row, lane, j);
        if (v.x >= edge) pick |= 1u << (4 * j);
        if (v.y >= edge) pick |= 2u << (4 * j);
        if (v.z >= edge) pick |= 4u << (4 * j);
        if (v.w >= edge) pick |= 8u << (4 * j);
    }
    int place = __popc(pick);
    const int mine = place;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int t = __shfl_up_sync(kFull, place, o);
        if (lane >= o) place += t;
    }
    li.n = __shfl_sync(kFull, place, 31);
    place -= mine;
    li.covers = li.n >= li.limit;
    // unless the list is covered a cut has to lie inside, and top-p's needs the list's sum
    if (li.n > 32 * K || !(li.covers || (a.top_p < 1.0f ? li.whole : a.min_p > 0.0f))) return kOutside;
#pragma unroll
    for (int j = 0; j < K; j += 4) reinterpret_cast<uint4 *>(cand)[lane + 8 * j] = make_uint4(~0u, ~0u, ~0u, ~0u);
    __syncwarp();
    uint32_t to = (uint32_t)__cvta_generic_to_shared(cand) + 4u * (uint32_t)place;
#pragma unroll
    for (int i = 0; i < 32; i++)   // predicated, without a branch per token
        asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %2, 0;\n\t@p st.shared.u32 [%0], %1;\n\t@p add.u32 %0, %0, 4;\n\t}"
                     : "+r"(to) : "r"(4 * lane + 128 * (i >> 2) + (i & 3)), "r"(pick & (1u << i)) : "memory");
    __syncwarp();
    // sort keys: the gap in 22 bits, then the token
    const float fine = __fdividef(4194303.0f * scale, (float)(last + 1));
    uint32_t key[K];
#pragma unroll
    for (int j = 0; j < K; j += 4) {
        const uint4 k4 = reinterpret_cast<uint4 *>(cand)[(K * lane + j) >> 2];
        key[j] = k4.x, key[j + 1] = k4.y, key[j + 2] = k4.z, key[j + 3] = k4.w;
    }
    float x[K];
#pragma unroll
    for (int j = 0; j < K; j++) {
        x[j] = -INFINITY;
        if (K * lane + j < li.n) {
            x[j] = row[row_at((int)key[j])];
            key[j] |= min((uint32_t)__fmul_rn(__fsub_rn(top, x[j]), fine), 4194302u) << 10;
        }
    }
    const bool f32 = a.log2_scale < 1e30f;
    if (f32 && li.covers && r.drafted && (unsigned)r.t < (unsigned)a.vocab) {
        // Without the order.  The kept sum lies below `upper`, the list's above `lower` (the
        // buckets before the one where the list ends).
        const float xt = row[row_at(r.t)];
        float upper = 0.0f, lower = 0.0f, ge = 0.0f;
#pragma unroll
        for (int j = 0; j < K; j++) {
            if (K * lane + j < li.n) {
                const float e = power<float>(a, x[j], top);
                upper += e;
                if (li.n == li.limit || gap_bucket(top, x[j], scale) < full) lower += e;
                if (x[j] >= xt) ge += e;
            }
        }
        if ((li.n == li.limit ? xt >= edge : gap_bucket(top, xt, scale) < full) &&
            surely_stands(a, r, power<float>(a, xt, top), warp_sum(ge), warp_sum(lower), warp_sum(upper))) {
            return r.t | kTaken;
        }
    }
    sort_keys<K>(key, lane);
    int token[K];
    float l[K];
#pragma unroll
    for (int j = 0; j < K; j++) {
        token[j] = (int)(key[j] & 1023u);
        l[j] = K * lane + j < li.n ? row[row_at(token[j])] : -INFINITY;
    }
    // keys of one quantum may stand in the wrong order: exchange neighbours until none do
    auto wrong = [](float la, int ta, float lb, int tb) {   // (la, ta) stands before (lb, tb)
        return la < lb || (la == lb && ta > tb && la > -INFINITY);
    };
    for (;;) {
        bool moved = false;
#pragma unroll
        for (int odd = 0; odd < 2; odd++) {
#pragma unroll
            for (int j = odd; j + 1 < K; j += 2) {
                if (wrong(l[j], token[j], l[j + 1], token[j + 1])) {
                    const float tl = l[j];
                    const int tt = token[j];
                    l[j] = l[j + 1], token[j] = token[j + 1];
                    l[j + 1] = tl, token[j + 1] = tt;
                    moved = true;
                }
            }
        }
        const float nl = __shfl_down_sync(kFull, l[0], 1), pl = __shfl_up_sync(kFull, l[K - 1], 1);
        const int nt = __shfl_down_sync(kFull, token[0], 1), pt = __shfl_up_sync(kFull, token[K - 1], 1);
        if (lane < 31 && wrong(l[K - 1], token[K - 1], nl, nt)) l[K - 1] = nl, token[K - 1] = nt, moved = true;
        if (lane > 0 && wrong(pl, pt, l[0], token[0])) l[0] = pl, token[0] = pt, moved = true;
        if (!__any_sync(kFull, moved)) break;
    }
    // (Without its sum where a whole row's last logit lay on the edge: then in f64, which takes it.)
    if (f32 && (li.covers || !(a.top_p < 1.0f) || all > 0.0f)) {
        const int code = decide<float, K>(a, r, li, l, token, all);
        if (code != kClose) return code;
    }
    Ordered<K> o;
#pragma unroll
    for (int j = 0; j < K; j++) o.l[j] = l[j], o.token[j] = token[j];
    return decide_exact<K>(a, r, li, o, row);
}

// As above with 256 candidates: for few rows, and apart, so that its registers cost the others none.
__device__ __noinline__ int by_more_candidates(const VerifyArgs &a, const Row r, const List li, const float *row,
                                               uint32_t *cand, float scale, int last, int full, float all)
{
    return by_candidates<8>(a, r, li, row, cand, scale, last, full, all);
}

// The row (s, d, c): its code, its flag, and whether the drafted code stands.
__device__ __forceinline__ int verify_row(const VerifyArgs &a, long long s, int d, int c, int pos,
                                          bool drafted, unsigned char *mem)
{
    const int lane = threadIdx.x & 31;
    float *row = reinterpret_cast<float *>(mem);
    uint16_t *tok = reinterpret_cast<uint16_t *>(row + kRowFloats);
    uint32_t *hist = reinterpret_cast<uint32_t *>(row + kRowFloats);
    uint32_t *cand = hist + 128;
    uint32_t *seen = cand + kMaxCand;
    const int V = a.vocab, D = a.n_draft, C = a.n_cb;
    const long long at = (s * (D + 1) + d) * C + c;
    const float *lg = a.logits + at * a.row_stride;

    float x[32];   // 0 past the vocabulary
    if (a.vec_logits) {
#pragma unroll
        for (int j = 0; j < 8; j++) {
            const int t = 4 * (lane + 32 * j);
            float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            if (t < V) v = __ldg(reinterpret_cast<const float4 *>(lg + t));
            x[4 * j] = v.x;
            x[4 * j + 1] = v.y;
            x[4 * j + 2] = v.z;
            x[4 * j + 3] = v.w;
        }
    } else {
#pragma unroll
        for (int i = 0; i < 32; i++) {
            const int t = 4 * (lane + 32 * (i >> 2)) + (i & 3);
            x[i] = t < V ? __ldg(lg + t) : 0.0f;
        }
    }

    Row r;
    r.drafted = drafted;
    r.t = drafted ? __ldg(a.drafts + (s * D + d) * C + c) : -1;
    r.q = drafted && a.probs ? a.probs + ((s * D + d) * C + c) * (long long)V : nullptr;
    r.u0 = __ldg(a.uniforms + 2 * at);
    r.u1 = __ldg(a.uniforms + 2 * at + 1);

    // the penalty's tokens: the ring without its d oldest entries, and the frames
    // drafted before (the newest of them where they fill the ring)
    uint32_t marks = 0;
    if (a.hist && a.rho != 1.0f) {
        const int H = a.hist_len;
        const int32_t *ring = a.hist + (s * C + c) * (long long)H;
        seen[lane] = 0;
        __syncwarp();
        auto mark = [&](int t) {
            if ((unsigned)t < (unsigned)V) atomicOr(&seen[(t >> 2) & 31], 1u << (4 * (t >> 7) + (t & 3)));
        };
        for (int i0 = lane; i0 < H; i0 += 256) {   // eight loads at a time, then their marks
            int t[8];
#pragma unroll
            for (int j = 0; j < 8; j++) t[j] = i0 + 32 * j < H ? ring[i0 + 32 * j] : -1;
#pragma unroll
            for (int j = 0; j < 8; j++) {
                const int i = i0 + 32 * j, age = i >= pos ? i - pos : i - pos + H;
                if (age >= d) mark(t[j]);
            }
        }
        for (int j = (d > H ? d - H : 0) + lane; j < d; j += 32) mark(__ldg(a.drafts + (s * D + j) * C + c));
        __syncwarp();
        marks = seen[lane];
    }
    uint32_t may = 0xffffffffu;
    if (a.allow) {
        const int words = (V + 31) >> 5;
        const uint32_t *w = a.allow + s * words;
        may = 0;
#pragma unroll
        for (int j = 0; j < 8; j++) {
            const int k = (lane >> 3) + 4 * j;
            if (k < words) may |= ((__ldg(w + k) >> (4 * (lane & 7))) & 15u) << (4 * j);
        }
    }
    if (a.delay_step >= 0 && (long long)a.delay_step + d < c) {   // only pad_id
        const int t = a.pad_id;
        may &= ((t >> 2) & 31) == lane ? 1u << (4 * (t >> 7) + (t & 3)) : 0u;
    }

    // 0 * x is not a number for an odd one (NaN, +inf) and for -inf
    bool odd = false;
    float nothing = 0.0f;
#pragma unroll
    for (int i = 0; i < 32; i++) nothing = fmaf(x[i], 0.0f, nothing);
    if (nothing != 0.0f) {
#pragma unroll
        for (int i = 0; i < 32; i++) {
            if (!(x[i] < INFINITY)) {
                odd = true;
                x[i] = -INFINITY;
            }
        }
    }
    if (a.hist && a.rho != 1.0f) {
#pragma unroll
        for (int i = 0; i < 32; i++) {
            const float pen = fminf(__fmul_rn(x[i], x[i] > 0.0f ? a.inv_rho : a.rho), 3.4028235e38f);
            x[i] = (marks >> i) & 1u ? pen : x[i];
        }
    }
    if (V < 1024) {
#pragma unroll
        for (int j = 0; j < 8; j++) {
            const int left = V - 4 * (lane + 32 * j);
            may &= ~((left <= 0 ? 15u : left < 4 ? 15u & (15u << left) : 0u) << (4 * j));
        }
    }
    if (!__all_sync(kFull, may == 0xffffffffu)) {
#pragma unroll
        for (int i = 0; i < 32; i++) x[i] = (may >> i) & 1u ? x[i] : -INFINITY;
    }
    float top = x[0];
#pragma unroll
    for (int i = 1; i < 32; i++) top = fmaxf(top, x[i]);
    top = warp_max(top);
    const int flag = __any_sync(kFull, odd) ? kNonfinite : 0;
    if (!(top >= kMaskedAll)) {   // all masked: pad_id is certain
        return a.pad_id | flag | kAllMasked | (r.t == a.pad_id && stands(r, V, 1.0, 1.0) ? kTaken : 0);
    }

    // ---- the row in shared memory, and the histogram of its gaps
    const float scale = fminf(8.0f * (float)a.inv_temp, 1e30f);
    reinterpret_cast<uint4 *>(hist)[lane] = make_uint4(0, 0, 0, 0);
#pragma unroll
    for (int j = 0; j < 8; j++)
        *reinterpret_cast<float4 *>(row + row_at(4 * (lane + 32 * j))) =
            make_float4(x[4 * j], x[4 * j + 1], x[4 * j + 2], x[4 * j + 3]);
    __syncwarp();
#pragma unroll
    for (int i = 0; i < 32; i++) atomicAdd(&hist[gap_bucket(top, x[i], scale)], 1u);
    __syncwarp();
    const uint4 h4 = reinterpret_cast<uint4 *>(hist)[lane];
    int c0 = (int)h4.x, c1 = c0 + (int)h4.y, c2 = c1 + (int)h4.z, c3 = c2 + (int)h4.w;
    int before = c3;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int t = __shfl_up_sync(kFull, before, o);
        if (lane >= o) before += t;
    }
    before -= c3;
    c0 += before;
    c1 += before;
    c2 += before;
    c3 += before;
    // the length of the top-k list; `whole` where that is all there is
    List li;
    li.top = top;
    li.limit = a.top_k;
    li.whole = false;
    if (a.top_k <= 0 || __shfl_sync(kFull, c2, 31) < a.top_k) {   // else the closed buckets hold it
        int alive = 0;
#pragma unroll
        for (int i = 0; i < 32; i++) alive += x[i] > -INFINITY;
        alive = __reduce_add_sync(kFull, alive);
        if (a.top_k <= 0 || alive <= a.top_k) {
            li.limit = alive;
            li.whole = true;
        }
    }
    // the first bucket whose cumulative count reaches the list's length, and the
    // last whose cumulative count fits the candidates; the open bucket is never taken
    const int limit = li.limit;
    const int full = __reduce_add_sync(kFull, (c0 < limit) + (c1 < limit) + (c2 < limit) + (c3 < limit));
    int last[2];
#pragma unroll
    for (int k = 0; k < 2; k++) {
        const int most = 128 << k;
        const int fits = __reduce_add_sync(kFull, (c0 <= most) + (c1 <= most) + (c2 <= most) +
                                                      (lane < 31 && c3 <= most)) - 1;
        last[k] = min(full, min(fits, kOpen - 1));
    }
    // With candidates that do not reach the list's end a cut has to lie inside, and top-p's
    // needs the list's sum.
    const bool cuts = a.top_p < 1.0f ? li.whole : a.min_p > 0.0f;
    bool try_first = last[0] >= 0 && (last[0] == full || cuts);
    bool try_second = last[1] > last[0] && (last[1] == full || cuts);
    float all = 0.0f;
    if (li.whole && a.top_p < 1.0f && last[0] < full && a.log2_scale < 1e30f) {
        // A nucleus of the whole row: the masses of the row, of either set of candidates, and
        // of the order up to the drafted code tell which of them it needs, or that the code stands.
        const float edge0 = bucket_edge(top, last[0], scale), edge1 = bucket_edge(top, last[1], scale);
        const bool in = r.drafted && (unsigned)r.t < (unsigned)V;
        const float xt = in ? row[row_at(r.t)] : INFINITY;
        float mass0 = 0.0f, mass1 = 0.0f, ge = 0.0f;
#pragma unroll
        for (int i = 0; i < 32; i++) {
            const float e = power<float>(a, x[i], top);
            all += e;
            if (x[i] >= edge0) mass0 += e;
            if (x[i] >= edge1) mass1 += e;
            if (x[i] >= xt) ge += e;
        }
        all = warp_sum(all);
        if (in && surely_stands(a, r, power<float>(a, xt, top), warp_sum(ge), all, all)) {
            return r.t | kTaken | flag;
        }
        const float least = (a.top_p - 2.0f * kMargin) * all;
        if (!(a.min_p > 0.0f)) {
            try_first = try_first && warp_sum(mass0) >= least;
            try_second = try_second && warp_sum(mass1) >= least;
        }
    }
#pragma unroll 1
    for (int k = 0; k < 2; k++) {
        if (!(k ? try_second : try_first)) continue;
        const int code = k ? by_more_candidates(a, r, li, row, cand, scale, last[1], full, all)
                           : by_candidates<4>(a, r, li, row, cand, scale, last[0], full, all);
        if (code >= 0) return code | flag;
        __syncwarp();
    }
    __syncwarp();
    return general_row(a, r, row, tok, top, limit) | flag;
}

__device__ __forceinline__ void cluster_barrier()
{
    __syncwarp();
    asm volatile("barrier.cluster.arrive.aligned;\n\tbarrier.cluster.wait.aligned;" ::: "memory");
}

// Block b: stream b / parts, the positions b % parts, + parts, ... of it; the `parts`
// blocks of a stream are a cluster.
template <int kMaxWarps, int kMinCtas>
__global__ void __launch_bounds__(32 * kMaxWarps, kMinCtas)
    verify_kernel(const __grid_constant__ VerifyArgs a, const int parts)
{
    extern __shared__ __align__(16) unsigned char smem[];
    __shared__ int refused[2];   // by the round's parity
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const int c = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const long long s = blockIdx.x / parts;
    const int part = blockIdx.x % parts;
    const int D = a.n_draft, C = a.n_cb, H = a.hist_len;
    unsigned char *mem = smem + c * kWarpBytes;
    int pos = 0;
    if (H > 0) {
        pos = a.hist_pos[s] % H;
        if (pos < 0) pos += H;
    }
    int drafted = D;
    if (a.n_drafts) drafted = min(max(__ldg(a.n_drafts + s), 0), D);
    int32_t *codes = a.codes + s * (D + 1) * C + c;
    int32_t *flags = a.flags ? a.flags + s * (D + 1) * C + c : nullptr;
    int32_t *ring = H > 0 ? a.hist + (s * C + c) * (long long)H : nullptr;
    // A frame with a refused code (the frame after the drafts counts as one) is the last.
    int last = -1, own = part;   // own: the first of this block's positions not yet written
    for (int round = 0; last < 0; round++, own += parts) {
        const int d = own;
        int flag = 0, code = -1;
        bool taken = false;
        if (d <= drafted) {
            code = verify_row(a, s, d, c, pos, d < drafted, mem);
            taken = code & kTaken;
            flag = code / kAllMasked & 3;
            code &= kAllMasked - 1;
        }
        const int no = __syncthreads_or(!taken);
        if (parts == 1) {
            if (no) last = d;
        } else {
            if (threadIdx.x == 0) refused[round & 1] = no;
            cluster_barrier();
            for (int p = parts - 1; p >= 0; p--) {
                uint32_t at = (uint32_t)__cvta_generic_to_shared(&refused[round & 1]);
                int n;
                asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(at), "r"(p));
                asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(n) : "r"(at) : "memory");
                if (n) last = round * parts + p;
            }
        }
        if (lane == 0 && d <= D) {
            const bool emitted = last < 0 || d <= last;
            codes[(long long)d * C] = emitted ? code : -1;
            if (flags) flags[(long long)d * C] = emitted ? flag : 0;
        }
    }
    // No block leaves before the others have read its flags.
    if (parts > 1) cluster_barrier();
    __syncwarp();
    for (long long k = own + (long long)lane * parts; k <= D; k += 32 * parts) {
        codes[k * C] = -1;
        if (flags) flags[k * C] = 0;
    }
    if (H > 0) {   // append the emitted frames: the ring's last H of them
        long long k = part + (long long)lane * parts;
        for (; k <= last; k += 32 * parts)
            if (k > last - H) ring[(pos + k) % H] = codes[k * C];
    }
    if (part == 0 && threadIdx.x == 0) {
        a.n_accepted[s] = last;
        if (H > 0) a.hist_pos[s] = (int)(((long long)pos + last + 1) % H);
    }
}

// The SMs of the current device.  A kernel's shared-memory limit is one value for all host
// threads: it is set to its most codebooks' on a device's first launch, and never lowered.
cudaError_t device_sms(int *sms)
{
    static std::mutex mu;
    static int known[64];
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (dev < 0 || dev >= 64) return cudaErrorInvalidDevice;
    std::lock_guard<std::mutex> lk(mu);
    if (!known[dev]) {
        constexpr auto kLimit = cudaFuncAttributeMaxDynamicSharedMemorySize;
        int n = 0;
        e = cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev);
        if (e == cudaSuccess) e = cudaFuncSetAttribute(verify_kernel<kSamplerCbMax, 1>, kLimit, kSamplerCbMax * kWarpBytes);
        if (e == cudaSuccess) e = cudaFuncSetAttribute(verify_kernel<9, 3>, kLimit, 9 * kWarpBytes);
        if (e == cudaSuccess) e = cudaFuncSetAttribute(verify_kernel<9, 2>, kLimit, 9 * kWarpBytes);
        if (e != cudaSuccess) return e;
        known[dev] = n;
    }
    *sms = known[dev];
    return cudaSuccess;
}

template <class Kernel>
cudaError_t launch(Kernel kernel, const VerifyArgs &a, int parts, cudaStream_t stream)
{
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)a.n_streams * (unsigned)parts);
    cfg.blockDim = dim3(32u * (unsigned)a.n_cb);
    cfg.dynamicSmemBytes = (size_t)(a.n_cb * kWarpBytes);
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = (unsigned)parts;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = parts > 1 ? 2 : 1;
    return cudaLaunchKernelEx(&cfg, kernel, a, parts);
}

}  // namespace

cudaError_t launch_verify(const VerifyArgs &a, cudaStream_t stream)
{
    if (a.n_streams == 0) return cudaSuccess;
    int sms = 0;
    const cudaError_t e = device_sms(&sms);
    if (e != cudaSuccess) return e;
    // A stream's positions at once where half the SMs hold them (8: the portable cluster): one
    // stream with 4 drafts 9.4 us, 16.1 us one after the other.  With more of them at work the
    // positions past a refusal cost the next call more than this one gains: 64 streams with 3
    // drafts 14.1 us in order, 18.1 us two and 18.5 us four at a time (37 and 33 us alone).
    const int parts = max(1, min(min(a.n_draft + 1, 8), sms / 2 / a.n_streams));
    if (a.n_cb > 9) return launch(verify_kernel<kSamplerCbMax, 1>, a, parts, stream);
    // Three blocks an SM (72 registers a thread, 96 with two; both spill, 120 and 180 bytes of
    // stores, more in the functions kept apart) where two do not hold nearly all: 300 streams 60.9 us with
    // three, 50.9 with two; 2048 streams 178 and 183.  Between those the crossover is not measured.
    return a.n_streams > 3 * sms ? launch(verify_kernel<9, 3>, a, parts, stream)
                                 : launch(verify_kernel<9, 2>, a, parts, stream);
}

}  // namespace z2
