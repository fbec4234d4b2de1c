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
// sums: differences to the mathematics are below 1e-14 relative.
//
// One warp per row, a CTA of n_cb warps per position.  Lane l holds the tokens
// 4 * (l + 32 * j) + e (j < 8, e < 4).  The row's top is found by a histogram of
// the gaps to its largest logit, at most 128 candidates are sorted in registers,
// and the cuts and the draw are prefix sums over them.  A row whose cuts lie
// outside its 128 largest logits sorts all of them in shared memory.
// A CTA goes through its stream's positions in order and stops at the first
// refusal: later logits are not read.
#include <math.h>

#include "common.cuh"
#include "sampler.cuh"
#include "verify.cuh"

namespace z2 {

namespace {

constexpr int kCand = 128;
constexpr float kOpen = 127.0f;       // the histogram's open-ended last bucket
constexpr float kMaskedAll = -1e9f;   // a row without a logit at or above this is all masked
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

__device__ __forceinline__ double warp_sum(double v)
{
#pragma unroll
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(kFull, v, o);
    return v;
}

// The sum of the lanes below this one.
__device__ __forceinline__ double warp_before(double v, int lane)
{
    double s = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const double t = __shfl_up_sync(kFull, s, o);
        if (lane >= o) s += t;
    }
    const double b = __shfl_up_sync(kFull, s, 1);
    return lane ? b : 0.0;
}

__device__ __forceinline__ float gap_bucket(float top, float x, float scale)
{
    return fminf(__fmul_rn(__fsub_rn(top, x), scale), kOpen);
}

struct Row {
    const float *q;     // the draft's probabilities of the row (nullptr: certain of t)
    int t;              // the drafted code
    bool drafted;
    double u0, u1;
};

__device__ __forceinline__ double weight(const Row &r, double e, double sum, int token)
{
    const double q = r.q ? (double)__ldg(r.q + token) : (token == r.t ? 1.0 : 0.0);
    const double w = e - q * sum;   // (p - q) * sum
    return w > 0.0 ? w : 0.0;
}

// Whether the drafted code, of weight e out of sum, stands.
__device__ __forceinline__ bool stands(const Row &r, int vocab, double e, double sum)
{
    if (!r.drafted || (unsigned)r.t >= (unsigned)vocab) return false;
    const double q = r.q ? (double)__ldg(r.q + r.t) : 1.0;
    return r.u0 * q * sum < e;
}

// The general path: the whole row sorted in shared memory (x at row_at, tokens at
// tok_at), each lane owning n / 32 consecutive positions of the order.
__device__ __noinline__ int general_row(const VerifyArgs &a, const Row &r, float *x, uint16_t *tok,
                                        float top, int limit, bool *taken)
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
    auto value = [&](int i) { return exp(((double)x[row_at(i)] - (double)top) * a.inv_temp); };
    double own = 0.0;
    for (int i = i0; i < i0 + per && i < limit; i++) own += value(i);
    double run = warp_before(own, lane);
    const double cut = (double)a.top_p * warp_sum(own);
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
    *taken = stands(r, a.vocab, et, sum);
    if (*taken) return r.t;
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
    const double goal = r.u1 * total;
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

// 128 keys, four per lane in lane order, into ascending order.
__device__ __forceinline__ void sort_keys(uint32_t (&key)[4], int lane)
{
#pragma unroll
    for (int k = 2; k <= kCand; k <<= 1) {
#pragma unroll
        for (int j = k >> 1; j; j >>= 1) {
            const bool up = k == 2 || (lane & (k >> 2)) == 0;
            if (j >= 4) {
                const bool low = (lane & (j >> 2)) == 0;
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const uint32_t o = __shfl_xor_sync(kFull, key[i], j >> 2);
                    key[i] = low == up ? min(key[i], o) : max(key[i], o);
                }
            } else {
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    if (i & j) continue;
                    const bool asc = k == 2 ? i == 0 : up;
                    const uint32_t lo = min(key[i], key[i + j]), hi = max(key[i], key[i + j]);
                    key[i] = asc ? lo : hi;
                    key[i + j] = asc ? hi : lo;
                }
            }
        }
    }
}

// The row (s, d, c): its code, its flag, and whether the drafted code stands.
__device__ __forceinline__ int verify_row(const VerifyArgs &a, long long s, int d, int c, int pos,
                                          bool drafted, unsigned char *mem, int *flag, bool *taken)
{
    const int lane = threadIdx.x & 31;
    float *row = reinterpret_cast<float *>(mem);
    uint16_t *tok = reinterpret_cast<uint16_t *>(row + kRowFloats);
    uint32_t *hist = reinterpret_cast<uint32_t *>(row + kRowFloats);
    uint32_t *cand = hist + 128;
    uint32_t *seen = cand + kCand;
    const int V = a.vocab, D = a.n_draft, C = a.n_cb;
    const long long at = (s * (D + 1) + d) * C + c;
    const float *lg = a.logits + at * a.row_stride;

    float x[32];
    if (a.vec_logits) {
#pragma unroll
        for (int j = 0; j < 8; j++) {
            const int t = 4 * (lane + 32 * j);
            float4 v = make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
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
            x[i] = t < V ? __ldg(lg + t) : -INFINITY;
        }
    }

    Row r;
    r.drafted = drafted;
    r.t = drafted ? __ldg(a.drafts + (s * D + d) * C + c) : -1;
    r.q = drafted && a.probs ? a.probs + ((s * D + d) * C + c) * (long long)V : nullptr;
    r.u0 = (double)__ldg(a.uniforms + 2 * at);
    r.u1 = (double)__ldg(a.uniforms + 2 * at + 1);

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
        for (int i = lane; i < H; i += 32) {
            const int age = i >= pos ? i - pos : i - pos + H;
            if (age >= d) mark(ring[i]);
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

    bool odd = false;
    float top = -INFINITY;
#pragma unroll
    for (int i = 0; i < 32; i++) {
        float v = x[i];
        if (!(v < INFINITY)) {   // NaN, +inf
            odd = true;
            v = -INFINITY;
        }
        const float pen = fminf(__fmul_rn(v, v > 0.0f ? a.inv_rho : a.rho), 3.4028235e38f);
        v = (marks >> i) & 1u ? pen : v;
        v = (may >> i) & 1u ? v : -INFINITY;
        x[i] = v;
        top = fmaxf(top, v);
    }
    top = warp_max(top);
    *flag = __any_sync(kFull, odd) ? 2 : 0;
    if (!(top >= kMaskedAll)) {   // all masked: pad_id is certain
        *flag |= 1;
        *taken = r.t == a.pad_id && stands(r, V, 1.0, 1.0);
        return a.pad_id;
    }

    // ---- the row in shared memory, and the histogram of its gaps
    const float scale = fminf(8.0f * (float)a.inv_temp, 1e30f);
    reinterpret_cast<uint4 *>(hist)[lane] = make_uint4(0, 0, 0, 0);
    int alive = 0;
#pragma unroll
    for (int j = 0; j < 8; j++)
        *reinterpret_cast<float4 *>(row + row_at(4 * (lane + 32 * j))) =
            make_float4(x[4 * j], x[4 * j + 1], x[4 * j + 2], x[4 * j + 3]);
    __syncwarp();
#pragma unroll
    for (int i = 0; i < 32; i++) {
        alive += x[i] > -INFINITY;
        atomicAdd(&hist[(int)gap_bucket(top, x[i], scale)], 1u);
    }
    alive = __reduce_add_sync(kFull, alive);
    __syncwarp();
    const int limit = a.top_k > 0 && a.top_k < alive ? a.top_k : alive;   // length of the top-k list
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
    // the first bucket whose cumulative count reaches the list's length, and the
    // last whose cumulative count is at most kCand; the open bucket is never taken
    const int full = __reduce_add_sync(kFull, (c0 < limit) + (c1 < limit) + (c2 < limit) + (c3 < limit));
    const int fits = __reduce_add_sync(kFull, (c0 <= kCand) + (c1 <= kCand) + (c2 <= kCand) +
                                                  (lane < 31 && c3 <= kCand)) - 1;
    const int last_bucket = min(full, min(fits, 126));
    bool closed = last_bucket >= 0;
    if (closed) {
        const int sel = last_bucket & 3;
        int n = sel == 0 ? c0 : sel == 1 ? c1 : sel == 2 ? c2 : c3;
        n = __shfl_sync(kFull, n, last_bucket >> 2);
        const bool covers = n >= limit;
        // the candidates as sort keys: the gap in 22 bits, then the token
        const float width = __fdiv_rn((float)(last_bucket + 1), scale);
        const float fine = __fdiv_rn(4194303.0f, width);
        uint32_t pick = 0;
#pragma unroll
        for (int i = 0; i < 32; i++)
            pick |= (gap_bucket(top, x[i], scale) < (float)(last_bucket + 1) ? 1u : 0u) << i;
        int place = __popc(pick);
        const int mine = place;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int t = __shfl_up_sync(kFull, place, o);
            if (lane >= o) place += t;
        }
        place -= mine;
        reinterpret_cast<uint4 *>(cand)[lane] = make_uint4(~0u, ~0u, ~0u, ~0u);
        __syncwarp();
        for (; pick; pick &= pick - 1) {
            const int i = __ffs(pick) - 1;
            const int t = 4 * (lane + 32 * (i >> 2)) + (i & 3);
            const float g = __fmul_rn(__fsub_rn(top, row[row_at(t)]), fine);
            if (place < kCand) cand[place] = (min((uint32_t)g, 4194302u) << 10) | (uint32_t)t;
            place++;
        }
        __syncwarp();
        const uint4 k4 = reinterpret_cast<uint4 *>(cand)[lane];
        uint32_t key[4] = {k4.x, k4.y, k4.z, k4.w};
        sort_keys(key, lane);
        int token[4];
        float l[4];
#pragma unroll
        for (int j = 0; j < 4; j++) {
            token[j] = (int)(key[j] & 1023u);
            l[j] = 4 * lane + j < n ? row[row_at(token[j])] : -INFINITY;
        }
        // keys of one quantum may stand in the wrong order: exchange neighbours until none do
        for (;;) {
            bool moved = false;
            auto exchange = [&](int i, int j) {
                if (l[i] < l[j] || (l[i] == l[j] && token[i] > token[j] && l[i] > -INFINITY)) {
                    const float tl = l[i];
                    const int tt = token[i];
                    l[i] = l[j];
                    token[i] = token[j];
                    l[j] = tl;
                    token[j] = tt;
                    moved = true;
                }
            };
            exchange(0, 1);
            exchange(2, 3);
            exchange(1, 2);
            const float nl = __shfl_down_sync(kFull, l[0], 1), pl = __shfl_up_sync(kFull, l[3], 1);
            const int nt = __shfl_down_sync(kFull, token[0], 1), pt = __shfl_up_sync(kFull, token[3], 1);
            if (lane < 31 && (l[3] < nl || (l[3] == nl && token[3] > nt && nl > -INFINITY))) {
                l[3] = nl;
                token[3] = nt;
                moved = true;
            }
            if (lane > 0 && (pl < l[0] || (pl == l[0] && pt > token[0] && pl > -INFINITY))) {
                l[0] = pl;
                token[0] = pt;
                moved = true;
            }
            if (!__any_sync(kFull, moved)) break;
        }
        double e[4];
        double own = 0.0;
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const int i = 4 * lane + j;
            e[j] = i < n && i < limit ? exp(((double)l[j] - (double)top) * a.inv_temp) : 0.0;
            own += e[j];
        }
        double run = warp_before(own, lane);
        bool keep[4];
#pragma unroll
        for (int j = 0; j < 4; j++) keep[j] = e[j] > 0.0 && e[j] >= (double)a.min_p;
        // min-p cuts inside the list if its last candidate is cut
        bool inside = a.min_p > 0.0f &&
                      __any_sync(kFull, (4 * lane <= n - 1 && n - 1 < 4 * lane + 4) &&
                                            [&] {
                                                bool k = true;
#pragma unroll
                                                for (int j = 0; j < 4; j++)
                                                    if (4 * lane + j == n - 1) k = keep[j];
                                                return !k;
                                            }());
        if (a.top_p < 1.0f && (covers || limit == alive)) {
            const double listed = warp_sum(own);
            double all = listed;
            if (!covers) {   // the list is the whole row: its sum
                all = 0.0;
#pragma unroll 4
                for (int i = 0; i < 32; i++)
                    all += exp(((double)row[row_at(4 * (lane + 32 * (i >> 2)) + (i & 3))] - (double)top) *
                               a.inv_temp);
                all = warp_sum(all);
            }
            const double cut = (double)a.top_p * all;
#pragma unroll
            for (int j = 0; j < 4; j++) {
                if (!(4 * lane + j == 0 || run < cut)) keep[j] = false;
                run += e[j];
            }
            inside = inside || listed >= cut;
        } else if (a.top_p < 1.0f) {
            inside = false;   // a top-k list longer than the candidates: its sum is not known
        }
        closed = covers || inside;
        if (closed) {
            double kept = 0.0;
#pragma unroll
            for (int j = 0; j < 4; j++) kept += keep[j] ? e[j] : 0.0;
            const double sum = warp_sum(kept);
            double et = 0.0;
#pragma unroll
            for (int j = 0; j < 4; j++)
                if (keep[j] && token[j] == r.t) et = e[j];
            et = warp_sum(et);   // one lane's, or none
            *taken = stands(r, V, et, sum);
            if (*taken) return r.t;
            double w[4], total = 0.0;
            if (drafted) {
                own = 0.0;
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    w[j] = keep[j] ? weight(r, e[j], sum, token[j]) : 0.0;
                    own += w[j];
                }
                total = warp_sum(own);
            }
            if (!(total > 0.0)) {   // after the last draft, or no weight is left: p
                own = kept;
                total = sum;
#pragma unroll
                for (int j = 0; j < 4; j++) w[j] = keep[j] ? e[j] : 0.0;
            }
            run = warp_before(own, lane);
            const double goal = r.u1 * total;
            int first = kCand, last = -1;
#pragma unroll
            for (int j = 0; j < 4; j++) {
                run += w[j];
                if (w[j] > 0.0) {
                    last = 4 * lane + j;
                    if (first == kCand && run >= goal) first = 4 * lane + j;
                }
            }
            first = __reduce_min_sync(kFull, first);
            last = __reduce_max_sync(kFull, last);
            const int i = first < kCand ? first : last;
            const int hit = (i & 3) == 0 ? token[0] : (i & 3) == 1 ? token[1] : (i & 3) == 2 ? token[2] : token[3];
            return __shfl_sync(kFull, hit, i >> 2);
        }
    }
    __syncwarp();
    return general_row(a, r, row, tok, top, limit, taken);
}

template <int kMaxWarps, int kMinCtas>
__global__ void __launch_bounds__(32 * kMaxWarps, kMinCtas) verify_kernel(const __grid_constant__ VerifyArgs a)
{
    extern __shared__ __align__(16) unsigned char smem[];
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const int c = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const long long s = blockIdx.x;
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
    int d = 0;
    for (;; d++) {
        int flag = 0;
        bool taken = false;
        const int code = verify_row(a, s, d, c, pos, d < drafted, mem, &flag, &taken);
        if (lane == 0) {
            codes[(long long)d * C] = code;
            if (flags) flags[(long long)d * C] = flag;
        }
        // a frame with a refused code (the frame after the drafts counts as one) is the last
        if (__syncthreads_or(!taken)) break;
    }
    for (int k = d + 1 + lane; k <= D; k += 32) {
        codes[(long long)k * C] = -1;
        if (flags) flags[(long long)k * C] = 0;
    }
    if (H > 0)   // append the emitted frames: the ring's last H of them
        for (int k = (d >= H ? d - H + 1 : 0) + lane; k <= d; k += 32)
            ring[((long long)pos + k) % H] = codes[(long long)k * C];
    if (threadIdx.x == 0) {
        a.n_accepted[s] = d;
        if (H > 0) a.hist_pos[s] = (int)(((long long)pos + d + 1) % H);
    }
}

template <class Kernel>
cudaError_t launch(Kernel kernel, const VerifyArgs &a, cudaStream_t stream)
{
    const int smem = a.n_cb * kWarpBytes;
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)a.n_streams);
    cfg.blockDim = dim3(32u * (unsigned)a.n_cb);
    cfg.dynamicSmemBytes = (size_t)smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kernel, a);
}

}  // namespace

cudaError_t launch_verify(const VerifyArgs &a, cudaStream_t stream)
{
    if (a.n_streams == 0) return cudaSuccess;
    return a.n_cb <= 9 ? launch(verify_kernel<9, 3>, a, stream)
                       : launch(verify_kernel<kSamplerCbMax, 1>, a, stream);
}

}  // namespace z2
