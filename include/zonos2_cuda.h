/*
 * zonos2_cuda.h -- C ABI of the B200 (sm_100a) per-decode-step output path of
 * zonos2.cpp: the 9-codebook output head (hidden 2048 -> 9 x 1024 logits), the
 * tanh softcap 15*tanh(x/15) and the sampler (repetition penalty, temperature,
 * top-k / top-p / min-p, token masks, seeded categorical draw).
 *
 * Conventions
 *   - Every entry point returns int: >= 0 on success (a token id where the
 *     reference returned one), a negative ZONOS2CU_E* code on failure.  No C++
 *     exception crosses this boundary.
 *   - "_dev" pointers are CUDA device pointers owned by the caller; calls that
 *     take them are asynchronous and ordered on the cudaStream_t passed as
 *     `stream` (NULL = the legacy default stream).  "_host" pointers are host
 *     memory; those calls copy in and out and return when the result is on the
 *     host.
 *   - Device memory is allocated only by these calls:
 *       zonos2cu_ctx_create, zonos2cu_set_head, zonos2cu_set_allow,
 *       zonos2cu_set_out_norm, zonos2cu_set_adapters, zonos2cu_set_cfg
 *       (with adapters), zonos2cu_set_embeddings, zonos2cu_gen_begin
 *         (owned by the context, freed by zonos2cu_ctx_destroy);
 *       the first zonos2cu_ctx_sample_host / zonos2cu_ctx_step_host of a
 *         context, and a later one with larger inputs (host-path staging,
 *         owned by the context);
 *       the first zonos2cu_sample_token on a device (a small per-device
 *         staging area, device and page-locked host memory, kept until exit);
 *       zonos2cu_comm_create and zonos2cu_comm_create_timeout (NCCL's own
 *         buffers, freed by zonos2cu_comm_destroy or zonos2cu_comm_abort);
 *       zonos2cu_ipc_alloc (freed by zonos2cu_ipc_free).
 *     Every other entry point, zonos2cu_step_noalloc included, allocates
 *     nothing.
 *   - Host buffers given to the "_host" calls are copied with
 *     cudaMemcpyAsync: page-locked memory (cudaHostAlloc, or
 *     cudaHostRegister on an existing buffer) copies at full PCIe speed,
 *     pageable memory (a plain std::vector) through a bounce buffer.
 *   - A context belongs to one device and is not thread-safe; use one per
 *     (device, host thread).
 *
 * Reference interfaces replaced (paths relative to the zonos2.cpp tree):
 *   sample_token(Xoshiro256&, const float*, int, float, int, float, float)
 *                                         src/zonos2_generate.cpp:36-93
 *   Xoshiro256 seeding / next / randf     src/zonos2_generate.cpp:11-33
 *   head: linear_forward(multi_output)    src/zonos2_model.cpp:200-216, :687-690
 *   softcap + [n_tok, 9, audio_vocab]     src/zonos2_model.cpp:692-703
 *   the per-step sampling loop            src/zonos2_generate.cpp:259-267
 */
#ifndef ZONOS2_CUDA_H
#define ZONOS2_CUDA_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* ---- status codes --------------------------------------------------------- */
#define ZONOS2CU_OK 0
#define ZONOS2CU_EINVAL (-1)       /* an argument is out of range or NULL          */
#define ZONOS2CU_ECUDA (-2)        /* a CUDA runtime / driver call failed          */
#define ZONOS2CU_ENOMEM (-3)       /* a device allocation failed                   */
#define ZONOS2CU_ESTATE (-4)       /* context not ready (e.g. no head weights set) */
#define ZONOS2CU_EUNSUPPORTED (-5) /* shape outside what the kernels implement     */
#define ZONOS2CU_EDEVICE (-6)      /* a kernel reported a bounded wait that expired */
#define ZONOS2CU_ETOOBIG (-7)      /* larger than zonos2cu_step_noalloc's fixed scratch */
#define ZONOS2CU_ENCCL (-8)        /* NCCL is missing or an NCCL call failed        */

/* ---- per-row flags written next to each sampled code ---------------------- */
#define ZONOS2CU_FLAG_ALL_MASKED 1 /* no logit >= -1e9 survived: code = pad_id     */
#define ZONOS2CU_FLAG_NONFINITE 2  /* a NaN / +inf logit was treated as masked     */

typedef enum { ZONOS2CU_F32 = 0, ZONOS2CU_BF16 = 1 } zonos2cu_dtype;

/* Sampler knobs.  Meaning and defaults follow Zonos2GenParams
 * (src/zonos2.h:244-254).  repetition_penalty is build-defined (the reference
 * declares it but never reads it): every distinct token of the row's history
 * window is scaled once, l > 0 ? l * RN(1/rho) : l * rho; 1.0 disables it.
 * pad_id is the code forced by the delay-pattern mask and returned for
 * all-masked rows. */
typedef struct {
    float temperature; /* > 0                                    default 0.7  */
    int top_k;         /* <= 0 or >= vocab: off                  default 50   */
    float top_p;       /* >= 1: off                              default 0.9  */
    float min_p;       /* in [0, 1]; 0: off                      default 0.02 */
    float repetition_penalty; /* > 0; 1: off                     default 1.0  */
    int pad_id;        /* in [0, vocab)                          default 1023 */
} zonos2cu_sample_params;

/* Fills *p with the defaults above. */
void zonos2cu_default_params(zonos2cu_sample_params *p);

/* Library version string and the last CUDA error text seen on this thread. */
const char *zonos2cu_version(void);
const char *zonos2cu_last_error(void);

/* ---- generator ------------------------------------------------------------ */

/* Xoshiro256** seeded as the reference does (src/zonos2_generate.cpp:13-19):
 * state[i] = seed ^ K_i, then 20 discarded outputs.  Host-side helper. */
void zonos2cu_rng_seed(uint64_t seed, uint64_t state[4]);

/* ---- the drop-in for sample_token (src/zonos2_generate.cpp:36-37) --------- */

/* Same arguments and result as the reference's
 *   static int sample_token(Xoshiro256& rng, const float* logits,
 *                           int vocab_size, float temp, int top_k,
 *                           float top_p, float min_p);
 * rng_state are the generator's four state words (host memory), advanced by
 * exactly one draw; logits are vocab_size host floats (1 <= vocab_size <=
 * 1024).  The uniform is drawn on the host, as the reference draws it; the
 * row is sampled on the current CUDA device (one copy in, one launch, one copy
 * out).  Equal probabilities are taken in ascending token order.  Returns the
 * token id, or a negative ZONOS2CU_E* code (temp <= 0, NaN knobs, min_p > 1,
 * or an all-masked row -- the cases where the reference is undefined; the
 * generator is left unadvanced when the arguments are rejected). */
int zonos2cu_sample_token(uint64_t rng_state[4], const float *logits, int vocab_size,
                          float temp, int top_k, float top_p, float min_p);

/* ---- stateless batched sampler (device pointers) -------------------------- */

/* One decode step over n_streams x n_cb rows.  Row (s, c) is
 * logits_dev[(s*n_cb + c) * row_stride .. + vocab) (row_stride >= vocab; the
 * reference's [n_tok, 9, 1026] layout is row_stride = 1026).
 *   rng_dev      [n_streams][4] u64, 16-byte aligned: stream s draws one
 *                uniform per codebook,
 *                in codebook order (the reference's order at
 *                src/zonos2_generate.cpp:259-267), and is advanced by n_cb.
 *   hist_dev     [n_streams][n_cb][hist_len] i32 ring (may be NULL when
 *                hist_len == 0): read for the repetition penalty, then the
 *                sampled code is written at hist_pos.  Entries outside
 *                [0, vocab) are ignored (use -1 for empty slots).
 *   allow_dev    [n_streams][ceil(vocab/32)] u32 or NULL: bit t of stream s
 *                clear masks token t for all its codebooks.
 *   delay_step   >= 0: codebook c with delay_step < c may only emit pad_id
 *                (the delay pattern); < 0: off.
 *   codes_dev    [n_streams][n_cb] i32 output; flags_dev the same or NULL.
 * Limits: 1 <= vocab <= 1024, 1 <= n_cb <= 16. */
int zonos2cu_sample_rows(const float *logits_dev, int n_streams, int n_cb, int vocab,
                         long long row_stride, const zonos2cu_sample_params *params,
                         uint64_t *rng_dev, int32_t *hist_dev, int hist_len, int hist_pos,
                         const uint32_t *allow_dev, int delay_step, int32_t *codes_dev,
                         int32_t *flags_dev, void *stream);

/* ---- stateless output head + softcap (device pointers) -------------------- */

/* logits_dev[b][c][v] = softcap * tanh(dot(hidden[b], W[c*rows_per_cb + v]) / softcap)
 * for b < batch, c < n_cb, v < vocab (softcap <= 0: no cap).  W_dev is the
 * head weight [n_cb*rows_per_cb][dim] row-major -- the reference's
 * multi_output / output.bin layout is rows_per_cb = 1026, vocab = 1024
 * (src/zonos2_loader.cpp:133-136) -- and hidden_dev is [batch][dim], both of
 * `dtype`.  F32 runs an f32-exact GEMV (f64 accumulation); BF16 runs the
 * tcgen05 tensor-core GEMM (f32 accumulation in TMEM) and needs
 * dim % 64 == 0, vocab % 64 == 0 and 16-byte aligned rows. */
int zonos2cu_head_softcap(const void *W_dev, zonos2cu_dtype dtype, int rows_per_cb, int n_cb,
                          int vocab, int dim, const void *hidden_dev, int batch, float softcap,
                          float *logits_dev, void *stream);

/* ---- the output head beside low-rank adapters (device pointers) ------------- */

/* zonos2cu_head_softcap with an adapter per hidden row (no counterpart in the
 * reference): with a = adapter_dev[b],
 *   logits[b][c][v] = softcap * tanh((W[n] . h + scale[a] * B[a][n] . (A[a] h)) / softcap)
 * where n = c*rows_per_cb + v and h = hidden_dev[b]; rows whose a lies outside
 * [0, n_adapters) have no adapter.  Rows may name their adapters in any order.
 *   A_dev        [n_adapters][rank][dim], B_dev [n_adapters][n_cb*rows_per_cb][rank],
 *                of `dtype` like W_dev and hidden_dev.
 *   scale_dev    [n_adapters] f32 or NULL (1).
 *   adapter_dev  [batch] i32.
 *   work_dev     work_bytes of scratch, 16-byte aligned, at least
 *                zonos2cu_head_adapters_work(dtype, batch, rank) (8 bytes per row and
 *                rank always suffice).  Calls that may overlap need scratch of their own.
 * A h is kept in f32 beside a bf16 head and in f64 beside an f32 one, whose result
 * is rounded once (its products are summed by fours in f32 before).  Any dim, vocab
 * and rank (<= ZONOS2CU_MAX_RANK); the bf16 tensor-core kernels run where dim % 8 ==
 * 0, rank % 8 == 0, n_adapters <= 4096 and W, hidden, A and B are 16-byte aligned.
 * Elsewhere, and for f32, a kernel runs that reads W again for every four hidden rows:
 * meant for a few rows, its time grows with their number.  A product past the range of f32 is
 * infinite, and its logit the end of the softcap. */
#define ZONOS2CU_MAX_RANK 256
long long zonos2cu_head_adapters_work(zonos2cu_dtype dtype, int batch, int rank);
int zonos2cu_head_adapters(const void *W_dev, zonos2cu_dtype dtype, int rows_per_cb, int n_cb,
                           int vocab, int dim, const void *hidden_dev, int batch, float softcap,
                           const void *A_dev, const void *B_dev, const float *scale_dev,
                           int n_adapters, int rank, const int32_t *adapter_dev, void *work_dev,
                           long long work_bytes, float *logits_dev, void *stream);

/* ---- the tail of a decoder block (device pointers) ------------------------- */

/* The norm of a block's output, its gate, the scaled residual sum, and the
 * RMSNorm that follows (the next block's, or the output norm ahead of the head),
 * in one pass over each row:
 *     y = block * post_weight / rms(block)    (post_eps >= 0; y = block below 0)
 *     r = resid + scale * g * y
 *     n = r * norm_weight / rms(r),           rms(x) = sqrt(mean(x^2) + eps)
 * in f32, r and n rounded once each to `dtype` (n from the unrounded r).
 *   resid_dev, block_dev  [rows] rows of dim elements of `dtype`, their starts
 *                resid_stride and block_stride elements apart (>= dim).
 *   gate_dev     NULL (g = 1), or the value of row r, column d at element
 *                r * gate_row_stride + d * gate_col_stride: (stride, 1) one per
 *                element, (stride, 0) one per row, (0, 1) one per column.  With
 *                gate_sigmoid g = 1 / (1 + exp(-gate)), else the value itself.
 *   post_weight_dev, norm_weight_dev  [dim] f32, or NULL for 1.
 *   resid_out_dev (r), normed_out_dev (n)  rows out_stride elements apart; one of
 *                them may be NULL.  Either may be resid_dev or block_dev itself, at
 *                the same row stride (out_stride); no other overlap is allowed.
 * Replaces, for a block with these parts, the residual sum and the
 * rms_norm_per_token behind it (src/zonos2_model.cpp:19-35, :684-685). */
int zonos2cu_block_norm(const void *resid_dev, const void *block_dev, zonos2cu_dtype dtype,
                        int rows, int dim, long long resid_stride, long long block_stride,
                        const float *post_weight_dev, float post_eps, const void *gate_dev,
                        long long gate_row_stride, int gate_col_stride, int gate_sigmoid,
                        float scale, const float *norm_weight_dev, float norm_eps,
                        void *resid_out_dev, void *normed_out_dev, long long out_stride,
                        void *stream);

/* ---- the output head in 8-bit integers (device pointers) ------------------- */

/* Rows of x (bf16 or f32, their starts x_stride elements apart) rounded to 8 bits with a
 * scale each (no counterpart in the reference):
 *     scale[r] = max_k |x[r][k]| / 127,   q[r][k] = x[r][k] * 127 / max_k |x[r][k]|,
 * q rounded once to the nearest integer, ties to even, so that |q| <= 127.  Rows have fewer
 * than 2^30 elements (ZONOS2CU_EUNSUPPORTED elsewhere).  A row of
 * zeros has scale 0; a row that holds a NaN or an infinity has q = 0 and scale NaN.
 *   q_dev        [rows][dim] i8; scale_dev [rows] f32.
 * For the weights of zonos2cu_head_i8 once, at set-up. */
int zonos2cu_quantize_rows(const void *x_dev, zonos2cu_dtype dtype, int rows, int dim,
                           long long x_stride, int8_t *q_dev, float *scale_dev, void *stream);

/* zonos2cu_head_softcap with 8-bit weights and hidden rows rounded to 8 bits on the way, as
 * zonos2cu_quantize_rows rounds them:
 *   logits[b][c][v] = softcap * tanh(scale_b * w_scale[n] * (q_b . W[n]) / softcap)
 * with n = c*rows_per_cb + v (softcap <= 0: no cap).  The products are summed exactly, in
 * 32-bit integers; the rest is f32.  A hidden row that holds a NaN or an infinity has NaN
 * logits.  With n_cb = 1 and no cap this is a plain product of 8-bit integers with a scale
 * per row of either side.
 *   W_dev        [n_cb*rows_per_cb][dim] i8, 16-byte aligned; w_scale_dev
 *                [n_cb*rows_per_cb] f32.
 *   hidden_dev   [batch][dim] of `dtype`, logits_dev [batch][n_cb][vocab].
 *   work_dev     work_bytes of scratch, 16-byte aligned, at least
 *                zonos2cu_head_i8_work(batch, dim).  Calls that may overlap need scratch of
 *                their own.
 * dim must be a multiple of 16, and batch and n_cb * rows_per_cb lie below 2^30
 * (ZONOS2CU_EUNSUPPORTED elsewhere); dim is at most ZONOS2CU_MAX_I8_DIM (no sum of products then passes 32 bits). */
#define ZONOS2CU_MAX_I8_DIM 131072
long long zonos2cu_head_i8_work(int batch, int dim);
int zonos2cu_head_i8(const int8_t *W_dev, const float *w_scale_dev, int rows_per_cb, int n_cb,
                     int vocab, int dim, const void *hidden_dev, zonos2cu_dtype dtype, int batch,
                     float softcap, void *work_dev, long long work_bytes, float *logits_dev,
                     void *stream);

/* ---- a paged cache of keys and values (device pointers) -------------------- */

/* The attention state of n_streams decode streams, for the decoder blocks ahead of the
 * head: pages of page_size tokens, and per stream a table of the pages its tokens lie on
 * (replaces, for a batch, the flat cache of src/zonos2_generate.cpp:115-126).  Token j of
 * stream s lies on page table[s][j / page_size] at slot j % page_size.
 *   k_dev, v_dev  pages of `dtype`, page p at element p * page_stride, and in it
 *                [n_kv_heads][page_size][head_dim] (page_stride >= their product: keys
 *                and values may share one buffer, page by page).
 *   table_dev     [n_streams][max_pages] i32.  An entry outside [0, n_pages) is no page:
 *                nothing is written there, and its tokens are not attended (entries
 *                behind a stream's last token have no effect; pages that a window has left
 *                behind may be given back and marked -1).
 *   kv_len_dev    [n_streams] i32, the stream's tokens, the new ones of the call among
 *                them (tokens past max_pages * page_size are nowhere).
 *   q_start_dev   [n_streams + 1] i32, rising: rows [q_start[s], q_start[s+1]) of the
 *                call's token rows are the last tokens of stream s, row i of its n at
 *                position kv_len[s] - n + i.  A stream may have none.  Rows outside
 *                [q_start[0], q_start[n_streams]) are not read and stay as they are.
 * k_dev and v_dev are 16-byte aligned, head_dim is a multiple of 8 up to
 * ZONOS2CU_MAX_HEAD_DIM, page_size a power of two from 8 to ZONOS2CU_MAX_PAGE, page_stride a
 * multiple of 8, n_kv_heads at most 4096 and n_heads 65535; of a stream the first 2^31 - 256
 * tokens count, and n_streams and rows times query heads per key head stay below 2^30 (ZONOS2CU_EUNSUPPORTED elsewhere). */
#define ZONOS2CU_MAX_HEAD_DIM 256
#define ZONOS2CU_MAX_PAGE 4096
typedef struct {
    void *k_dev, *v_dev;
    zonos2cu_dtype dtype;
    int n_pages, page_size, n_kv_heads, head_dim;
    long long page_stride;
    const int32_t *table_dev;
    int n_streams, max_pages;
    const int32_t *kv_len_dev;
    const int32_t *q_start_dev;
} zonos2cu_cache;

/* The new tokens' queries and keys normalised and rotated, their keys and values written to
 * the pages (the QK-norm, rotation and cache write of the attention, src/zonos2_model.cpp:221, for a batch).
 * Per token at position p and per head:
 *     x' = x * weight / sqrt(mean(x^2) + eps)      (eps >= 0; x' = x below 0)
 *     (a, b) -> (a cos(p f) - b sin(p f), b cos(p f) + a sin(p f))
 * for the rot_dim / 2 pairs of the head's first rot_dim elements: neighbours
 * (2i, 2i + 1), or with rot_halves (i, i + rot_dim / 2); f = freq[i].  In f32 (the angle
 * in f64), rounded once to the cache's type.  Values are copied.
 *   q_dev, k_dev, v_dev  [rows] token rows of n_heads, n_kv_heads and n_kv_heads heads
 *                of head_dim elements, of the cache's type, their starts q_stride,
 *                k_stride and v_stride elements apart.  q_dev may be NULL (keys and
 *                values alone).
 *   q_weight_dev, k_weight_dev  [head_dim] f32 or NULL (1).
 *   freq_dev     [rot_dim / 2] f32, radians per position.  rot_dim = 0: no rotation.
 *   q_out_dev    as q_dev, at q_out_stride; may be q_dev itself at the same stride.
 * Rows are 16-byte aligned (ZONOS2CU_EUNSUPPORTED elsewhere).  No two streams' new tokens
 * may lie on one page's slot.  No other overlap of buffers is allowed. */
int zonos2cu_cache_append(const zonos2cu_cache *cache, int rows, int n_heads, const void *q_dev,
                          long long q_stride, const void *k_dev, long long k_stride,
                          const void *v_dev, long long v_stride, const float *q_weight_dev,
                          const float *k_weight_dev, float eps, const float *freq_dev, int rot_dim,
                          int rot_halves, void *q_out_dev, long long q_out_stride, void *stream);

/* Attention of the new tokens over the pages, after zonos2cu_cache_append on the same stream
 * (the attention's scores, softmax, values and head gate, src/zonos2_model.cpp:221, for a batch).
 * Query head h of a token at position p, with key head h / (n_heads / n_kv_heads):
 *     o = g * sum_j softmax_j(scale * q . k_j) v_j
 * over the stream's tokens j <= p (j > p - window with 0 < window < 2^30) that lie on a
 * page; zero where there is none, whatever the gate.  What lies elsewhere, a NaN among it, has no part
 * in it.  An infinite value that the row sees makes its element infinite, or a NaN (as 0 times it) where its weight or the gate
 * is zero in f32.
 * g = 1 / (1 + exp(-gate)) (1 without gates).  Scores, sums and softmax are f32.  With a
 * bf16 cache the softmax's weights are rounded to bf16 before they meet the values (each
 * is at most 1 beside the row's largest; their sum is taken unrounded): for normal values the error is then 2.0e-3 to 2.3e-3 in
 * the 2-norm, 1.7e-3 of it the result's own rounding.  With an f32 cache and more than 16 rows (tokens times query heads of a key
 * head) products are taken in three parts of 11 bits, to 2^-20 of each: 9e-7 in the 2-norm, 5.7e-7 in f32 throughout.
 *   q_dev, out_dev  [rows] token rows of n_heads heads of head_dim elements of the cache's
 *                type, q_stride and out_stride elements apart, 16-byte aligned
 *                (ZONOS2CU_EUNSUPPORTED elsewhere).  out_dev must not overlap the others.
 *   gate_dev     NULL, or the gate of row r, head h at r * gate_stride + h.
 *   max_new      the most new tokens that a stream has, as far as the caller knows (0:
 *                not at all).  It chooses between kernels; chunks longer than it says are
 *                still attended.
 * n_heads is a multiple of n_kv_heads; scale is positive, and finite also times log2(e).  The sum of the values'
 * sizes, times 256, must lie within f32.  Sums are taken in an
 * order that the sizes alone give. */
int zonos2cu_cache_attend(const zonos2cu_cache *cache, int rows, int n_heads, const void *q_dev,
                          long long q_stride, float scale, int window, const void *gate_dev,
                          long long gate_stride, int max_new, void *out_dev, long long out_stride,
                          void *stream);

/* ---- drafted frames against the target (device pointers) -------------------- */

/* No counterpart in the reference.  A stream has up to n_draft drafted frames of
 * n_cb codes, and the target's logits at each of their positions and at the one
 * after them: row (s, d, c) is logits_dev[((s*(n_draft+1) + d)*n_cb + c) *
 * row_stride .. + vocab), the head's output for n_streams * (n_draft + 1) hidden
 * rows.  Per row, p is the distribution zonos2cu_sample_rows draws from (penalty,
 * masks, temperature, top-k, top-p, min-p, in that order; tokens ordered by logit
 * descending, then token ascending) and q the draft's.  With the row's uniforms
 * u0, u1 in [0, 1):
 *   - the drafted code t stands iff u0 * q(t) < p(t) (never outside [0, vocab));
 *   - a refused code is drawn from max(p - q, 0), or from p where that is zero
 *     everywhere: the first token in the order above that has weight and whose
 *     cumulative weight reaches u1 of the total;
 *   - a stream's first frame with a refused code is its last emitted one; if all
 *     its drafts stand, the frame after them is drawn from p and is the last.
 * The emitted frames then have the distribution the sampler would have given them
 * one at a time.  Decisions are made in f64.
 *   drafts_dev   [n_streams][n_draft][n_cb].
 *   draft_probs_dev  q, [n_streams][n_draft][n_cb][vocab] f32, or NULL: the drafts
 *                are certain (q(t) = 1; looked up rather than drawn).  A NaN in q
 *                refuses the code it belongs to and gives it no weight.
 *   n_drafts_dev [n_streams] how many of the n_draft frames each stream has
 *                (clamped to [0, n_draft]), or NULL: all of them.
 *   uniforms_dev [n_streams][n_draft + 1][n_cb][2]: u0, u1 (u0 of the position
 *                after the drafts is not used).
 *   hist_dev     [n_streams][n_cb][hist_len] ring (may be NULL when hist_len == 0)
 *                and hist_pos_dev [n_streams], each stream's next write position
 *                (taken mod hist_len).  Position d's penalty sees the ring with
 *                the d frames drafted before it appended; the emitted frames are
 *                appended and hist_pos_dev advanced by their number, mod hist_len.
 *   allow_dev, delay_step  as in zonos2cu_sample_rows; position d counts as
 *                delay step delay_step + d.
 *   codes_dev    [n_streams][n_draft + 1][n_cb]: the emitted frames, -1 after them.
 *   n_accepted_dev  [n_streams]: drafted frames that stand whole; n_accepted + 1
 *                frames are emitted.
 *   flags_dev    as codes_dev or NULL: ZONOS2CU_FLAG_* of each emitted code, 0 after.
 * No two of the buffers may overlap.
 * Limits: 1 <= vocab <= 1024, 1 <= n_cb <= 16, n_draft <= ZONOS2CU_MAX_DRAFTS. */
#define ZONOS2CU_MAX_DRAFTS 4095
int zonos2cu_verify_drafts(const float *logits_dev, int n_streams, int n_draft, int n_cb,
                           int vocab, long long row_stride, const zonos2cu_sample_params *params,
                           const int32_t *drafts_dev, const float *draft_probs_dev,
                           const int32_t *n_drafts_dev, const float *uniforms_dev,
                           int32_t *hist_dev, int hist_len, int32_t *hist_pos_dev,
                           const uint32_t *allow_dev, int delay_step, int32_t *codes_dev,
                           int32_t *n_accepted_dev, int32_t *flags_dev, void *stream);

/* ---- context: device-resident state for a batch of decode streams --------- */

typedef struct zonos2cu_ctx zonos2cu_ctx;

typedef struct {
    int n_streams;   /* decode streams held by this context (this device's shard) */
    int n_cb;        /* codebooks per frame: 9                                     */
    int vocab;       /* sampled tokens per codebook: 1024                          */
    int dim;         /* hidden size for the fused head: 2048 (0: sampler only)     */
    int hist_len;    /* repetition-history window per row (0: none; <= 65535)      */
    uint64_t seed;   /* stream s uses Xoshiro256(seed + first_stream + s)          */
    uint64_t first_stream; /* global index of this shard's first stream           */
} zonos2cu_dims;

int zonos2cu_ctx_create(int device, const zonos2cu_dims *dims, zonos2cu_ctx **out);
int zonos2cu_ctx_destroy(zonos2cu_ctx *ctx);

/* The setters and getters below synchronise the device: they are set-up calls,
 * safe against steps enqueued on any stream, not per-step calls. */

/* Head weights from host memory, [n_cb*rows_per_cb][dim] of dtype
 * (rows_per_cb = 1026 for the reference's output.bin; only the first vocab
 * rows of each codebook are kept on the device).  After a call that fails past
 * its argument checks steps return ZONOS2CU_ESTATE. */
int zonos2cu_set_head(zonos2cu_ctx *ctx, const void *W_host, zonos2cu_dtype dtype,
                      int rows_per_cb);
/* History ring [n_streams][n_cb][hist_len] and its write position.  The
 * context also keeps, per row, how often each token occurs in the ring and a
 * bitmap of the tokens present, updated by every step for the token it evicts
 * and the one it appends: the penalty reads 128 bytes per row instead of the
 * whole ring. */
int zonos2cu_set_history(zonos2cu_ctx *ctx, const int32_t *hist_host, int hist_pos);
int zonos2cu_get_history(zonos2cu_ctx *ctx, int32_t *hist_host, int *hist_pos);
/* Generator states [n_streams][4]. */
int zonos2cu_set_rng(zonos2cu_ctx *ctx, const uint64_t *state_host);
int zonos2cu_get_rng(zonos2cu_ctx *ctx, uint64_t *state_host);
/* Allow bitmask [n_streams][ceil(vocab/32)]; NULL clears it. */
int zonos2cu_set_allow(zonos2cu_ctx *ctx, const uint32_t *bits_host);

/* The output RMSNorm ahead of the head in zonos2cu_ctx_step: replaces
 * rms_norm_per_token(x, dim, n, eps, out_norm.weight) applied to the last hidden
 * states before the multi_output head (src/zonos2_model.cpp:684-685, :19-35).
 * With it enabled, ctx_step takes the un-normalised hidden states.  weight_host
 * is [dim] f32, or NULL for no scale weight; enable = 0 turns it off.  With an
 * f32 head the norm is the reference's, exactly; with a bf16 head it is folded
 * into the head (the weight into W's columns, rounded to bf16 once; each row's
 * 1 / rms into the GEMM's epilogue), within the bf16 path's tolerance.  Where that
 * folding fails, here or in zonos2cu_set_head, ctx_step returns ZONOS2CU_ESTATE
 * until the norm is set again or turned off. */
int zonos2cu_set_out_norm(zonos2cu_ctx *ctx, int enable, const float *weight_host, float eps);
/* Classifier-free guidance in zonos2cu_ctx_step: the blend
 * uncond + scale * (cond - uncond) of softcapped logits that the reference
 * applies to its prefill logits (src/zonos2_generate.cpp:157-183), here on every
 * step.  With it enabled, ctx_step and ctx_step_host take [2*n_streams][dim]
 * hidden states, row 2s the conditional and row 2s+1 the unconditional state
 * of stream s; logits and codes stay [n_streams][...].  enable = 0 turns it off. */
int zonos2cu_set_cfg(zonos2cu_ctx *ctx, int enable, float scale);

/* Low-rank adapters beside the head in zonos2cu_ctx_step, as in
 * zonos2cu_head_adapters: A [n_adapters][rank][dim], B [n_adapters][n_cb*rows_per_cb]
 * [rank] (the first vocab rows of each codebook are kept) and scale [n_adapters] f32
 * (NULL: 1) from host memory, `dtype` the head's (a step with another head type
 * returns ZONOS2CU_ESTATE).  Every stream starts without one;
 * zonos2cu_set_stream_adapters gives each stream its adapter (-1: none; NULL: none
 * anywhere).  With guidance on, both rows of a stream use it; with the output norm's
 * weight folded into a bf16 head it is folded into A as well.  n_adapters = 0 removes
 * them, and so does a call that fails past its argument checks (head, norm and
 * guidance stay as they were).  While adapters are set, streams without one take the
 * adapters' kernels as well: slower than the plain head's, and with its own roundings
 * (an f32 head's products are summed by fours in f32), so that their logits may differ
 * in the last bits.  A captured step holds the adapters' buffers: capture it again after
 * this call (after zonos2cu_set_stream_adapters it reads the new ids). */
int zonos2cu_set_adapters(zonos2cu_ctx *ctx, const void *A_host, const void *B_host,
                          const float *scale_host, int n_adapters, int rank,
                          zonos2cu_dtype dtype, int rows_per_cb);
int zonos2cu_set_stream_adapters(zonos2cu_ctx *ctx, const int32_t *ids_host);

/* One sampling step from device logits [n_streams][n_cb][row_stride] on
 * `stream` (NULL = the legacy default stream, like every "_dev" call); the
 * history position advances by one (mod hist_len) on success.  The host-path
 * calls below run on the context's own stream (zonos2cu_ctx_stream): work a
 * caller enqueues on other streams is not ordered with them, so synchronise
 * between the two kinds of call.  Each step reads what the step before it wrote
 * (generator states, history, the uniforms drawn ahead): a context's steps go on
 * one stream, or on streams the caller orders with events. */
int zonos2cu_ctx_sample(zonos2cu_ctx *ctx, const float *logits_dev, long long row_stride,
                        const zonos2cu_sample_params *params, int delay_step,
                        int32_t *codes_dev, int32_t *flags_dev, void *stream);
/* The same from host logits [n_streams][n_cb][row_stride] to host codes/flags
 * (flags may be NULL): copies in, samples, copies out, returns when done. */
int zonos2cu_ctx_sample_host(zonos2cu_ctx *ctx, const float *logits_host, long long row_stride,
                             const zonos2cu_sample_params *params, int delay_step,
                             int32_t *codes_host, int32_t *flags_host);
/* One fused step: hidden [n_streams][dim] (device, dtype; [2*n_streams][dim] with
 * guidance on) -> output RMSNorm if set -> head + softcap -> guidance blend if
 * set -> sampler.  logits_out_dev ([n_streams][n_cb][vocab] f32) may be NULL. */
int zonos2cu_ctx_step(zonos2cu_ctx *ctx, const void *hidden_dev, zonos2cu_dtype dtype,
                      const zonos2cu_sample_params *params, int delay_step, int32_t *codes_dev,
                      int32_t *flags_dev, float *logits_out_dev, void *stream);
/* The same from host hidden states to host codes. */
int zonos2cu_ctx_step_host(zonos2cu_ctx *ctx, const void *hidden_host, zonos2cu_dtype dtype,
                           const zonos2cu_sample_params *params, int delay_step,
                           int32_t *codes_host, int32_t *flags_host);
/* The context's CUDA stream (cudaStream_t), for callers that order work on it. */
void *zonos2cu_ctx_stream(zonos2cu_ctx *ctx);

/* ---- the generation loop around the step ------------------------------------
 * Replaces the frame bookkeeping of zonos2_generate's loop
 * (src/zonos2_generate.cpp:203-279) for a batch: between zonos2cu_gen_begin and
 * zonos2cu_gen_end, every zonos2cu_ctx_sample / zonos2cu_ctx_step (and their
 * host variants) also keeps the step's frame on the device, on the step's
 * stream: codes clamped to vocab - 1 (:214, :264), the stream ended after the
 * first frame holding eoa_id (:218-224, :269-276; that frame is kept), at most
 * max_frames frames per stream, and the next step's input frame (the codes,
 * then text_pad_id; :238-243).  With the reference's constants (1024 sampled
 * tokens, eoa_id 1024) no frame can hold eoa_id, so streams run to max_frames,
 * as in the reference.  gen_begin clears the state; before the first frame the
 * next input frame is audio_pad_id codes and text_pad_id. */
int zonos2cu_gen_begin(zonos2cu_ctx *ctx, int max_frames, int eoa_id, int audio_pad_id,
                       int text_pad_id);
int zonos2cu_gen_end(zonos2cu_ctx *ctx);
/* Frames [n_streams][max_frames][n_cb] (entries past a stream's count are -1),
 * frame counts [n_streams], end-of-audio frame [n_streams] (-1: none); any
 * pointer may be NULL.  Synchronises the device. */
int zonos2cu_gen_read(zonos2cu_ctx *ctx, int32_t *frames_host, int32_t *n_frames_host,
                      int32_t *eos_at_host);
/* Device pointer to the next step's input frames [n_streams][n_cb + 1] (NULL
 * before gen_begin). */
const int32_t *zonos2cu_gen_next_input(zonos2cu_ctx *ctx);
/* shear_up of every stream's frames (scripts/dac_decode.py:23-30): out_dev
 * [n_streams][max_frames][n_cb], out[s][t][j] = frames[s][t + j][j] while
 * t + j < the stream's frame count, audio_pad_id elsewhere. */
int zonos2cu_gen_shear_up(zonos2cu_ctx *ctx, int32_t *out_dev, void *stream);
/* The model's input embedding tables, f32 row-major: codebook tables
 * [n_cb][audio_vocab][dim] (Zonos2Weights::codebook_embeds) and the text table
 * [text_vocab + 1][dim] (text_embed, padding row last). */
int zonos2cu_set_embeddings(zonos2cu_ctx *ctx, const float *codebook_tables_host,
                            const float *text_table_host, int audio_vocab, int text_vocab);
/* embedding_sum (src/zonos2_model.cpp:116-151) of the next input frames into
 * out_dev [n_streams][dim] f32: the next model step's input. */
int zonos2cu_gen_embed_next(zonos2cu_ctx *ctx, float *out_dev, void *stream);
/* The same on caller buffers: ids_dev [n_frames][n_cb + 1], out_dev [n_frames][dim]. */
int zonos2cu_embed_frames(const float *codebook_tables_dev, const float *text_table_dev,
                          int n_cb, int audio_vocab, int text_vocab, int dim,
                          const int32_t *ids_dev, int n_frames, float *out_dev, void *stream);
/* Writes frames_host [n_frames][n_cb] in the reference's codes.bin format
 * (decode_dac_to_wav, src/zonos2_generate.cpp:285-306): int32 n_frames, int32
 * n_cb, then the codes frame by frame. */
int zonos2cu_write_codes_bin(const char *path, const int32_t *frames_host, int n_frames,
                             int n_cb);

/* Reads and clears the device-side error word that bounded waits set when
 * they expire (synchronises the current device).  0 = no error. */
int zonos2cu_device_error(void);

/* ---- several GPUs: batch-sharded streams, codes collected on one rank --------
 * One process per GPU.  Rank r of n owns the contiguous slice [first, first +
 * count) of the global batch that zonos2cu_shard_range gives (the first
 * n_streams % n_ranks ranks own one stream more) and creates its context with
 * that count and first_stream = first: its generators and codes then equal the
 * same streams of a one-GPU run of the whole batch.  Nothing crosses GPUs but
 * the codes, which the writer rank collects -- the frame collection of
 * src/zonos2_generate.cpp:278, for a batch.  NCCL is loaded at run time
 * (libnccl.so.2, or the copy the process already holds); without it these
 * calls return ZONOS2CU_ENCCL and the rest of the library is unaffected. */
int zonos2cu_shard_range(long long n_streams, int n_ranks, int rank, long long *first,
                         long long *count);
/* An NCCL communicator over the job's ranks (a ncclComm_t, as void *): rank 0
 * makes the id, the caller hands it to every rank out of band (MPI, a file, a
 * socket), then every rank calls zonos2cu_comm_create with it -- collectively,
 * as ncclCommInitRank is.  A caller that has its own NCCL communicator passes
 * that to zonos2cu_gather_codes instead. */
int zonos2cu_comm_unique_id(unsigned char id[128]);
int zonos2cu_comm_create(int device, int n_ranks, int rank, const unsigned char id[128],
                         void **nccl_comm_out);
/* The same communicator, set up without blocking (ncclCommInitRankConfig with
 * blocking = 0) and polled: if every rank has not joined within timeout_ms the
 * set-up is aborted (ncclCommAbort) and ZONOS2CU_ENCCL returned, so a rank that
 * died or never started cannot hang the others in set-up.  Its gathers wait at
 * most 120 s for connections and its destroy at most 60 s for the flush (then
 * aborts).  Needs NCCL >= 2.14; otherwise ZONOS2CU_ENCCL. */
int zonos2cu_comm_create_timeout(int device, int n_ranks, int rank, const unsigned char id[128],
                                 int timeout_ms, void **nccl_comm_out);
/* Flushes (a communicator from zonos2cu_comm_create_timeout, within 60 s) and
 * frees a communicator. */
int zonos2cu_comm_destroy(void *nccl_comm);
/* Frees a communicator at once, ending the operations still in flight on it
 * (ncclCommAbort): the error path when a peer rank is known to be gone. */
int zonos2cu_comm_abort(void *nccl_comm);
/* Collects n_steps steps of codes on rank `root`, called by every rank of the
 * communicator with the same root, n_steps, n_streams (the global batch) and
 * n_cb, on `stream` (asynchronous; nothing is synchronised).  codes_dev is this
 * rank's block [n_steps][count][n_cb] (e.g. a ring of per-step codes); out_dev
 * (root only; others may pass NULL) receives every rank's block in rank
 * order: rank r's at element n_steps * first_r * n_cb.  For n_steps = 1 that
 * is the global [n_streams][n_cb].  Only the root receives: the other ranks
 * send and return. */
int zonos2cu_gather_codes(void *nccl_comm, int root, const int32_t *codes_dev, int n_steps,
                          long long n_streams, int n_cb, int32_t *out_dev, void *stream);

/* The same collection by the copy engines, for a loop that must not give SMs or
 * a collective to it: the root allocates its output with zonos2cu_ipc_alloc
 * (device memory of the library's own, freed by zonos2cu_ipc_free) and hands
 * the 64-byte handle to every other rank out of band; each of those maps it
 * once with zonos2cu_ipc_open (a pointer into the root's GPU, valid in this
 * process until zonos2cu_ipc_close) and, after each block of steps, enqueues
 * zonos2cu_push_codes of its codes to their place in the root's output, on a
 * stream ordered after those steps.  The copies run on the copy engines over
 * NVLink while the SMs run the next steps; no rank waits for another in the
 * loop.  The caller orders the reuse of its source buffer after the copy (an
 * event) and, before the root reads its output, the completion of every rank's
 * copies (each rank synchronises its copy stream, then a barrier).  All on one
 * node. */
int zonos2cu_ipc_alloc(int device, long long bytes, void **dev_ptr_out, unsigned char handle[64]);
int zonos2cu_ipc_free(void *dev_ptr);
int zonos2cu_ipc_open(int device, const unsigned char handle[64], void **dev_ptr_out);
int zonos2cu_ipc_close(void *dev_ptr);
/* n_steps blocks of elems_per_step int32 codes, contiguous in codes_dev (e.g.
 * [n_steps][count][n_cb] of a ring), to dst_dev + k * dst_stride for block k
 * (e.g. rank r's place, first_r * n_cb, in the root's [n_steps][n_streams][n_cb]
 * output: dst_stride = n_streams * n_cb), one strided copy asynchronous on
 * `stream`.  Pushing a block of steps at a time keeps the step stream free of
 * per-step event waits, which would cut the programmatic overlap of one step's
 * launch with the step before. */
int zonos2cu_push_codes(const int32_t *codes_dev, int n_steps, long long elems_per_step,
                        int32_t *dst_dev, long long dst_stride, void *stream);

/* ---- one decode step that allocates nothing -------------------------------- */

/* No counterpart in the reference.  For callers that may not allocate device
 * memory -- a host application whose device memory belongs to another
 * framework's pool, or a real-time decode loop where an allocation could
 * block or synchronise the device.  It runs zonos2cu_head_softcap and then
 * zonos2cu_sample_rows (same arguments, same results) with the intermediate
 * logits in a fixed device array compiled into the library: every GPU that
 * loads the library holds ZONOS2CU_NOALLOC_MAX_LOGITS floats (2.25 MiB) of it
 * until the process exits, and no call allocates or frees anything.
 *   - n_streams * n_cb * vocab must not exceed ZONOS2CU_NOALLOC_MAX_LOGITS
 *     (64 streams of 9 x 1024): larger requests return ZONOS2CU_ETOOBIG.
 *   - The array's device address belongs to the CUDA context current at the
 *     call.  Outside stream capture each call looks it up (cudaGetSymbolAddress,
 *     which allocates nothing); a call made while `stream` is capturing uses
 *     the address found by the last call outside capture in the same context,
 *     and returns ZONOS2CU_ESTATE if that context has made none.  So make one
 *     call in a context before capturing it, and again after cudaDeviceReset.
 *   - All calls on a device share the one array: calls whose work overlaps on
 *     the GPU race.  Order them on one stream, or synchronise between them.
 *   - Every argument is checked before anything is launched, as the two entry
 *     points would check it (n_streams = 0 included).
 * Arguments are those of the two entry points it combines (softcap 15 in
 * the model; row stride of the logits = vocab). */
#define ZONOS2CU_NOALLOC_MAX_LOGITS (64 * 9 * 1024)
int zonos2cu_step_noalloc(const void *W_dev, zonos2cu_dtype dtype, int rows_per_cb, int n_cb,
                          int vocab, int dim, const void *hidden_dev, int n_streams, float softcap,
                          const zonos2cu_sample_params *params, uint64_t *rng_dev,
                          int32_t *hist_dev, int hist_len, int hist_pos,
                          const uint32_t *allow_dev, int delay_step, int32_t *codes_dev,
                          int32_t *flags_dev, void *stream);

#ifdef __cplusplus
}
#endif
#endif /* ZONOS2_CUDA_H */
