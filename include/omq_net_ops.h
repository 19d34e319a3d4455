/*
 * omq_net_ops.h -- C ABI of the MI355X (gfx950) operators of a policy network over board tokens
 * (libomq_net_ops.so): the token embedding and its gradient, the root-mean-square norm of a
 * residual sum with dropout, its 8-bit output and its gradients, dropout, the clipped policy
 * loss over legal actions with its gradient, the norm of queries and keys with the rotation by
 * their positions and its gradients, attention and its gradients, and the log-probabilities of
 * given tokens with the entropy, the best alternatives and their gradient.
 *
 * Conventions, those of omq_tree_ops.h: every array is a DEVICE pointer owned by the caller;
 * an entry point launches on the HIP stream it is given and returns without synchronising, keeps
 * nothing between calls and allocates nothing.  It returns OMQ_NET_OK or a negative code, and
 * omq_net_last_error() then holds a message for the calling thread.  Nothing is launched when an
 * argument is refused.  Every result is a function of the arguments alone: the sums run in a
 * fixed order (no floating-point atomics).
 *
 * Arrays of rows are given with a row stride in ELEMENTS; the elements of a row are adjacent.
 * No alignment beyond the element's own is needed, but workspaces (and `stats`) begin on a 16-byte
 * boundary.  Sums, statistics and intermediate values are
 * float32; a result is rounded to its type once.
 */
#ifndef OMQ_NET_OPS_H
#define OMQ_NET_OPS_H

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define OMQ_NET_ABI_VERSION 2

#define OMQ_NET_OK 0
#define OMQ_NET_E_ARG (-1)    /* invalid argument (size, type, null pointer, workspace) */
#define OMQ_NET_E_LAUNCH (-2) /* HIP launch or runtime error */
#define OMQ_NET_E_LIMIT (-3)  /* size beyond a limit of this build */

/* element types */
#define OMQ_NET_F32 0
#define OMQ_NET_BF16 1
#define OMQ_NET_F16 2

#define OMQ_NET_STATS 8 /* floats that a policy loss's row leaves for its gradient */

/* limits of this build */
#define OMQ_NET_MAX_NORM_DIM 16384    /* columns of a normed row (a row is held in registers) */
#define OMQ_NET_MAX_DIM (1 << 20)     /* columns of an embedding row, of a dropout row */
#define OMQ_NET_MAX_ACTIONS (1 << 30) /* columns of a policy loss's row */
#define OMQ_NET_MAX_COUNT 2147483647  /* rows, tokens, vocabulary */
#define OMQ_NET_MAX_ROTARY_DIM 256    /* columns of a rotated head */
#define OMQ_NET_MAX_AXES 4            /* axes of its positions */
#define OMQ_NET_MAX_HEAD_DIM 128      /* columns of a head of the attention */
#define OMQ_NET_MAX_TOP 32            /* alternatives of a row */

int omq_net_abi_version(void);
const char* omq_net_last_error(void);

/* out[t] = scale * weight[ids[t]], rounded once.  An id outside [0, vocab) gives a row of zeros.
 *   ids     int32 or int64 [tokens] (ids_are_64)
 *   weight  [vocab, dim] rows of `dtype`, weight_stride apart
 *   out     [tokens, dim] of `dtype`, contiguous */
int omq_token_embedding(const void* ids, int ids_are_64, int64_t tokens, const void* weight,
                        int64_t weight_stride, int64_t vocab, int64_t dim, int dtype, float scale,
                        void* out, void* stream);

/* Bytes of workspace of omq_token_embedding_grad; negative for sizes it refuses. */
int64_t omq_token_embedding_grad_workspace(int64_t tokens, int64_t vocab, int64_t dim);

/* out[v] = scale * sum over the tokens t with ids[t] == v, in ascending t, of grad[t]; zero for
 * a row without tokens.  Ids outside [0, vocab) take no part.
 *   grad  [tokens, dim] rows of `dtype`, grad_stride apart
 *   out   [vocab, dim] of `out_dtype` (`dtype` or OMQ_NET_F32), contiguous; every element written */
int omq_token_embedding_grad(const void* grad, int64_t grad_stride, int dtype, const void* ids,
                             int ids_are_64, int64_t tokens, int64_t vocab, int64_t dim,
                             float scale, void* out, int out_dtype, void* workspace,
                             int64_t workspace_bytes, void* stream);

/* Dropout of [rows, dim], contiguous: out = x * 65536/(65536 - t) where the element is kept, 0
 * (whatever x holds) where it is not; t = floor(p * 65536 + 1/2), p in [0, 1].
 *
 * Element (r, c) is kept when the 16 bits c % 4 (from the low end) of
 *     splitmix64(key + 0x9E3779B97F4A7C15 * (r * ceil(dim/4) + c/4))
 * are at least t, with key = splitmix64(splitmix64(seed) ^ offset) and
 *     splitmix64(x): z = x + 0x9E3779B97F4A7C15; z = (z ^ z>>30) * 0xBF58476D1CE4E5B9;
 *                    z = (z ^ z>>27) * 0x94D049BB133111EB; z ^ z>>31
 * in 64-bit arithmetic: the mask is a function of (seed, offset, position) and is formed again
 * where it is needed.  The gradient is the same call on the gradient.  out may be x. */
int omq_dropout(const void* x, int64_t rows, int64_t dim, int dtype, double p, uint64_t seed,
                uint64_t offset, void* out, void* stream);

/* h = residual + dropout(x), y = h / sqrt(mean(h^2) + eps) * weight.
 * y is formed from the unrounded h.  residual may be NULL (zeros); h may be NULL when the sum is
 * not wanted.  h may be residual or x, and y may be x, when their strides are dim.
 *   x, residual  [rows, dim] rows of `dtype`, their strides apart
 *   weight       [dim] of `weight_dtype` (`dtype` or OMQ_NET_F32)
 *   y, h         [rows, dim] of `dtype`, contiguous */
int omq_add_rms_norm(const void* x, int64_t x_stride, const void* residual,
                     int64_t residual_stride, const void* weight, int weight_dtype, int64_t rows,
                     int64_t dim, int dtype, float eps, double p, uint64_t seed, uint64_t offset,
                     void* y, void* h, void* stream);

/* The same without dropout, y in 8 bits (OCP e4m3): y = q * scale, with one scale for a row
 * (group 0) or for each `group` columns of it (128; the last group may be shorter):
 * scale = max(largest |y| of the group / 448, 2^-126).  A row whose y are NaN has NaN in q.
 *   q       [rows, dim] bytes, contiguous
 *   scales  [rows, groups] float32, contiguous, groups = 1 or ceil(dim/128) */
int omq_add_rms_norm_fp8(const void* x, int64_t x_stride, const void* residual,
                         int64_t residual_stride, const void* weight, int weight_dtype,
                         int64_t rows, int64_t dim, int dtype, float eps, int group, uint8_t* q,
                         float* scales, void* h, void* stream);

/* Bytes of workspace of omq_add_rms_norm_grad; negative for sizes it refuses. */
int64_t omq_add_rms_norm_grad_workspace(int64_t rows, int64_t dim);

/* Gradients of omq_add_rms_norm from its h: with n = h / sqrt(mean(h^2) + eps),
 *   grad_residual = grad_h + (g - n * mean(g * n)) / sqrt(mean(h^2) + eps),  g = grad_y * weight
 *   grad_x        = dropout(grad_residual)
 *   grad_weight   = sum over rows of grad_y * n
 *   grad_h       [rows, dim] or NULL (zeros): the gradient that reaches h by its other use
 *   grad_x       NULL when p == 0 (it is grad_residual then); grad_residual NULL when not wanted
 *   grad_weight  [dim] of weight_dtype, or NULL
 * The outputs are contiguous. */
int omq_add_rms_norm_grad(const void* grad_y, int64_t grad_y_stride, const void* grad_h,
                          int64_t grad_h_stride, const void* h, int64_t h_stride,
                          const void* weight, int weight_dtype, int64_t rows, int64_t dim,
                          int dtype, float eps, double p, uint64_t seed, uint64_t offset,
                          void* grad_x, void* grad_residual, void* grad_weight, void* workspace,
                          int64_t workspace_bytes, void* stream);

/* The rows of a policy loss.  With L the legal actions of a row, logq = log_softmax of its logits
 * over L, and a its action:
 *   logp  = logq[a]
 *   ratio = exp(logp - old_logp)
 *   loss  = -min(ratio * adv, clamp(ratio, 1 - clip_low, 1 + clip_high) * adv) + kl_coef * kl
 *   kl    = d' - 1 - log d' with d' = exp(ref_logp - logp)           (ref_logp given)
 *         = sum over L of target * (log target - logq)               (target given)
 *         = 0                                                        (neither)
 * A row whose action lies outside [0, actions) or is not legal has logp 0 and neither the first
 * term nor a sampled kl; the kl against a target stays.  A row without a legal action whose
 * logit is above -infinity has loss, logp, kl and gradient 0.  Logits and targets of illegal
 * actions are never used, whatever they hold; a target that is not positive adds nothing whatever
 * its logq.  A row that adds nothing to the loss (padding) has gradient 0 whatever its logits
 * hold; elsewhere a NaN among the legal logits reaches the row's results.  A legal action whose
 * logit is -infinity has logp -infinity when it is taken, and a sampled kl of +infinity; where
 * kl_coef is 0 the kl reaches neither loss nor gradient, whatever it is. */
typedef struct omq_policy_rows {
  int64_t rows;
  int64_t actions;        /* columns */
  const void* logits;     /* [rows, actions] of dtype */
  int64_t logits_stride;
  const uint8_t* legal;   /* [rows, actions], non-zero = legal; NULL: all are */
  int64_t legal_stride;
  const float* target;    /* [rows, actions] probabilities, or NULL */
  int64_t target_stride;
  const void* taken;      /* [rows] the actions, int32 or int64 */
  const float* advantages;  /* [rows] */
  const float* old_logp;    /* [rows] */
  const float* ref_logp;    /* [rows] or NULL; not together with target */
  int32_t dtype;
  int32_t taken_are_64;
  float clip_low, clip_high, kl_coef;
  float reserved;
} omq_policy_rows;

/* Bytes of workspace of the two loss entry points; negative for sizes they refuse. */
int64_t omq_clipped_policy_loss_workspace(int64_t rows, int64_t actions);

/* loss, logp, kl: float32 [rows].  stats: float32 [rows, OMQ_NET_STATS] on a 16-byte boundary for
 * omq_clipped_policy_loss_grad, or NULL. */
int omq_clipped_policy_loss(const omq_policy_rows* r, float* loss, float* logp, float* kl,
                            float* stats, void* workspace, int64_t workspace_bytes, void* stream);

/* grad [rows, actions] of the logits' type, contiguous: row_weight[row] (NULL: 1) times the
 * gradient of the row's loss; 0 at illegal actions.  stats: from omq_clipped_policy_loss on the
 * same rows. */
int omq_clipped_policy_loss_grad(const omq_policy_rows* r, const float* stats,
                                 const float* row_weight, void* grad, void* stream);

/* Both at once.  Rows of up to 16384 actions (8192 with a target) are read once, longer ones
 * twice. */
int omq_clipped_policy_loss_with_grad(const omq_policy_rows* r, const float* row_weight,
                                      float* loss, float* logp, float* kl, void* grad,
                                      void* workspace, int64_t workspace_bytes, void* stream);

/* Heads of queries and keys, normed each over its columns and rotated by the token's position:
 *   n = x / sqrt(mean(x^2) + eps) * weight       (n = x where there are no weights)
 *   out: pair j of the first 2 * pairs columns of n, (a, b), becomes
 *        (a cos t - b sin t, b cos t + a sin t),  t = position[axis of j] * frequencies[j];
 *        the columns behind them stay.
 * Pair j is the columns (j, j + pairs), or (2j, 2j + 1) with `interleaved`.  Axis a holds the pairs
 * from section_end[a-1] (0 for the first) to section_end[a]; the last section ends at `pairs`.
 * The angle is formed in 64 bits and reduced to one turn before it is rounded.
 *   q, k        [tokens, heads, dim] of dtype; a token's heads and the tokens at their strides
 *   weights     [dim] of weight_dtype (dtype or OMQ_NET_F32), both or neither
 *   positions   int32 or int64 [position_rows, axes]; token i has row i % position_rows
 *   frequencies float64 [pairs], radians per unit of the position */
typedef struct omq_rotary {
  int64_t tokens, position_rows;
  const void *q, *k;
  int64_t q_token_stride, q_head_stride, k_token_stride, k_head_stride;
  const void *q_weight, *k_weight;
  const void* positions;
  const double* frequencies;
  int32_t q_heads, k_heads, dim, pairs, axes;
  int32_t section_end[OMQ_NET_MAX_AXES];
  int32_t positions_are_64, interleaved, dtype, weight_dtype;
  float eps;
} omq_rotary;

/* q_out, k_out: [tokens, heads, dim] of dtype, contiguous. */
int omq_head_norm_rotary(const omq_rotary* r, void* q_out, void* k_out, void* stream);

/* Bytes of workspace of omq_head_norm_rotary_grad; negative for what it refuses. */
int64_t omq_head_norm_rotary_grad_workspace(const omq_rotary* r);

/* Gradients from the same q and k and the gradients of the outputs (contiguous):
 *   grad_q, grad_k              [tokens, heads, dim] of dtype, contiguous
 *   grad_q_weight, grad_k_weight  [dim] of weight_dtype; NULL where there are no weights */
int omq_head_norm_rotary_grad(const omq_rotary* r, const void* grad_q_out, const void* grad_k_out,
                              void* grad_q, void* grad_k, void* grad_q_weight,
                              void* grad_k_weight, void* workspace, int64_t workspace_bytes,
                              void* stream);

/* Attention of sequences: with the query i and the key j of a sequence of lq queries and lk keys,
 *   out_i = sum_j p_ij v_j,  p_ij = exp(scale q_i.k_j - lse_i),  lse_i = log sum_j exp(scale q_i.k_j)
 * over the keys that i sees: all, or j <= i + lk - lq with `causal` (the last query sees every
 * key).  A query that sees none has out 0 and lse -infinity, and so have rows of no sequence.
 * Query head h attends to key head h / (q_heads / k_heads).
 *
 * Either a batch (q_starts NULL): sequence s has the queries q + s * q_seq_stride, q_len of them,
 * and room for k_len keys at k + s * k_seq_stride.  Or packed (q_starts and k_starts given, int32
 * [sequences + 1], not falling): sequence s has the rows q_starts[s] to q_starts[s + 1] of q and
 * k_starts[s] to k_starts[s + 1] of k; q_len and k_len are the rows of all.  k_lengths (int32
 * [sequences] or NULL) gives how many of a sequence's keys are in use, from the first.  Starts
 * and lengths out of range are cut to the range; what rows behind a sequence's keys hold is never
 * used.
 *   q       rows of [q_heads, dim], at q_row_stride; its heads at q_head_stride; k, v alike
 *   out     [rows of q, q_heads, dim], contiguous
 *   lse     float32 [rows of q, q_heads], contiguous
 * Products are formed from the elements' type and summed in float32; p is rounded to the elements'
 * type before it multiplies v, as are the gradients of the scores before they multiply q (for k they
 * have twice its bits); float16 takes both times powers of two, so that small ones
 * keep their bits.  Rows of heads of queries (q_len times q_heads, of all sequences) and k_len are
 * at most OMQ_NET_MAX_COUNT - 4095 each. */
typedef struct omq_attention_args {
  int64_t sequences, q_len, k_len;
  const void *q, *k, *v;
  int64_t q_seq_stride, q_row_stride, q_head_stride;
  int64_t k_seq_stride, k_row_stride, k_head_stride;
  int64_t v_seq_stride, v_row_stride, v_head_stride;
  const int32_t *q_starts, *k_starts, *k_lengths;
  int32_t q_heads, k_heads, dim, dtype, causal;
  float scale; /* above 0, at most 2^127 */
} omq_attention_args;

/* Bytes of workspace of omq_attention_forward; negative for what it refuses. */
int64_t omq_attention_forward_workspace(const omq_attention_args* a);

/* lse may be NULL when it is not wanted. */
int omq_attention_forward(const omq_attention_args* a, void* out, float* lse, void* workspace,
                          int64_t workspace_bytes, void* stream);

/* Bytes of workspace of omq_attention_grad; negative for what it refuses. */
int64_t omq_attention_grad_workspace(const omq_attention_args* a);

/* Gradients of sum(grad_out * out) from the forward pass's out and lse.  Those may be of more keys
 * than the call's (a part of a row's keys, whose parts were joined by their lse): then they are the
 * part's share.
 *   grad_out, out, grad_q  as out above
 *   grad_k, grad_v         [rows of k (all of them), k_heads, dim], contiguous; 0 for rows of no
 *                          sequence and behind a sequence's keys */
int omq_attention_grad(const omq_attention_args* a, const void* grad_out, const void* out,
                       const float* lse, void* grad_q, void* grad_k, void* grad_v,
                       void* workspace, int64_t workspace_bytes, void* stream);

/* What a policy says of given tokens.  With logq the log-softmax of a row over its legal tokens L:
 *   logp     = logq[token]; 0 for a token outside [0, vocab) or not legal
 *   entropy  = -sum over L of e^logq logq
 *   top      the `top` most probable tokens of L, by falling logit and rising index among equals:
 *            their logq and their indices; -infinity and -1 where L has fewer of probability
 *            above 0
 * A row without a legal token whose logit is above -infinity has logp and entropy 0 and no
 * alternatives.  What the logits of other tokens hold is never used.  A NaN or +infinity among the
 * legal logits makes the row's logp (of a legal token), entropy and top_logp NaN, its alternatives
 * being those of its other logits (a NaN is never one).
 *   logits  [rows, vocab] of dtype, logits_stride apart
 *   legal   [rows, vocab], non-zero = legal, legal_stride apart; NULL: all are
 *   tokens  int32 or int64 [rows] */
typedef struct omq_logprob_rows {
  int64_t rows, vocab;
  const void* logits;
  int64_t logits_stride;
  const uint8_t* legal;
  int64_t legal_stride;
  const void* tokens;
  int32_t dtype, tokens_are_64;
} omq_logprob_rows;

/* logp, entropy: float32 [rows].  top_logp float32, top_tokens int64 [rows, top] (0 <= top <=
 * OMQ_NET_MAX_TOP; NULL for 0).  stats: float32 [rows, OMQ_NET_STATS] on a 16-byte boundary for
 * omq_token_logprobs_grad, or NULL. */
int omq_token_logprobs(const omq_logprob_rows* r, int32_t top, float* logp, float* entropy,
                       float* top_logp, int64_t* top_tokens, float* stats, void* stream);

/* grad [rows, vocab] of the logits' type, contiguous: the gradient of sum(logp_weight * logp +
 * entropy_weight * entropy); 0 at tokens that are not legal, and in a row whose two weights are 0.
 * Weights float32 [rows]; NULL: 0.  stats: from omq_token_logprobs on the same rows. */
int omq_token_logprobs_grad(const omq_logprob_rows* r, const float* stats,
                            const float* logp_weight, const float* entropy_weight, void* grad,
                            void* stream);

/* Both at once; rows of up to 16384 tokens are read once. */
int omq_token_logprobs_with_grad(const omq_logprob_rows* r, const float* logp_weight,
                                 const float* entropy_weight, float* logp, float* entropy,
                                 void* grad, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* OMQ_NET_OPS_H */
