/*
 * ns_losses.h -- C ABI of the operators on the logits of sampled tokens:
 * token log-probabilities (with entropies and their gradient), a clipped
 * policy loss with a KL term, and a preference loss on paired sequences.
 *
 * No counterpart in nano-inference (it samples, sampling/sampler.py:11-133,
 * and neither returns log-probabilities nor trains).  They are what comes after
 * the draw: a serving loop reports the log-probability of the id ns_sample
 * chose, and a training step scores rollouts and learns from them.
 *
 * Conventions, in addition to ns_sampler.h's (device pointers, asynchronous on
 * `stream`, which belongs to the current device, ns_status results)
 *   - One row of logits holds one token: logits [rows, vocab] of `dtype`,
 *     `row_stride` elements from row to row, element-aligned; rows and vocab
 *     up to 2^24.  The distribution of a row is softmax(logits / T) without
 *     penalties and without top-k or top-p.
 *   - targets int64 [rows]: the row's token id, ns_sample's out_ids as they
 *     are.  A negative target (padding, a prompt position, a failed draw's
 *     status) marks a row that holds no token: its logits are not read, its
 *     log-probability, entropy, loss and KL are 0 and its gradient row is 0.
 *     A target >= vocab makes the row's results NaN.
 *   - T: temperature fp32 [rows], or NULL and every row uses temperature_all.
 *     0 (a greedy row) stands for 1: a greedy draw is scored under the
 *     unscaled logits.  A temperature that is negative, infinite or NaN makes
 *     the row's results NaN (temperature_all: NS_ERR_INVALID_ARGUMENT).  Where
 *     T is so small that a coefficient / T passes 2^127 (an entropy's 2^119),
 *     that is what it counts as in the columns other than the target.
 *   - -inf logits have probability 0.  A row that holds a NaN, a +inf or
 *     nothing but -inf has no distribution; its results are NaN.
 *   - Gradients have the logits' dtype and are `grad_stride` elements from row
 *     to row.  grad_logits may be the logits themselves (same pointer and same
 *     stride): the gradient then takes their place.  No other overlap.  The
 *     columns past vocab are left as they are.
 *   - Sums are fp32 per thread and joined in a fixed order: equal inputs give
 *     equal bits (of rows that start on the same 16-byte boundaries; others are
 *     added up in another order).  No call needs a workspace or leaves state
 *     for the next.
 *
 *   stats fp32 [rows][2], written by the forward calls and read by the
 *   gradient: an offset c (a logit of the row) and log2 of sum exp((x - c) / T).
 */
#ifndef NS_LOSSES_H
#define NS_LOSSES_H

#include "ns_sampler.h"

#ifdef __cplusplus
extern "C" {
#endif

/*
 * logprobs fp32 [rows]: ln p(target).  entropy fp32 [rows] or NULL:
 * -sum p ln p in nats.  stats fp32 [rows][2] or NULL.
 */
int ns_token_logprobs(const void* logits, int dtype, int64_t rows, int64_t vocab, int64_t row_stride,
                      const int64_t* targets, const float* temperature, float temperature_all,
                      float* logprobs, float* entropy, float* stats, ns_stream_t stream);

/*
 * grad_logits = d/dlogits of sum_i a_i logprob_i + h_i entropy_i:
 *   (a_i (1{j = target} - p_j) - h_i p_j (ln p_j + entropy_i)) / T.
 * grad_logprobs (a) and grad_entropy (h) fp32 [rows] or NULL for 0; h needs the
 * forward call's entropy.  A row with a = h = 0 is written as zeros without
 * reading its logits.
 */
int ns_token_logprobs_grad(const void* logits, int dtype, int64_t rows, int64_t vocab, int64_t row_stride,
                           const int64_t* targets, const float* temperature, float temperature_all,
                           const float* stats, const float* entropy, const float* grad_logprobs,
                           const float* grad_entropy, void* grad_logits, int64_t grad_stride, ns_stream_t stream);

/*
 * Clipped policy loss: loss = sum_i w_i row_loss_i over the rows that hold a
 * token, with r_i = exp(logprob_i - old_logprobs_i), A_i the advantage,
 *   row_loss_i = -min(r_i A_i, clip(r_i, 1 - clip_low, 1 + clip_high) A_i)
 *                + kl_coef kl_i - entropy_coef entropy_i,
 *   kl_i = exp(d_i) - d_i - 1,  d_i = ref_logprobs_i - logprob_i.
 * A_i = 0 leaves no policy term, whatever r_i is.
 *
 * old_logprobs, advantages fp32 [rows]; ref_logprobs fp32 [rows], or NULL when
 * kl_coef is 0; weights fp32 [rows], or NULL for 1 / rows.  A row of weight 0
 * counts as holding no token.
 * clip_low in [0, 1], clip_high >= 0; kl_coef and entropy_coef finite.
 * loss fp32 [1]; row_loss, logprobs fp32 [rows]; entropy fp32 [rows] or NULL
 * when entropy_coef is 0; kl fp32 [rows] or NULL (it needs ref_logprobs);
 * stats as above; row_grad fp32 [2][rows]: dloss/dlogprob, then dloss/dentropy
 * (what ns_token_logprobs_grad takes).  grad_logits: dloss/dlogits, or NULL.
 */
int ns_policy_loss(const void* logits, int dtype, int64_t rows, int64_t vocab, int64_t row_stride,
                   const int64_t* targets, const float* temperature, float temperature_all,
                   const float* old_logprobs, const float* ref_logprobs, const float* advantages,
                   const float* weights, float clip_low, float clip_high, float kl_coef, float entropy_coef,
                   float* loss, float* row_loss, float* logprobs, float* entropy, float* kl, float* stats,
                   float* row_grad, void* grad_logits, int64_t grad_stride, ns_stream_t stream);

/*
 * ns_policy_loss in which one wait inside the kernel that holds rows on chip
 * counts as run out at row `give_up`: for tests of what a call leaves then.  A
 * wait runs out after 200 ms, which takes a fault elsewhere.  The rows of the
 * blocks concerned that hold a token are then NaN in all results, and so is the
 * loss.  Without grad_logits, or with rows too short or too long to be held,
 * there are no such waits, and the results are ns_policy_loss's.
 */
int ns_policy_loss_debug(const void* logits, int dtype, int64_t rows, int64_t vocab, int64_t row_stride,
                         const int64_t* targets, const float* temperature, float temperature_all,
                         const float* old_logprobs, const float* ref_logprobs, const float* advantages,
                         const float* weights, float clip_low, float clip_high, float kl_coef, float entropy_coef,
                         float* loss, float* row_loss, float* logprobs, float* entropy, float* kl, float* stats,
                         float* row_grad, void* grad_logits, int64_t grad_stride, int64_t give_up,
                         ns_stream_t stream);

/*
 * Preference loss on pairs of sequences whose tokens are packed row after row:
 * sequence s holds rows [seq_offsets[s], seq_offsets[s + 1]) (int64 [2 pairs +
 * 1], ascending, within rows); 2 p is pair p's chosen sequence and 2 p + 1 the
 * rejected one.  With g_i = logprob_i - ref_logprobs_i (ref NULL: 0),
 *   reward_s = beta * sum of g_i over the sequence's tokens (average != 0:
 *              their mean; an empty sequence has reward 0),
 *   h_p = reward_2p - reward_2p+1,
 *   pair_loss_p = -(1 - e) ln sigmoid(h_p) - e ln sigmoid(-h_p),
 * e = label_smoothing in [0, 1), beta finite, and loss is the pairs' mean (0
 * without pairs).  Rows outside every sequence count as holding no token.
 * loss fp32 [1]; pair_loss fp32 [pairs]; rewards fp32 [pairs][2]; logprobs
 * fp32 [rows]; stats as above; row_grad fp32 [rows]: dloss/dlogprob.
 * grad_logits: dloss/dlogits, or NULL.
 */
int ns_preference_loss(const void* logits, int dtype, int64_t rows, int64_t vocab, int64_t row_stride,
                       const int64_t* targets, const float* temperature, float temperature_all,
                       const int64_t* seq_offsets, int64_t pairs, const float* ref_logprobs, float beta,
                       float label_smoothing, int average, float* loss, float* pair_loss, float* rewards,
                       float* logprobs, float* stats, float* row_grad, void* grad_logits, int64_t grad_stride,
                       ns_stream_t stream);

#ifdef __cplusplus
}
#endif

#endif /* NS_LOSSES_H */
