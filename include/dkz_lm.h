/*
 * dkz_lm.h -- C ABI of libdkz_lm.so: what a token model needs beside the dense end
 * of dkz_dense.h, as fused gfx950 kernels over fp32 or bf16 tensors: gated
 * feed-forward blocks with their backward pass, log probabilities of given tokens
 * with the entropy and the top alternatives, and distillation from a teacher's top
 * logits. A companion of libdkz.so (dkz_ops.h), beside which it is installed and
 * which it loads; the reference has no counterpart.
 *
 * The conventions are dkz_dense.h's: element types, rounding, sizes, refusals,
 * overlaps, workspaces, streams, captured graphs, the same bits from the same call.
 * dkz_lm_last_error_context has the text of the last nonzero return of this
 * library's calls on this host thread. Deltas are the negative gradients of a loss,
 * as everywhere in the framework.
 *
 * A workspace of a gated block goes by the call's own sizes, as dkz_dense.h's do: fewer
 * rows can need more. What the queries of the calls on logits give does for any number
 * of rows up to theirs.
 *
 * Logits are rows of `classes` elements, each row `pitch` elements after the one
 * before (pitch >= classes); what lies between a row's end and the next row is
 * neither read nor written. rows, classes and pitch are 2^26 at most and
 * rows * pitch is 2^38: a tensor of logits may be larger than others. Rows that
 * start on 16-byte boundaries run fastest. A class whose logit is -infinity is
 * masked: its probability is 0.
 */
#ifndef DKZ_LM_H
#define DKZ_LM_H

#include "dkz_dense.h"

#if defined(__GNUC__)
#pragma GCC visibility push(default)
#endif

#ifdef __cplusplus
extern "C" {
#endif

/* What failed in this library's last nonzero return on this host thread, or "". */
const char *dkz_lm_last_error_context(void);

/* ------------------------------------------------------------------------ */
/* Gated feed-forward block                                                   */
/* ------------------------------------------------------------------------ */

/* A gate's activations: dkz_activation's DKZ_LOGISTIC, DKZ_RELU and DKZ_LINEAR, and
 *     DKZ_SILU  g * logistic(g)
 *     DKZ_GELU  g / 2 * (1 + tanh(sqrt(2 / pi) * (g + 0.044715 * g^3))) */
enum dkz_gate { DKZ_SILU = 14, DKZ_GELU = 15 };

/* For row r and hidden unit j, with weights [2 * hidden, inputs] (the gate's rows,
 * then the others) and biases [2 * hidden] (or NULL)
 *     s(r, o) = sum over k of input(r, k) * weights(o, k) + biases[o]
 *     output(r, j) = activation(s(r, j)) * s(r, hidden + j).
 * sums [rows, 2 * hidden], if not NULL, receives s: the backward pass needs it. The
 * block's last layer is dkz_linear_forward's, on output. */
int dkz_gated_forward_workspace(int type, int rows, int inputs, int hidden, size_t *bytes);
int dkz_gated_forward(int type, int rows, int inputs, int hidden, int activation, const void *input, const void *weights,
                      const float *biases, void *sums, void *output, void *workspace, size_t workspace_bytes);

/* Its backward pass, with delta the delta of output and s the forward's sums as they
 * are stored:
 *     d(r, j) = delta(r, j) * s(r, hidden + j) * activation'(s(r, j))
 *     d(r, hidden + j) = delta(r, j) * activation(s(r, j))
 *     bias_updates[o] = beta * bias_updates[o] + sum over r of d(r, o)
 *     weight_updates(o, k) = beta * weight_updates(o, k) + sum over r of d(r, o) * input(r, k)
 *     input_delta(r, k) = sum over o of d(r, o) * weights(o, k) + input_residual(r, k).
 * NULL results, beta and input_residual are dkz_linear_backward's. A bf16 pass takes
 * d rounded to bf16 into the two products, the bias sums take it unrounded. */
int dkz_gated_backward_workspace(int type, int rows, int inputs, int hidden, size_t *bytes);
int dkz_gated_backward(int type, int rows, int inputs, int hidden, int activation, const void *input, const void *weights,
                       const void *sums, const void *delta, const void *input_residual, float beta, float *bias_updates,
                       void *weight_updates, void *input_delta, void *workspace, size_t workspace_bytes);

/* ------------------------------------------------------------------------ */
/* Log probabilities of tokens                                                */
/* ------------------------------------------------------------------------ */

/* With y(r, c) = logits(r, c) / temperature, m(r) the largest logit of row r and
 *     l(r) = log(sum over c of exp(y(r, c) - m(r) / temperature))
 * the log probability of class c is (logits(r, c) - m(r)) / temperature - l(r).
 *     log_probs[r * given + j]   that of class tokens[r * given + j]; 0 where that is
 *                                no class (-1, say). given is 0 .. 256.
 *     entropy[r]                 -(sum over c of p * log p); may be NULL.
 *     stats[2 * r], [2 * r + 1]  m(r) and l(r): the backward pass needs them, and the
 *                                logarithm of the sum of exp(y) is m / temperature + l.
 *     top_tokens[r * top + i]    the class of the (i + 1)th largest logit, of equal ones
 *                                the lowest first, and its log probability in
 *     top_log_probs[r * top + i] ; top is 0 .. 64. Masked classes are no alternatives:
 *                                past the last other one the token is -1 and its log
 *                                probability -infinity.
 * tokens and log_probs may be NULL where given is 0, as top_tokens and top_log_probs
 * where top is. temperature is 2^-64 .. 2^64. (fp32: what passes its range, the
 * difference of two logits too, is infinite.) A row that has no class left has
 * m and l -infinity, log probabilities -infinity and entropy 0. A row with a NaN or
 * +infinity logit has NaN for l, log probabilities and entropy, and no alternatives:
 * tokens -1 with NaN. m passes over NaNs. */
int dkz_token_log_probs_workspace(int type, int rows, int classes, int top, size_t *bytes);
int dkz_token_log_probs(int type, int rows, int classes, int pitch, const void *logits, float temperature, int given,
                        const int *tokens, int top, float *log_probs, float *entropy, float *stats, int *top_tokens,
                        float *top_log_probs, void *workspace, size_t workspace_bytes);

/* The delta of the logits from those of log_probs, a(r, j), and of entropy, e(r)
 * (entropy_deltas NULL: 0, and entropy may be NULL). With p the probabilities, from the
 * forward's stats, A(r) the sum of a(r, j) over the tokens that are classes, and H(r)
 * the forward's entropy
 *     d(r, c) = (sum over j of a(r, j) * (tokens(r, j) == c)
 *                - p(r, c) * (A(r) + e(r) * (log p(r, c) + H(r)))) / temperature
 *     logits_delta(r, c) = beta * logits_delta(r, c) + d(r, c)
 * (beta == 0 does not read it). logits_delta has the logits' type and pitch and may be
 * logits if beta is 0. A row without a class left has d 0. */
int dkz_token_log_probs_backward(int type, int rows, int classes, int pitch, const void *logits, float temperature, int given,
                                 const int *tokens, const float *stats, const float *entropy, const float *log_prob_deltas,
                                 const float *entropy_deltas, float beta, void *logits_delta);

/* ------------------------------------------------------------------------ */
/* Distillation                                                               */
/* ------------------------------------------------------------------------ */

/* A teacher's `top` (1 .. 256) entries a row, class teacher_tokens[r * top + j] with
 * logit teacher_logits[r * top + j], have the probabilities
 *     p(r, j) = softmax over j of teacher_logits(r, j) / temperature;
 * entries that are no class (-1, say) have none, and one class may have several. With
 * q = softmax over all classes of logits / temperature
 *     loss[r] = temperature^2 * sum over j of p(r, j) * (log p(r, j) - log q(r, teacher_tokens(r, j)))
 *     logits_delta(r, c) = s(r) * temperature * (sum over j of p(r, j) * (teacher_tokens(r, j) == c) - q(r, c)),
 * the delta of scale(r) * loss[r] with s(r) = scale * row_scales[r] (row_scales NULL:
 * scale). logits_delta may be NULL (the loss alone) or logits; it has their pitch. A row
 * without an entry, or whose entries are all -infinity, has loss 0 and delta 0, a row
 * whose s is 0 has delta 0. A masked class that an entry has makes the loss +infinity, and
 * a row without a class left has that and delta 0. NaN and +infinity logits make the
 * row's loss and delta NaN (a teacher's: the delta of its entries). temperature is 2^-64 .. 2^64. */
int dkz_distillation_workspace(int type, int rows, int classes, size_t *bytes);
int dkz_distillation(int type, int rows, int classes, int pitch, const void *logits, float temperature, int top,
                     const int *teacher_tokens, const float *teacher_logits, const float *row_scales, float scale, float *loss,
                     void *logits_delta, void *workspace, size_t workspace_bytes);

#ifdef __cplusplus
}
#endif

#if defined(__GNUC__)
#pragma GCC visibility pop
#endif

#endif /* DKZ_LM_H */
