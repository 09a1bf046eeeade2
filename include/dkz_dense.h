/*
 * dkz_dense.h -- C ABI of libdkz_dense.so: the dense end of a network (connected
 * layers with their bias, activation, dropout and residual, and a softmax
 * cross-entropy over many classes) as fused gfx950 kernels over fp32 or bf16
 * tensors. A companion of libdkz.so (dkz_ops.h), beside which it is installed
 * and which it loads: ops are issued on dkz_set_stream's stream -- all launches
 * of a call on the one that is set as it begins --, wait for their kernels under
 * dkz_set_sync_after_launch, and return 0 or a hipError_t that dkz_error_string
 * decodes. dkz_dense_last_error_context has the text of the last nonzero return
 * of this library's calls on this host thread.
 *
 * The reference runs these as separate ops: a connected layer's gemm, addBias
 * and activateArray, randUniform + dropout with the draws kept for the backward
 * pass (layers/misc.zig:105-127), and softmax + softmaxCrossEntropy over stored
 * logits (layers/misc.zig:63-76).
 *
 * Conventions:
 *   - `type` is the element type of the tensors given as void *: fp32 or bf16.
 *     Biases, bias gradients, losses and log-sums are fp32. Sums are fp32 or
 *     wider; a bf16 result is rounded to nearest even once.
 *   - Matrices are row-major without gaps: input [rows, inputs], weights
 *     [outputs, inputs], output [rows, outputs]. Any size and element
 *     alignment will do; sizes that are multiples of eight, on 16-byte
 *     boundaries, run fastest. A tensor holds at most 2^31 - 4 elements; rows,
 *     inputs, outputs and classes are 2^26 at most, and rows * classes 2^38.
 *   - A negative size, an unknown type or activation, a null pointer where
 *     elements must be touched or a workspace that is too small returns
 *     hipErrorInvalidValue (1) and launches nothing. An output may not overlap
 *     an input, but for the places named below.
 *   - The ops keep no scratch of their own: what they need is the caller's
 *     workspace (16-byte aligned device memory, contents irrelevant before and
 *     after; null where 0 bytes are needed). How much goes by a call's own sizes:
 *     fewer rows can need more, since a product that leaves the chip empty is cut
 *     into pieces, so that a workspace for several batch sizes is the largest of
 *     theirs. Calls with workspaces of their own
 *     may overlap on any streams, host threads and captured graphs. (The stream is
 *     the process's: host threads that set streams of their own take a lock from
 *     dkz_set_stream to the call's return.) Nothing is allocated, copied to the
 *     host or waited for, and every op may be captured in a graph. Pointers belong
 *     to the current device.
 *   - Sums are taken in an order that depends on sizes, the tensors' alignment and
 *     the workspace's size alone: the same call gives the same bits.
 */
#ifndef DKZ_DENSE_H
#define DKZ_DENSE_H

#include <stddef.h>

#include "dkz_ops.h"

#if defined(__GNUC__)
#pragma GCC visibility push(default)
#endif

#ifdef __cplusplus
extern "C" {
#endif

/* Element types. */
enum dkz_type { DKZ_F32 = 0, DKZ_BF16 = 1 };

/* What failed in this library's last nonzero return on this host thread, or "". */
const char *dkz_dense_last_error_context(void);

/* ------------------------------------------------------------------------ */
/* Dropout without a stored mask                                              */
/* ------------------------------------------------------------------------ */

/* y[i] = (draw(seed, first + i) < prob ? 0 : x[i] * scale) + residual[i], with
 * draw(seed, j) = (hash(seed ^ hash(j mod 2^32) ^ hash(0x9e3779b9 * (j >> 32)))
 * >> 8) * 2^-24 and dkz_rand_uniform's hash: for j < 2^32 its element j. So
 * with first == 0 and no residual the fp32 result is that of dkz_rand_uniform
 * followed by dkz_dropout, bit for bit. residual (y's type) may be NULL, and
 * nothing is added; y may be residual, or x if the types are the same. The
 * backward pass is the same call on the gradient. prob 0 keeps everything:
 * with scale 1 the call converts from one type to the other. */
int dkz_seeded_dropout(int n, int x_type, const void *x, const void *residual, float prob, float scale,
                       unsigned int seed, unsigned long long first, int y_type, void *y);

/* ------------------------------------------------------------------------ */
/* A linear layer                                                             */
/* ------------------------------------------------------------------------ */

/* For row r and output o
 *     a(r, o) = activation(sum over k of input(r, k) * weights(o, k) + biases[o])
 *     output(r, o) = dropout(a(r, o)) + residual(r, o)
 * where dropout is dkz_seeded_dropout's with element first + r * outputs + o
 * (prob 0 and scale 1: none). biases and residual may be NULL. activated, if
 * not NULL, receives a: the backward pass needs it where the activation is not
 * linear and a dropout or residual follows (else output is a). output may be
 * residual. activation is an enum dkz_activation code; fp32 values are those of
 * dkz_activate_array. */
int dkz_linear_forward_workspace(int type, int rows, int inputs, int outputs, size_t *bytes);
int dkz_linear_forward(int type, int rows, int inputs, int outputs, int activation, float prob, float scale,
                       unsigned int seed, unsigned long long first, const void *input, const void *weights,
                       const float *biases, const void *residual, void *activated, void *output, void *workspace,
                       size_t workspace_bytes);

/* Its backward pass. With delta the delta of output and activated the forward's a
 *     d(r, o) = dropout(delta(r, o)) * gradient(activated(r, o))
 *     bias_updates[o] = beta * bias_updates[o] + sum over r of d(r, o)
 *     weight_updates(o, k) = beta * weight_updates(o, k) + sum over r of d(r, o) * input(r, k)
 *     input_delta(r, k) = sum over o of d(r, o) * weights(o, k) + input_residual(r, k)
 * with dkz_gradient_array's gradient and the draws of the forward. beta == 0
 * does not read the updates. Each of the three results may be NULL: it is not
 * computed. activated may be NULL for the linear activation; input_residual (a
 * second path's delta, or input_delta itself to add to it) may be NULL. A bf16
 * pass takes d / scale rounded to bf16 into the two products, and multiplies
 * their sums by the scale: exact where the gradient is 0 or 1, else the results
 * are off by this rounding and their own (for a scale of 2^-8 to 2^8; beyond, d
 * itself is rounded). The bias sums take d unrounded. */
int dkz_linear_backward_workspace(int type, int rows, int inputs, int outputs, size_t *bytes);
int dkz_linear_backward(int type, int rows, int inputs, int outputs, int activation, float prob, float scale,
                        unsigned int seed, unsigned long long first, const void *input, const void *weights,
                        const void *activated, const void *delta, const void *input_residual, float beta,
                        float *bias_updates, void *weight_updates, void *input_delta, void *workspace,
                        size_t workspace_bytes);

/* ------------------------------------------------------------------------ */
/* Softmax cross-entropy of a linear layer, without its logits                */
/* ------------------------------------------------------------------------ */

/* For row r with logits z(r, c) = sum over k of input(r, k) * weights(c, k) +
 * biases[c] (biases may be NULL) and target class t = targets[r]
 *     lse[r] = log(sum over c of exp(z(r, c))),  loss[r] = lse[r] - z(r, t).
 * A target outside 0 .. classes - 1 (-1, say) is none: the row's loss is 0 and
 * it has no gradient. A class whose bias is -infinity has probability 0; a row
 * with no class left has lse -infinity, loss +infinity if it has a target, and
 * no gradient. A row with a NaN or +infinity logit has lse NaN, and with a target
 * NaN loss and gradient.
 *
 * The classes are taken in pieces, as many at a time as the workspace has room
 * for: *best is what the fastest way takes, *least what any call of this shape
 * needs. A piece holds its logits, or the deltas d below, in the tensors' type: half a
 * gigabyte of them at most, but at least 256 classes (256 * rows elements). A bf16
 * forward pass takes all classes at once: a pair of floats for every 16 to 128
 * classes of a row, *least and *best the same. */
int dkz_linear_cross_entropy_forward_workspace(int type, int rows, int inputs, int classes, size_t *least,
                                               size_t *best);
int dkz_linear_cross_entropy_forward(int type, int rows, int inputs, int classes, const void *input,
                                     const void *weights, const float *biases, const int *targets, float *loss,
                                     float *lse, void *workspace, size_t workspace_bytes);

/* Its gradient, from the forward's lse. With s(r) = scale * row_scales[r]
 * (row_scales NULL: scale; 0 for a row without a target) and p(r, c) =
 * exp(z(r, c) - lse[r])
 *     d(r, c) = s(r) * ((c == targets[r]) - p(r, c))
 * -- the delta truth - probability, as dkz_softmax_cross_entropy's -- and
 * bias_updates, weight_updates and input_delta follow from d as in
 * dkz_linear_backward, without an input_residual. A bf16 pass takes d rounded to
 * bf16 into the two products, the bias sums take it unrounded. */
int dkz_linear_cross_entropy_backward_workspace(int type, int rows, int inputs, int classes, size_t *least,
                                                size_t *best);
int dkz_linear_cross_entropy_backward(int type, int rows, int inputs, int classes, const void *input,
                                      const void *weights, const float *biases, const int *targets, const float *lse,
                                      const float *row_scales, float scale, float beta, float *bias_updates,
                                      void *weight_updates, void *input_delta, void *workspace,
                                      size_t workspace_bytes);

#ifdef __cplusplus
}
#endif

#if defined(__GNUC__)
#pragma GCC visibility pop
#endif

#endif /* DKZ_DENSE_H */
