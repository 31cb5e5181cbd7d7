/*
 * mlease_operators.h -- C-ABI of the operators on token ids, logits and pairs of answers (libmlease_hip.so).
 *
 * They stand beside the trainer's own operators (mlease_admm.h), which do not call them, and keep their conventions where those apply:
 *   mlx_embedding_lookup / _gradient   rows of a table by id, each by itself (mlx_score_rows sums a row's coefficients), and the
 *                                      gradient by sorted ids; an id the table does not hold (-1) is absent
 *   mlx_token_loglik / _gradient       a log-likelihood as mlx_test_loglik's, for one of many classes
 *   mlx_preference_loss                the logistic loss and gradient with weight and offset, on the margins of pairs
 *
 * Conventions
 *   - C linkage, plain pointers and sizes, no exceptions cross the boundary. MLX_OK (0) or a negative MLX_ERR_* code;
 *     mlx_last_error(NULL) gives the calling thread's message. Arguments are checked before any HIP call is made.
 *   - No handle and no state: `device` is the HIP device index, `stream` a hipStream_t of that device (NULL = its null stream).
 *     A call enqueues its kernels and returns; nothing is allocated, copied to the host or waited for, so calls may be
 *     captured into a HIP graph and made from several threads at once. The calling thread's current device is left as it was.
 *     Each launch's own status counts, not the thread's last error (hipGetLastError), which is left to whom it belongs; behind a
 *     launch that fails nothing more is enqueued.
 *   - All data pointers are DEVICE pointers of `device` (or memory it can reach). A matrix is row-major with `ld` elements from one
 *     row to the next; outputs need ld >= the row's length, inputs may repeat rows (ld = 0). Pointers need the alignment of their
 *     element only. Outputs may not overlap inputs, except where a call says so.
 *   - type: MLX_F32, MLX_BF16 or MLX_F16. id_type: MLX_I32 or MLX_I64. Arithmetic is done in 32 bits or more; results are
 *     rounded to `type` once. Rows (ids, tokens) and table rows / classes are fewer than 2^31 - 1; offsets are 64 bits throughout.
 *   - A workspace is device memory of the size the _workspace call names, 256-byte aligned, held by one call at a time: concurrent
 *     calls (also two captured graphs that replay at the same time) need one each. Its contents mean nothing between calls.
 *   - Results do not depend on the stream, the workspace or what else runs: the same inputs give the same bits.
 */
#ifndef MLEASE_OPERATORS_H
#define MLEASE_OPERATORS_H

#include "mlease_admm.h"

#ifdef __cplusplus
extern "C" {
#endif

enum { MLX_F32 = 0, MLX_BF16 = 1, MLX_F16 = 2 };
enum { MLX_I32 = 0, MLX_I64 = 1 };

/* out[t][j] = scale * table[ids[t]][j] for t < n_ids, j < width. An id outside [0, n_rows) is absent: its row of out is zero. */
int mlx_embedding_lookup(int32_t device, void *stream, int32_t type, const void *table, int64_t n_rows, int64_t width, int64_t ld_table,
                         int32_t id_type, const void *ids, int64_t n_ids, float scale, void *out, int64_t ld_out);

/* grad[v][j] = scale * sum over the t with ids[t] == v of grad_out[t][j], summed in 32 bits in an order that the
 * sizes and ids decide. accumulate == 0: grad [n_rows][width] is written whole (rows without an id are zero); accumulate != 0: the sums are
 * added to what grad holds (32-bit sum, rounded once) and rows without an id are not touched. grad_type is `type` or MLX_F32. */
int mlx_embedding_gradient_workspace(int64_t n_rows, int64_t width, int64_t n_ids, size_t *bytes);
int mlx_embedding_gradient(int32_t device, void *stream, int32_t type, const void *grad_out, int64_t ld_grad_out, int32_t id_type, const void *ids,
                           int64_t n_ids, float scale, int32_t accumulate, int32_t grad_type, void *grad, int64_t n_rows, int64_t width,
                           int64_t ld_grad, void *workspace, size_t workspace_bytes);

/* logp[t] = logits[t][target[t]] - log sum_j exp(logits[t][j]), and stats[t] = { max_j, log sum_j exp(logits[t][j] - max_j) } for the
 * gradient. A target outside [0, n_classes) is absent: logp[t] = 0, the row is not read and stats[t] is { 0, 0 }. Logits of -infinity
 * are classes of probability 0; a row of nothing else has logp = -infinity. A NaN or +infinity in a row makes its logp NaN. */
int mlx_token_loglik_workspace(int64_t n_tokens, int64_t n_classes, size_t *bytes);
int mlx_token_loglik(int32_t device, void *stream, int32_t type, const void *logits, int64_t n_tokens, int64_t n_classes, int64_t ld_logits,
                     int32_t id_type, const void *target, float *logp, float *stats, void *workspace, size_t workspace_bytes);

/* dlogits[t][j] = grad_logp[t] * ([j == target[t]] - exp(logits[t][j] - log sum)), with the stats of mlx_token_loglik. Rows whose target is
 * absent, whose grad_logp is 0 or whose logits are all -infinity are zero (and not read). dlogits may be logits itself (same ld). */
int mlx_token_loglik_gradient(int32_t device, void *stream, int32_t type, const void *logits, int64_t n_tokens, int64_t n_classes, int64_t ld_logits,
                              int32_t id_type, const void *target, const float *stats, const float *grad_logp, void *dlogits, int64_t ld_dlogits);

/* Loss and gradient of n_pairs pairs of sequences, packed one behind the other: sequence s holds the tokens
 * [seq_ptr[s], seq_ptr[s+1]), s < 2 n_pairs, pair p prefers sequence p to sequence n_pairs + p. seq_ptr[2 n_pairs + 1] has to be ascending,
 * within [0, n_tokens]. Bounds are on the device and cannot be refused: values outside are read as the nearest bound, and where they descend
 * every access stays within the arrays, a sequence that ends before it begins counts as empty for ratio, margin and loss, and grad is unspecified
 * (a token can then be of two sequences, or be taken for one of none).
 *   ratio[s] = sum over its tokens of logp - ref_logp   (mean != 0: divided by their number; an empty sequence has ratio 0)
 *   margin[p] = beta (ratio[p] - ratio[n_pairs + p]) + offset[p]
 *   pair_loss[p] = (1 - smoothing) log(1 + exp(-margin)) + smoothing log(1 + exp(margin))
 *   loss = sum_p scale weight[p] pair_loss[p],   grad[t] = d loss / d logp[t]   (0 for tokens of no sequence)
 * ref_logp NULL = 0; mask (one byte per token, 0 = the token does not count: its logp and ref_logp are not looked at, grad 0) NULL = all
 * count; weight (>= 0; a pair of weight 0 adds nothing) NULL = 1; offset NULL = 0. margin, ratio and grad may be NULL. Sums are in 64 bits.
 * loss is one float, pair_loss and margin n_pairs, ratio 2 n_pairs, grad n_tokens. The workspace is never more than 16384 + 8 n_pairs bytes. */
int mlx_preference_loss_workspace(int64_t n_tokens, int64_t n_pairs, size_t *bytes);
int mlx_preference_loss(int32_t device, void *stream, const float *logp, const float *ref_logp, int64_t n_tokens, const int64_t *seq_ptr,
                        int64_t n_pairs, float beta, float smoothing, float scale, int32_t mean, const uint8_t *mask, const float *weight,
                        const float *offset, float *loss, float *pair_loss, float *margin, float *ratio, float *grad, void *workspace,
                        size_t workspace_bytes);

#ifdef __cplusplus
}
#endif
#endif /* MLEASE_OPERATORS_H */
