/*
 * distlr_losses.h -- C-ABI of the softmax losses on device data (gfx950):
 * lib/libdistlr_losses.so.
 *
 * The many-class counterparts of the engine's margin / residual / log-loss
 * (lr.cc:35-40, 47-63), for models whose output layer is a softmax: the
 * log-probabilities of given classes and their gradient, the paired logistic
 * loss over sequences of them, the clipped policy loss, and log-probabilities
 * straight from hidden states and the output layer's weights.  (The reference
 * has no such calls.)
 *
 * Conventions
 *   - They need no dlr_ctx and keep no state.  Every array is DEVICE memory
 *     of HIP device `device`; the work is enqueued on `stream` (a hipStream_t
 *     of that device; NULL: its default stream) and the call returns without
 *     waiting.  Calls may be captured into a graph.  The calling thread's
 *     current device is unchanged on return.
 *   - Scratch memory is the caller's (dlr_logits_workspace,
 *     dlr_head_logprob_workspace; 256-byte aligned device memory, not
 *     initialised, free for other use once the call's work is done): two calls
 *     that may run at the same time, or two captured graphs that do, need two
 *     workspaces.
 *   - Rows: `data` (the hidden states, the weights) is row-major with
 *     contiguous elements in a row; rows start row_stride elements apart, at
 *     any alignment of the element type.
 *   - target: rows class indices (target_bits 32 or 64).  A NEGATIVE target
 *     marks a row that takes no part: its logits are not read (NaN there does
 *     no harm), its results are 0 and its gradient's row is 0.  A target >=
 *     vocab gives NaN (nothing is read out of range).
 *   - The arrays of a call do not overlap, except where a call says so.
 *   - -inf logits (classes masked out) have probability 0.  A row of -inf
 *     only has lse -inf and logprob NaN; NaN or +inf in a row make it NaN.
 *   - Row statistics are held in 32 bits and finished in 64; gradients are
 *     rounded to the logits' type once, to nearest.  Results do not depend on
 *     timing (no atomics): the same call gives the same bits.
 *   - Errors: DLR_E_ARG for arguments that do not fit (message through
 *     dlr_losses_last_error()), nothing is enqueued then; DLR_E_HIP if the launch
 *     fails.  rows = 0 is a valid call that does nothing.
 *   - Up to 2^31 - 1 rows; from 2^21 (dlr_head_logprob: 2^35 logits) on a
 *     call is several launches, which a failing one ends.
 *   - A library of its own: it needs neither the engine nor RCCL, and it
 *     shares its caller's HIP runtime, whose streams and tensors it takes.  It
 *     is linked to the name "libamdhip64.so", under which torch loads its
 *     runtime.  A process that also runs the engine imports torch before
 *     distlr_amd (libdistlr_amd.so then takes torch's runtime too): of two HIP
 *     runtimes in a process only one sees the GPU.
 */
#ifndef DISTLR_LOSSES_H_
#define DISTLR_LOSSES_H_

#include <stddef.h>
#include <stdint.h>

#include "distlr_amd.h" /* DLR_OK, DLR_E_* */

#ifdef __cplusplus
extern "C" {
#endif

/* The message of the calling thread's last failure in this library. */
const char *dlr_losses_last_error(void);
/* The file of the HIP runtime this library is bound to. */
const char *dlr_losses_runtime(void);

#define DLR_DTYPE_F32 0
#define DLR_DTYPE_BF16 1
#define DLR_DTYPE_F16 2

/* z[t][j] = data[t * row_stride + j], t < rows, j < vocab; probabilities are
 * softmax(z / temperature). */
typedef struct dlr_logits {
    const void *data;
    const void *target;     /* rows class indices; < 0: the row takes no part */
    int64_t rows;
    int64_t vocab;          /* classes, 1 .. 2^30                             */
    int64_t row_stride;     /* elements, >= vocab (0: one row for all)        */
    int32_t dtype;          /* DLR_DTYPE_*                                    */
    int32_t target_bits;    /* 32 or 64                                       */
    double temperature;     /* 1e-6 .. 1e6                                    */
} dlr_logits;

/* Bytes of the scratch memory of dlr_token_logprob and dlr_policy_loss, or < 0:
 * 0 (then the workspace may be NULL) but for few long rows, at most 128 of
 * 32,768 classes and more, whose chunks meet there. */
int64_t dlr_logits_workspace(int64_t rows, int64_t vocab, int dtype);

/* lse[t] = log sum_j exp(z_tj / temperature), logprob[t] = z_ty / temperature
 * - lse[t], y = target[t].  Each logit is read once. */
int dlr_token_logprob(int device, void *stream, const dlr_logits *x, void *workspace, int64_t workspace_bytes,
                      float *logprob, float *lse);

/* The gradient of sum_t grad[t] * logprob[t] with respect to the logits (the
 * softmax residual): grad_logits[t][j] = grad[t] / temperature * (1[j = y] -
 * exp(z_tj / temperature - lse[t])), in the logits' type, rows
 * grad_row_stride (>= vocab) elements apart.  lse is dlr_token_logprob's, or of
 * more classes than these (of which target[t] is one).  32 bits are coarse for
 * an lse beyond +-128: one that is the row's own up to its last bit is taken
 * again from the row, any other as it is given.  A row with grad[t] = 0 is 0
 * whatever its logits hold.  grad_logits may be x->data itself with the same
 * stride (the logits are then overwritten); any other overlap is refused (rows
 * between the logits' rows, at the same stride, are none). */
int dlr_token_logprob_grad(int device, void *stream, const dlr_logits *x, const float *lse, const float *grad,
                           void *grad_logits, int64_t grad_row_stride);

/* The clipped policy loss.  Per row, with l = logprob[t], A = advantage[t]:
 *   ratio   = exp(l - old_logprob[t])
 *   kl      = exp(ref_logprob[t] - l) - (ref_logprob[t] - l) - 1
 *   loss[t] = -min(ratio A, clip(ratio, 1 - clip_low, 1 + clip_high) A) + kl_coef kl
 * The objective is sum_t weight[t] * loss[t]; grad_logits is its gradient.
 * A row of weight 0 takes no part (like a negative target).  clipped[t] = 1
 * where the clip holds the surrogate (its gradient is 0 there).  One pass over
 * the logits, which are read once where a row fits a CU's registers. */
typedef struct dlr_policy {
    const float *old_logprob;   /* rows                                       */
    const float *ref_logprob;   /* rows; NULL: no KL term (kl_coef must be 0) */
    const float *advantage;     /* rows                                       */
    const float *weight;        /* rows; NULL: 1                              */
    double clip_low;            /* in [0, 1]                                  */
    double clip_high;           /* >= 0                                       */
    double kl_coef;             /* >= 0                                       */
} dlr_policy;
/* loss, logprob, kl, clipped: rows each.  grad_logits: NULL for no gradient,
 * else as for dlr_token_logprob_grad (x->data itself is allowed). */
int dlr_policy_loss(int device, void *stream, const dlr_logits *x, const dlr_policy *p, void *workspace,
                    int64_t workspace_bytes, float *loss, float *logprob, float *kl, uint8_t *clipped,
                    void *grad_logits, int64_t grad_row_stride);

/* The paired logistic (preference) loss over packed ragged sequences.
 * Sequence i is tokens [offsets[i], offsets[i+1]); sequences 0 .. pairs-1
 * are the preferred ones, pairs .. 2 pairs - 1 the others, pair by pair.
 *   score_i  = sum over i's tokens with mask: logprob - ref_logprob
 *   reward_i = beta * score_i  (average: / max(1, its tokens with mask))
 *   u        = reward_p - reward_{pairs+p} - margin
 *   loss[p]  = -(1 - label_smoothing) log sigma(u) - label_smoothing log sigma(-u)
 * The objective is sum_p weight[p] * loss[p]; grad is its gradient with
 * respect to logprob: tokens without mask and tokens of no sequence get 0,
 * whatever their log-probabilities hold.  A sequence that leaves the tokens
 * gives NaN for its pair and its pair's tokens; offsets that descend anywhere
 * (sequences would overlap) give NaN for every pair and token. */
typedef struct dlr_preference {
    const float *logprob;       /* tokens                                     */
    const float *ref_logprob;   /* tokens; NULL: 0                            */
    const uint8_t *mask;        /* tokens, 0 = does not count; NULL: all do   */
    const int64_t *offsets;     /* 2 * pairs + 1, ascending                   */
    const float *weight;        /* pairs; NULL: 1                             */
    int64_t pairs;              /* 0 .. 2^22 - 1                              */
    int64_t tokens;             /* 0 .. 2^40                                  */
    double beta;                /* > 0                                        */
    double label_smoothing;     /* in [0, 1]                                  */
    double margin;
    int32_t average;            /* 1: rewards per counted token               */
    int32_t reserved;
} dlr_preference;
/* loss, chosen_reward, rejected_reward: pairs each.  grad: tokens, or NULL. */
int dlr_preference_loss(int device, void *stream, const dlr_preference *p, float *loss, float *chosen_reward,
                        float *rejected_reward, float *grad);

/* dlr_token_logprob of the logits hidden . head^T, which are never written
 * out: for scoring (a reference model's or an earlier policy's
 * log-probabilities); there is no gradient.  DLR_DTYPE_BF16 or DLR_DTYPE_F16
 * (hidden and head alike), products and sums in 32 bits on the matrix cores. */
typedef struct dlr_head {
    const void *hidden;         /* rows x dim                                 */
    const void *head;           /* vocab x dim: one row of weights per class  */
    const void *target;
    int64_t rows, vocab, dim;   /* vocab 1 .. 2^28, dim 1 .. 2^20,            */
                                /* rows * vocab <= 2^44                       */
    int64_t hidden_stride;      /* elements between rows                      */
    int64_t head_stride;
    int32_t dtype;
    int32_t target_bits;
    double temperature;
} dlr_head;
/* Bytes of dlr_head_logprob's scratch memory, or < 0. */
int64_t dlr_head_logprob_workspace(int64_t rows, int64_t vocab, int64_t dim);
int dlr_head_logprob(int device, void *stream, const dlr_head *h, void *workspace, int64_t workspace_bytes,
                     float *logprob, float *lse);

#ifdef __cplusplus
}
#endif

#endif /* DISTLR_LOSSES_H_ */
