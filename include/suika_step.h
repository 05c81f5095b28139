/*
 * suika_step.h -- operators of a training step over sharded state
 * (libsuika_reshard.so).
 *
 * Between two plan changes a job trains on the state that a reshard moves:
 * bf16 or f32 parameters, f32 master weights and Adam moments, with the
 * vocabulary of the embedding cut over the tensor-parallel ranks.  These are
 * the parts of a step that work on that state's own layouts:
 *
 *   sr_square_sum, sr_clip, sr_clip_norm, sr_adamw, sr_adamw_norm
 *       the gradients' global norm over all tensors of a share, clipping by
 *       it, and the AdamW update of every state field.  In the reference
 *       these are torch.optim.AdamW on the model's parameters
 *       (tasks/task.py:72-73, 94)
 *   sr_embedding, sr_embedding_grad
 *       rows of a vocabulary shard for the tokens that lie in it, and the
 *       gradient of its rows.  In the reference the embedding is an
 *       nn.Embedding (Suika/models/llama_model.py:108-157)
 *   sr_logprob, sr_logprob_grad, sr_logprob_pair, sr_logprob_pair_grad
 *       log probabilities of given tokens, entropy and the best alternatives
 *       from the head's logits, and the gradient of the logits
 *
 * Conventions
 *   - All device memory, workspaces included, belongs to the caller.
 *   - Calls are asynchronous and stream-ordered, allocate nothing, and keep
 *     nothing from one call for the next.  They launch kernels only, so they
 *     can be captured into a HIP graph; sr_adamw and sr_adamw_norm refuse
 *     (SR_EINVAL), because their step number is a host value.
 *   - Data may be aligned to its element size only.  Workspaces are aligned
 *     to 16 bytes.
 *   - Sums, statistics and updates are computed in 32 bits or more and
 *     rounded once, to nearest even, where they are stored.  Results do not
 *     depend on the order in which workgroups run.
 *   - Status codes are the sr_status values of suika_reshard.h;
 *     sr_last_error() describes the last failure.  Arguments are checked
 *     before anything is launched.  Element types are sr_dtype codes.
 */
#ifndef SUIKA_STEP_H
#define SUIKA_STEP_H

#include <stdint.h>

#include "suika_reshard.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Most elements of one array; most tokens, rows or columns of one call. */
#define SR_STEP_MAX_ELEMENTS ((uint64_t)1 << 34)
#define SR_STEP_MAX_ROWS ((uint64_t)1 << 23)

/* A dense array of n elements (n may be 0). */
typedef struct sr_array {
  void* data;
  uint64_t n;
  int32_t dtype;      /* SR_DT_F32, SR_DT_BF16 or SR_DT_F16 */
  int32_t reserved;   /* must be 0 */
} sr_array;

/*
 * The sum of the squares of all elements, in 64 bits: *sum on the device, and
 * its root, *norm, where norm is not NULL.  Ranks that hold other shards add
 * their sums before clipping.  workspace: sr_square_sum_workspace bytes.  *sum,
 * *norm and the workspace overlap nothing else (SR_EOVERLAP).
 */
int sr_square_sum_workspace(const sr_array* arrays, int32_t count, uint64_t* bytes);
int sr_square_sum(const sr_array* arrays, int32_t count, int32_t read_again, void* workspace, uint64_t workspace_bytes,
                  double* sum, float* norm, hipStream_t stream);

/*
 * dst[i] = src[i] * min(1, max_norm / (sqrt(*square_sum) + 1e-6)), array by
 * array.  dst NULL: in place, where a factor of 1 leaves the memory as it is.
 * Arrays that are written overlap no others, nor *square_sum or *norm (SR_EOVERLAP).
 * norm (may be NULL) gets sqrt(*square_sum).
 */
int sr_clip(const sr_array* src, const sr_array* dst, int32_t count, const double* square_sum, float max_norm,
            float* norm, hipStream_t stream);

/* The norm that gradients are clipped by: of a sum of squares on the device
 * (square_sum; sum and workspace are not used then), or, where square_sum is
 * NULL, of the call's own gradients, whose sum goes to *sum. */
typedef struct sr_norm {
  const double* square_sum;
  double* sum;
  void* workspace;          /* sr_square_sum_workspace bytes of the gradients */
  uint64_t workspace_bytes;
  float* norm;              /* gets the sum's root; may be NULL */
} sr_norm;

/* sr_clip by such a norm: the gradients' sum of squares and the clipping in one
 * call, whose arguments are all checked before the first launch. */
int sr_clip_norm(const sr_array* src, const sr_array* dst, int32_t count, float max_norm, const sr_norm* norm,
                 hipStream_t stream);

/* One parameter's fields.  param is the bf16 copy of an f32 weight (master),
 * NULL where the weight is the parameter itself. */
typedef struct sr_adamw_tensor {
  void* weight;          /* master, or the parameter: f32 or bf16 */
  void* exp_avg;
  void* exp_avg_sq;
  void* param;           /* bf16 copy, or NULL */
  const void* grad;      /* f32 or bf16 */
  uint64_t n;
  int32_t weight_dtype;  /* SR_DT_F32 or SR_DT_BF16 (no param then) */
  int32_t moment_dtype;  /* SR_DT_F32 or SR_DT_BF16 */
  int32_t grad_dtype;
  int32_t reserved;      /* must be 0 */
} sr_adamw_tensor;

typedef struct sr_adamw_options {
  double lr;
  double beta1;
  double beta2;
  double eps;
  double weight_decay;
  int64_t step;          /* number of this update, from 1 */
  double max_norm;       /* with square_sum or norm: the gradients are clipped to it */
} sr_adamw_options;

/*
 * One AdamW update in place (decoupled weight decay, bias corrections of
 * `step`).  square_sum: the sum that clipping goes by, on the device; NULL: no
 * clipping.  Fields that are written overlap no others, nor *square_sum
 * (SR_EOVERLAP).
 */
int sr_adamw(const sr_adamw_tensor* tensors, int32_t count, const sr_adamw_options* options, const double* square_sum,
             hipStream_t stream);

/* The same with the norm in the call: clipped by `norm`, or not where it is
 * NULL.  steps[i] is the number of tensors[i]'s update (a parameter that had no
 * gradient for a while has had fewer); steps NULL: options->step for all.  All
 * arguments are checked before the first launch. */
int sr_adamw_norm(const sr_adamw_tensor* tensors, const int64_t* steps, int32_t count,
                  const sr_adamw_options* options, const sr_norm* norm, hipStream_t stream);

/* The tokens and the shard of an embedding: row r of the shard is token
 * vocab_start + r.  Tokens outside the shard (negative ones among them) give
 * rows of zeros and no gradient.  Outputs overlap no inputs (SR_EOVERLAP). */
typedef struct sr_embedding_shape {
  const void* tokens;    /* SR_DT_I32 or SR_DT_I64, dense */
  int32_t token_dtype;
  int32_t dtype;         /* of the weight and of the outputs' gradient */
  uint64_t n_tokens;
  uint64_t rows;         /* of the shard */
  uint64_t cols;
  int64_t vocab_start;   /* 0 or more */
  float scale;
  int32_t reserved;      /* must be 0 */
} sr_embedding_shape;

/* out[i] = scale * weight[tokens[i] - vocab_start]; weight's rows are
 * weight_stride elements apart, out is dense and of the same type. */
int sr_embedding(const sr_embedding_shape* shape, const void* weight, uint64_t weight_stride, void* out,
                 hipStream_t stream);

/* grad[r] = scale * sum of grad_out[i] over the tokens of row r, in the order
 * of i, plus grad[r] where accumulate is not 0.  grad_out's rows are
 * grad_out_stride elements apart, grad is dense.  workspace:
 * sr_embedding_grad_workspace bytes. */
int sr_embedding_grad_workspace(const sr_embedding_shape* shape, uint64_t* bytes);
int sr_embedding_grad(const sr_embedding_shape* shape, const void* grad_out, uint64_t grad_out_stride, void* grad,
                      int32_t grad_dtype, int32_t accumulate, void* workspace, uint64_t workspace_bytes,
                      hipStream_t stream);

#define SR_LOGPROB_MAX_TOP 64

/* Logits of `rows` positions, `columns` each, of which the first `vocab` are
 * tokens (the rest pads the head). */
typedef struct sr_logprob_shape {
  const void* logits;
  const void* targets;   /* SR_DT_I32 or SR_DT_I64, dense */
  int32_t target_dtype;
  int32_t dtype;         /* SR_DT_F32, SR_DT_BF16 or SR_DT_F16 */
  uint64_t rows;
  uint64_t columns;
  uint64_t vocab;
  uint64_t stride;       /* elements between rows of logits */
} sr_logprob_shape;

/*
 * Per row: lse = ln sum exp(x), logprob = x[target] - lse, entropy, and the
 * `top` largest log probabilities in falling order with their columns (equal
 * logits: the lower column first).  A negative target is not scored: logprob
 * 0.  A target of vocab or more has logprob -inf.  A row whose logits are all
 * -inf has lse and logprobs -inf and entropy 0.  A row with NaN or +inf has NaN
 * statistics; its alternatives are ordered with NaN above +inf.  workspace:
 * sr_logprob_workspace bytes.
 */
int sr_logprob_workspace(const sr_logprob_shape* shape, int32_t top, uint64_t* bytes);
int sr_logprob(const sr_logprob_shape* shape, int32_t top, float* logprob, float* entropy, float* lse,
               float* top_logprob, int64_t* top_index, void* workspace, uint64_t workspace_bytes, hipStream_t stream);

/*
 * grad[row][j] = g_logprob[row] * ([j = target] - p_j)
 *                - g_entropy[row] * p_j * (ln p_j + entropy[row])
 * with p_j = exp(x_j - lse[row]); 0 in the padded columns, in rows that are
 * all -inf, and for the first term in rows that are not scored.  g_logprob or
 * g_entropy may be NULL (0).  grad has the logits' type and rows of
 * grad_stride elements; it may be the logits themselves, and overlaps no
 * other input (SR_EOVERLAP).  lse is rounded to a float32: beside the error of
 * the sum and of the exponential, p_j is off by up to |lse| 2^-24 of itself, so
 * logits of a large common offset want the pair below.
 */
int sr_logprob_grad(const sr_logprob_shape* shape, const float* lse, const float* entropy, const float* g_logprob,
                    const float* g_entropy, void* grad, uint64_t grad_stride, hipStream_t stream);

/*
 * The same with the log of the sum as two floats: lse_low is what the rounding
 * of lse lost (0 where lse is not finite), and p_j = exp((x_j - lse) - lse_low)
 * does not depend on a common offset of the logits.
 */
int sr_logprob_pair(const sr_logprob_shape* shape, int32_t top, float* logprob, float* entropy, float* lse,
                    float* lse_low, float* top_logprob, int64_t* top_index, void* workspace, uint64_t workspace_bytes,
                    hipStream_t stream);
int sr_logprob_pair_grad(const sr_logprob_shape* shape, const float* lse, const float* lse_low, const float* entropy,
                         const float* g_logprob, const float* g_entropy, void* grad, uint64_t grad_stride,
                         hipStream_t stream);

#ifdef __cplusplus
}
#endif

#endif /* SUIKA_STEP_H */
