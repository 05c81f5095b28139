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
 *   sr_ffn, sr_ffn_grad
 *       the gated feed-forward block of a share and its gradients.  In the
 *       reference it is the blocks' mlp, gate and up column parallel and down
 *       row parallel (Suika/models/llama_model.py:16-35)
 *   sr_orthogonalize, sr_muon
 *       matrices made orthogonal by Newton-Schulz products, and the Muon update
 *       of a share's matrices, beside the reference's torch.optim.AdamW
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

/* Activations: a s(a), a Phi(a) and a s(2 z) with z = sqrt(2/pi) (a + 0.044715
 * a^3), where s(a) = 1 / (1 + exp(-a)) and Phi is the normal distribution. */
#define SR_ACT_SILU 0
#define SR_ACT_GELU 1
#define SR_ACT_GELU_TANH 2

/* A gated feed-forward block: x [tokens][hidden], this rank's rows of gate and
 * up [ffn][hidden] and columns of down [hidden][ffn], of one type, with rows of
 * dense elements `*_stride` apart.  hidden and ffn are at most 2^20, and any of
 * the three sizes may be 0. */
typedef struct sr_ffn_shape {
  const void* x;
  const void* gate;
  const void* up;
  const void* down;
  uint64_t tokens;
  uint64_t hidden;
  uint64_t ffn;
  uint64_t x_stride;
  uint64_t gate_stride;
  uint64_t up_stride;
  uint64_t down_stride;
  int32_t dtype;        /* SR_DT_F32, SR_DT_BF16 or SR_DT_F16 */
  int32_t activation;   /* SR_ACT_* */
} sr_ffn_shape;

/*
 * out = (act(x gate^T) * (x up^T)) down^T, dense [tokens][hidden]; the ranks'
 * outputs add up.  The product in brackets is rounded to the operands' type on
 * the way, sums are in 32 bits.  gate_out and up_out (both or neither, floats,
 * dense [tokens][ffn]) keep x gate^T and x up^T for sr_ffn_grad.  workspace:
 * sr_ffn_workspace bytes, for a call that keeps them or does not.  What is
 * written overlaps nothing else (SR_EOVERLAP).
 */
int sr_ffn_workspace(const sr_ffn_shape* shape, int32_t keep, uint64_t* bytes);
int sr_ffn(const sr_ffn_shape* shape, void* out, float* gate_out, float* up_out, void* workspace,
           uint64_t workspace_bytes, hipStream_t stream);

/* Where the gradients go, dense; NULL: not wanted. */
typedef struct sr_ffn_grads {
  void* x;        /* [tokens][hidden] */
  void* gate;     /* [ffn][hidden] */
  void* up;       /* [ffn][hidden] */
  void* down;     /* [hidden][ffn] */
} sr_ffn_grads;

/*
 * The gradients of a block from that of its output (grad_out, rows
 * grad_out_stride apart) and what sr_ffn kept.  The gradients of the two
 * projections are rounded to the operands' type on the way, sums are in 32
 * bits.  workspace: sr_ffn_grad_workspace bytes for the same gradients.  What
 * is written overlaps nothing else (SR_EOVERLAP).
 */
int sr_ffn_grad_workspace(const sr_ffn_shape* shape, const void* grad_out, uint64_t grad_out_stride,
                          const sr_ffn_grads* grads, uint64_t* bytes);
int sr_ffn_grad(const sr_ffn_shape* shape, const float* gate_out, const float* up_out, const void* grad_out,
                uint64_t grad_out_stride, const sr_ffn_grads* grads, void* workspace, uint64_t workspace_bytes,
                hipStream_t stream);

#define SR_MAX_NEWTON_SCHULZ 64

/* Sums count values (SR_DT_F32 or SR_DT_F64) at data over the ranks, in place
 * and in the order of the stream.  Not 0: the call ends with SR_EINVAL. */
typedef int (*sr_reduce)(void* context, void* data, uint64_t count, int32_t dtype, hipStream_t stream);

/* X = G / max(|G|, eps) with the norm of all elements, then steps times X <-
 * a X + b (X X^T) X + c (X X^T)^2 X, with a, b and c from coefficients
 * [steps][3].  The singular values of X, 1 at most at first, have to stay at
 * 1.9 or less, and a + b s^2 + c s^4 within +-15 (SR_EINVAL).  Values of X below
 * 2^-38 count as 0. */
typedef struct sr_newton_schulz {
  int32_t steps;                /* 1 to SR_MAX_NEWTON_SCHULZ */
  int32_t reserved;             /* must be 0 */
  const double* coefficients;   /* in host memory */
  double eps;
  sr_reduce reduce;             /* NULL: no matrix is split */
  void* reduce_context;
} sr_newton_schulz;

/* A matrix with rows of dense elements.  split: -1, or the dimension (0: rows,
 * 1: columns) that is cut over the ranks, of which this is one's part.  All
 * ranks then call with the same list, and reduce is called equally often on
 * each, also where a part has no elements. */
typedef struct sr_matrix {
  void* data;
  uint64_t rows;
  uint64_t cols;
  uint64_t stride;    /* elements between rows */
  int32_t dtype;      /* SR_DT_F32, SR_DT_BF16 or SR_DT_F16 */
  int32_t split;
} sr_matrix;

/*
 * dst[i] = the last X of G = src[i]; sides of at most 2^19.  Products are of 22
 * bits a value in sums of 32 bits.  A matrix may be its own result; otherwise
 * what is written overlaps nothing else (SR_EOVERLAP).  workspace:
 * sr_orthogonalize_workspace bytes: 8 for a value of X and 8 for one of X X^T, of as
 * many matrices as go through the steps together, 48 with 8 GiB of these at most, or
 * one.  Of split matrices 12 for a value of X X^T, the 8 GiB are of these alone and
 * X's come on top.  split of dst is not read.
 */
int sr_orthogonalize_workspace(const sr_matrix* src, const sr_matrix* dst, int32_t count, const sr_newton_schulz* ns,
                               uint64_t* bytes);
int sr_orthogonalize(const sr_matrix* src, const sr_matrix* dst, int32_t count, const sr_newton_schulz* ns, void* workspace,
                     uint64_t workspace_bytes, hipStream_t stream);

/* One parameter's fields, dense [rows][cols]; param as in sr_adamw_tensor. */
typedef struct sr_muon_tensor {
  void* weight;          /* master, or the parameter: f32 or bf16 */
  void* exp_avg;
  void* param;           /* bf16 copy, or NULL */
  const void* grad;
  uint64_t rows;
  uint64_t cols;
  double scale;          /* of this matrix's update, times lr */
  int32_t weight_dtype;  /* SR_DT_F32 or SR_DT_BF16 (no param then) */
  int32_t moment_dtype;  /* SR_DT_F32 or SR_DT_BF16 */
  int32_t grad_dtype;    /* SR_DT_F32 or SR_DT_BF16 */
  int32_t split;         /* as in sr_matrix */
  int64_t reserved;      /* must be 0 */
} sr_muon_tensor;

typedef struct sr_muon_options {
  double lr;
  double weight_decay;
  double momentum;
  int32_t nesterov;
  int32_t reserved;           /* must be 0 */
  double max_norm;            /* with square_sum: the gradients are clipped to it */
  const double* square_sum;   /* as for sr_adamw */
} sr_muon_options;

/*
 * One Muon update in place: exp_avg = momentum exp_avg + (1 - momentum) g; G =
 * momentum exp_avg + (1 - momentum) g with nesterov, else exp_avg, as it is
 * stored; weight = weight (1 - lr weight_decay) - lr scale X with the last X of
 * G.  Fields that are written overlap no others (SR_EOVERLAP).  It holds no
 * step number and can be captured where reduce can.  Where a reduce fails, all
 * moments are updated, and of the weights those of matrices that are not split
 * and of groups of split ones that came before (at most 48 matrices go through
 * the steps together), each as a whole.  workspace: sr_muon_workspace bytes; that
 * call makes all of sr_muon's checks.
 */
int sr_muon_workspace(const sr_muon_tensor* tensors, int32_t count, const sr_muon_options* options, const sr_newton_schulz* ns,
                      uint64_t* bytes);
int sr_muon(const sr_muon_tensor* tensors, int32_t count, const sr_muon_options* options, const sr_newton_schulz* ns,
            void* workspace, uint64_t workspace_bytes, hipStream_t stream);

#ifdef __cplusplus
}
#endif

#endif /* SUIKA_STEP_H */
