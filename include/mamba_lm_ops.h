/*
 * mamba_lm_ops.h — operators of recurrent language models beside the
 * selective scan: linear attention with a decay for each head and the gated
 * delta rule (a prompt, and one token at a time), the log probabilities of
 * given tokens, and the loss of a language model's head with its gradients.
 *
 * Not part of the reference's plugin interface (the reference ships only the
 * scan op). Same conventions as mamba_scan.h: DEVICE pointers, enqueued on
 * `stream` (a cudaStream_t; NULL = the legacy default stream) of the current
 * device, nothing allocated, a mamba_scan_status returned and
 * mamba_scan_last_error() describing a failure (nothing enqueued then).
 * Addresses are multiples of their element's size.
 */
#ifndef MAMBA_LM_OPS_H_
#define MAMBA_LM_OPS_H_

#include <stddef.h>
#include <stdint.h>

#include "mamba_scan.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Element types of the tensors declared `const void*` below. */
typedef enum mamba_dtype {
  MAMBA_DTYPE_F32 = 0,
  MAMBA_DTYPE_F16 = 1,
  MAMBA_DTYPE_BF16 = 2,
} mamba_dtype;

/*
 * Linear attention with a decay for each head, over whole sequences:
 *   S[b,h,t] = exp(log_decay[b,t,h]) S[b,h,t-1] + k[b,t,g] v[b,t,h]^T
 *   out[b,t,h] = scale * q[b,t,g] S[b,h,t]
 * with a dk x dv state S for each sequence and head, S[b,h,-1] = h0[b,h] (0
 * when h0 is NULL), and head h reading the queries and keys of group g =
 * h / (heads / groups) (groups divides heads).
 *
 * q, k are [batch][seqlen][groups][dk], v is [batch][seqlen][heads][dv], of
 * type `dtype`, the last dimension contiguous and the others with any
 * non-negative strides (in elements). log_decay is float32 with any
 * non-negative strides over [batch][seqlen][heads] (0, 0, 1: one fixed decay
 * for each head): values at most 0 in ordinary use; -inf clears the state.
 * The state is kept in fp32. out is [batch][seqlen][heads][dv], contiguous, of
 * type `dtype`; h0 and h_last (NULL: not written) are fp32
 * [batch][heads][dk][dv], contiguous.
 *
 * lengths (NULL: all seqlen): [batch] int32, clamped to 0..seqlen. What rows at
 * or past lengths[b] hold does not matter (up to 63 of them may be read, within
 * seqlen, and are not used), their out rows are set to 0, and h_last[b] is the
 * state after the last row that counts (h0[b], or 0, for a length of 0).
 *
 * Accuracy. Up to 16 rows (32 with dk over 128) run in fp32 throughout. Longer
 * prompts go through tensor-core products of half-precision parts with fp32
 * sums: relative to the sum of the magnitudes an output or state element adds
 * up, about 2^-20 for float32 tensors (operands, scores and states of 22 bits)
 * and 2^-16 for 16-bit ones (scores and states of at least 16 bits), before the
 * one rounding of a 16-bit output; the state itself stays fp32 for every type.
 * Except for bf16 tensors with 16-byte aligned rows and dk up to 128, very
 * uneven rows add an absolute error: operands keep to 2^-39 of the largest
 * element of their row (q, k), of the largest |k||v| of 64 rows (v), of the
 * largest element of their column (the state), so with elements of q, k or v
 * more than about 2^17 times smaller than others that meet zeros in the
 * product, what the small ones contribute is not exact to 22 bits.
 *
 * The address ranges of out and h_last must not overlap the inputs', each
 * other's or the workspace's.
 * q, k, v, log_decay and h0 have to be finite where they count (log_decay may
 * be -inf): one infinity or NaN spoils the outputs of its sequence and head,
 * up to 63 rows before it among them. dk and dv: 1..256. All strides are in
 * elements, the order [batch, row, group or head].
 */
typedef struct mamba_linear_attention_args {
  const void* q;
  const void* k;
  const void* v;
  const float* log_decay;
  const float* h0;
  const int32_t* lengths;
  void* out;
  float* h_last;
  int64_t batch, seqlen, heads, groups, dk, dv;
  int64_t q_stride[3];
  int64_t k_stride[3];
  int64_t v_stride[3];
  int64_t decay_stride[3];
  float scale;
  int32_t dtype; /* mamba_dtype of q, k, v, out */
} mamba_linear_attention_args;

/*
 * Workspace bytes mamba_linear_attention uses for this shape when it gets
 * them: nonzero when there are too few (sequence, head) pairs to fill the
 * GPU, so that each sequence is split into segments whose states are joined
 * through the workspace, and for 16-bit outputs of more than 128 keys, whose
 * two halves are added there in fp32 (4 bytes for each element of out;
 * without it the recurrence runs token by token, about ten times slower).
 * Depends on the current device's SM count. 0 for a bad shape.
 */
MAMBA_SCAN_API size_t mamba_linear_attention_workspace_size(int64_t batch, int64_t seqlen,
                                                            int64_t heads, int64_t groups,
                                                            int64_t dk, int64_t dv, int32_t dtype);

/*
 * workspace: NULL, to run each sequence in one piece, or at least
 * mamba_linear_attention_workspace_size() bytes, 16-byte aligned, its
 * contents not needing initialisation (fewer bytes: MAMBA_SCAN_ERR_WORKSPACE).
 * Calls that share a workspace must be ordered on the GPU. The result is
 * deterministic for one choice of workspace.
 */
MAMBA_SCAN_API int mamba_linear_attention(const mamba_linear_attention_args* args, void* workspace,
                                          size_t workspace_bytes, void* stream);

/*
 * One token of the same recurrence for each sequence:
 *   state_out[b,h] = exp(log_decay[b,h]) state[b,h] + k[b,g] v[b,h]^T
 *   out[b,h] = scale * q[b,g] state_out[b,h]
 * q, k [batch][groups][dk] and v [batch][heads][dv] with the last dimension
 * contiguous and strides (in elements) for the other two; log_decay float32
 * with strides over [batch][heads] (0, 1: one decay for each head); state and
 * state_out fp32 [batch][heads][dk][dv], contiguous; state_out may be state
 * itself (updated in place) and must not overlap it otherwise; out
 * [batch][heads][dv], contiguous, of type `dtype`. Neither out nor state_out
 * may overlap another argument.
 */
typedef struct mamba_linear_attention_step_args {
  const void* q;
  const void* k;
  const void* v;
  const float* log_decay;
  const float* state;
  float* state_out;
  void* out;
  int64_t batch, heads, groups, dk, dv;
  int64_t q_stride[2];
  int64_t k_stride[2];
  int64_t v_stride[2];
  int64_t decay_stride[2];
  float scale;
  int32_t dtype;
} mamba_linear_attention_step_args;

MAMBA_SCAN_API int mamba_linear_attention_step(const mamba_linear_attention_step_args* args,
                                               void* stream);

/*
 * The gated delta rule: linear attention whose state forgets by a factor for
 * each head and replaces, instead of adding to, what it holds under a key:
 *   S'       = exp(log_decay[b,t,h]) S[b,h,t-1]
 *   S[b,h,t] = S' + beta[b,t,h] k[b,t,g] (v[b,t,h] - k[b,t,g] S')^T
 *   out[b,t,h] = scale * q[b,t,g] S[b,h,t]
 * Shapes, strides, groups, types, states and lengths are those of
 * mamba_linear_attention (so both may serve layers of one model); beta is
 * float32 with any non-negative strides over [batch][seqlen][heads]. The rule
 * is meant for keys of norm 1 and beta in 0..1 (up to 2 is stable); with
 * beta |k|^2 above 2 the recurrence itself grows from token to token. Rows at
 * or past a length may be read (up to the next 63 before seqlen) and have no
 * effect, whatever they hold.
 *
 * Accuracy. Up to 16 rows (48 of float32), dk over 128, and calls without a
 * workspace run token by token in fp32. Longer prompts run in chunks of 64 rows
 * through tensor-core products of half-precision parts with fp32 sums, the inverse
 * of a chunk's triangular system among them, every operand to 22 bits, those of
 * 16-bit tensors to 21: nearly as mamba_linear_attention for float32 tensors,
 * whatever the type, before the one rounding of a 16-bit output. The parts keep
 * to 2^-39 of the largest element of their row of q or k, of a chunk's scores or
 * its inverse, and of their column of the state, the values or the updates of a
 * chunk: with positive decays, all bits of all factors while a state grows no more
 * than 2^17 within 64 rows (what grows more, token by token).
 * q, k, v, beta and h0 have to be finite where they count, log_decay too or
 * -inf: one infinity or NaN spoils the outputs of its sequence and head, up to
 * 63 rows before it among them.
 */
typedef struct mamba_gated_delta_args {
  const void* q;
  const void* k;
  const void* v;
  const float* log_decay;
  const float* beta;
  const float* h0;
  const int32_t* lengths;
  void* out;
  float* h_last;
  int64_t batch, seqlen, heads, groups, dk, dv;
  int64_t q_stride[3];
  int64_t k_stride[3];
  int64_t v_stride[3];
  int64_t decay_stride[3];
  int64_t beta_stride[3];
  float scale;
  int32_t dtype; /* mamba_dtype of q, k, v, out */
} mamba_gated_delta_args;

/*
 * Workspace bytes mamba_gated_delta_rule uses for this shape on the current
 * device: the inverses, scores and weights of the chunks in flight. 0 when
 * it needs none, and for a bad shape.
 */
MAMBA_SCAN_API size_t mamba_gated_delta_rule_workspace_size(int64_t batch, int64_t seqlen,
                                                            int64_t heads, int64_t groups,
                                                            int64_t dk, int64_t dv, int32_t dtype);

/*
 * workspace: NULL, to run token by token, or at least
 * mamba_gated_delta_rule_workspace_size() bytes, 16-byte aligned, its contents
 * not needing initialisation (fewer bytes: MAMBA_SCAN_ERR_WORKSPACE). Calls
 * that share a workspace must be ordered on the GPU. No address range of out,
 * h_last and workspace may overlap another argument's. The result is
 * deterministic for one choice of workspace.
 */
MAMBA_SCAN_API int mamba_gated_delta_rule(const mamba_gated_delta_args* args, void* workspace,
                                          size_t workspace_bytes, void* stream);

/*
 * One token of the same recurrence for each sequence, in fp32: shapes as in
 * mamba_linear_attention_step, beta float32 with strides over [batch][heads].
 * state_out may be state itself and must not overlap it otherwise; neither out
 * nor state_out may overlap another argument.
 */
typedef struct mamba_gated_delta_step_args {
  const void* q;
  const void* k;
  const void* v;
  const float* log_decay;
  const float* beta;
  const float* state;
  float* state_out;
  void* out;
  int64_t batch, heads, groups, dk, dv;
  int64_t q_stride[2];
  int64_t k_stride[2];
  int64_t v_stride[2];
  int64_t decay_stride[2];
  int64_t beta_stride[2];
  float scale;
  int32_t dtype;
} mamba_gated_delta_step_args;

MAMBA_SCAN_API int mamba_gated_delta_rule_step(const mamba_gated_delta_step_args* args,
                                               void* stream);

/* Most alternatives mamba_token_logprobs returns for a row. */
#define MAMBA_LOGPROBS_MAX_TOP 64

/*
 * Log probabilities under softmax(logits[r]) for each of `rows` rows of
 * `vocab` logits (type `dtype`, row_stride elements apart, row_stride >=
 * vocab or 0):
 *   logprob[r] = logits[r][target[r]] - log(sum_i exp(logits[r][i]))
 *   entropy[r] = -sum_i p_i log p_i, with 0 log 0 = 0
 *   top_logprob[r][0..top), top_id[r][0..top): the `top` largest logits' log
 *     probabilities and ids, in falling order, equal logits by rising id
 * target [rows] int64: a negative one gives logprob 0 (padding), one past the
 * vocabulary gives NaN. logprob, entropy [rows] and top_logprob [rows][top]
 * are fp32, top_id [rows][top] int64; each output may be NULL (top_logprob
 * and top_id together), and so may target when logprob is. Logits of -inf
 * have probability 0 (their top_logprob is -inf); a row of -inf alone, or one
 * with a NaN or +inf, has no distribution: its logprob (of a target within
 * the vocabulary), entropy and top_logprob are NaN, and its top_id are
 * ordered with NaN above +inf, equal ones by rising id. vocab: 1..2^30; top:
 * 0..min(vocab, 64). No output may overlap an input or another output. Sums
 * are fp32, of terms scaled by the row's maximum; deterministic. Where a row's
 * `top` largest are not told apart from more than 1000 others (a mask that
 * leaves fewer tokens than `top`, one value nearly everywhere), it is read once
 * for each alternative.
 */
MAMBA_SCAN_API int mamba_token_logprobs(const void* logits, int64_t row_stride, int32_t dtype,
                                        const int64_t* target, float* logprob, float* entropy,
                                        float* top_logprob, int64_t* top_id, int64_t rows,
                                        int64_t vocab, int64_t top, void* stream);

/*
 * The loss of a language model from its last hidden states and the weights of
 * its head, the logits z[r][v] = hidden[r] . weight[v] formed a tile at a time
 * and never stored:
 *   loss[r] = log(sum_v exp(z[r][v])) - z[r][target[r]]
 * hidden [rows][width] and weight [vocab][width], of type `dtype`, rows
 * contiguous and hidden_stride, weight_stride (>= width) elements apart;
 * target [rows] int64: a negative one marks a row that does not count (loss 0;
 * whatever its hidden state holds leaves no trace), one past the vocabulary
 * gives NaN. loss [rows] fp32. stats [rows][2] fp32, contiguous: the row's
 * largest logit and sum_v exp(z[r][v] - it), which the gradients need (and
 * log(stats[1]) + stats[0] is the normaliser); NULL: not wanted. Logits,
 * statistics and sums are fp32; 16-bit operands enter the products as they
 * are, float32 ones in two half-precision parts scaled by a power of two (22
 * bits; the parts keep to 2^-39 of a matrix's largest finite element, and a logit
 * of an infinite one is NaN), or, for few rows, as they are.
 * Deterministic. rows: 0..2^31-257, vocab: 1..2^30, width: 1..65536. No output
 * may overlap an input, another output or the workspace.
 */
typedef struct mamba_linear_cross_entropy_args {
  const void* hidden;
  const void* weight;
  const int64_t* target;
  float* loss;
  float* stats;
  int64_t rows, vocab, width;
  int64_t hidden_stride, weight_stride;
  int32_t dtype; /* mamba_dtype of hidden, weight and their gradients */
  int32_t reserved; /* 0 */
} mamba_linear_cross_entropy_args;

/* Workspace bytes mamba_linear_cross_entropy uses on the current device (0 for
 * bad arguments): partial sums of the vocabulary's tiles, the operands' parts
 * for float32, and a copy of an operand whose rows do not start at 16 bytes. */
MAMBA_SCAN_API size_t
mamba_linear_cross_entropy_workspace_size(const mamba_linear_cross_entropy_args* args);

/* workspace: that many bytes, 16-byte aligned, not needing initialisation
 * (fewer: MAMBA_SCAN_ERR_WORKSPACE). Calls that share one must be ordered on
 * the GPU. */
MAMBA_SCAN_API int mamba_linear_cross_entropy(const mamba_linear_cross_entropy_args* args,
                                              void* workspace, size_t workspace_bytes,
                                              void* stream);

/*
 * Its gradients: with p = softmax(z) and dz[r][v] = grad[r] (p[r][v] - [v =
 * target[r]]),
 *   d_hidden = dz weight,   d_weight = dz^T hidden,
 * contiguous, of type `dtype`; either may be NULL. `forward` as for the loss
 * (its loss is not used, stats are those the loss gave); grad [rows] fp32 with
 * grad_stride >= 0 elements between rows. dz goes through the products in
 * pieces of the vocabulary, relative to the largest finite |grad| and rounded to the
 * operands' type (bf16: 2^-8 of each; fp16: 2^-11, and 2^-39 absolute; float32:
 * two half-precision parts; fp32 for few rows); sums are fp32 with one rounding at
 * the end. Rows that do not count add nothing and have d_hidden 0. Deterministic.
 */
typedef struct mamba_linear_cross_entropy_grad_args {
  mamba_linear_cross_entropy_args forward;
  const float* grad;
  int64_t grad_stride;
  void* d_hidden;
  void* d_weight;
} mamba_linear_cross_entropy_grad_args;

MAMBA_SCAN_API size_t mamba_linear_cross_entropy_grad_workspace_size(
    const mamba_linear_cross_entropy_grad_args* args);

MAMBA_SCAN_API int mamba_linear_cross_entropy_grad(
    const mamba_linear_cross_entropy_grad_args* args, void* workspace, size_t workspace_bytes,
    void* stream);

#ifdef __cplusplus
}
#endif

#endif /* MAMBA_LM_OPS_H_ */
