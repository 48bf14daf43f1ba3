/*
 * mamba_lm_ops.h — operators of recurrent language models beside the
 * selective scan: linear attention with a decay for each head (a prompt, and
 * one token at a time) and the log probabilities of given tokens.
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

#ifdef __cplusplus
}
#endif

#endif /* MAMBA_LM_OPS_H_ */
