// Internal interface between the two halves of linear attention: the host
// checks and recurrent kernels (linear_attention.cu) and the tensor-core
// kernel for prompts (linear_attention_mma.cu).
#pragma once

#include <cuda_runtime.h>
#include <stddef.h>
#include <stdint.h>

#include "../../include/mamba_lm_ops.h"

namespace mamba_la {

// Whether the tensor-core kernel takes a prompt of this shape.
bool mma_takes(int64_t seqlen, int64_t dk, int64_t dv);

// Whether it runs only with a workspace: the fp32 sums of outputs of more than
// 128 keys, unless out itself can hold them.
bool mma_needs_workspace(int64_t dk, int32_t dtype);

// Workspace bytes the tensor-core kernel's plan uses for this shape on the
// current device (0: every sequence in one piece).
size_t mma_workspace_size(int64_t batch, int64_t seqlen, int64_t heads, int64_t dk, int64_t dv,
                          int32_t dtype);

// Enqueues the tensor-core kernel (and, with a workspace, the passes that
// split sequences). `workspace` is NULL or holds mma_workspace_size() bytes.
cudaError_t launch_mma(const mamba_linear_attention_args& a, void* workspace, cudaStream_t st);

// The kernel's error word (a bounded wait that gave up): its code, or -1 when
// it cannot be read; cleared when set.
int read_and_clear_error();

}  // namespace mamba_la
