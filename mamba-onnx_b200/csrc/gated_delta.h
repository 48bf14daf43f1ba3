// Internal interface between the two halves of the gated delta rule: the host
// checks and recurrent kernels (gated_delta.cu) and the tensor-core kernels
// for prompts (gated_delta_mma.cu).
#pragma once

#include <cuda_runtime.h>
#include <stddef.h>
#include <stdint.h>

#include "../../include/mamba_lm_ops.h"

namespace mamba_gd {

// Whether the tensor-core kernels take a prompt of this shape.
bool mma_takes(int64_t seqlen, int64_t dk, int64_t dv, int32_t dtype);

// Workspace bytes they use for this shape on the current device.
size_t mma_workspace_size(int64_t batch, int64_t seqlen, int64_t heads, int64_t dk, int64_t dv,
                          int32_t dtype);

// Enqueues them; `workspace` holds mma_workspace_size() bytes.
cudaError_t launch_mma(const mamba_gated_delta_args& a, void* workspace, cudaStream_t st);

// Their error word (a bounded wait that gave up): its code, or -1 when it
// cannot be read; cleared when set.
int read_and_clear_error();

}  // namespace mamba_gd
