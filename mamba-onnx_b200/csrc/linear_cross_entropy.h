// Internal interface of the loss from hidden states (linear_cross_entropy.cu, and
// linear_cross_entropy_few.cu for a few rows).
#pragma once

#include <cuda_runtime.h>
#include <stddef.h>
#include <stdint.h>

#include "../../include/mamba_lm_ops.h"

namespace mamba_lce {

// The kernels' error word (a bounded wait that gave up): its code, or -1 when
// it cannot be read; cleared when set.
int read_and_clear_error();

// Partial (m, s) [part][row] and the targets' logits -> loss and (unless NULL) stats.
cudaError_t launch_combine(const float2* partial, const float* target_logit, const int64_t* target,
                           float* loss, float* stats, int rows, int parts, int64_t vocab,
                           cudaStream_t st);

// Whether a call has few rows, its workspace and its launches.
bool few_rows(const mamba_linear_cross_entropy_args& a, bool grad);
size_t few_forward_bytes(const mamba_linear_cross_entropy_args& a);
size_t few_grad_bytes(const mamba_linear_cross_entropy_grad_args& g);
cudaError_t few_forward(const mamba_linear_cross_entropy_args& a, void* workspace, cudaStream_t st);
cudaError_t few_backward(const mamba_linear_cross_entropy_grad_args& g, void* workspace,
                         cudaStream_t st);

}  // namespace mamba_lce
