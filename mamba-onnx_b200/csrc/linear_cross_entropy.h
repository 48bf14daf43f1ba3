// Internal interface of the loss from hidden states (linear_cross_entropy.cu, and
// linear_cross_entropy_few.cu for a few rows).
#pragma once

#include <cuda_runtime.h>
#include <stddef.h>
#include <stdint.h>

#include "../../include/mamba_lm_ops.h"
#include "scan_device.cuh"

namespace mamba_lce {

constexpr float kLog2e = 1.4426950408889634f;

// What exponents are taken relative to where the largest logit so far is m: -inf,
// of no logit or of logits of -inf alone, leaves sums of 0, not of inf - inf.
__device__ __forceinline__ float finite_max(float m) { return m == -INFINITY ? 0.f : m; }

// (m, s), a largest logit and the sum of exp(z - m), joined with another's.
__device__ __forceinline__ void merge_sums(float& m, float& s, float om, float os) {
  const float top = fmaxf(m, om), from = finite_max(top);
  s = s * mamba_scan::ex2_approx((m - from) * kLog2e) +
      os * mamba_scan::ex2_approx((om - from) * kLog2e);
  m = top;
}

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
