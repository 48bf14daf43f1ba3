// Log probabilities of given tokens, entropies and the most likely
// alternatives from rows of logits (include/mamba_lm_ops.h): what a program
// does with the logits of a language model's head (the reference leaves the
// model around its scan op to the caller, benchmarks/profiler.py:18-150).
//
// With m = max x, s = sum e^(x - m), t = sum (x - m) e^(x - m):
//   log p_i = (x_i - m) - log s,   entropy = log s - t / s.
#include <cuda_runtime.h>
#include <float.h>
#include <stdint.h>

#include <string>

#include "../../include/mamba_lm_ops.h"
#include "lm_device.cuh"
#include "scan_device.cuh"
#include "scan_kernels.h"

namespace {

using mamba_lm::to_f32;
using mamba_scan::launch_pdl;

constexpr int kThreads = 256;

struct LogprobParams {
  const void* logits;
  int64_t row_stride;
  const int64_t* target;
  float* logprob;
  float* entropy;
  float* top_logprob;
  int64_t* top_id;
  int vocab, top;
};

// A logit's place in the order of the alternatives, as one integer: larger
// values first (NaN above +inf), equal values by rising index.
__device__ __forceinline__ uint64_t order_key(float x, int index) {
  uint32_t u = __float_as_uint(x);
  if ((u & 0x7fffffffu) > 0x7f800000u) u = 0x7fffffffu;     // any NaN
  if (u == 0x80000000u) u = 0;                              // -0 equals 0
  u = (u & 0x80000000u) ? ~u : (u | 0x80000000u);
  return ((uint64_t)u << 32) | (uint32_t)~index;
}

// Running (m, s, t) over some of a row's logits. m starts at the lowest
// finite value, so that logits of -inf add nothing (e^-inf = 0) and NaN or
// +inf turn s into NaN.
struct Stats {
  float m = -FLT_MAX, s = 0.f, t = 0.f;

  // to a maximum m2 >= m: s and t of the same terms
  __device__ __forceinline__ void rescale(float m2) {
    const float d = fmaxf(m - m2, -200.f), f = expf(d);  // e^-200 is 0 in fp32
    t = f * fmaf(d, s, t);
    s *= f;
    m = m2;
  }
  __device__ __forceinline__ void add(float x) {
    if (x > m) rescale(x);
    const float d = x - m, e = expf(d);
    s += e;
    t = fmaf(e, fmaxf(d, -200.f), t);  // 0 * -inf does not arise
  }
  __device__ __forceinline__ void merge(Stats o) {
    const float m2 = fmaxf(m, o.m);
    rescale(m2);
    o.rescale(m2);
    s += o.s;
    t += o.t;
  }
};

template <typename T>
__global__ void __launch_bounds__(kThreads) logprobs_kernel(const LogprobParams p) {
  __shared__ Stats stats[kThreads / 32];
  __shared__ uint64_t keys[kThreads / 32];
  mamba_scan::pdl_trigger();
  mamba_scan::pdl_wait();
  const int64_t row = blockIdx.x;
  const T* x = static_cast<const T*>(p.logits) + row * p.row_stride;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  Stats st;
  for (int i = threadIdx.x; i < p.vocab; i += kThreads) st.add(to_f32(x[i]));
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    Stats other;
    other.m = __shfl_xor_sync(0xffffffffu, st.m, o);
    other.s = __shfl_xor_sync(0xffffffffu, st.s, o);
    other.t = __shfl_xor_sync(0xffffffffu, st.t, o);
    st.merge(other);
  }
  if (lane == 0) stats[warp] = st;
  __syncthreads();
  st = stats[0];
  for (int w = 1; w < kThreads / 32; ++w) st.merge(stats[w]);
  const float log_s = logf(st.s);
  if (threadIdx.x == 0) {
    if (p.entropy) p.entropy[row] = log_s - st.t / st.s;
    if (p.logprob) {
      const int64_t y = p.target[row];
      p.logprob[row] = y < 0 ? 0.f
                       : y >= p.vocab ? __int_as_float(0x7fc00000)
                                      : (to_f32(x[y]) - st.m) - log_s;
    }
  }
  // the alternatives: the largest key below the last one, `top` times
  uint64_t last = ~(uint64_t)0;
  for (int j = 0; j < p.top; ++j) {
    uint64_t best = 0;
    for (int i = threadIdx.x; i < p.vocab; i += kThreads) {
      const uint64_t key = order_key(to_f32(x[i]), i);
      if (key < last && key > best) best = key;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const uint64_t other = __shfl_xor_sync(0xffffffffu, best, o);
      best = other > best ? other : best;
    }
    __syncthreads();
    if (lane == 0) keys[warp] = best;
    __syncthreads();
    for (int w = 0; w < kThreads / 32; ++w) best = keys[w] > best ? keys[w] : best;
    if (threadIdx.x == 0) {
      const int id = (int)~(uint32_t)best;
      p.top_id[row * p.top + j] = id;
      p.top_logprob[row * p.top + j] = (to_f32(x[id]) - st.m) - log_s;
    }
    last = best;
  }
}

}  // namespace

extern "C" {

int mamba_token_logprobs(const void* logits, int64_t row_stride, int32_t dtype,
                         const int64_t* target, float* logprob, float* entropy,
                         float* top_logprob, int64_t* top_id, int64_t rows, int64_t vocab,
                         int64_t top, void* stream) try {
  using mamba_lm::Range;
  using mamba_lm::overlap;
  using mamba_lm::range_of;
  using mamba_scan::set_last_error;
  set_last_error(MAMBA_SCAN_OK, "");
  const int64_t size = dtype == MAMBA_DTYPE_F32 ? 4
                       : dtype == MAMBA_DTYPE_F16 || dtype == MAMBA_DTYPE_BF16 ? 2 : 0;
  if (size == 0)
    return set_last_error(MAMBA_SCAN_ERR_INVALID_ARGUMENT, "token_logprobs: unknown dtype");
  if (rows < 0 || rows >= (int64_t)1 << 31 || vocab < 1 || vocab >= (int64_t)1 << 31)
    return set_last_error(MAMBA_SCAN_ERR_INVALID_ARGUMENT,
                          "token_logprobs: rows must be 0..2^31-1 and vocab 1..2^31-1");
  if (top < 0 || top > MAMBA_LOGPROBS_MAX_TOP || top > vocab)
    return set_last_error(MAMBA_SCAN_ERR_INVALID_ARGUMENT,
                          "token_logprobs: top must be 0..64 and at most vocab");
  if (row_stride < 0 || row_stride > (int64_t)1 << 40 || (row_stride != 0 && row_stride < vocab))
    return set_last_error(MAMBA_SCAN_ERR_INVALID_ARGUMENT,
                          "token_logprobs: row_stride must be 0 or vocab..2^40");
  if (rows == 0) return MAMBA_SCAN_OK;
  if (!logits || (logprob && !target) || (top > 0 && (!top_logprob != !top_id)))
    return set_last_error(MAMBA_SCAN_ERR_INVALID_ARGUMENT,
                          "token_logprobs: logits is NULL, or logprob without target, or only "
                          "one of top_logprob and top_id");
  if (!top_logprob || !top_id) top = 0;
  const int64_t n[1] = {rows}, s1[1] = {1}, st[1] = {top}, sl[1] = {row_stride};
  const Range ins[] = {range_of(logits, size, vocab, n, sl, 1), range_of(target, 8, 1, n, s1, 1)};
  const Range outs[] = {range_of(logprob, 4, 1, n, s1, 1), range_of(entropy, 4, 1, n, s1, 1),
                        range_of(top > 0 ? top_logprob : nullptr, 4, top, n, st, 1),
                        range_of(top > 0 ? top_id : nullptr, 8, top, n, st, 1)};
  for (int i = 0; i < 4; ++i) {
    for (const Range& in : ins)
      if (overlap(outs[i], in))
        return set_last_error(MAMBA_SCAN_ERR_ALIASING, "token_logprobs: an output overlaps an input");
    for (int j = 0; j < i; ++j)
      if (overlap(outs[i], outs[j]))
        return set_last_error(MAMBA_SCAN_ERR_ALIASING, "token_logprobs: outputs overlap");
  }
  LogprobParams p{logits, row_stride, target, logprob, entropy, top_logprob, top_id, (int)vocab,
                  (int)top};
  const dim3 grid((unsigned)rows), block(kThreads);
  cudaStream_t cs = static_cast<cudaStream_t>(stream);
  cudaError_t e;
  switch (dtype) {
    case MAMBA_DTYPE_F32: e = launch_pdl(logprobs_kernel<float>, grid, block, 0, cs, p); break;
    case MAMBA_DTYPE_F16: e = launch_pdl(logprobs_kernel<__half>, grid, block, 0, cs, p); break;
    default: e = launch_pdl(logprobs_kernel<__nv_bfloat16>, grid, block, 0, cs, p); break;
  }
  if (e != cudaSuccess) return set_last_error(MAMBA_SCAN_ERR_CUDA, cudaGetErrorString(e));
  return MAMBA_SCAN_OK;
} catch (...) {
  return MAMBA_SCAN_ERR_CUDA;
}

}  // extern "C"
