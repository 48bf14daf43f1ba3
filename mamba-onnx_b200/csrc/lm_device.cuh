// Element types and host helpers shared by the kernels of
// include/mamba_lm_ops.h.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <atomic>
#include <initializer_list>

namespace mamba_lm {

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }

// The one rounding of an output: fp32 to the tensor's type, to nearest even.
template <typename T> __device__ __forceinline__ T from_f32(float v);
template <> __device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ __half from_f32<__half>(float v) {
  return __float2half_rn(v);
}
template <> __device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) {
  return __float2bfloat16_rn(v);
}

// SMs of the current device, which the rules that split work count with.
inline int sm_count() {
  static std::atomic<int> cache[64];
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 148;
  int v = cache[dev].load(std::memory_order_relaxed);
  if (v > 0) return v;
  if (cudaDeviceGetAttribute(&v, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || v <= 0)
    v = 148;
  cache[dev].store(v, std::memory_order_relaxed);
  return v;
}

// All of these addresses a multiple of `size` (1, 2, 4 or 8; NULL is one).
inline bool aligned_to(int64_t size, std::initializer_list<const void*> all) {
  uintptr_t bits = 0;
  for (const void* p : all) bits |= reinterpret_cast<uintptr_t>(p);
  return (bits & (uintptr_t)(size - 1)) == 0;
}

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

// A tensor's address range: the elements (n0-1) s0 + (n1-1) s1 + ... + inner
// of `size` bytes each, for overlap checks. Strides are non-negative.
struct Range {
  uintptr_t begin = 0;
  unsigned __int128 bytes = 0;
};

inline Range range_of(const void* p, int64_t size, int64_t inner, const int64_t* n,
                      const int64_t* stride, int dims) {
  Range r;
  if (p == nullptr || inner <= 0) return r;
  unsigned __int128 last = (unsigned __int128)inner;
  for (int i = 0; i < dims; ++i) {
    if (n[i] <= 0) return r;
    last += (unsigned __int128)(n[i] - 1) * (unsigned __int128)stride[i];
  }
  r.begin = reinterpret_cast<uintptr_t>(p);
  r.bytes = last * (unsigned __int128)size;
  return r;
}

inline bool overlap(const Range& a, const Range& b) {
  return a.bytes != 0 && b.bytes != 0 && a.begin < b.begin + b.bytes &&
         b.begin < a.begin + a.bytes;
}

}  // namespace mamba_lm
