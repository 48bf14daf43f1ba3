// The loss from hidden states and its gradients for a few rows
// (linear_cross_entropy.cu states the mathematics and serves the others).
//
// Up to 16 rows use a weight 16 times at most, so reading the weights bounds the
// call, not products: fp32 multiply-adds on the weights as they are, where the
// tensor cores' tiles of 256 rows would be nearly empty and float32 weights would
// first have to be found a scale for and split (twice the weights read, once
// written, once read again).
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <type_traits>

#include "../../include/mamba_lm_ops.h"
#include "linear_cross_entropy.h"
#include "lm_device.cuh"
#include "scan_device.cuh"
#include "scan_kernels.h"

namespace mamba_lce {

using mamba_lm::from_f32;
using mamba_lm::to_f32;

namespace {

constexpr int kWarps = 16;       // of logits_kernel
constexpr int kCols = 4;         // vocabulary rows of a warp at a time; columns of a thread
constexpr int kThreads = 128;    // of grads_kernel

// Four elements of a row from column k on, zeros past the width. kVec: rows in
// fours, the width too (the load then is not in a branch, so that several are under
// way).
template <bool kVec, typename T>
__device__ __forceinline__ void load4(float (&x)[4], const T* row, int k, int width) {
  if constexpr (kVec) {
    struct alignas(4 * sizeof(T)) Four { T e[4]; };
    const Four f = *reinterpret_cast<const Four*>(row + min(k, width - 4));
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = k < width ? to_f32(f.e[i]) : 0.f;
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = k + i < width ? to_f32(row[k + i]) : 0.f;
  }
}
template <typename T>
__device__ __forceinline__ void store4(T* row, const float (&x)[4], int k, int width, bool vec) {
  if (vec && k + 4 <= width) {
    struct alignas(4 * sizeof(T)) Four { T e[4]; } f;
#pragma unroll
    for (int i = 0; i < 4; ++i) f.e[i] = from_f32<T>(x[i]);
    *reinterpret_cast<Four*>(row + k) = f;
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (k + i < width) row[k + i] = from_f32<T>(x[i]);
  }
}

struct LogitsParams {
  const void* hidden;
  const void* weight;
  const int64_t* target;
  const float2* stats;       // kGrad
  const float* grad;         // kGrad
  float2* partial;           // [CTA][row]: (m, s)
  float* target_logit;
  float* dz;                 // kGrad: [vocabulary][R]
  int64_t hidden_stride, weight_stride, grad_stride;
  int rows, vocab, width, padded;  // padded: width in shared memory
  int vec;
};

// z of R rows, four vocabulary rows a warp at a time: the hidden states lie in
// shared memory, a lane has every 32nd piece of four columns, and the 4 R sums over
// the lanes come about by halves, so that each lane ends with one or two logits of
// one row. Then (m, s) of its row, or dz. 100000 x 2048 in float32: 163 us for a row
// (5.0 TB/s), 281 for 16, whose multiply-adds and reads of shared memory bound it.
template <typename T, int R, bool kGrad>
__global__ void __launch_bounds__(32 * kWarps, 1) logits_kernel(const LogitsParams p) {
  extern __shared__ __align__(16) float h[];  // [R][padded]
  __shared__ float2 joined[kWarps][R];
  mamba_scan::pdl_trigger();
  mamba_scan::pdl_wait();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (int i = threadIdx.x; i < R * p.padded; i += 32 * kWarps) {
    const int r = i / p.padded, k = i % p.padded;
    // (rows that do not count leave no trace)
    const bool on = r < p.rows && k < p.width && p.target[min(r, p.rows - 1)] >= 0;
    h[i] = on ? to_f32(static_cast<const T*>(p.hidden)[r * p.hidden_stride + k]) : 0.f;
  }
  __syncthreads();
  // what this lane ends with: logits of row `r`, vocabulary rows v0 + j0 (and + 1)
  constexpr int kSums = 4 * R, kMine = kSums == 64 ? 2 : 1;
  const int at = kSums == 64 ? 2 * lane : lane >> 1, r = at >> 2, j0 = at & 3;
  const int64_t target = r < p.rows ? p.target[r] : -1;
  const bool counts = r < p.rows && (kSums == 64 || lane % 2 == 0);
  float m = kGrad ? 0.f : -INFINITY, s = 0.f, scale = 0.f, g = 0.f;
  if constexpr (kGrad) {
    if (r < p.rows && target >= 0) {
      const float2 st = p.stats[r];
      g = p.grad[r * p.grad_stride];
      if (target >= p.vocab) g = __int_as_float(0x7fc00000);
      m = st.x;
      scale = g / st.y;
    }
  }
  for (int64_t v0 = kCols * ((int64_t)blockIdx.x * kWarps + warp); v0 < p.vocab;
       v0 += (int64_t)kCols * kWarps * gridDim.x) {
    const T* row[kCols];
#pragma unroll
    for (int j = 0; j < kCols; ++j)
      row[j] = static_cast<const T*>(p.weight) + min(v0 + j, (int64_t)p.vocab - 1) * p.weight_stride;
    float2 sum[R][kCols / 2];
#pragma unroll
    for (int i = 0; i < R; ++i)
#pragma unroll
      for (int j = 0; j < kCols / 2; ++j) sum[i][j] = make_float2(0.f, 0.f);
    auto add = [&](auto vec, int k) {
      float w[kCols][4];
#pragma unroll
      for (int j = 0; j < kCols; ++j) load4<decltype(vec)::value>(w[j], row[j], k, p.width);
#pragma unroll
      for (int i = 0; i < R; ++i) {
        const float4 x4 = *reinterpret_cast<const float4*>(h + i * p.padded + k);
        const float x[4] = {x4.x, x4.y, x4.z, x4.w};
#pragma unroll
        for (int c = 0; c < 4; ++c)
#pragma unroll
          for (int j = 0; j < kCols / 2; ++j)
            sum[i][j] = __ffma2_rn(make_float2(w[2 * j][c], w[2 * j + 1][c]), make_float2(x[c], x[c]),
                                   sum[i][j]);
      }
    };
    if (p.vec) {
#pragma unroll(R == 4 ? 4 : 1)
      for (int k = 4 * lane; k < p.padded; k += 128) add(std::true_type(), k);
    } else {
#pragma unroll 1
      for (int k = 4 * lane; k < p.padded; k += 128) add(std::false_type(), k);
    }
    float z[kSums];
#pragma unroll
    for (int i = 0; i < R; ++i)
#pragma unroll
      for (int j = 0; j < kCols / 2; ++j) {
        z[4 * i + 2 * j] = sum[i][j].x;
        z[4 * i + 2 * j + 1] = sum[i][j].y;
      }
    // each step keeps the half that the lane's bit says
#pragma unroll
    for (int step = 0; step < 5; ++step) {
      const int d = 16 >> step, n = kSums >> (step + 1);
      if (n > 0) {
#pragma unroll
        for (int i = 0; i < n; ++i) {
          const bool upper = lane & d;
          const float keep = upper ? z[i + n] : z[i], send = upper ? z[i] : z[i + n];
          z[i] = keep + __shfl_xor_sync(0xffffffffu, send, d);
        }
      } else {
        z[0] += __shfl_xor_sync(0xffffffffu, z[0], d);
      }
    }
#pragma unroll
    for (int i = 0; i < kMine; ++i) {
      const int64_t v = v0 + j0 + i;
      if (v >= p.vocab) continue;
      if constexpr (kGrad) {
        float dz = mamba_scan::ex2_approx((z[i] - m) * kLog2e) * scale;
        if (v == target) dz -= g;
        if (kSums == 64 || lane % 2 == 0) p.dz[v * R + r] = target >= 0 ? dz : 0.f;
      } else if (counts) {
        merge_sums(m, s, z[i], 1.f);
        if (v == target) p.target_logit[r] = z[i];
      }
    }
  }
  if constexpr (!kGrad) {
    // the lanes of a row are neighbours: 2 of them (R = 16) or 8
    auto merge = [&](float2 o) { merge_sums(m, s, o.x, o.y); };
#pragma unroll
    for (int d = 1; d < 32 / R; d <<= 1) {
      const float om = __shfl_xor_sync(0xffffffffu, m, d), os = __shfl_xor_sync(0xffffffffu, s, d);
      merge(make_float2(om, os));
    }
    if (lane % (32 / R) == 0) joined[warp][r] = make_float2(m, s);
    __syncthreads();
    if (threadIdx.x < p.rows) {
      const float2 first = joined[0][threadIdx.x];
      m = first.x, s = first.y;
      for (int i = 1; i < kWarps; ++i) merge(joined[i][threadIdx.x]);
      p.partial[(int64_t)blockIdx.x * p.rows + threadIdx.x] = make_float2(m, s);
    }
  }
}

struct GradsParams {
  const void* hidden;
  const void* weight;
  const int64_t* target;
  const float* dz;           // [vocabulary][R]
  float* sums;               // [part][row][width], or NULL
  void* d_weight;            // or NULL
  int64_t hidden_stride, weight_stride;
  int rows, vocab, width, per_part;
  int vec, out_vec;
};

// d_weight = dz^T H of a part of the vocabulary, and that part's sum of d_hidden =
// dz W: a thread has four columns of H and of the sums in registers and goes through
// the vocabulary's rows, whose dz all threads read. Reading W and writing d_weight
// bound it: 100000 x 2048 in float32 250 us for a row (6.5 TB/s); for 16 rows, 420 us,
// the multiply-adds and what two CTAs on an SM hide. (dz read by each thread from
// memory instead of shared memory 1200, no rows of W read ahead 580.)
template <typename T, int R>
__global__ void __launch_bounds__(kThreads) grads_kernel(const GradsParams p) {
  mamba_scan::pdl_trigger();
  mamba_scan::pdl_wait();
  constexpr int kBatch = R > 4 ? 4 : 8;        // rows of W under way
  constexpr int kHeld = 4 * kThreads / R;      // rows of dz in shared memory at a time
  __shared__ __align__(16) float dz[2][kHeld][R];
  const int k = 4 * ((int)blockIdx.x * kThreads + (int)threadIdx.x);
  const bool on = k < p.width;
  float2 h[R][2], sum[R][2];
#pragma unroll
  for (int i = 0; i < R; ++i) {
    float x[4] = {0.f, 0.f, 0.f, 0.f};
    if (on && i < p.rows && p.target[i] >= 0)
      load4<false>(x, static_cast<const T*>(p.hidden) + i * p.hidden_stride, k, p.width);
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      h[i][c] = make_float2(x[2 * c], x[2 * c + 1]);
      sum[i][c] = make_float2(0.f, 0.f);
    }
  }
  const int64_t from = (int64_t)blockIdx.y * p.per_part, to = min(from + p.per_part, (int64_t)p.vocab);
  const T* weight = static_cast<const T*>(p.weight);
  // four of the next rows' dz, a thread (zeros past the end)
  auto fetch = [&](int64_t v) {
    const int64_t at = v * R + 4 * threadIdx.x;
    return at < to * R ? *reinterpret_cast<const float4*>(p.dz + at) : make_float4(0.f, 0.f, 0.f, 0.f);
  };
  auto rows_of = [&](float (&w)[kBatch][4], int64_t v) {
    if (p.sums == nullptr || !on) return;
    if (p.vec) {
#pragma unroll
      for (int b = 0; b < kBatch; ++b)
        load4<true>(w[b], weight + min(v + b, to - 1) * p.weight_stride, k, p.width);
    } else {
#pragma unroll
      for (int b = 0; b < kBatch; ++b)
        load4<false>(w[b], weight + min(v + b, to - 1) * p.weight_stride, k, p.width);
    }
  };
  // (16 rows' registers leave two CTAs on an SM: there the next rows of W are read
  // while these are worked on)
  constexpr bool kAhead = R > 4;
  float w[kBatch][4], ahead[kAhead ? kBatch : 1][4];
  if constexpr (kAhead) rows_of(w, from);
  float4 next = fetch(from);
  int buffer = 0;
  for (int64_t v1 = from; v1 < to; v1 += kHeld, buffer ^= 1) {
    *reinterpret_cast<float4*>(&dz[buffer][0][0] + 4 * threadIdx.x) = next;
    __syncthreads();  // (the other buffer's readers are past it)
    next = fetch(v1 + kHeld);
    if (!on) continue;
    const int held = (int)min((int64_t)kHeld, to - v1);
#pragma unroll 1
    for (int b0 = 0; b0 < held; b0 += kBatch) {
      if constexpr (kAhead) rows_of(ahead, v1 + b0 + kBatch);
      else rows_of(w, v1 + b0);
#pragma unroll
      for (int b = 0; b < kBatch; ++b) {
        if (b0 + b >= held) break;
        float2 d[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
#pragma unroll
        for (int i = 0; i < R; i += 4) {
          const float4 f4 = *reinterpret_cast<const float4*>(&dz[buffer][b0 + b][i]);
          const float f[4] = {f4.x, f4.y, f4.z, f4.w};
#pragma unroll
          for (int r = 0; r < 4; ++r)
#pragma unroll
            for (int c = 0; c < 2; ++c) {
              d[c] = __ffma2_rn(make_float2(f[r], f[r]), h[i + r][c], d[c]);
              if (p.sums != nullptr)
                sum[i + r][c] = __ffma2_rn(make_float2(f[r], f[r]),
                                           make_float2(w[b][2 * c], w[b][2 * c + 1]), sum[i + r][c]);
            }
        }
        if (p.d_weight != nullptr) {
          const float x[4] = {d[0].x, d[0].y, d[1].x, d[1].y};
          store4(static_cast<T*>(p.d_weight) + (v1 + b0 + b) * p.width, x, k, p.width, p.out_vec);
        }
      }
      if constexpr (kAhead)
#pragma unroll
        for (int b = 0; b < kBatch; ++b)
#pragma unroll
          for (int c = 0; c < 4; ++c) w[b][c] = ahead[b][c];
    }
  }
  if (!on) return;
  if (p.sums != nullptr)
#pragma unroll
    for (int i = 0; i < R; ++i) {
      if (i >= p.rows) break;
      const float x[4] = {sum[i][0].x, sum[i][0].y, sum[i][1].x, sum[i][1].y};
      store4(p.sums + ((int64_t)blockIdx.y * p.rows + i) * p.width, x, k, p.width, false);
    }
}

// d_hidden = the parts' sums; 0 where a row does not count. 8 warps share an
// element's parts.
template <typename T>
__global__ void __launch_bounds__(256)
    join_kernel(const float* sums, const int64_t* target, T* out, int parts, int rows, int width) {
  mamba_scan::pdl_trigger();
  mamba_scan::pdl_wait();
  __shared__ float part[8][32];
  const int64_t all = (int64_t)rows * width;
  const int64_t at = (int64_t)blockIdx.x * 32 + (threadIdx.x & 31);
  float s = 0.f;
  if (at < all)
#pragma unroll 4
    for (int i = threadIdx.x >> 5; i < parts; i += 8) s += sums[i * all + at];
  part[threadIdx.x >> 5][threadIdx.x & 31] = s;
  __syncthreads();
  if (threadIdx.x >= 32 || at >= all) return;
#pragma unroll
  for (int i = 1; i < 8; ++i) s += part[i][threadIdx.x];
  out[at] = from_f32<T>(target[at / width] < 0 ? 0.f : s);
}

// -------------------------------------------------------------------- host

using Args = mamba_linear_cross_entropy_args;
using GradArgs = mamba_linear_cross_entropy_grad_args;

constexpr int kMostRows = 16;
constexpr size_t kMostShared = 200 * 1024;
constexpr int64_t kMostDz = (int64_t)96 << 20;  // (in tiles it is formed a piece at a time)

int rows_held(const Args& a) { return a.rows <= 4 ? 4 : 16; }
int64_t padded(const Args& a) { return (a.width + 127) / 128 * 128; }

// Rows of multiples of four elements that start at such.
bool in_fours(const void* p, int64_t stride, int64_t width, int64_t size) {
  return stride % 4 == 0 && width % 4 == 0 && reinterpret_cast<uintptr_t>(p) % (4 * size) == 0;
}

int64_t logits_ctas(const Args& a) {
  const int64_t units = (a.vocab + kCols * kWarps - 1) / (kCols * kWarps);
  return std::min<int64_t>(units, mamba_lm::sm_count());  // (one takes an SM's registers)
}

struct Parts {
  int64_t parts, per_part;
};
// About four CTAs to an SM, of at least 32 rows of the vocabulary.
Parts grads_parts(const Args& a) {
  const int64_t across = (a.width + 4 * kThreads - 1) / (4 * kThreads);
  const int64_t want = std::max<int64_t>(1, 4 * mamba_lm::sm_count() / across);
  const int64_t per = std::max<int64_t>(32, (a.vocab + want - 1) / want);
  return {(a.vocab + per - 1) / per, per};
}

struct Space {
  size_t at = 0;
  uint8_t* base;
  template <typename P> P* take(int64_t count) {
    P* p = reinterpret_cast<P*>(base + at);
    at += (size_t)((count * (int64_t)sizeof(P) + 255) / 256 * 256);
    return p;
  }
};
struct ForwardSpace {
  float2* partial;
  float* target_logit;
  size_t bytes;
};
ForwardSpace forward_space(const Args& a, void* workspace) {
  Space s{0, static_cast<uint8_t*>(workspace)};
  ForwardSpace f;
  f.partial = s.take<float2>(logits_ctas(a) * a.rows);
  f.target_logit = s.take<float>(a.rows);
  f.bytes = s.at;
  return f;
}
struct GradSpace {
  float* dz;
  float* sums;
  size_t bytes;
};
GradSpace grad_space(const GradArgs& g, void* workspace) {
  const Args& a = g.forward;
  Space s{0, static_cast<uint8_t*>(workspace)};
  GradSpace f;
  f.dz = s.take<float>(a.vocab * rows_held(a));
  f.sums = g.d_hidden ? s.take<float>(grads_parts(a).parts * a.rows * a.width) : nullptr;
  f.bytes = s.at;
  return f;
}

template <typename T, int R, bool kGrad>
cudaError_t launch_logits(const Args& a, LogitsParams p, cudaStream_t st) {
  p.hidden = a.hidden;
  p.weight = a.weight;
  p.target = a.target;
  p.hidden_stride = a.hidden_stride;
  p.weight_stride = a.weight_stride;
  p.rows = (int)a.rows;
  p.vocab = (int)a.vocab;
  p.width = (int)a.width;
  p.padded = (int)padded(a);
  p.vec = in_fours(a.weight, a.weight_stride, a.width, sizeof(T));
  const size_t bytes = (size_t)R * p.padded * 4;
  auto kernel = logits_kernel<T, R, kGrad>;
  const cudaError_t e =
      cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
  if (e != cudaSuccess) return e;
  return mamba_scan::launch_pdl(kernel, dim3((unsigned)logits_ctas(a)), dim3(32 * kWarps), bytes, st,
                                p);
}

template <typename T, int R>
cudaError_t forward(const Args& a, void* workspace, cudaStream_t st) {
  const ForwardSpace f = forward_space(a, workspace);
  LogitsParams p = {};
  p.partial = f.partial;
  p.target_logit = f.target_logit;
  const cudaError_t e = launch_logits<T, R, false>(a, p, st);
  if (e != cudaSuccess) return e;
  return launch_combine(f.partial, f.target_logit, a.target, a.loss, a.stats, (int)a.rows,
                        (int)logits_ctas(a), a.vocab, st);
}

template <typename T, int R>
cudaError_t backward(const GradArgs& g, void* workspace, cudaStream_t st) {
  const Args& a = g.forward;
  const GradSpace f = grad_space(g, workspace);
  LogitsParams p = {};
  p.stats = reinterpret_cast<const float2*>(a.stats);
  p.grad = g.grad;
  p.grad_stride = g.grad_stride;
  p.dz = f.dz;
  cudaError_t e = launch_logits<T, R, true>(a, p, st);
  if (e != cudaSuccess) return e;
  const Parts parts = grads_parts(a);
  GradsParams q = {};
  q.hidden = a.hidden;
  q.weight = a.weight;
  q.target = a.target;
  q.dz = f.dz;
  q.sums = f.sums;
  q.d_weight = g.d_weight;
  q.hidden_stride = a.hidden_stride;
  q.weight_stride = a.weight_stride;
  q.rows = (int)a.rows;
  q.vocab = (int)a.vocab;
  q.width = (int)a.width;
  q.per_part = (int)parts.per_part;
  q.vec = in_fours(a.weight, a.weight_stride, a.width, sizeof(T));
  q.out_vec = in_fours(g.d_weight, a.width, a.width, sizeof(T));
  const dim3 grid((unsigned)((a.width + 4 * kThreads - 1) / (4 * kThreads)), (unsigned)parts.parts);
  e = mamba_scan::launch_pdl(grads_kernel<T, R>, grid, dim3(kThreads), 0, st, q);
  if (e != cudaSuccess || !g.d_hidden) return e;
  return mamba_scan::launch_pdl(join_kernel<T>, dim3((unsigned)((a.rows * a.width + 31) / 32)),
                                dim3(256), 0, st, static_cast<const float*>(f.sums), a.target,
                                static_cast<T*>(g.d_hidden), (int)parts.parts, (int)a.rows,
                                (int)a.width);
}

}  // namespace

bool few_rows(const Args& a, bool grad) {
  // 100000 x 2048, here and in tiles: float32 losses of 1 row 163 and 665 us, of 16
  // 281 and 674, with gradients 580 and 1766, 973 and 1720; bf16 losses of 4 rows 132
  // and 149, of 16 270 and 147, with gradients 448 and 944, 964 and 935 (50280 x 768:
  // 337 and 567). Past 16 rows the multiply-adds would take longer than the tiles.
  const int64_t most = a.dtype == MAMBA_DTYPE_F32 || grad ? kMostRows : 4;
  return a.rows <= most && (size_t)rows_held(a) * padded(a) * 4 <= kMostShared &&
         (!grad || a.vocab * rows_held(a) * 4 <= kMostDz);
}

size_t few_forward_bytes(const Args& a) { return forward_space(a, nullptr).bytes; }
size_t few_grad_bytes(const GradArgs& g) { return grad_space(g, nullptr).bytes; }

cudaError_t few_forward(const Args& a, void* workspace, cudaStream_t st) {
  const bool four = rows_held(a) == 4;
  switch (a.dtype) {
    case MAMBA_DTYPE_F32:
      return four ? forward<float, 4>(a, workspace, st) : forward<float, 16>(a, workspace, st);
    case MAMBA_DTYPE_F16:
      return four ? forward<__half, 4>(a, workspace, st) : forward<__half, 16>(a, workspace, st);
    default:
      return four ? forward<__nv_bfloat16, 4>(a, workspace, st)
                  : forward<__nv_bfloat16, 16>(a, workspace, st);
  }
}

cudaError_t few_backward(const GradArgs& g, void* workspace, cudaStream_t st) {
  const bool four = rows_held(g.forward) == 4;
  switch (g.forward.dtype) {
    case MAMBA_DTYPE_F32:
      return four ? backward<float, 4>(g, workspace, st) : backward<float, 16>(g, workspace, st);
    case MAMBA_DTYPE_F16:
      return four ? backward<__half, 4>(g, workspace, st) : backward<__half, 16>(g, workspace, st);
    default:
      return four ? backward<__nv_bfloat16, 4>(g, workspace, st)
                  : backward<__nv_bfloat16, 16>(g, workspace, st);
  }
}

}  // namespace mamba_lce
