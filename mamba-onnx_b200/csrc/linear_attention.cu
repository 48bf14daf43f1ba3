// Linear attention with a decay for each head (include/mamba_lm_ops.h): the
// recurrence itself, token by token, for prompts, and its single-token step.
//
// The recurrence is that of the successors of the selective scan this library
// is built around (the reference has only the scan, src/native/cpp/
// selective_scan.cc:163-230): a scalar decay for each head and token in place
// of one for each channel and state, S <- exp(g) S + k v^T, out = scale q S.
#include <cuda_runtime.h>
#include <stdint.h>

#include <algorithm>
#include <string>
#include <type_traits>

#include "linear_attention.h"
#include "lm_device.cuh"
#include "scan_device.cuh"
#include "scan_kernels.h"

namespace {

using mamba_lm::from_f32;
using mamba_lm::to_f32;
using mamba_scan::launch_pdl;

constexpr int kMaxDim = 256;   // largest dk and dv
constexpr int kCols = 32;      // dv columns per CTA of the recurrent kernels
constexpr int kWarps = 8;

// Lets the next kernel be scheduled, then waits for the previous one: every
// kernel here is launched as a programmatic dependent launch.
__device__ __forceinline__ void pdl_enter() {
  mamba_scan::pdl_trigger();
  mamba_scan::pdl_wait();
}

__device__ __forceinline__ int clamped_length(const int32_t* lengths, int b, int seqlen) {
  if (lengths == nullptr) return seqlen;
  const int n = lengths[b];
  return n < 0 ? 0 : (n > seqlen ? seqlen : n);
}

// ------------------------------------------------- prompts, token by token

struct RecurrentParams {
  mamba_linear_attention_args a;
  int tiles;  // ceil(dv / kCols)
};

// One CTA = (sequence, head, 32 dv columns); lane = column, warp w holds the
// state rows [w R, (w+1) R) of that column in registers (R = dk / 8 rounded
// up to a power of two), so a token is R fused multiply-adds for the state
// and R for the output, from k and q rows broadcast out of shared memory.
// Tokens are staged kTok at a time as fp32; the 8 warps' partial outputs are
// added in warp order after each batch of tokens. The fused multiply-adds
// bound it (2 dk dv for a token and head, 8x2048 tokens of 40 heads of 128x128
// 2.85 ms), so it serves prompts of up to 16 tokens, where its one launch
// does as well (16 tokens of 40 heads of 64 6.6 us, the tensor-core kernel 6.6
// us from 17 tokens on); with dk over 128, which takes the tensor cores two
// launches, up to 32 (16 heads of 256 x 256, bf16: 23 us for 32 tokens, 43
// against 22 for 64), and 16-bit calls without the workspace that those need.
template <typename T, int R>
__global__ void __launch_bounds__(32 * kWarps) recurrent_kernel(const RecurrentParams p) {
  constexpr int kTok = R <= 16 ? 16 : 8;
  constexpr int kRows = R * kWarps;
  __shared__ __align__(16) float qs[kTok][kRows];
  __shared__ __align__(16) float ks[kTok][kRows];
  __shared__ float vs[kTok][kCols];
  __shared__ float as[kTok];
  __shared__ float part[kWarps][kTok][kCols];
  pdl_enter();
  const mamba_linear_attention_args& a = p.a;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int H = (int)a.heads, dk = (int)a.dk, dv = (int)a.dv, L = (int)a.seqlen;
  const int tile = (int)(blockIdx.x % (unsigned)p.tiles);
  const int64_t bh = blockIdx.x / (unsigned)p.tiles;
  const int b = (int)(bh / H), h = (int)(bh % H), g = h / (int)(a.heads / a.groups);
  const int col0 = tile * kCols, col = col0 + lane;
  const bool col_ok = col < dv;
  const int len = clamped_length(a.lengths, b, L);
  const T* q = static_cast<const T*>(a.q) + b * a.q_stride[0] + g * a.q_stride[2];
  const T* k = static_cast<const T*>(a.k) + b * a.k_stride[0] + g * a.k_stride[2];
  const T* v = static_cast<const T*>(a.v) + b * a.v_stride[0] + h * a.v_stride[2];
  const float* ld = a.log_decay + b * a.decay_stride[0] + h * a.decay_stride[2];
  T* out = static_cast<T*>(a.out) + ((int64_t)b * L * H + h) * dv;

  float s[R];
#pragma unroll
  for (int i = 0; i < R; ++i) {
    const int r = warp * R + i;
    s[i] = (a.h0 && r < dk && col_ok) ? a.h0[(bh * dk + r) * dv + col] : 0.f;
  }
  for (int t0 = 0; t0 < len; t0 += kTok) {
    const int n = min(kTok, len - t0);
    for (int i = threadIdx.x; i < n * kRows; i += 32 * kWarps) {
      const int t = i / kRows, r = i % kRows;
      const bool ok = r < dk;
      qs[t][r] = ok ? to_f32(q[(int64_t)(t0 + t) * a.q_stride[1] + r]) : 0.f;
      ks[t][r] = ok ? to_f32(k[(int64_t)(t0 + t) * a.k_stride[1] + r]) : 0.f;
    }
    for (int i = threadIdx.x; i < n * kCols; i += 32 * kWarps) {
      const int t = i / kCols, c = i % kCols;
      vs[t][c] = col0 + c < dv ? to_f32(v[(int64_t)(t0 + t) * a.v_stride[1] + col0 + c]) : 0.f;
    }
    if (threadIdx.x < n) as[threadIdx.x] = expf(ld[(int64_t)(t0 + threadIdx.x) * a.decay_stride[1]]);
    __syncthreads();
    for (int t = 0; t < n; ++t) {
      const float decay = as[t], vv = vs[t][lane];
      float acc = 0.f;
#pragma unroll
      for (int i = 0; i < R; i += 4) {
        const float4 kk = *reinterpret_cast<const float4*>(&ks[t][warp * R + i]);
        const float4 qq = *reinterpret_cast<const float4*>(&qs[t][warp * R + i]);
        s[i] = fmaf(kk.x, vv, decay * s[i]);
        s[i + 1] = fmaf(kk.y, vv, decay * s[i + 1]);
        s[i + 2] = fmaf(kk.z, vv, decay * s[i + 2]);
        s[i + 3] = fmaf(kk.w, vv, decay * s[i + 3]);
        acc = fmaf(qq.x, s[i], acc);
        acc = fmaf(qq.y, s[i + 1], acc);
        acc = fmaf(qq.z, s[i + 2], acc);
        acc = fmaf(qq.w, s[i + 3], acc);
      }
      part[warp][t][lane] = acc;
    }
    __syncthreads();
    for (int i = threadIdx.x; i < n * kCols; i += 32 * kWarps) {
      const int t = i / kCols, c = i % kCols;
      float sum = 0.f;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) sum += part[w][t][c];
      if (col0 + c < dv)
        out[(int64_t)(t0 + t) * H * dv + col0 + c] = from_f32<T>(a.scale * sum);
    }
    // the next batch's loads write qs, ks, vs and as (read above, before the
    // barrier) and its sums write part only after another barrier
  }
  for (int64_t i = threadIdx.x; i < (int64_t)(L - len) * kCols; i += 32 * kWarps) {
    const int64_t t = len + i / kCols;
    const int c = (int)(i % kCols);
    if (col0 + c < dv) out[t * H * dv + col0 + c] = from_f32<T>(0.f);
  }
  if (a.h_last && col_ok) {
#pragma unroll
    for (int i = 0; i < R; ++i) {
      const int r = warp * R + i;
      if (r < dk) a.h_last[(bh * dk + r) * dv + col] = s[i];
    }
  }
}

template <typename T>
cudaError_t launch_recurrent(const mamba_linear_attention_args& a, cudaStream_t st) {
  RecurrentParams p;
  p.a = a;
  p.tiles = (int)((a.dv + kCols - 1) / kCols);
  const dim3 grid((unsigned)(a.batch * a.heads * p.tiles)), block(32 * kWarps);
  if (a.dk <= 32) return launch_pdl(recurrent_kernel<T, 4>, grid, block, 0, st, p);
  if (a.dk <= 64) return launch_pdl(recurrent_kernel<T, 8>, grid, block, 0, st, p);
  if (a.dk <= 128) return launch_pdl(recurrent_kernel<T, 16>, grid, block, 0, st, p);
  return launch_pdl(recurrent_kernel<T, 32>, grid, block, 0, st, p);
}

// ------------------------------------------------------------ one token

struct StepParams {
  mamba_linear_attention_step_args a;
  int tiles;  // ceil(dv / kCols)
};

// One CTA = (sequence, head, kC dv columns). The state is read and written
// once and nothing else is large, so HBM bounds it. kVec: kC / 4 threads x
// float4 cover the columns and the other threads stride over dk; otherwise (dv
// not a multiple of 4, or a state that is not 16-byte aligned) a lane per
// column (kC = 32) and a warp per row. 64 sequences of 40 states of 128x128:
// 58 us, 5.8 TB/s (0.89 of the measured copy rate); one sequence of 24 states
// of 64x64 2.5 us.
template <typename T, int kC, bool kVec>
__global__ void __launch_bounds__(32 * kWarps) step_kernel(const StepParams p) {
  constexpr int kLanes = kVec ? kC / 4 : 32;       // threads across the columns
  constexpr int kRowStep = 32 * kWarps / kLanes;   // rows in flight per iteration
  constexpr int kPer = kVec ? 4 : 1, kBatch = 4;
  __shared__ float part[kWarps][kC];
  pdl_enter();
  const mamba_linear_attention_step_args& a = p.a;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int H = (int)a.heads, dk = (int)a.dk, dv = (int)a.dv;
  const int tile = (int)(blockIdx.x % (unsigned)p.tiles);
  const int64_t bh = blockIdx.x / (unsigned)p.tiles;
  const int b = (int)(bh / H), h = (int)(bh % H), g = h / (int)(a.heads / a.groups);
  const int col = tile * kC + (int)(threadIdx.x % kLanes) * kPer;
  const int row0 = (int)threadIdx.x / kLanes;
  const T* q = static_cast<const T*>(a.q) + b * a.q_stride[0] + g * a.q_stride[1];
  const T* k = static_cast<const T*>(a.k) + b * a.k_stride[0] + g * a.k_stride[1];
  const T* v = static_cast<const T*>(a.v) + b * a.v_stride[0] + h * a.v_stride[1];
  const float* ld = a.log_decay + b * a.decay_stride[0] + h * a.decay_stride[1];
  const bool ok = col < dv;
  float acc[kPer];
#pragma unroll
  for (int j = 0; j < kPer; ++j) acc[j] = 0.f;
  if (ok) {
    const float* s = a.state + bh * dk * dv + col;
    float* so = a.state_out + bh * dk * dv + col;
    // A batch of the state's loads goes out before anything that waits for a
    // value (instructions issue in order), and before the batch's stores:
    // state_out may be state, so the compiler cannot move loads over them.
    using V = typename std::conditional<kVec, float4, float>::type;
    float vv[kPer], decay = 0.f;
    for (int r0 = row0; r0 < dk; r0 += kBatch * kRowStep) {
      V x[kBatch];
      T kt[kBatch], qt[kBatch];
#pragma unroll
      for (int i = 0; i < kBatch; ++i) {
        const int r = min(r0 + i * kRowStep, dk - 1);  // (past the end: not used)
        x[i] = __ldcs(reinterpret_cast<const V*>(s + (int64_t)r * dv));
      }
#pragma unroll
      for (int i = 0; i < kBatch; ++i) {
        const int r = min(r0 + i * kRowStep, dk - 1);
        kt[i] = k[r];
        qt[i] = q[r];
      }
      if (r0 == row0) {
        T vt[kPer];
#pragma unroll
        for (int j = 0; j < kPer; ++j) vt[j] = v[col + j];
        const float g = *ld;
#pragma unroll
        for (int j = 0; j < kPer; ++j) vv[j] = to_f32(vt[j]);
        decay = expf(g);
      }
#pragma unroll
      for (int i = 0; i < kBatch; ++i) {
        const int r = r0 + i * kRowStep;
        if (r >= dk) break;
        const float kk = to_f32(kt[i]), qq = to_f32(qt[i]);
        float* e = reinterpret_cast<float*>(&x[i]);
#pragma unroll
        for (int j = 0; j < kPer; ++j) {
          e[j] = fmaf(kk, vv[j], decay * e[j]);
          acc[j] = fmaf(qq, e[j], acc[j]);
        }
        __stcs(reinterpret_cast<V*>(so + (int64_t)r * dv), x[i]);
      }
    }
  }
#pragma unroll
  for (int o = 16; o >= kLanes; o >>= 1)
#pragma unroll
    for (int j = 0; j < kPer; ++j) acc[j] += __shfl_xor_sync(0xffffffffu, acc[j], o);
  if (lane < kLanes)
#pragma unroll
    for (int j = 0; j < kPer; ++j) part[warp][lane * kPer + j] = acc[j];
  __syncthreads();
  if (threadIdx.x < kC && tile * kC + (int)threadIdx.x < dv) {
    float sum = 0.f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) sum += part[w][threadIdx.x];
    static_cast<T*>(a.out)[bh * dv + tile * kC + threadIdx.x] = from_f32<T>(a.scale * sum);
  }
}

template <typename T, int kC, bool kVec>
cudaError_t launch_step_tiles(const mamba_linear_attention_step_args& a, cudaStream_t st) {
  StepParams p;
  p.a = a;
  p.tiles = (int)((a.dv + kC - 1) / kC);
  return launch_pdl(step_kernel<T, kC, kVec>, dim3((unsigned)(a.batch * a.heads * p.tiles)),
                    dim3(32 * kWarps), 0, st, p);
}

template <typename T>
cudaError_t launch_step(const mamba_linear_attention_step_args& a, cudaStream_t st) {
  if (a.dv % 4 != 0 || !mamba_lm::aligned16(a.state) || !mamba_lm::aligned16(a.state_out))
    return launch_step_tiles<T, kCols, false>(a, st);
  // The widest tile whose rows are contiguous reads, narrowed while the CTAs
  // do not make one full wave (8 per SM) and a tile keeps more than 8 KB.
  // Measured (us, tiles of 32 / 64 / 128 columns): 64x40 states of 128x128
  // 64.9 / 57.6 / 57.8 (5.8 TB/s), of 64x64 26.6 / 17.8 / -, of 32x128 40.5 /
  // 26.1 / 17.2; 16x40 of 128x128 18.4 / 17.4 / 19.1, 1x40 3.6 / 4.6 / 4.6,
  // 8x24 of 64x64 3.4 / 2.6 / -.
  const int64_t sms = mamba_lm::sm_count();
  int64_t cols = a.dv > 64 ? 128 : a.dv > 32 ? 64 : 32;
  while (cols > 32 && a.batch * a.heads * ((a.dv + cols - 1) / cols) < 8 * sms &&
         cols / 2 * a.dk > 2048)
    cols /= 2;
  if (cols == 128) return launch_step_tiles<T, 128, true>(a, st);
  if (cols == 64) return launch_step_tiles<T, 64, true>(a, st);
  return launch_step_tiles<T, 32, true>(a, st);
}

// ------------------------------------------------------------- host checks

int element_size(int32_t dtype) {
  return dtype == MAMBA_DTYPE_F32 ? 4 : (dtype == MAMBA_DTYPE_F16 || dtype == MAMBA_DTYPE_BF16) ? 2 : 0;
}

constexpr int64_t kMaxCount = (int64_t)1 << 31;   // batch, seqlen, heads
constexpr int64_t kMaxStride = (int64_t)1 << 40;

bool strides_ok(const int64_t* s, int n) {
  for (int i = 0; i < n; ++i)
    if (s[i] < 0 || s[i] > kMaxStride) return false;
  return true;
}

// NULL, or what is wrong with the sizes.
const char* bad_shape(int64_t batch, int64_t seqlen, int64_t heads, int64_t groups, int64_t dk,
                      int64_t dv, int32_t dtype) {
  if (batch < 0 || seqlen < 0 || heads < 1 || groups < 1) return "batch, seqlen, heads, groups";
  if (batch >= kMaxCount || seqlen >= kMaxCount - 1024 || heads >= kMaxCount)
    return "dimension exceeds 2^31 - 1024";
  if (heads % groups != 0) return "groups must divide heads";
  if (dk < 1 || dk > kMaxDim || dv < 1 || dv > kMaxDim) return "dk and dv must be 1..256";
  if (element_size(dtype) == 0) return "unknown dtype";
  if (batch > 0 && heads > (kMaxCount - 1) / ((dv + kCols - 1) / kCols) / batch)
    return "batch x heads x dv is too large";
  return nullptr;
}

}  // namespace

extern "C" {

size_t mamba_linear_attention_workspace_size(int64_t batch, int64_t seqlen, int64_t heads,
                                             int64_t groups, int64_t dk, int64_t dv,
                                             int32_t dtype) {
  if (bad_shape(batch, seqlen, heads, groups, dk, dv, dtype) || batch == 0 ||
      !mamba_la::mma_takes(seqlen, dk, dv))
    return 0;
  return mamba_la::mma_workspace_size(batch, seqlen, heads, dk, dv, dtype);
}

int mamba_linear_attention(const mamba_linear_attention_args* a, void* workspace,
                           size_t workspace_bytes, void* stream) try {
  using mamba_lm::Range;
  using mamba_lm::overlap;
  using mamba_lm::range_of;
  using mamba_scan::set_last_error;
  set_last_error(MAMBA_SCAN_OK, "");
  if (a == nullptr) return set_last_error(MAMBA_SCAN_ERR_INVALID_ARGUMENT, "args is NULL");
  if (const char* bad = bad_shape(a->batch, a->seqlen, a->heads, a->groups, a->dk, a->dv, a->dtype))
    return set_last_error(MAMBA_SCAN_ERR_INVALID_ARGUMENT, std::string("linear_attention: ") + bad);
  if (!strides_ok(a->q_stride, 3) || !strides_ok(a->k_stride, 3) || !strides_ok(a->v_stride, 3) ||
      !strides_ok(a->decay_stride, 3))
    return set_last_error(MAMBA_SCAN_ERR_INVALID_ARGUMENT,
                          "linear_attention: strides must be 0..2^40");
  if (a->batch == 0) return MAMBA_SCAN_OK;
  if (a->seqlen > 0 && (!a->q || !a->k || !a->v || !a->log_decay || !a->out))
    return set_last_error(MAMBA_SCAN_ERR_INVALID_ARGUMENT,
                          "linear_attention: q, k, v, log_decay and out must be non-NULL");
  const int64_t size = element_size(a->dtype);
  if (!mamba_lm::aligned_to(size, {a->q, a->k, a->v, a->out}) ||
      !mamba_lm::aligned_to(4, {a->log_decay, a->h0, a->lengths, a->h_last}))
    return set_last_error(MAMBA_SCAN_ERR_INVALID_ARGUMENT,
                          "linear_attention: an address is not a multiple of its type's size");
  const int64_t gd[3] = {a->batch, a->seqlen, a->groups}, hd[3] = {a->batch, a->seqlen, a->heads};
  const int64_t one[1] = {1}, packed[1] = {0};
  const int64_t n_out = a->batch * a->seqlen, n_state = a->batch * a->heads;
  const int64_t out_n[2] = {n_out, a->heads}, out_s[2] = {a->heads * a->dv, a->dv};
  const int64_t st_n[1] = {n_state}, st_s[1] = {a->dk * a->dv};
  const Range out = range_of(a->out, size, a->dv, out_n, out_s, 2);
  const Range h_last = range_of(a->h_last, 4, a->dk * a->dv, st_n, st_s, 1);
  const Range ws = range_of(workspace, 1, (int64_t)workspace_bytes, one, packed, 1);
  const Range ins[] = {range_of(a->q, size, a->dk, gd, a->q_stride, 3),
                       range_of(a->k, size, a->dk, gd, a->k_stride, 3),
                       range_of(a->v, size, a->dv, hd, a->v_stride, 3),
                       range_of(a->log_decay, 4, 1, hd, a->decay_stride, 3),
                       range_of(a->h0, 4, a->dk * a->dv, st_n, st_s, 1),
                       range_of(a->lengths, 4, a->batch, one, packed, 1)};
  for (const Range& in : ins) {
    if (overlap(out, in))
      return set_last_error(MAMBA_SCAN_ERR_ALIASING, "linear_attention: out overlaps an input");
    if (overlap(h_last, in))
      return set_last_error(MAMBA_SCAN_ERR_ALIASING, "linear_attention: h_last overlaps an input");
    if (overlap(ws, in))
      return set_last_error(MAMBA_SCAN_ERR_ALIASING, "linear_attention: workspace overlaps an input");
  }
  if (overlap(out, h_last) || overlap(ws, out) || overlap(ws, h_last))
    return set_last_error(MAMBA_SCAN_ERR_ALIASING,
                          "linear_attention: out, h_last and workspace must not overlap");
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  cudaError_t e;
  if (mamba_la::mma_takes(a->seqlen, a->dk, a->dv) &&
      (workspace != nullptr || !mamba_la::mma_needs_workspace(a->dk, a->dtype))) {
    const size_t need = workspace == nullptr ? 0
                        : mamba_la::mma_workspace_size(a->batch, a->seqlen, a->heads, a->dk, a->dv,
                                                       a->dtype);
    if (workspace_bytes < need)
      return set_last_error(MAMBA_SCAN_ERR_WORKSPACE,
                            "linear_attention: workspace holds " + std::to_string(workspace_bytes) +
                                " bytes; this shape needs " + std::to_string(need));
    if (need > 0 && !mamba_lm::aligned16(workspace))
      return set_last_error(MAMBA_SCAN_ERR_WORKSPACE,
                            "linear_attention: workspace must be 16-byte aligned");
    e = mamba_la::launch_mma(*a, need > 0 ? workspace : nullptr, st);
  } else {
    switch (a->dtype) {
      case MAMBA_DTYPE_F32: e = launch_recurrent<float>(*a, st); break;
      case MAMBA_DTYPE_F16: e = launch_recurrent<__half>(*a, st); break;
      default: e = launch_recurrent<__nv_bfloat16>(*a, st); break;
    }
  }
  if (e != cudaSuccess) return set_last_error(MAMBA_SCAN_ERR_CUDA, cudaGetErrorString(e));
  return MAMBA_SCAN_OK;
} catch (...) {
  return MAMBA_SCAN_ERR_CUDA;
}

int mamba_linear_attention_step(const mamba_linear_attention_step_args* a, void* stream) try {
  using mamba_lm::Range;
  using mamba_lm::overlap;
  using mamba_lm::range_of;
  using mamba_scan::set_last_error;
  set_last_error(MAMBA_SCAN_OK, "");
  if (a == nullptr) return set_last_error(MAMBA_SCAN_ERR_INVALID_ARGUMENT, "args is NULL");
  if (const char* bad = bad_shape(a->batch, 1, a->heads, a->groups, a->dk, a->dv, a->dtype))
    return set_last_error(MAMBA_SCAN_ERR_INVALID_ARGUMENT,
                          std::string("linear_attention_step: ") + bad);
  if (!strides_ok(a->q_stride, 2) || !strides_ok(a->k_stride, 2) || !strides_ok(a->v_stride, 2) ||
      !strides_ok(a->decay_stride, 2))
    return set_last_error(MAMBA_SCAN_ERR_INVALID_ARGUMENT,
                          "linear_attention_step: strides must be 0..2^40");
  if (a->batch == 0) return MAMBA_SCAN_OK;
  if (!a->q || !a->k || !a->v || !a->log_decay || !a->state || !a->state_out || !a->out)
    return set_last_error(MAMBA_SCAN_ERR_INVALID_ARGUMENT,
                          "linear_attention_step: every tensor must be non-NULL");
  const int64_t size = element_size(a->dtype);
  if (!mamba_lm::aligned_to(size, {a->q, a->k, a->v, a->out}) ||
      !mamba_lm::aligned_to(4, {a->log_decay, a->state, a->state_out}))
    return set_last_error(MAMBA_SCAN_ERR_INVALID_ARGUMENT,
                          "linear_attention_step: an address is not a multiple of its type's size");
  const int64_t gd[2] = {a->batch, a->groups}, hd[2] = {a->batch, a->heads};
  const int64_t st_n[1] = {a->batch * a->heads}, st_s[1] = {a->dk * a->dv}, out_s[1] = {a->dv};
  const Range out = range_of(a->out, size, a->dv, st_n, out_s, 1);
  const Range state = range_of(a->state, 4, a->dk * a->dv, st_n, st_s, 1);
  const Range next = range_of(a->state_out, 4, a->dk * a->dv, st_n, st_s, 1);
  const Range ins[] = {range_of(a->q, size, a->dk, gd, a->q_stride, 2),
                       range_of(a->k, size, a->dk, gd, a->k_stride, 2),
                       range_of(a->v, size, a->dv, hd, a->v_stride, 2),
                       range_of(a->log_decay, 4, 1, hd, a->decay_stride, 2)};
  for (const Range& in : ins)
    if (overlap(out, in) || overlap(next, in))
      return set_last_error(MAMBA_SCAN_ERR_ALIASING,
                            "linear_attention_step: out or state_out overlaps an input");
  if (overlap(out, state) || overlap(out, next))
    return set_last_error(MAMBA_SCAN_ERR_ALIASING, "linear_attention_step: out overlaps a state");
  if (a->state_out != a->state && overlap(next, state))
    return set_last_error(MAMBA_SCAN_ERR_ALIASING,
                          "linear_attention_step: state_out must be state or not overlap it");
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  cudaError_t e;
  switch (a->dtype) {
    case MAMBA_DTYPE_F32: e = launch_step<float>(*a, st); break;
    case MAMBA_DTYPE_F16: e = launch_step<__half>(*a, st); break;
    default: e = launch_step<__nv_bfloat16>(*a, st); break;
  }
  if (e != cudaSuccess) return set_last_error(MAMBA_SCAN_ERR_CUDA, cudaGetErrorString(e));
  return MAMBA_SCAN_OK;
} catch (...) {
  return MAMBA_SCAN_ERR_CUDA;
}

}  // extern "C"
