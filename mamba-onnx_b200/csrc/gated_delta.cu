// The gated delta rule (include/mamba_lm_ops.h): the recurrence itself, token
// by token, for prompts, and its single-token step.
//
// Like linear attention (linear_attention.cu) a successor of the selective
// scan this library is built around (the reference has only the scan,
// src/native/cpp/selective_scan.cc:163-230): with S' = exp(g) S,
//   S <- S' + beta k (v - k S')^T,   out = scale q S.
// Two sums over the keys a token, the second after the first has gone into
// the state; since q S = q S' + (q k) beta (v - k S'), both are formed from S'
// at once and a token needs one reduction.
#include <cuda_runtime.h>
#include <stdint.h>

#include <string>

#include "gated_delta.h"
#include "lm_device.cuh"
#include "scan_device.cuh"
#include "scan_kernels.h"

namespace {

using mamba_lm::from_f32;
using mamba_lm::to_f32;
using mamba_scan::launch_pdl;

constexpr int kMaxDim = 256;   // largest dk and dv
constexpr int kCols = 32;      // dv columns per CTA of the recurrent kernel
constexpr int kWarps = 8;      // of the step kernel

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
  mamba_gated_delta_args a;
  int tiles;  // ceil(dv / kCols)
};

// One CTA = (sequence, head, 32 dv columns), 4 warps of 8 columns; 4 lanes
// share a column, each with R = dk / 4 of its state rows in registers (rows
// 16 j + 4 part .. + 3), so a token is two dot products over R rows, two
// shuffles and the update, with no barrier but the staging of kTok tokens.
// The chain of dependent instructions bounds it (0.4 us a token of 24 heads of 64 x
// 64, 0.7 of 384 of them), so it serves short prompts, heads of more than 128 keys
// and calls without a workspace. Short are those for which chunks take no less: 16
// rows, 48 of float32 (24 heads of 64 x 64, 16 bits: 18 us for 16 rows, 31 for 32,
// chunks 20 for either; float32: 20 us for 32 rows, 33 for 64, chunks 27 and 29).
template <typename T, int R>
__global__ void __launch_bounds__(128) recurrent_kernel(const RecurrentParams p) {
  constexpr int kTok = 16;
  constexpr int kRows = 4 * R;
  __shared__ __align__(16) float qs[kTok][kRows];
  __shared__ __align__(16) float ks[kTok][kRows];
  __shared__ float vs[kTok][kCols];
  __shared__ float as[kTok], bs[kTok], qk[kTok];
  pdl_enter();
  const mamba_gated_delta_args& a = p.a;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, part = lane & 3;
  const int H = (int)a.heads, dk = (int)a.dk, dv = (int)a.dv, L = (int)a.seqlen;
  const int tile = (int)(blockIdx.x % (unsigned)p.tiles);
  const int64_t bh = blockIdx.x / (unsigned)p.tiles;
  const int b = (int)(bh / H), h = (int)(bh % H), g = h / (int)(a.heads / a.groups);
  const int col0 = tile * kCols, c = warp * 8 + (lane >> 2), col = col0 + c;
  const bool col_ok = col < dv;
  const int len = clamped_length(a.lengths, b, L);
  const T* q = static_cast<const T*>(a.q) + b * a.q_stride[0] + g * a.q_stride[2];
  const T* k = static_cast<const T*>(a.k) + b * a.k_stride[0] + g * a.k_stride[2];
  const T* v = static_cast<const T*>(a.v) + b * a.v_stride[0] + h * a.v_stride[2];
  const float* ld = a.log_decay + b * a.decay_stride[0] + h * a.decay_stride[2];
  const float* be = a.beta + b * a.beta_stride[0] + h * a.beta_stride[2];
  T* out = static_cast<T*>(a.out) + ((int64_t)b * L * H + h) * dv;

  float s[R];
#pragma unroll
  for (int i = 0; i < R; ++i) {
    const int r = (i >> 2) * 16 + part * 4 + (i & 3);
    s[i] = (a.h0 && r < dk && col_ok) ? a.h0[(bh * dk + r) * dv + col] : 0.f;
  }
  for (int t0 = 0; t0 < len; t0 += kTok) {
    const int n = min(kTok, len - t0);
    __syncthreads();
    for (int i = threadIdx.x; i < n * kRows; i += 128) {
      const int t = i / kRows, r = i % kRows;
      const bool ok = r < dk;
      qs[t][r] = ok ? to_f32(q[(int64_t)(t0 + t) * a.q_stride[1] + r]) : 0.f;
      ks[t][r] = ok ? to_f32(k[(int64_t)(t0 + t) * a.k_stride[1] + r]) : 0.f;
    }
    for (int i = threadIdx.x; i < n * kCols; i += 128) {
      const int t = i / kCols, cc = i % kCols;
      vs[t][cc] = col0 + cc < dv ? to_f32(v[(int64_t)(t0 + t) * a.v_stride[1] + col0 + cc]) : 0.f;
    }
    if (threadIdx.x < n) {
      as[threadIdx.x] = expf(ld[(int64_t)(t0 + threadIdx.x) * a.decay_stride[1]]);
      bs[threadIdx.x] = be[(int64_t)(t0 + threadIdx.x) * a.beta_stride[1]];
    }
    __syncthreads();
    for (int t = warp; t < n; t += 4) {
      float sum = 0.f;
      for (int r = lane; r < kRows; r += 32) sum = fmaf(qs[t][r], ks[t][r], sum);
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
      if (lane == 0) qk[t] = sum;
    }
    __syncthreads();
    for (int t = 0; t < n; ++t) {
      float ksum[4] = {}, qsum[4] = {};  // over S before the decay
#pragma unroll
      for (int i = 0; i < R; i += 4) {
        const float4 kk = *reinterpret_cast<const float4*>(&ks[t][i * 4 + part * 4]);
        const float4 qq = *reinterpret_cast<const float4*>(&qs[t][i * 4 + part * 4]);
        ksum[0] = fmaf(kk.x, s[i], ksum[0]);
        ksum[1] = fmaf(kk.y, s[i + 1], ksum[1]);
        ksum[2] = fmaf(kk.z, s[i + 2], ksum[2]);
        ksum[3] = fmaf(kk.w, s[i + 3], ksum[3]);
        qsum[0] = fmaf(qq.x, s[i], qsum[0]);
        qsum[1] = fmaf(qq.y, s[i + 1], qsum[1]);
        qsum[2] = fmaf(qq.z, s[i + 2], qsum[2]);
        qsum[3] = fmaf(qq.w, s[i + 3], qsum[3]);
      }
      float held = (ksum[0] + ksum[1]) + (ksum[2] + ksum[3]);
      float o = (qsum[0] + qsum[1]) + (qsum[2] + qsum[3]);
      held += __shfl_xor_sync(0xffffffffu, held, 1);
      o += __shfl_xor_sync(0xffffffffu, o, 1);
      held += __shfl_xor_sync(0xffffffffu, held, 2);
      o += __shfl_xor_sync(0xffffffffu, o, 2);
      const float decay = as[t], u = bs[t] * fmaf(-decay, held, vs[t][c]);
#pragma unroll
      for (int i = 0; i < R; i += 4) {
        const float4 kk = *reinterpret_cast<const float4*>(&ks[t][i * 4 + part * 4]);
        s[i] = fmaf(kk.x, u, decay * s[i]);
        s[i + 1] = fmaf(kk.y, u, decay * s[i + 1]);
        s[i + 2] = fmaf(kk.z, u, decay * s[i + 2]);
        s[i + 3] = fmaf(kk.w, u, decay * s[i + 3]);
      }
      if (part == 0 && col_ok)
        out[(int64_t)(t0 + t) * H * dv + col] = from_f32<T>(a.scale * fmaf(qk[t], u, decay * o));
    }
  }
  for (int64_t i = threadIdx.x; i < (int64_t)(L - len) * kCols; i += 128) {
    const int64_t t = len + i / kCols;
    const int cc = (int)(i % kCols);
    if (col0 + cc < dv) out[t * H * dv + col0 + cc] = from_f32<T>(0.f);
  }
  if (a.h_last && col_ok) {
#pragma unroll
    for (int i = 0; i < R; ++i) {
      const int r = (i >> 2) * 16 + part * 4 + (i & 3);
      if (r < dk) a.h_last[(bh * dk + r) * dv + col] = s[i];
    }
  }
}

template <typename T>
cudaError_t launch_recurrent(const mamba_gated_delta_args& a, cudaStream_t st) {
  RecurrentParams p;
  p.a = a;
  p.tiles = (int)((a.dv + kCols - 1) / kCols);
  const dim3 grid((unsigned)(a.batch * a.heads * p.tiles)), block(128);
  if (a.dk <= 64) return launch_pdl(recurrent_kernel<T, 16>, grid, block, 0, st, p);
  if (a.dk <= 128) return launch_pdl(recurrent_kernel<T, 32>, grid, block, 0, st, p);
  return launch_pdl(recurrent_kernel<T, 64>, grid, block, 0, st, p);
}

// ------------------------------------------------------------ one token

struct StepParams {
  mamba_gated_delta_step_args a;
  int tiles;  // ceil(dv / kC)
};

// One CTA = (sequence, head, kC dv columns), its part of the state in
// registers: all loads go out at once, one barrier joins the two sums over the
// keys, and the updated state is written. The state once in, once out bounds it:
// 64 sequences of 40 states of 128 x 128 take 57 us, 5.9 TB/s (0.90 of the
// measured copy rate); 7 of 12 of 80 x 72 take 8. kVec: kC / 4 threads of float4
// cover the columns, the others stride over dk; otherwise (dv not a multiple of 4,
// or a state that is not 16-byte aligned) a lane per column (kC = 32) and a warp
// per row. NR rows per thread, and registers for three CTAs on an SM where they
// are float4 or few (with four 7% more: their registers hold fewer loads).
template <typename T, int kC, bool kVec, int NR>
__global__ void __launch_bounds__(32 * kWarps, NR <= 8 ? 3 : 1) step_kernel(const StepParams p) {
  constexpr int kLanes = kVec ? kC / 4 : 32;       // threads across the columns
  constexpr int kRowStep = 32 * kWarps / kLanes;   // rows between a thread's rows
  constexpr int kPer = kVec ? 4 : 1;
  __shared__ float part[2][kWarps][kC];
  __shared__ float part_qk[kWarps];
  pdl_enter();
  const mamba_gated_delta_step_args& a = p.a;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int H = (int)a.heads, dk = (int)a.dk, dv = (int)a.dv;
  const int tile = (int)(blockIdx.x % (unsigned)p.tiles);
  const int64_t bh = blockIdx.x / (unsigned)p.tiles;
  const int b = (int)(bh / H), h = (int)(bh % H), g = h / (int)(a.heads / a.groups);
  const int c0 = (int)(threadIdx.x % kLanes) * kPer, col = tile * kC + c0;
  const int row0 = (int)threadIdx.x / kLanes;
  const T* q = static_cast<const T*>(a.q) + b * a.q_stride[0] + g * a.q_stride[1];
  const T* k = static_cast<const T*>(a.k) + b * a.k_stride[0] + g * a.k_stride[1];
  const T* v = static_cast<const T*>(a.v) + b * a.v_stride[0] + h * a.v_stride[1];
  const bool ok = col < dv;
  float x[NR][kPer], kk[NR], held[kPer] = {}, o[kPer] = {};
  // (a thread past the columns, or a row past the keys, holds zeros)
#pragma unroll
  for (int i = 0; i < NR; ++i) {
    const int r = row0 + i * kRowStep;
#pragma unroll
    for (int j = 0; j < kPer; ++j) x[i][j] = 0.f;
    if (ok && r < dk) {
      const float* s = a.state + (bh * dk + r) * dv + col;
      if constexpr (kVec) {
        const float4 w = __ldcs(reinterpret_cast<const float4*>(s));
        x[i][0] = w.x, x[i][1] = w.y, x[i][2] = w.z, x[i][3] = w.w;
      } else {
        x[i][0] = __ldcs(s);
      }
    }
  }
  float qq[NR];
#pragma unroll
  for (int i = 0; i < NR; ++i) {
    const int r = row0 + i * kRowStep;
    kk[i] = r < dk ? to_f32(k[r]) : 0.f;
    qq[i] = r < dk ? to_f32(q[r]) : 0.f;
  }
  float vv[kPer];
#pragma unroll
  for (int j = 0; j < kPer; ++j) vv[j] = ok ? to_f32(v[col + j]) : 0.f;
  const float decay = expf(a.log_decay[b * a.decay_stride[0] + h * a.decay_stride[1]]);
  const float beta = a.beta[b * a.beta_stride[0] + h * a.beta_stride[1]];
  float qk = 0.f;
#pragma unroll
  for (int i = 0; i < NR; ++i) {
    qk = fmaf(qq[i], kk[i], qk);
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
      held[j] = fmaf(kk[i], x[i][j], held[j]);
      o[j] = fmaf(qq[i], x[i][j], o[j]);
    }
  }
  // over the warp's rows: lanes that differ in bits of kLanes and above
#pragma unroll
  for (int d = 16; d >= kLanes; d >>= 1) {
    qk += __shfl_xor_sync(0xffffffffu, qk, d);
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
      held[j] += __shfl_xor_sync(0xffffffffu, held[j], d);
      o[j] += __shfl_xor_sync(0xffffffffu, o[j], d);
    }
  }
  if (lane < kLanes) {
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
      part[0][warp][c0 + j] = held[j];
      part[1][warp][c0 + j] = o[j];
    }
  }
  if (lane == 0) part_qk[warp] = qk;
  __syncthreads();
  float u[kPer];
#pragma unroll
  for (int j = 0; j < kPer; ++j) {
    float sum = 0.f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) sum += part[0][w][c0 + j];
    u[j] = beta * fmaf(-decay, sum, vv[j]);
  }
  if (ok) {
#pragma unroll
    for (int i = 0; i < NR; ++i) {
      const int r = row0 + i * kRowStep;
      if (r >= dk) break;
      float* s = a.state_out + (bh * dk + r) * dv + col;
      float y[kPer];
#pragma unroll
      for (int j = 0; j < kPer; ++j) y[j] = fmaf(kk[i], u[j], decay * x[i][j]);
      if constexpr (kVec) {
        __stcs(reinterpret_cast<float4*>(s), make_float4(y[0], y[1], y[2], y[3]));
      } else {
        __stcs(s, y[0]);
      }
    }
  }
  if (row0 == 0 && ok) {
    float all_qk = 0.f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) all_qk += part_qk[w];
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
      float sum = 0.f;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) sum += part[1][w][c0 + j];
      static_cast<T*>(a.out)[bh * dv + col + j] =
          from_f32<T>(a.scale * fmaf(all_qk, u[j], decay * sum));
    }
  }
}

template <typename T, int kC, bool kVec, int NR>
cudaError_t launch_step_kernel(const mamba_gated_delta_step_args& a, cudaStream_t st) {
  StepParams p;
  p.a = a;
  p.tiles = (int)((a.dv + kC - 1) / kC);
  return launch_pdl(step_kernel<T, kC, kVec, NR>, dim3((unsigned)(a.batch * a.heads * p.tiles)),
                    dim3(32 * kWarps), 0, st, p);
}

template <typename T>
cudaError_t launch_step(const mamba_gated_delta_step_args& a, cudaStream_t st) {
  if (a.dv % 4 != 0 || !mamba_lm::aligned16(a.state) || !mamba_lm::aligned16(a.state_out)) {
    if (a.dk <= 64) return launch_step_kernel<T, 32, false, 8>(a, st);
    if (a.dk <= 128) return launch_step_kernel<T, 32, false, 16>(a, st);
    return launch_step_kernel<T, 32, false, 32>(a, st);
  }
  // 32 KB of the state to a CTA, so that others' loads are under way while one
  // joins its sums: 128 columns of up to 64 rows, 64 of 128, 32 of 256 (5120
  // states of 64 x 128, 2560 of 128 x 128 and 768 of 256 x 256: with tiles half as
  // wide 1.25, 1.36 and - times as long, with twice as wide -, 1.15 and 1.16 times).
  // Narrower while there are not two CTAs to an SM and 8 KB are left (96 states of
  // 128 x 128: 8 us with 384 CTAs, 10 with 192; 192 states: 12 with 768, 10 with 384).
  const int64_t sms = mamba_lm::sm_count();
  int64_t cols = a.dk <= 64 ? 128 : a.dk <= 128 ? 64 : 32;
  while (cols > 32 && (cols / 2 >= a.dv ||
                       (a.batch * a.heads * ((a.dv + cols - 1) / cols) < 2 * sms &&
                        cols / 2 * a.dk > 2048)))
    cols /= 2;
  if (cols == 128) return launch_step_kernel<T, 128, true, 8>(a, st);
  if (cols == 64)
    return a.dk <= 64 ? launch_step_kernel<T, 64, true, 4>(a, st)
                      : launch_step_kernel<T, 64, true, 8>(a, st);
  if (a.dk <= 64) return launch_step_kernel<T, 32, true, 2>(a, st);
  if (a.dk <= 128) return launch_step_kernel<T, 32, true, 4>(a, st);
  return launch_step_kernel<T, 32, true, 8>(a, st);
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
  // (grids: at most one CTA for each 16 columns)
  if (batch > 0 && heads > (kMaxCount - 1) / ((dv + 15) / 16) / batch)
    return "batch x heads x dv is too large";
  return nullptr;
}

}  // namespace

extern "C" {

size_t mamba_gated_delta_rule_workspace_size(int64_t batch, int64_t seqlen, int64_t heads,
                                             int64_t groups, int64_t dk, int64_t dv,
                                             int32_t dtype) {
  if (bad_shape(batch, seqlen, heads, groups, dk, dv, dtype) || batch == 0 ||
      !mamba_gd::mma_takes(seqlen, dk, dv, dtype))
    return 0;
  return mamba_gd::mma_workspace_size(batch, seqlen, heads, dk, dv, dtype);
}

int mamba_gated_delta_rule(const mamba_gated_delta_args* a, void* workspace,
                           size_t workspace_bytes, void* stream) try {
  using mamba_lm::Range;
  using mamba_lm::overlap;
  using mamba_lm::range_of;
  using mamba_scan::set_last_error;
  set_last_error(MAMBA_SCAN_OK, "");
  if (a == nullptr) return set_last_error(MAMBA_SCAN_ERR_INVALID_ARGUMENT, "args is NULL");
  if (const char* bad = bad_shape(a->batch, a->seqlen, a->heads, a->groups, a->dk, a->dv, a->dtype))
    return set_last_error(MAMBA_SCAN_ERR_INVALID_ARGUMENT, std::string("gated_delta_rule: ") + bad);
  if (!strides_ok(a->q_stride, 3) || !strides_ok(a->k_stride, 3) || !strides_ok(a->v_stride, 3) ||
      !strides_ok(a->decay_stride, 3) || !strides_ok(a->beta_stride, 3))
    return set_last_error(MAMBA_SCAN_ERR_INVALID_ARGUMENT,
                          "gated_delta_rule: strides must be 0..2^40");
  if (a->batch == 0) return MAMBA_SCAN_OK;
  if (a->seqlen > 0 && (!a->q || !a->k || !a->v || !a->log_decay || !a->beta || !a->out))
    return set_last_error(MAMBA_SCAN_ERR_INVALID_ARGUMENT,
                          "gated_delta_rule: q, k, v, log_decay, beta and out must be non-NULL");
  const int64_t size = element_size(a->dtype);
  if (!mamba_lm::aligned_to(size, {a->q, a->k, a->v, a->out}) ||
      !mamba_lm::aligned_to(4, {a->log_decay, a->beta, a->h0, a->lengths, a->h_last}))
    return set_last_error(MAMBA_SCAN_ERR_INVALID_ARGUMENT,
                          "gated_delta_rule: an address is not a multiple of its type's size");
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
                       range_of(a->beta, 4, 1, hd, a->beta_stride, 3),
                       range_of(a->h0, 4, a->dk * a->dv, st_n, st_s, 1),
                       range_of(a->lengths, 4, a->batch, one, packed, 1)};
  for (const Range& in : ins) {
    if (overlap(out, in))
      return set_last_error(MAMBA_SCAN_ERR_ALIASING, "gated_delta_rule: out overlaps an input");
    if (overlap(h_last, in))
      return set_last_error(MAMBA_SCAN_ERR_ALIASING, "gated_delta_rule: h_last overlaps an input");
    if (overlap(ws, in))
      return set_last_error(MAMBA_SCAN_ERR_ALIASING, "gated_delta_rule: workspace overlaps an input");
  }
  if (overlap(out, h_last) || overlap(ws, out) || overlap(ws, h_last))
    return set_last_error(MAMBA_SCAN_ERR_ALIASING,
                          "gated_delta_rule: out, h_last and workspace must not overlap");
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  cudaError_t e;
  if (workspace != nullptr && mamba_gd::mma_takes(a->seqlen, a->dk, a->dv, a->dtype)) {
    const size_t need = mamba_gd::mma_workspace_size(a->batch, a->seqlen, a->heads, a->dk, a->dv,
                                                     a->dtype);
    if (workspace_bytes < need)
      return set_last_error(MAMBA_SCAN_ERR_WORKSPACE,
                            "gated_delta_rule: workspace holds " + std::to_string(workspace_bytes) +
                                " bytes; this shape needs " + std::to_string(need));
    if (!mamba_lm::aligned16(workspace))
      return set_last_error(MAMBA_SCAN_ERR_WORKSPACE,
                            "gated_delta_rule: workspace must be 16-byte aligned");
    e = mamba_gd::launch_mma(*a, workspace, st);
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

int mamba_gated_delta_rule_step(const mamba_gated_delta_step_args* a, void* stream) try {
  using mamba_lm::Range;
  using mamba_lm::overlap;
  using mamba_lm::range_of;
  using mamba_scan::set_last_error;
  set_last_error(MAMBA_SCAN_OK, "");
  if (a == nullptr) return set_last_error(MAMBA_SCAN_ERR_INVALID_ARGUMENT, "args is NULL");
  if (const char* bad = bad_shape(a->batch, 1, a->heads, a->groups, a->dk, a->dv, a->dtype))
    return set_last_error(MAMBA_SCAN_ERR_INVALID_ARGUMENT,
                          std::string("gated_delta_rule_step: ") + bad);
  if (!strides_ok(a->q_stride, 2) || !strides_ok(a->k_stride, 2) || !strides_ok(a->v_stride, 2) ||
      !strides_ok(a->decay_stride, 2) || !strides_ok(a->beta_stride, 2))
    return set_last_error(MAMBA_SCAN_ERR_INVALID_ARGUMENT,
                          "gated_delta_rule_step: strides must be 0..2^40");
  if (a->batch == 0) return MAMBA_SCAN_OK;
  if (!a->q || !a->k || !a->v || !a->log_decay || !a->beta || !a->state || !a->state_out || !a->out)
    return set_last_error(MAMBA_SCAN_ERR_INVALID_ARGUMENT,
                          "gated_delta_rule_step: every tensor must be non-NULL");
  const int64_t size = element_size(a->dtype);
  if (!mamba_lm::aligned_to(size, {a->q, a->k, a->v, a->out}) ||
      !mamba_lm::aligned_to(4, {a->log_decay, a->beta, a->state, a->state_out}))
    return set_last_error(MAMBA_SCAN_ERR_INVALID_ARGUMENT,
                          "gated_delta_rule_step: an address is not a multiple of its type's size");
  const int64_t gd[2] = {a->batch, a->groups}, hd[2] = {a->batch, a->heads};
  const int64_t st_n[1] = {a->batch * a->heads}, st_s[1] = {a->dk * a->dv}, out_s[1] = {a->dv};
  const Range out = range_of(a->out, size, a->dv, st_n, out_s, 1);
  const Range state = range_of(a->state, 4, a->dk * a->dv, st_n, st_s, 1);
  const Range next = range_of(a->state_out, 4, a->dk * a->dv, st_n, st_s, 1);
  const Range ins[] = {range_of(a->q, size, a->dk, gd, a->q_stride, 2),
                       range_of(a->k, size, a->dk, gd, a->k_stride, 2),
                       range_of(a->v, size, a->dv, hd, a->v_stride, 2),
                       range_of(a->log_decay, 4, 1, hd, a->decay_stride, 2),
                       range_of(a->beta, 4, 1, hd, a->beta_stride, 2)};
  for (const Range& in : ins)
    if (overlap(out, in) || overlap(next, in))
      return set_last_error(MAMBA_SCAN_ERR_ALIASING,
                            "gated_delta_rule_step: out or state_out overlaps an input");
  if (overlap(out, state) || overlap(out, next))
    return set_last_error(MAMBA_SCAN_ERR_ALIASING, "gated_delta_rule_step: out overlaps a state");
  if (a->state_out != a->state && overlap(next, state))
    return set_last_error(MAMBA_SCAN_ERR_ALIASING,
                          "gated_delta_rule_step: state_out must be state or not overlap it");
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
