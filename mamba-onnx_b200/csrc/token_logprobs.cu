// Log probabilities of given tokens, entropies and the most likely
// alternatives from rows of logits (include/mamba_lm_ops.h): what a program
// does with the logits of a language model's head (the reference leaves the
// model around its scan op to the caller, benchmarks/profiler.py:18-150).
//
// With m = max x, s = sum e^(x - m), t = sum (x - m) e^(x - m):
//   log p_i = (x_i - m) - log s,   entropy = log s - t / s.
// One pass over the logits: each thread keeps a running (m, s, t), merged at
// the end, so HBM bounds it: 4096 rows of 50280 bf16 in 69.7 us, 5.9 TB/s
// (0.90 of the measured copy rate; one 2^x for each of 3e12 logits a second is
// two thirds of the exponential unit's rate), 1024 rows in fp32 39.7 us (0.79:
// 1024 CTAs on 888 places). CTAs of 256 threads, 6 on an SM, hide each other's
// starts and ends better than 512-thread ones did (88 us). (Calls in a row.)
//
// Alternatives. A pass that keeps ordered lists would wait on insertions;
// instead the pass keeps only each thread's largest logit, which the sums
// need anyway. The top-th largest of the group maxima (pairs of threads) is no
// more than the top-th largest logit, so all alternatives lie in the about
// `top` groups whose maximum reaches it: only their logits are read
// again (out of L2), and the few that reach the bound are ranked by counting.
// More of them than fit, or a row with NaN or +inf, goes through one pass per
// alternative instead (a mask that leaves fewer tokens than alternatives does:
// 5 of 50280, 20 alternatives, 1024 bf16 rows take 1.07 ms). 20 alternatives
// cost the 4096 rows 29 us (98 us in all; 104 among other work): no HBM traffic but a fifth more instructions, and five barriers and a
// second trip to L2 in each row's tail.
//
// A row is one CTA's, or a cluster's of up to 8 when there are too few rows
// to fill the GPU; the first CTA then merges the others' sums and
// alternatives through distributed shared memory.
#include <cooperative_groups.h>
#include <cuda_runtime.h>
#include <float.h>
#include <stdint.h>

#include <string>
#include <type_traits>

#include "../../include/mamba_lm_ops.h"
#include "lm_device.cuh"
#include "scan_device.cuh"
#include "scan_kernels.h"

namespace {

using mamba_lm::to_f32;
namespace cg = cooperative_groups;

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kGroups = kThreads / 2;   // threads 2g and 2g + 1 are group g
constexpr int kBatch = 4;               // 16-byte loads in flight per thread
constexpr int kCandidates = 1024;       // alternatives' candidates of a CTA
constexpr int kMaxTop = MAMBA_LOGPROBS_MAX_TOP;
static_assert(kGroups >= kMaxTop && kGroups <= kThreads - 32 && kMaxTop <= kThreads, "roles of threads");
constexpr int kMaxCluster = 8;
constexpr int64_t kMaxVocab = (int64_t)1 << 30;  // indices and their steps stay within an int
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

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
// values first (NaN above +inf), equal values by rising index. Never 0 or all
// ones, which stand for none and for the place before the first.
__device__ __forceinline__ uint64_t order_key(float x, int index) {
  uint32_t u = __float_as_uint(x);
  if ((u & 0x7fffffffu) > 0x7f800000u) u = 0x7f800001u;     // any NaN
  if (u == 0x80000000u) u = 0;                              // -0 equals 0
  u = (u & 0x80000000u) ? ~u : (u | 0x80000000u);
  return ((uint64_t)u << 32) | (uint32_t)~index;
}
__device__ __forceinline__ int key_index(uint64_t key) { return (int)~(uint32_t)key; }
__device__ __forceinline__ float key_value(uint64_t key) {  // (the logit, but for the sign of 0)
  const uint32_t u = (uint32_t)(key >> 32);
  return __uint_as_float((u & 0x80000000u) ? (u & 0x7fffffffu) : ~u);
}

__device__ __forceinline__ float max_nan(float a, float b) {  // NaN if either is
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// Running m, s = sum 2^y and t = sum y 2^y, y = (x - m) log2(e), over some of
// a row's logits. m starts at the lowest finite value, so logits of -inf add
// nothing; y is held at -300 (2^-300 is 0 in fp32), which keeps 0 times -inf
// out of t; NaN and +inf turn s into NaN.
struct Stats {
  float m, s, t;

  static __device__ __forceinline__ Stats none() { return Stats{-FLT_MAX, 0.f, 0.f}; }
  // to a maximum m2 >= m: s and t of the same terms
  __device__ __forceinline__ void rescale(float m2) {
    const float y = fmaxf((m - m2) * kLog2e, -300.f), f = mamba_scan::ex2_approx(y);
    t = f * fmaf(y, s, t);
    s *= f;
    m = m2;
  }
  __device__ __forceinline__ void merge(Stats o) {
    const float m2 = fmaxf(m, o.m);
    rescale(m2);
    o.rescale(m2);
    s += o.s;
    t += o.t;
  }
  __device__ __forceinline__ Stats shuffled(int lane_mask) const {
    Stats o;
    o.m = __shfl_xor_sync(0xffffffffu, m, lane_mask);
    o.s = __shfl_xor_sync(0xffffffffu, s, lane_mask);
    o.t = __shfl_xor_sync(0xffffffffu, t, lane_mask);
    return o;
  }
};

template <typename T> struct Vec { static constexpr int n = 16 / (int)sizeof(T); };

// Element i (of Vec<T>::n) of 16 bytes, as a float.
template <typename T> __device__ __forceinline__ void unpack(const uint4& w, float (&f)[Vec<T>::n]) {
  const uint32_t r[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (sizeof(T) == 4) {
      f[i] = __uint_as_float(r[i]);
    } else if constexpr (std::is_same<T, __half>::value) {
      const float2 x = __half22float2(*reinterpret_cast<const __half2*>(&r[i]));
      f[2 * i] = x.x, f[2 * i + 1] = x.y;
    } else {
      f[2 * i] = __uint_as_float(r[i] << 16), f[2 * i + 1] = __uint_as_float(r[i] & 0xffff0000u);
    }
  }
}

// The largest of a batch's logits (NaN ignored).
template <typename T, int n> __device__ __forceinline__ float batch_max(const uint4 (&w)[n]) {
  if constexpr (sizeof(T) == 4) {
    float m = -INFINITY;
#pragma unroll
    for (int b = 0; b < n; ++b)
      m = fmaxf(fmaxf(m, fmaxf(__uint_as_float(w[b].x), __uint_as_float(w[b].y))),
                fmaxf(__uint_as_float(w[b].z), __uint_as_float(w[b].w)));
    return m;
  } else {
    using T2 = typename std::conditional<std::is_same<T, __half>::value, __half2, __nv_bfloat162>::type;
    T2 m;
#pragma unroll
    for (int b = 0; b < n; ++b) {
      const T2* h = reinterpret_cast<const T2*>(&w[b]);
      const T2 x = __hmax2(__hmax2(h[0], h[1]), __hmax2(h[2], h[3]));
      m = b == 0 ? x : __hmax2(m, x);
    }
    return fmaxf(to_f32(m.x), to_f32(m.y));  // (NaN only where both halves of a pair were)
  }
}

// This CTA's share [begin, end) of a row: whole 16-byte vectors from element
// `body` on, and fewer than 2 vectors' worth of single elements around them.
template <typename T> struct Share {
  const T* x;
  int begin, end, body, n_vec;

  __device__ __forceinline__ Share(const T* row, int vocab, int rank, int ranks) : x(row) {
    constexpr int V = Vec<T>::n;
    const int head = (int)((16u - ((uint32_t)reinterpret_cast<uintptr_t>(row) & 15u)) & 15u) / (int)sizeof(T);
    const int per = ((vocab + ranks - 1) / ranks + V - 1) / V * V;
    // cut where vectors start, so that only the row's own ends are ragged
    const int64_t lo = (int64_t)rank * per, hi = lo + per;
    begin = rank == 0 ? 0 : (int)min((int64_t)vocab, lo + head);
    end = rank == ranks - 1 ? vocab : (int)min((int64_t)vocab, hi + head);
    body = min(end, rank == 0 ? head : begin);
    n_vec = (end - body) / V;
  }
  // the i-th single element's index, or -1
  __device__ __forceinline__ int single(int i) const {
    if (i < body - begin) return begin + i;
    const int at = body + n_vec * Vec<T>::n + (i - (body - begin));
    return at < end ? at : -1;
  }
  __device__ __forceinline__ uint4 vec(int v) const {
    return *reinterpret_cast<const uint4*>(x + body + (int64_t)v * Vec<T>::n);
  }
};

struct Shared {
  Stats stats[kWarps];
  Stats total;                 // this CTA's, then (first CTA) the row's
  __align__(16) float group_max[kGroups];
  int selected[kGroups];
  int n_selected, n_candidates;
  float bound;
  uint64_t warp_key[kWarps];
  uint64_t top[kMaxTop];       // this CTA's alternatives, in order (0: none)
  uint64_t merged[kMaxCluster * kMaxTop];
  uint64_t candidates[kCandidates];
};

// The `top` largest of n keys (distinct but for 0) in order, by counting the
// larger ones, into out, which holds zeros.
__device__ __forceinline__ void rank_keys(const uint64_t* keys, int n, uint64_t* out, int top) {
  for (int i = threadIdx.x; i < n; i += kThreads) {
    const uint64_t key = keys[i];
    if (key == 0) continue;
    int rank = 0;
    for (int j = 0; j < n; ++j) rank += keys[j] > key;
    if (rank < top) out[rank] = key;
  }
  __syncthreads();
}

// A lower bound of the top-th largest group maximum, close enough to leave
// few more groups than that: the longest prefix, as an ordered integer, that
// `top` of the maxima reach, found bit by bit until exactly `top` do. By one
// warp (counting larger ones for every maximum took four warps 7 times the
// instructions).
__device__ __forceinline__ void find_bound(Shared& sh, int top) {
  const int lane = threadIdx.x & 31;
  uint32_t key[kGroups / 32];
#pragma unroll
  for (int i = 0; i < kGroups / 32; ++i)
    key[i] = (uint32_t)(order_key(sh.group_max[i * 32 + lane], 0) >> 32);
  uint32_t prefix = 0;
#pragma unroll 1
  for (int bit = 31; bit >= 0; --bit) {
    const uint32_t next = prefix | (1u << bit);
    int count = 0;
#pragma unroll
    for (int i = 0; i < kGroups / 32; ++i)
      count += __popc(__ballot_sync(0xffffffffu, key[i] >= next));
    if (count < top) continue;
    prefix = next;
    if (count == top) break;
  }
  // (no lower than -inf's place: below it are no numbers)
  if (lane == 0) sh.bound = key_value((uint64_t)max(prefix, 0x007fffffu) << 32);
}

// This CTA's alternatives -> sh.top (zeros before). single: this thread's
// logit outside the vectors, at index single_at (-1: none); clean: no NaN or
// +inf in the share.
template <typename T>
__device__ __forceinline__ void local_top(Shared& sh, const Share<T>& s, int top, float single,
                                          int single_at, bool clean) {
  constexpr int V = Vec<T>::n;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (clean) {
    const float bound = sh.bound;
    if (threadIdx.x < kGroups && sh.group_max[threadIdx.x] >= bound)
      sh.selected[atomicAdd(&sh.n_selected, 1)] = threadIdx.x;
    if (single_at >= 0 && single >= bound)
      sh.candidates[atomicAdd(&sh.n_candidates, 1)] = order_key(single, single_at);
    __syncthreads();
    // A warp per selected group, a lane per vector; four loads in flight (two
    // groups, 64 vectors of each): one at a time, their latencies added up to
    // most of what the alternatives cost.
    const int per = 2 * ((s.n_vec + kThreads - 1) / kThreads), n_selected = sh.n_selected;
    for (int i = warp; i < n_selected; i += 2 * kWarps)
      for (int l0 = lane; l0 < per; l0 += 64) {
        uint4 w[4];
        int v[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const int g = i + u / 2 * kWarps, l = l0 + u % 2 * 32;
          v[u] = g < n_selected && l < per ? l / 2 * kThreads + sh.selected[g] * 2 + l % 2 : s.n_vec;
          if (v[u] < s.n_vec) w[u] = s.vec(v[u]);
        }
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          if (v[u] >= s.n_vec) continue;
          const uint4 one[1] = {w[u]};
          if (!(batch_max<T, 1>(one) >= bound)) continue;
          float x[V];
          unpack<T>(w[u], x);
#pragma unroll
          for (int e = 0; e < V; ++e)
            if (x[e] >= bound) {
              const int at = atomicAdd(&sh.n_candidates, 1);
              if (at < kCandidates) sh.candidates[at] = order_key(x[e], s.body + v[u] * V + e);
            }
        }
      }
    __syncthreads();
    if (sh.n_candidates <= kCandidates) {
      rank_keys(sh.candidates, sh.n_candidates, sh.top, top);
      return;
    }
  }
  // the largest key below the last one, `top` times
  uint64_t last = ~(uint64_t)0;
  for (int j = 0; j < top; ++j) {
    uint64_t best = 0;
    for (int i = s.begin + (int)threadIdx.x; i < s.end; i += kThreads) {
      const uint64_t key = order_key(to_f32(s.x[i]), i);
      if (key < last && key > best) best = key;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const uint64_t other = __shfl_xor_sync(0xffffffffu, best, o);
      best = other > best ? other : best;
    }
    __syncthreads();
    if (lane == 0) sh.warp_key[warp] = best;
    __syncthreads();
    for (int w = 0; w < kWarps; ++w) best = sh.warp_key[w] > best ? sh.warp_key[w] : best;
    if (threadIdx.x == 0) sh.top[j] = best;
    if (best != 0) last = best;
  }
  __syncthreads();
}

template <typename T>
__global__ void __launch_bounds__(kThreads, 6) logprobs_kernel(const LogprobParams p) {
  constexpr int V = Vec<T>::n;
  __shared__ Shared sh;
  mamba_scan::pdl_trigger();
  mamba_scan::pdl_wait();
  cg::cluster_group cluster = cg::this_cluster();
  const int ranks = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
  const int64_t row = blockIdx.x / ranks;
  const Share<T> s(static_cast<const T*>(p.logits) + row * p.row_stride, p.vocab, rank, ranks);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  // the target's logit, on its way while the row is summed
  int64_t target = -1;
  float target_logit = 0.f;
  if (p.logprob && rank == 0 && threadIdx.x == 0) {
    target = p.target[row];
    if (target >= 0 && target < p.vocab) target_logit = to_f32(s.x[target]);
  }

  Stats st = Stats::none();
  float thread_max = -INFINITY;
  auto add = [&](const float2 x) {  // two logits, neither above st.m: 2^y and y
    const float2 m2 = make_float2(-st.m, -st.m), l2 = make_float2(kLog2e, kLog2e);
    float2 y = __fmul2_rn(__fadd2_rn(x, m2), l2);
    y = make_float2(max_nan(y.x, -300.f), max_nan(y.y, -300.f));
    const float2 e = make_float2(mamba_scan::ex2_approx(y.x), mamba_scan::ex2_approx(y.y));
    return make_float4(e.x, e.y, y.x, y.y);
  };
  auto add_vectors = [&](auto count, int v0) {  // vectors v0, v0 + kThreads, ...
    constexpr int n = decltype(count)::value;
    uint4 w[n];
#pragma unroll
    for (int b = 0; b < n; ++b) w[b] = s.vec(v0 + b * kThreads);
    const float m = batch_max<T, n>(w);
    thread_max = fmaxf(thread_max, m);
    if (m > st.m) st.rescale(m);
    float2 sum = make_float2(st.s, 0.f), sum_t = make_float2(st.t, 0.f);
#pragma unroll
    for (int b = 0; b < n; ++b) {
      float x[V];
      unpack<T>(w[b], x);
#pragma unroll
      for (int i = 0; i < V; i += 2) {
        const float4 ey = add(make_float2(x[i], x[i + 1]));
        sum = __fadd2_rn(sum, make_float2(ey.x, ey.y));
        sum_t = __ffma2_rn(make_float2(ey.x, ey.y), make_float2(ey.z, ey.w), sum_t);
      }
    }
    st.s = sum.x + sum.y;
    st.t = sum_t.x + sum_t.y;
  };
  int v0 = threadIdx.x;
  for (; v0 + (kBatch - 1) * kThreads < s.n_vec; v0 += kBatch * kThreads)
    add_vectors(std::integral_constant<int, kBatch>(), v0);
  for (; v0 < s.n_vec; v0 += kThreads) add_vectors(std::integral_constant<int, 1>(), v0);
  const int single_at = threadIdx.x < 2 * V ? s.single(threadIdx.x) : -1;
  float single = 0.f;
  if (single_at >= 0) {
    single = to_f32(s.x[single_at]);
    if (single > st.m) st.rescale(single);
    const float4 ey = add(make_float2(single, -INFINITY));
    st.s += ey.x;
    st.t = fmaf(ey.x, ey.z, st.t);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) st.merge(st.shuffled(o));
  if (lane == 0) sh.stats[warp] = st;
  if (p.top > 0) {
    const float g = fmaxf(thread_max, __shfl_xor_sync(0xffffffffu, thread_max, 1));
    if ((threadIdx.x & 1) == 0) sh.group_max[threadIdx.x >> 1] = g;
    if (threadIdx.x == 0) sh.n_selected = sh.n_candidates = 0;
    if (threadIdx.x < p.top) sh.top[threadIdx.x] = 0;
  }
  __syncthreads();
  if (warp == kWarps - 1) {  // (lanes past the warps' sums hold empty ones)
    Stats all = lane < kWarps ? sh.stats[lane] : Stats::none();
#pragma unroll
    for (int o = kWarps / 2; o > 0; o >>= 1) all.merge(all.shuffled(o));
    if (lane == 0) sh.total = all;
  } else if (p.top > 0 && warp == 0) {
    find_bound(sh, p.top);
  }
  __syncthreads();
  st = sh.total;
  if (p.top > 0) local_top(sh, s, p.top, single, single_at, st.s == st.s);

  const uint64_t* keys = sh.top;
  if (ranks > 1) {
    cluster.sync();
    if (rank == 0) {
      st = Stats::none();
      for (int r = 0; r < ranks; ++r) st.merge(*cluster.map_shared_rank(&sh.total, r));
      if (threadIdx.x < p.top) sh.candidates[threadIdx.x] = 0;
      for (int i = threadIdx.x; i < ranks * p.top; i += kThreads)
        sh.merged[i] = cluster.map_shared_rank(sh.top, i / p.top)[i % p.top];
    }
    cluster.sync();  // the others may leave: their shared memory has been read
    if (rank != 0) return;
    if (p.top > 0) {
      // (sh.merged was filled before the second cluster.sync)
      rank_keys(sh.merged, ranks * p.top, sh.candidates, p.top);
      keys = sh.candidates;
    }
  }
  const float log_s = logf(st.s);
  if (threadIdx.x == 0) {
    if (p.entropy) p.entropy[row] = log_s - kLn2 * (st.t / st.s);
    if (p.logprob) {
      p.logprob[row] = target < 0 ? 0.f
                       : target >= p.vocab ? __int_as_float(0x7fc00000)
                                           : (target_logit - st.m) - log_s;
    }
  }
  for (int j = threadIdx.x; j < p.top; j += kThreads) {
    p.top_id[row * p.top + j] = key_index(keys[j]);
    p.top_logprob[row * p.top + j] = (key_value(keys[j]) - st.m) - log_s;
  }
}

// CTAs per row: doubled while the grid stays within 3 CTAs per SM (6 are
// resident), up to 8, each with at least 2048 logits (below that the merge
// costs more than the shorter share saves). Measured, bf16 rows of 50280 with
// 20 alternatives: 100 rows 17.4 us with 2 CTAs each, 14.8 with 4, 19.5 with
// 8; 296 rows 15.4 with 1, 20.3 with 2, 27.4 with 4.
int cluster_size(int64_t rows, int64_t vocab) {
  const int64_t sms = mamba_lm::sm_count();
  int n = 1;
  while (n < kMaxCluster && rows * n * 2 <= 3 * sms && vocab >= 2 * n * 2048) n *= 2;
  return n;
}

template <typename T>
cudaError_t launch(const LogprobParams& p, int64_t rows, cudaStream_t st) {
  const int n = cluster_size(rows, p.vocab);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(rows * n));
  cfg.blockDim = dim3(kThreads);
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = (unsigned)n;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = n > 1 ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, logprobs_kernel<T>, p);
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
  if (rows < 0 || rows >= (int64_t)1 << 31 || vocab < 1 || vocab > kMaxVocab)
    return set_last_error(MAMBA_SCAN_ERR_INVALID_ARGUMENT,
                          "token_logprobs: rows must be 0..2^31-1 and vocab 1..2^30");
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
  if (!mamba_lm::aligned_to(size, {logits}) || !mamba_lm::aligned_to(8, {target, top_id}) ||
      !mamba_lm::aligned_to(4, {logprob, entropy, top_logprob}))
    return set_last_error(MAMBA_SCAN_ERR_INVALID_ARGUMENT,
                          "token_logprobs: an address is not a multiple of its type's size");
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
  cudaStream_t cs = static_cast<cudaStream_t>(stream);
  cudaError_t e;
  switch (dtype) {
    case MAMBA_DTYPE_F32: e = launch<float>(p, rows, cs); break;
    case MAMBA_DTYPE_F16: e = launch<__half>(p, rows, cs); break;
    default: e = launch<__nv_bfloat16>(p, rows, cs); break;
  }
  if (e != cudaSuccess) return set_last_error(MAMBA_SCAN_ERR_CUDA, cudaGetErrorString(e));
  return MAMBA_SCAN_OK;
} catch (...) {
  return MAMBA_SCAN_ERR_CUDA;
}

}  // extern "C"
