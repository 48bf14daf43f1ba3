// Linear attention over prompts on the sm_100a tensor cores, in chunks of 64
// rows (include/mamba_lm_ops.h states the operator).
//
// Mathematics. With G_i the running sum of the chunk's log decays (base 2),
// S the state before the chunk, C its last row:
//   out_i = scale (2^G_i q_i S + sum_{j <= i} (q_i k_j) 2^(G_i - G_j) v_j)
//   S'    = 2^G_C S + sum_j 2^(G_C - G_j) k_j v_j^T
// which is four matrix products per chunk. Everything is held transposed,
// with the dv axis on the 128 lanes of tensor memory: S^T (dv x dk) lives in
// the threads' registers in fp32, and its split parts, like the weighted
// values', go to tensor memory as the A operand:
//   scores  [64 rows x 64]  = q k^T                  (A, B in shared memory)
//   O1^T    [dv x 64 rows]  = S^T q^T                (A in tensor memory)
//   O2^T    [dv x 64 rows]  = v^T P^T                (A, B in shared memory)
//   dS^T    [dv x dk]       = (weighted v)^T k       (A in tensor memory)
//
// Two kernels compute this: prompt_kernel for any type and layout, described
// here, and prompt_direct_kernel (further down) for bf16 tensors that TMA can
// take. 64 rows: the intra-chunk products and their weights grow with the
// chunk, the state's conversion shrinks with it, and at 128 rows neither
// tensor memory (640 columns) nor shared memory would hold a chunk.
//
// Numbers. All products are fp16 x fp16 with fp32 accumulation, of operands
// scaled by powers of two and split where fp16's 11 bits are too few: a
// float32 operand is hi + lo (22 bits; hi hi + hi lo + lo hi, a relative
// error of about 3 * 2^-22, the tensor core's TF32 form at half its cost); a
// 16-bit operand is exact in one part. Every row of q, k and v has its own
// power of two (largest element to 2^14..2^15), so rows of very different
// sizes keep their relative accuracy; within a row the parts' smallest step,
// 2^-24, is 2^-39 to 2^-38 of its largest element: a float32 element below
// 2^-17 of that, a bf16 one below 2^-31, loses bits. In the same way a score
// keeps to 2^-39 of the largest that its row's sizes allow, a value to 2^-39 of
// the chunk's largest |k||v|, the state to 2^-39 of its column's largest. (The
// kernel for bf16 further down has none of this.) The weighted values are always split in
// two: the state is fp32, whatever the inputs are. So are the scores and the
// state on their way into an output: one part (11 bits) of them put as large
// an error, 2^-12 of a term, into fp16 outputs as their own rounding does.
//
// Decays. G is summed in fixed point; the score of (i, j) is weighted by
// 2^(x_j - U_i - frac G_j) with x_j = er_j - floor G_j (er_j the exponent that
// undoes row j's scaling) and U_i the running maximum of x up to i: never
// more than 1, so nothing overflows whatever the decays, and the rest,
// 2^(G_i + U_i), is one factor for each output row.
#include <cudaTypedefs.h>

#include <algorithm>
#include <cstring>
#include <mutex>
#include <type_traits>

#include "linear_attention.h"
#include "lm_device.cuh"
#include "scan_device.cuh"
#include "scan_kernels.h"

namespace mamba_la {

using mamba_lm::from_f32;
using mamba_lm::sm_count;
using mamba_lm::to_f32;
using mamba_scan::smem_u32;

constexpr int kChunk = 64;
constexpr int kLanes = 128;      // dv columns per CTA: the lanes of tensor memory
constexpr int kSlab = 64 * 128;  // bytes of 64 rows x 64 fp16 in the 128-byte swizzle

__device__ int g_error = 0;

template <typename T> struct Parts { static constexpr int n = 1; };
template <> struct Parts<float> { static constexpr int n = 2; };

// Of one chunk, from scan_decays; read 16 bytes at a time. G is the running
// log2 decay, from the chunk's first row on.
struct __align__(16) DecayWeights {
  float2 gg[kChunk];                        // floor G and G - floor G
  __align__(16) float from_start[kChunk];   // 2^G_j
  __align__(16) float to_end[kChunk];       // 2^(G_last - G_j)
  int64_t total;                            // G_last, 32 fraction bits
};

struct __align__(16) Decays : DecayWeights {
  int Gi[kChunk];                           // floor G
  float Gf[kChunk];                         // G - floor G
  float up[kChunk], down[kChunk];           // 2^Gf and 2^-Gf
};

struct __align__(16) Small {
  Decays dec[2];                // this chunk's and the next one's
  __align__(16) float2 xg[kChunk];  // (er_j - floor G_j, G_j - floor G_j)
  float U[kChunk];              // U_i + kShift
  __align__(16) float2 c12[kChunk]; // factors of O1 and O2 for each row
  __align__(16) float fv[16][kChunk / 2];  // each warp's weights of its value rows
  int eq[kChunk], ek[kChunk], ev[kChunk];  // the rows' exponents
  float gamma, cs;              // 2^G_C, and the factor of dS
  uint32_t rowmax[4][kLanes];   // |S| maxima of the dk quarters (bit patterns)
  uint64_t full, v_full;         // q and k, v have landed
  uint64_t scores, o1, ds, o2;   // products are done
  int gave_up;                   // a wait ran out
  uint32_t tmem;
};

// Sizes of one kernel: DKP / DVP = dk / dv tile rounded up to 64 or 128.
template <typename T, int DKP_, int DVP_>
struct Cfg {
  static constexpr int DKP = DKP_, DVP = DVP_, NP = Parts<T>::n;  // (P and S: always two)
  static constexpr int kRawQ = kChunk * DKP * (int)sizeof(T), kRawV = kChunk * DVP * (int)sizeof(T);
  static constexpr int kPartQ = DKP / 64 * kSlab, kPartV = DVP / 64 * kSlab;
  // shared memory: raw q, k, v as TMA delivers them, then their parts, P's
  // parts, and the small arrays
  static constexpr int kOffK = kRawQ, kOffV = 2 * kRawQ, kOffQP = kOffV + kRawV;
  static constexpr int kOffKP = kOffQP + NP * kPartQ, kOffVP = kOffKP + NP * kPartQ;
  // With DKP = 64 two CTAs share an SM: the weighted values take the place of
  // S's parts in tensor memory, and, where q has two parts, P that of q in
  // shared memory, once O1 is done.
  static constexpr bool kShareSV = DKP == 64;
  static constexpr int kEndV = kOffVP + NP * kPartV;
  static constexpr bool kShareQP = kShareSV && NP == 2;
  static constexpr int kOffP = kShareQP ? kOffQP : kEndV;
  static constexpr int kOffSmall = kShareQP ? kEndV : kEndV + 2 * kSlab;
  // (the products' A operands are 128 rows: with 64 real ones they read up to
  // one slab past their own tile, rows whose results nobody looks at)
  static constexpr int kBytes = kOffSmall + (int)std::max<size_t>(sizeof(Small), kSlab) + 1024;
  static constexpr int kColS = 0, kColV = kShareSV ? 0 : DKP;
  static constexpr int kColAcc = kShareSV ? 64 : kColV + 64, kColO1 = kColAcc + 64;
  static constexpr int kColD = kColO1 + 64;
  static constexpr int kTmemCols = kColD + DKP <= 256 ? 256 : 512;
  static_assert(kColD + DKP <= kTmemCols, "tensor memory");
};

struct Params {
  mamba_linear_attention_args a;
  float* ws;        // [tail unit][segment][DKP][128] states, then decays
  float* ws_decay;  // [tail unit][segment]
  int tiles;        // dv tiles of 128
  int n_full, n_tail, n_seg;
  int seg_len;      // rows per segment, a multiple of 64
  int aggregate;    // 1: only the segments' end states from zero
  int tma;          // q, k and v come by TMA
  // dk over 128: a launch for each half of the key columns. a holds the half's
  // q, k, dk, h0 and h_last; the first half's outputs wait in acc.
  int64_t state_rows;  // dk of the whole head
  float* acc;          // [batch][seqlen][heads][dv]
  int half;            // 0 or 1
};

struct Maps {
  CUtensorMap q, k, v;
};

// ------------------------------------------------------------ PTX wrappers

__device__ __forceinline__ void tma_load_4d(void* dst, const CUtensorMap* map, uint64_t* bar,
                                            int c0, int c1, int c2, int c3) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%3, %4, %5, %6}], [%2];" ::"r"(smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(smem_u32(bar)), "r"(c0), "r"(c1), "r"(c2), "r"(c3)
      : "memory");
}

__device__ __forceinline__ void tc_fence_before() {
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
}
__device__ __forceinline__ void tc_fence_after() {
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
}
__device__ __forceinline__ void tmem_wait_ld() {
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tmem_wait_st() {
  asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
}

__device__ __forceinline__ void tmem_ld16(uint32_t addr, float (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, "
      "%12, %13, %14, %15}, [%16];"
      : "=f"(r[0]), "=f"(r[1]), "=f"(r[2]), "=f"(r[3]), "=f"(r[4]), "=f"(r[5]), "=f"(r[6]),
        "=f"(r[7]), "=f"(r[8]), "=f"(r[9]), "=f"(r[10]), "=f"(r[11]), "=f"(r[12]), "=f"(r[13]),
        "=f"(r[14]), "=f"(r[15])
      : "r"(addr));
}

__device__ __forceinline__ void tmem_st8(uint32_t addr, const uint32_t (&r)[8]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"r"(addr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
      : "memory");
}

// Shared-memory matrix descriptors of tiles in the 128-byte swizzle (64 fp16
// = 128 bytes per row, groups of 8 rows 1024 bytes apart), as the low word
// (start address >> 4 in bits [0,14), leading byte offset >> 4 in [16,30))
// and the high one (stride byte offset >> 4, descriptor version 1 in bit 14,
// layout SWIZZLE_128B = 2 in [29,32)). K-major: the rows are M or N. MN-major:
// the rows are K, and the leading byte offset is the distance of the next 64
// columns of M or N (one slab). A step of `bytes` adds bytes >> 4.
constexpr uint32_t kDescHigh = (1024u >> 4) | (1u << 14) | (2u << 29);
__device__ __forceinline__ uint32_t desc_k(uint32_t addr) { return (addr >> 4) | (1u << 16); }
__device__ __forceinline__ uint32_t desc_mn(uint32_t addr) {
  return (addr >> 4) | ((uint32_t)(kSlab >> 4) << 16);
}

// Instruction descriptor of kind::f16: D fp32 (bit 4), A and B fp16 (0), A and
// B MN-major in bits 15 and 16, N >> 3 in [17,23), M >> 4 in [24,29); M = 128.
__host__ __device__ constexpr uint32_t idesc(int n, bool a_mn, bool b_mn) {
  return (1u << 4) | ((uint32_t)a_mn << 15) | ((uint32_t)b_mn << 16) | ((uint32_t)(n >> 3) << 17) |
         ((uint32_t)(128 >> 4) << 24);
}

// The products are issued by a whole warp, converged, with one lane's
// predicate on the instruction itself: operands and control flow stay uniform
// (behind a divergent branch each product took about 100 clocks to issue).
__device__ __forceinline__ uint32_t elect_one() {
  uint32_t leader;
  asm volatile(
      "{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}\n"
      : "=r"(leader));
  return leader;
}

__device__ __forceinline__ void mma_ss(uint32_t leader, uint32_t d, uint32_t a, uint32_t b,
                                       uint32_t desc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t.reg .b64 da, db;\n\t"
      "setp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %6, 0;\n\t"
      "mov.b64 da, {%1, %5};\n\tmov.b64 db, {%2, %5};\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %3, p;\n\t}\n" ::"r"(d),
      "r"(a), "r"(b), "r"(desc), "r"(accumulate), "r"(kDescHigh), "r"(leader)
      : "memory");
}

__device__ __forceinline__ void mma_ts(uint32_t leader, uint32_t d, uint32_t a, uint32_t b,
                                       uint32_t desc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t.reg .b64 db;\n\t"
      "setp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %6, 0;\n\t"
      "mov.b64 db, {%2, %5};\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], db, %3, p;\n\t}\n" ::"r"(d),
      "r"(a), "r"(b), "r"(desc), "r"(accumulate), "r"(kDescHigh), "r"(leader)
      : "memory");
}

__device__ __forceinline__ void mma_commit(uint32_t leader, uint64_t* bar) {
  asm volatile(
      "{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %1, 0;\n\t"
      "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}\n" ::"r"(
          smem_u32(bar)),
      "r"(leader)
      : "memory");
}

// A bounded wait that also ends when another thread's has run out. Each try
// may park the warp for up to 2 us (the hint) instead of spinning on issue
// slots that the other groups need; 2^20 tries without one are far beyond any
// wait here. (Few instructions: the roles' code competes for the instruction
// caches.)
__device__ __forceinline__ bool wait_or_leave(uint64_t* bar, uint32_t parity, int* gave_up) {
#pragma unroll 1
  for (int tries = 0; tries < (1 << 20); ++tries) {
    uint32_t done;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, 2000;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}\n"
        : "=r"(done)
        : "r"(smem_u32(bar)), "r"(parity)
        : "memory");
    if (done) return true;
    if (*reinterpret_cast<volatile int*>(gave_up)) return false;
  }
  *reinterpret_cast<volatile int*>(gave_up) = 1;
  atomicExch(&g_error, 6);  // MAMBA_SCAN_ERR_DEVICE_TIMEOUT
  return false;
}

// ------------------------------------------------------------- small pieces

// The exponent e with |x| 2^e in [2^14, 2^15) for the largest |x| of a row,
// from the exponent field of its fp32 form (at most 126: rows of tiny values
// stay finite).
__device__ __forceinline__ int scale_exponent(int field) { return min(141 - field, 126); }

__device__ __forceinline__ float pow2i(int e) { return __int_as_float((e + 127) << 23); }

// x 2^e for x in [1/2, 2): 0 below fp32's normal range, infinity above it.
__device__ __forceinline__ float shift2(float x, int e) {
  return e < -125 ? x * 0.f : x * (e > 127 ? __int_as_float(0x7f800000) : pow2i(max(e, -126)));
}

__device__ __forceinline__ uint32_t pack_half2(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// A pair as fp16 hi + lo: hi to nearest, lo the rest to nearest.
__device__ __forceinline__ void split_half2(float2 x, uint32_t& hi, uint32_t& lo) {
  const __half2 h = __floats2half2_rn(x.x, x.y);
  const float2 f = __half22float2(h);
  hi = *reinterpret_cast<const uint32_t*>(&h);
  x = __fadd2_rn(x, make_float2(-f.x, -f.y));
  lo = pack_half2(x.x, x.y);
}

__device__ __forceinline__ float2 twice(float x) { return make_float2(x, x); }

// Sixteen bytes of a raw row as floats.
template <typename T>
__device__ __forceinline__ void unpack16(const uint4& w, float (&f)[16 / sizeof(T)]) {
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

// The largest magnitude among sixteen bytes of a row, as its bit pattern (of
// T, in the low bits): patterns without the sign order like the magnitudes.
template <typename T> __device__ __forceinline__ uint32_t max_bits(const uint4& w) {
  if constexpr (sizeof(T) == 4) {
    // (as floats: absolute values cost nothing there. NaN is skipped: a row
    // with one is spoilt whatever its scale)
    return __float_as_uint(fmaxf(fmaxf(fabsf(__uint_as_float(w.x)), fabsf(__uint_as_float(w.y))),
                                 fmaxf(fabsf(__uint_as_float(w.z)), fabsf(__uint_as_float(w.w)))));
  } else {
    const uint32_t m = __vmaxu2(__vmaxu2(w.x & 0x7fff7fffu, w.y & 0x7fff7fffu),
                                __vmaxu2(w.z & 0x7fff7fffu, w.w & 0x7fff7fffu));
    return max(m & 0xffffu, m >> 16);
  }
}

// The fp32 exponent field of a magnitude of type T.
template <typename T> __device__ __forceinline__ int exponent_field(uint32_t bits) {
  if constexpr (sizeof(T) == 4) return (int)(bits >> 23);
  if constexpr (std::is_same<T, __half>::value) return (int)(bits >> 10) + 112;
  return (int)(bits >> 7);
}

// One raw tile [64][W] -> fp16 parts in the 128-byte swizzle, and each row's
// exponent, in two steps so that the caller can load several tiles first. A
// warp's lanes hold 16 bytes each of kRows rows at once.
template <typename T, int W, int kWarps>
struct TileConverter {
  static constexpr int NP = Parts<T>::n, kE = 16 / (int)sizeof(T);
  static constexpr int kRowLanes = W / kE, kRows = 32 / kRowLanes;
  static constexpr int kIter = kChunk / (kWarps * kRows);
  static constexpr int kPart = W / 64 * kSlab;
  uint4 w[kIter];

  // rows at or past n become zeros whatever the tile holds
  __device__ __forceinline__ void load(const uint8_t* raw, int n) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
#pragma unroll
    for (int i = 0; i < kIter; ++i) {
      const int r = (i * kWarps + warp) * kRows + lane / kRowLanes;
      w[i] = *reinterpret_cast<const uint4*>(raw + r * W * (int)sizeof(T) + lane % kRowLanes * 16);
      if (r >= n) w[i] = make_uint4(0, 0, 0, 0);
    }
  }

  __device__ __forceinline__ void store(uint8_t* parts, int* exps) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    uint32_t m[kIter];
#pragma unroll
    for (int i = 0; i < kIter; ++i) m[i] = max_bits<T>(w[i]);
    if constexpr (kRowLanes == 32) {
#pragma unroll
      for (int i = 0; i < kIter; ++i) m[i] = __reduce_max_sync(0xffffffffu, m[i]);
    } else {
#pragma unroll
      for (int o = kRowLanes / 2; o > 0; o >>= 1)
#pragma unroll
        for (int i = 0; i < kIter; ++i) m[i] = max(m[i], __shfl_xor_sync(0xffffffffu, m[i], o));
    }
    const int col = lane % kRowLanes * kE;
#pragma unroll
    for (int i = 0; i < kIter; ++i) {
      const int r = (i * kWarps + warp) * kRows + lane / kRowLanes;
      const int e = scale_exponent(exponent_field<T>(m[i]));
      const float s = pow2i(e);
      if (lane % kRowLanes == 0) exps[r] = e;
      float f[kE];
      unpack16<T>(w[i], f);
      uint32_t hi[kE / 2], lo[kE / 2];
#pragma unroll
      for (int j = 0; j < kE / 2; ++j) {
        const float2 x = __fmul2_rn(make_float2(f[2 * j], f[2 * j + 1]), twice(s));
        if constexpr (NP == 2) split_half2(x, hi[j], lo[j]);
        else hi[j] = pack_half2(x.x, x.y);
      }
      const int off = col / 64 * kSlab + r * 128 + ((col % 64 * 2) ^ ((r & 7) << 4));
      if constexpr (NP == 2) {
        *reinterpret_cast<uint2*>(parts + off) = make_uint2(hi[0], hi[1]);
        *reinterpret_cast<uint2*>(parts + kPart + off) = make_uint2(lo[0], lo[1]);
      } else {
        *reinterpret_cast<uint4*>(parts + off) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
      }
    }
  }
};

// A raw tile without TMA, by kN threads: n rows of `cols` elements with any
// strides and alignment, zeros outside. Rows that start and end on 8 bytes
// come by asynchronous copies (cp.async), others element by element.
template <typename T, int W, int kN>
__device__ __forceinline__ void load_tile(uint8_t* raw, const T* src, int64_t row_stride, int n,
                                          int cols) {
  constexpr int kE = 8 / (int)sizeof(T);
  const uint32_t odd = (uint32_t)reinterpret_cast<uintptr_t>(src) |
                       (uint32_t)(row_stride * (int64_t)sizeof(T)) | (uint32_t)(cols * (int)sizeof(T));
  if ((odd & 7u) == 0) {
#pragma unroll 4
    for (int i = threadIdx.x; i < kChunk * W / kE; i += kN) {
      const int r = i / (W / kE), c = i % (W / kE) * kE;
      uint8_t* dst = raw + i * 8;
      if (r < n && c < cols)
        asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(smem_u32(dst)),
                     "l"(src + r * row_stride + c)
                     : "memory");
      else
        *reinterpret_cast<uint2*>(dst) = make_uint2(0, 0);
    }
  } else {
    T* dst = reinterpret_cast<T*>(raw);
#pragma unroll 4
    for (int i = threadIdx.x; i < kChunk * W; i += kN) {
      const int r = i / W, c = i % W;
      dst[i] = (r < n && c < cols) ? src[r * row_stride + c] : from_f32<T>(0.f);
    }
  }
}

__device__ __forceinline__ void async_copies_done() {
  asm volatile("cp.async.wait_all;" ::: "memory");
}

// Decays, by one warp, two rows per lane: load_decays reads rows t.. (0 past
// the n-th), scan_decays forms their running sums. The sums are fixed point
// with 32 fraction bits: exact to 2^-33 per row whatever their size, and
// split into integer and fraction for nothing. Decays below 2^-200 are 0 in
// fp32 and are clamped there; NaN and +inf spoil the chunk.
__device__ __forceinline__ float2 load_decays(const float* g, int64_t stride, int64_t t, int n) {
  const int j = 2 * (threadIdx.x & 31);
  return make_float2(j < n ? g[(t + j) * stride] : 0.f, j + 1 < n ? g[(t + j + 1) * stride] : 0.f);
}

__device__ __forceinline__ int64_t fixed_log2(float g) {
  g = fminf(fmaxf(g, -138.f), 1e6f);
  // g log2(e) as the sum of two floats
  const float hi = g * 1.44269502162933349609f;
  const float lo = fmaf(g, 1.92596299112661746887e-8f, fmaf(g, 1.44269502162933349609f, -hi));
  return __float2ll_rn(hi * 4294967296.f) + __float2ll_rn(lo * 4294967296.f);
}

template <typename D>
__device__ __forceinline__ void scan_decays(D& d, float2 g) {
  const int lane = threadIdx.x & 31, j = 2 * lane;
  const bool bad = __any_sync(0xffffffffu, !(g.x < 3e38f) || !(g.y < 3e38f));
  const int64_t x0 = fixed_log2(g.x), x1 = fixed_log2(g.y);
  int64_t sum = x0 + x1;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t up = __shfl_up_sync(0xffffffffu, sum, o);
    if (lane >= o) sum += up;
  }
  const int64_t G[2] = {sum - x1, sum};
  const int64_t last = __shfl_sync(0xffffffffu, sum, 31);
  const float last_up = exp2f((float)(uint32_t)last * 2.3283064365386963e-10f);
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const float f = bad ? __int_as_float(0x7fc00000) : (float)(uint32_t)G[i] * 2.3283064365386963e-10f;
    const float up = exp2f(f), down = exp2f(-f);
    d.gg[j + i] = make_float2((float)(int)(G[i] >> 32), f);
    if constexpr (std::is_same<D, Decays>::value) {
      d.Gi[j + i] = (int)(G[i] >> 32);
      d.Gf[j + i] = f;
      d.up[j + i] = up;
      d.down[j + i] = down;
    }
    d.from_start[j + i] = shift2(up, (int)(G[i] >> 32));
    d.to_end[j + i] = last_up * shift2(down, (int)(last >> 32) - (int)(G[i] >> 32));
  }
  if (lane == 31) d.total = sum;
}

// ------------------------------------------------------------------ kernel

// One CTA's unit (sequence, head, tile of 128 dv columns) and segment.
struct Work {
  int unit, seg = 0, tail = -1;  // tail: the unit's place among the split ones
  int b, h, g, d0, bh;

  __device__ __forceinline__ explicit Work(const Params& p) {
    const int x = (int)blockIdx.x;
    if (p.aggregate) {
      tail = x / (p.n_seg - 1);
      seg = x % (p.n_seg - 1);
    } else if (x >= p.n_full) {
      tail = (x - p.n_full) / p.n_seg;
      seg = (x - p.n_full) % p.n_seg;
    }
    unit = tail >= 0 ? p.n_full + tail : x;
    const int H = (int)p.a.heads;
    bh = unit / p.tiles;
    d0 = unit % p.tiles * kLanes;
    b = bh / H;
    h = bh % H;
    g = h / (H / (int)p.a.groups);
  }
};

// Its rows: [begin, end) count, [end, limit) are padding.
struct Rows {
  int begin = 0, end, limit;

  __device__ __forceinline__ Rows(const Params& p, const Work& w) {
    const int L = (int)p.a.seqlen;
    limit = L;
    if (w.tail >= 0) {
      begin = (int)min((int64_t)w.seg * p.seg_len, (int64_t)L);
      limit = (int)min((int64_t)begin + p.seg_len, (int64_t)L);
    }
    end = limit;
    if (p.a.lengths) end = max(begin, min(end, p.a.lengths[w.b]));
  }
  __device__ __forceinline__ int chunks() const { return (end - begin + kChunk - 1) / kChunk; }
};

// A thread's columns [col0, col0 + N) of the state entering its rows: h0, or
// what the join left for a later segment, or 0.
template <int DKP, int N>
__device__ __forceinline__ void load_state(float (&S)[N], const Params& p, const Work& w, int col0,
                                           int row, bool d_ok) {
  const float* src = nullptr;
  int64_t step = 0;
  if (w.tail >= 0 && w.seg > 0 && !p.aggregate) {
    src = p.ws + ((int64_t)w.tail * (p.n_seg - 1) + w.seg - 1) * DKP * kLanes + row;
    step = kLanes;
  } else if (p.a.h0 && !p.aggregate && d_ok) {
    src = p.a.h0 + (int64_t)w.bh * p.state_rows * p.a.dv + w.d0 + row;
    step = p.a.dv;
  }
#pragma unroll
  for (int i = 0; i < N; ++i) S[i] = src && col0 + i < p.a.dk ? src[(col0 + i) * step] : 0.f;
}

// The state after them: to h_last, or a segment's end state to the workspace.
template <int DKP, int N>
__device__ __forceinline__ void store_state(const float (&S)[N], const Params& p, const Work& w,
                                            int col0, int row, bool d_ok) {
  if (p.aggregate) {
    float* dst = p.ws + ((int64_t)w.tail * (p.n_seg - 1) + w.seg) * DKP * kLanes + row;
#pragma unroll
    for (int i = 0; i < N; ++i) dst[(col0 + i) * kLanes] = S[i];
  } else if (p.a.h_last && d_ok && (w.tail < 0 || w.seg == p.n_seg - 1)) {
    float* dst = p.a.h_last + (int64_t)w.bh * p.state_rows * p.a.dv + w.d0 + row;
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (col0 + i < p.a.dk) dst[(col0 + i) * p.a.dv] = S[i];
  }
}

// A segment's whole decay, from its fixed-point log2.
__device__ __forceinline__ void store_total(const Params& p, const Work& w, int64_t total) {
  p.ws_decay[w.tail * (p.n_seg - 1) + w.seg] =
      shift2(exp2f((float)(uint32_t)total * 2.3283064365386963e-10f),
             (int)max(min(total >> 32, (int64_t)1000), (int64_t)-1000));
}

// Warps besides the compute warps: two that work, filled up to a group of four
// for setmaxnreg where one CTA has the SM to itself.
__host__ __device__ constexpr int issue_warps(int compute_warps) {
  return compute_warps == 16 ? 4 : 2;
}

// kWarps compute warps (warp w holds tensor memory lanes 32 (w % 4).. and the
// (w / 4)-th share of the columns) work in step; two more issue: the first the
// loads, the scores and O2, the second O1 and dS, and the decays one chunk
// ahead. (A product of 128 x 64 x 16 takes the tensor core 32 clocks and its
// issuing warp about 70: one warp issuing all of a float32 chunk's 72 held the
// others up for a third of the time.)
//
// Measured on one B200, one CTA per SM: 6.3 us a chunk of 64 rows for fp32
// heads of 128 x 128 (HBM alone would take 3.0), 5.3 in fp16, about a sixth each in the
// conversion, the values, the scores, the state and the outputs; the tensor
// core is busy 21% and the warps issue in 44% of the clocks, so what bounds it
// is the latency of the steps in sequence, then their instructions. One
// sequence of 2048 rows and 40 heads takes 106 us in fp16, 4 of them 272 us in
// fp32 (254 where the next call's first CTAs fill the last wave).
//
// kHalves: heads with more than 128 keys, whose state tensor memory does not
// hold. Outputs and states are sums over the keys, so a launch serves the
// first 128 and a second one the others and adds the first's outputs, in fp32.
// 4 sequences of 2048 rows, 16 heads of 256 x 256: 454 us in bf16 (token by
// token 4.7 ms), 487 us in fp32.
template <typename T, int DKP, int DVP, int kWarps, bool kHalves = false>
__global__ void __launch_bounds__(32 * (kWarps + issue_warps(kWarps)), 16 / kWarps)
    prompt_kernel(const __grid_constant__ Maps maps, const __grid_constant__ Params p) {
  using C = Cfg<T, DKP, DVP>;
  constexpr int NP = C::NP, kThreads = 32 * (kWarps + issue_warps(kWarps));
  constexpr int kSplit = kWarps / 4;             // warps per lane quarter
  constexpr int kSCols = DKP / kSplit;           // state columns of a thread
  constexpr int kTok = kChunk / kSplit;          // rows of a thread in the value and output steps
  constexpr int kShift = 15 + (DKP == 128 ? 7 : 6);  // scores < dk 2^30 to below 2^15
  extern __shared__ uint8_t smem_raw[];
  uint8_t* sm = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  Small& s = *reinterpret_cast<Small*>(sm + C::kOffSmall);
  const mamba_linear_attention_args& a = p.a;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int quarter = warp & 3, part = warp >> 2;

  const Work w(p);
  const int row = quarter * 32 + lane, d = w.d0 + row;
  const bool d_ok = d < (int)a.dv && row < DVP;

  if (threadIdx.x == 0) {
    mamba_scan::mbar_init(&s.full, 1);
    mamba_scan::mbar_init(&s.v_full, 1);
    s.gave_up = 0;
    mamba_scan::mbar_init(&s.scores, 1);
    mamba_scan::mbar_init(&s.o1, 1);
    mamba_scan::mbar_init(&s.ds, 1);
    mamba_scan::mbar_init(&s.o2, 1);
    mamba_scan::fence_mbarrier_init();
  }
  if (warp == 0) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                     smem_u32(&s.tmem)),
                 "r"(C::kTmemCols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = __shfl_sync(0xffffffffu, s.tmem, 0), leader = elect_one();
  // The dependents' CTAs come only after every CTA here holds its tensor
  // memory. Whole units of a split plan do not wait for the segments' passes:
  // those began after everything before them had ended.
  mamba_scan::pdl_trigger();
  if (w.tail >= 0 || p.n_tail == 0) mamba_scan::pdl_wait();

  const Rows rows(p, w);
  const int row0 = rows.begin, row1 = rows.end;
  const int n_chunks = rows.chunks();

  const float* decay = a.log_decay + w.b * a.decay_stride[0] + w.h * a.decay_stride[2];

  auto load_qk = [&](int t) {  // one thread
    mamba_scan::mbar_arrive_expect_tx(&s.full, C::kRawQ + (p.aggregate ? 0 : C::kRawQ));
    if (!p.aggregate) tma_load_4d(sm, &maps.q, &s.full, 0, w.g, t, w.b);
    tma_load_4d(sm + C::kOffK, &maps.k, &s.full, 0, w.g, t, w.b);
  };
  auto load_v = [&](int t) {
    mamba_scan::mbar_arrive_expect_tx(&s.v_full, C::kRawV);
    tma_load_4d(sm + C::kOffV, &maps.v, &s.v_full, w.d0, w.h, t, w.b);
  };
  auto wait = [&](uint64_t* bar, uint32_t phase) { return wait_or_leave(bar, phase, &s.gave_up); };

  const uint32_t lane_base = tmem + ((uint32_t)(quarter * 32) << 16);
  const uint32_t qp = smem_u32(sm + C::kOffQP), kp = smem_u32(sm + C::kOffKP);
  const uint32_t vp = smem_u32(sm + C::kOffVP), pp = smem_u32(sm + C::kOffP);

  // The roles meet at barriers: (1) parts and state ready, (2) values in
  // tensor memory, (3) P in shared memory.
  if (warp >= kWarps) {
    if constexpr (kWarps == 16) asm volatile("setmaxnreg.dec.sync.aligned.u32 64;");
    const bool issues_a = warp == kWarps, issues_b = warp == kWarps + 1;
    bool left = false;
    if (n_chunks > 0 && issues_a && p.tma && lane == 0) {
      load_qk(row0);
      load_v(row0);
    }
    if (n_chunks > 0 && issues_b)
      scan_decays(s.dec[0], load_decays(decay, a.decay_stride[1], row0, min(kChunk, row1 - row0)));
    __syncwarp();
    for (int c = 0; c < n_chunks; ++c) {
      const int t0 = row0 + c * kChunk;
      const bool more = c + 1 < n_chunks;
      float2 g_next = make_float2(0.f, 0.f);
      if (!p.tma) __syncthreads();  // (the compute warps' own loads)
      if (__syncthreads_or(0)) {  // (1); a wait gave up: every thread leaves
        left = true;
        break;
      }
      if (issues_a) {
        // the next chunk's q and k (the raw ones are used up), then the scores
        if (p.tma && more && lane == 0) load_qk(t0 + kChunk);
        __syncwarp();
        if (!p.aggregate) {
          tc_fence_after();
          uint32_t acc = 0;
#pragma unroll 1
          for (int pr = NP == 2 ? 0 : 2; pr < 3; ++pr) {  // lo hi, hi lo, hi hi
            uint32_t ad = desc_k(qp + (pr == 0 ? C::kPartQ : 0));
            uint32_t bd = desc_k(kp + (pr == 1 ? C::kPartQ : 0));
#pragma unroll 1
            for (int kk = 0; kk < DKP / 16; ++kk) {
              mma_ss(leader, tmem + C::kColAcc, ad, bd, idesc(64, false, false), acc);
              const uint32_t step = (kk & 3) == 3 ? (kSlab - 96) >> 4 : 2;  // 16 columns on
              ad += step;
              bd += step;
              acc = 1;
            }
          }
          mma_commit(leader, &s.scores);
        }
      } else if (issues_b) {
        // O1, of the state before this chunk
        if (more) g_next = load_decays(decay, a.decay_stride[1], t0 + kChunk,
                                       min(kChunk, row1 - t0 - kChunk));
        if (!p.aggregate) {
          tc_fence_after();
          uint32_t acc = 0;
#pragma unroll 1
          for (int pr = 0; pr < 3; ++pr) {  // lo hi, (hi lo), hi hi
            if (pr == 1 && NP == 1) continue;
            uint32_t ac = tmem + C::kColS + (pr == 0 ? DKP / 2 : 0);
            uint32_t bd = desc_k(qp + (pr == 1 ? C::kPartQ : 0));
#pragma unroll 1
            for (int kk = 0; kk < DKP / 16; ++kk) {
              mma_ts(leader, tmem + C::kColO1, ac, bd, idesc(64, false, false), acc);
              ac += 8;
              bd += (kk & 3) == 3 ? (kSlab - 96) >> 4 : 2;
              acc = 1;
            }
          }
          mma_commit(leader, &s.o1);
        }
      }
      // The rows' factors, by a warp that has nothing to issue or, of two, by
      // the one whose product is not waited for next.
      if (warp == (kWarps == 16 ? kWarps + 2 : kWarps + 1) && !p.aggregate) {
        // U_i, the running maximum of the row factors
        // er_j - floor G_j; lane l looks at rows l and l + 32.
        const Decays& dec = s.dec[c & 1];
        const int n = min(kChunk, row1 - t0);
        int m[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int j = lane + 32 * i;
          m[i] = j < n ? -(s.ek[j] + s.ev[j]) - dec.Gi[j] : -1000000;
        }
#pragma unroll 1
        for (int o = 1; o < 32; o <<= 1) {
          const int up0 = __shfl_up_sync(0xffffffffu, m[0], o), up1 = __shfl_up_sync(0xffffffffu, m[1], o);
          if (lane >= o) m[0] = max(m[0], up0), m[1] = max(m[1], up1);
        }
        m[1] = max(m[1], __shfl_sync(0xffffffffu, m[0], 31));
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int j = lane + 32 * i, e = dec.Gi[j] - s.eq[j];
          s.U[j] = (float)(m[i] + kShift);
          s.c12[j] = make_float2(a.scale * shift2(dec.up[j], e),
                                 a.scale * shift2(dec.up[j], e + m[i] + kShift + 32));
        }
      }
      __syncthreads();  // (2)
      if (issues_a && p.tma && more) {
        if (lane == 0) load_v(t0 + kChunk);
        __syncwarp();
      }
      if (issues_b) {
        // dS; the next chunk's decays
        tc_fence_after();
        uint32_t acc = 0;
#pragma unroll 1
        for (int pr = 0; pr < 3; ++pr) {  // lo hi, (hi lo), hi hi
          if (pr == 1 && NP == 1) continue;
          uint32_t ac = tmem + C::kColV + (pr == 0 ? kChunk / 2 : 0);
          uint32_t bd = desc_mn(kp + (pr == 1 ? C::kPartQ : 0));
#pragma unroll 1
          for (int kk = 0; kk < kChunk / 16; ++kk) {
            mma_ts(leader, tmem + C::kColD, ac, bd, idesc(DKP, false, true), acc);
            ac += 8;
            bd += 128;
            acc = 1;
          }
        }
        mma_commit(leader, &s.ds);
        if (more) scan_decays(s.dec[(c + 1) & 1], g_next);
      }
      if (p.aggregate) continue;
      __syncthreads();  // (3)
      if (issues_a) {  // O2, over the scores
        tc_fence_after();
        uint32_t acc = 0;
#pragma unroll 1
        for (int pr = NP == 2 ? 0 : 1; pr < 3; ++pr) {  // (lo hi), hi lo, hi hi
          uint32_t ad = desc_mn(vp + (pr == 0 ? C::kPartV : 0));
          uint32_t bd = desc_k(pp + (pr == 1 ? kSlab : 0));
#pragma unroll 1
          for (int kk = 0; kk < kChunk / 16; ++kk) {
            mma_ss(leader, tmem + C::kColAcc, ad, bd, idesc(64, true, false), acc);
            ad += 128;
            bd += 2;
            acc = 1;
          }
        }
        mma_commit(leader, &s.o2);
      }
    }
    if (left && p.tma && issues_a && lane == 0) {
      // the loads in flight have to land before the memory goes
      for (uint32_t phase = 0; phase < 2; ++phase) {
        mamba_scan::mbar_wait(&s.full, phase, &g_error);
        mamba_scan::mbar_wait(&s.v_full, phase, &g_error);
      }
    }
    __syncwarp();
  } else {
    // 512 x 104 + 128 x 64 registers of the launch's 640 x 96
    if constexpr (kWarps == 16) asm volatile("setmaxnreg.inc.sync.aligned.u32 104;");
    // S^T: this thread's dv lane, columns [part * kSCols, +kSCols)
    float2 S[kSCols / 2];
    load_state<DKP>(reinterpret_cast<float(&)[kSCols]>(S), p, w, part * kSCols, row, d_ok);
    float inv_s = 0.f;  // 1 / scale of the parts of S in tensor memory
    // writes the parts of S (scaled so that the lane's largest is near 2^15)
    auto store_state_parts = [&]() {
      float m = 0.f;
#pragma unroll
      for (int i = 0; i < kSCols / 2; ++i) m = fmaxf(m, fmaxf(fabsf(S[i].x), fabsf(S[i].y)));
      s.rowmax[part][row] = __float_as_uint(m);
      asm volatile("bar.sync %0, %1;" ::"r"(1 + quarter), "n"(32 * kSplit) : "memory");
      uint32_t bits = 0;
#pragma unroll
      for (int i = 0; i < kSplit; ++i) bits = max(bits, s.rowmax[i][row]);
      const int e = scale_exponent((int)(bits >> 23));
      const float sc = pow2i(e);
      inv_s = pow2i(-e);
#pragma unroll
      for (int i0 = 0; i0 < kSCols; i0 += 16) {
        uint32_t hi[8], lo[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float2 x = __fmul2_rn(S[i0 / 2 + i], twice(sc));
          split_half2(x, hi[i], lo[i]);
        }
        const uint32_t col = (uint32_t)(C::kColS + (part * kSCols + i0) / 2);
        tmem_st8(lane_base + col, hi);
        tmem_st8(lane_base + col + DKP / 2, lo);
      }
      tmem_wait_st();
    };

    const int64_t out_stride = a.heads * a.dv;
    T* out = static_cast<T*>(a.out) +
             (((int64_t)w.b * a.seqlen + row0) * a.heads + w.h) * a.dv + d;  // of the chunk's first row
    // loads without TMA, issued at the same places as TMA's
    auto copy_qk = [&](int t) {
      const int n = min(kChunk, row1 - t);
      const T* q = static_cast<const T*>(a.q) + w.b * a.q_stride[0] + w.g * a.q_stride[2];
      const T* k = static_cast<const T*>(a.k) + w.b * a.k_stride[0] + w.g * a.k_stride[2];
      if (!p.aggregate)
        load_tile<T, DKP, 32 * kWarps>(sm, q + t * a.q_stride[1], a.q_stride[1], n, (int)a.dk);
      load_tile<T, DKP, 32 * kWarps>(sm + C::kOffK, k + t * a.k_stride[1], a.k_stride[1], n,
                                     (int)a.dk);
    };
    auto copy_v = [&](int t) {
      const T* v = static_cast<const T*>(a.v) + w.b * a.v_stride[0] + w.h * a.v_stride[2] + w.d0;
      load_tile<T, DVP, 32 * kWarps>(sm + C::kOffV, v + t * a.v_stride[1], a.v_stride[1],
                                     min(kChunk, row1 - t), min((int)a.dv - w.d0, DVP));
    };
    bool ok = true;
    int64_t total = 0;  // log2 decay of the rows so far (aggregate pass)
    if (n_chunks > 0 && !p.tma) {
      copy_qk(row0);
      copy_v(row0);
    }
    if (n_chunks > 0 && !p.aggregate) store_state_parts();
    for (int c = 0; c < n_chunks; ++c) {
      const int t0 = row0 + c * kChunk, n = min(kChunk, row1 - t0);
      const uint32_t parity = (uint32_t)c & 1u;
      const Decays& dec = s.dec[c & 1];
      const bool more = c + 1 < n_chunks;
      // ---- 1: raw rows -> scaled fp16 parts
      if (p.tma) {
        ok = wait(&s.full, parity) && wait(&s.v_full, parity) && ok;
      } else {
        async_copies_done();
        __syncthreads();
      }
      // (one tile at a time: more rows in flight spill, and with shared memory
      // taking nearly all of the L1 cache a spill is a trip to L2)
      TileConverter<T, DKP, kWarps> cqk;
      TileConverter<T, DVP, kWarps> cv;
      if (!p.aggregate) {
        cqk.load(sm, n);
        cqk.store(sm + C::kOffQP, s.eq);
      }
      cqk.load(sm + C::kOffK, n);
      cqk.store(sm + C::kOffKP, s.ek);
      cv.load(sm + C::kOffV, n);
      cv.store(sm + C::kOffVP, s.ev);
      mamba_scan::fence_proxy_async_smem();
      tc_fence_before();
      if (__syncthreads_or(!ok)) break;  // (1)
      if (!p.tma && more) copy_qk(t0 + kChunk);
      total += dec.total;
      // ---- 2: weighted values -> tensor memory, two parts. Each warp finds
      // the largest row factor, er_j - floor G_j, and its own rows' weights.
      int x[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int j = lane + 32 * i;
        x[i] = j < n ? -(s.ek[j] + s.ev[j]) - dec.Gi[j] : -1000000;
      }
      const int last = __reduce_max_sync(0xffffffffu, max(x[0], x[1]));
      if (lane < kTok) {
        const int j = part * kTok + lane;
        // (of the raw values: their row's exponent is not in them)
        const int e = j < n ? -s.ek[j] - dec.Gi[j] - last : -1000000;
        s.fv[warp][lane] = shift2(dec.down[j], e);
      }
      if (warp == 1) {
        s.xg[lane] = make_float2((float)x[0], dec.Gf[lane]);
        s.xg[lane + 32] = make_float2((float)x[1], dec.Gf[lane + 32]);
        if (lane == 0) {
          s.gamma = shift2(dec.up[kChunk - 1], dec.Gi[kChunk - 1]);
          s.cs = shift2(dec.up[kChunk - 1], dec.Gi[kChunk - 1] + last + 32);
        }
      }
      __syncwarp();
      if (C::kShareSV && !p.aggregate) {
        ok = wait(&s.o1, parity) && ok;
        tc_fence_after();
      }
      const T* raw = reinterpret_cast<const T*>(sm + C::kOffV) + (row < DVP ? row : 0);
      auto value_block = [&](int j0, auto partial) {
        uint32_t hi[8], lo[8];
#pragma unroll
        for (int i = 0; i < 16; i += 4) {
          const float4 f = *reinterpret_cast<const float4*>(&s.fv[warp][j0 + i]);
          float x[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int j = part * kTok + j0 + i + e;
            x[e] = to_f32(raw[j * DVP]);
            // (rows past the n-th may hold anything)
            if (decltype(partial)::value && j >= n) x[e] = 0.f;
          }
          split_half2(__fmul2_rn(make_float2(x[0], x[1]), make_float2(f.x, f.y)), hi[i / 2], lo[i / 2]);
          split_half2(__fmul2_rn(make_float2(x[2], x[3]), make_float2(f.z, f.w)), hi[i / 2 + 1],
                      lo[i / 2 + 1]);
        }
        const uint32_t col = (uint32_t)(C::kColV + (part * kTok + j0) / 2);
        tmem_st8(lane_base + col, hi);
        tmem_st8(lane_base + col + kChunk / 2, lo);
      };
#pragma unroll 1
      for (int j0 = 0; j0 < kTok; j0 += 16) {
        if (n == kChunk) value_block(j0, std::false_type());
        else value_block(j0, std::true_type());
      }
      tmem_wait_st();
      tc_fence_before();
      __syncthreads();  // (2)
      if (!p.tma && more) copy_v(t0 + kChunk);
      if (!p.aggregate) {
        // ---- 3: weighted scores -> shared memory (lanes 0..63 hold the rows)
        if (quarter < 2) {
          const float Ui = s.U[row];
          ok = wait(&s.scores, parity) && ok;
          tc_fence_after();
          uint8_t* P = sm + C::kOffP + row * 128;
#pragma unroll 1
          for (int j0 = 0; j0 < kTok; j0 += 16) {
            const int jb = part * kTok + j0;
            uint32_t hi[8], lo[8];
            if (jb > quarter * 32 + 31) {  // above the diagonal for the whole warp
#pragma unroll
              for (int i = 0; i < 8; ++i) hi[i] = lo[i] = 0;
            } else {
              float x[16];
              tmem_ld16(lane_base + (uint32_t)(C::kColAcc + jb), x);
              tmem_wait_ld();
#pragma unroll
              for (int i = 0; i < 16; i += 2) {
                const float4 xg = *reinterpret_cast<const float4*>(&s.xg[jb + i]);
                const float w0 = mamba_scan::ex2_approx((xg.x - Ui) - xg.y);
                const float w1 = mamba_scan::ex2_approx((xg.z - Ui) - xg.w);
                x[i] = jb + i <= row ? x[i] * w0 : 0.f;
                x[i + 1] = jb + i + 1 <= row ? x[i + 1] * w1 : 0.f;
              }
#pragma unroll
              for (int i = 0; i < 8; ++i)
                split_half2(make_float2(x[2 * i], x[2 * i + 1]), hi[i], lo[i]);
            }
#pragma unroll
            for (int hlf = 0; hlf < 2; ++hlf) {
              const int off = ((jb / 8 + hlf) ^ (row & 7)) << 4;
              *reinterpret_cast<uint4*>(P + off) =
                  make_uint4(hi[4 * hlf], hi[4 * hlf + 1], hi[4 * hlf + 2], hi[4 * hlf + 3]);
              *reinterpret_cast<uint4*>(P + kSlab + off) =
                  make_uint4(lo[4 * hlf], lo[4 * hlf + 1], lo[4 * hlf + 2], lo[4 * hlf + 3]);
            }
          }
          mamba_scan::fence_proxy_async_smem();
          tc_fence_before();
        }
        __syncthreads();  // (3)
      }
      // ---- 4: the new state
      const float inv_old = inv_s;
      ok = wait(&s.ds, parity) && ok;
      // (the state's parts give way to the new ones, and O1 is read below)
      if (!p.aggregate) ok = wait(&s.o1, parity) && ok;
      tc_fence_after();
      const float gamma = s.gamma, cs = s.cs;
#pragma unroll
      for (int i0 = 0; i0 < kSCols; i0 += 16) {
        float x[16];
        tmem_ld16(lane_base + (uint32_t)(C::kColD + part * kSCols + i0), x);
        tmem_wait_ld();
#pragma unroll
        for (int i = 0; i < 8; ++i)
          S[i0 / 2 + i] = __ffma2_rn(
              __fmul2_rn(make_float2(x[2 * i], x[2 * i + 1]), twice(2.3283064365386963e-10f)),
              twice(cs), __fmul2_rn(twice(gamma), S[i0 / 2 + i]));  // 2^-32
      }
      if (!p.aggregate) {
        if (more) store_state_parts();
        // ---- 5: the outputs
        ok = wait(&s.o2, parity) && ok;
        tc_fence_after();
        T* o = out + part * kTok * out_stride;
        out += kChunk * out_stride;
#pragma unroll 1
        for (int j0 = 0; j0 < kTok; j0 += 16) {
          const int jb = part * kTok + j0;
          float x[16], y[16];
          tmem_ld16(lane_base + (uint32_t)(C::kColO1 + jb), x);
          tmem_ld16(lane_base + (uint32_t)(C::kColAcc + jb), y);
          tmem_wait_ld();
#pragma unroll
          for (int i = 0; i < 16; i += 2) {
            const float4 f = *reinterpret_cast<const float4*>(&s.c12[jb + i]);  // c1, c2 of two rows
            const float2 xs = __fmul2_rn(make_float2(x[i], x[i + 1]), twice(inv_old));
            const float2 ys = __fmul2_rn(make_float2(y[i], y[i + 1]), twice(2.3283064365386963e-10f));
            const float2 r = __ffma2_rn(ys, make_float2(f.y, f.w), __fmul2_rn(xs, make_float2(f.x, f.z)));
            x[i] = r.x, x[i + 1] = r.y;
          }
          if constexpr (kHalves) {
            // (acc may be out: its loads go first)
            float* acc = p.acc + (o - static_cast<T*>(a.out));
            if (p.half == 1) {
#pragma unroll
              for (int i = 0; i < 16; ++i) y[i] = d_ok && jb + i < n ? acc[i * out_stride] : 0.f;
            }
#pragma unroll
            for (int i = 0; i < 16; ++i, o += out_stride) {
              if (!d_ok || jb + i >= n) continue;
              if (p.half == 0) acc[i * out_stride] = x[i];
              else *o = from_f32<T>(y[i] + x[i]);
            }
          } else if (d_ok) {
            if (n == kChunk) {
#pragma unroll
              for (int i = 0; i < 16; ++i, o += out_stride) *o = from_f32<T>(x[i]);
            } else {
#pragma unroll
              for (int i = 0; i < 16; ++i, o += out_stride)
                if (jb + i < n) *o = from_f32<T>(x[i]);
            }
          }
        }
      }
      tc_fence_before();
    }
    store_state<DKP>(reinterpret_cast<float(&)[kSCols]>(S), p, w, part * kSCols, row, d_ok);
    if (!p.aggregate && d_ok) {  // padded rows
      out = static_cast<T*>(a.out) + ((int64_t)w.b * a.seqlen * a.heads + w.h) * a.dv + d;
      for (int t = row1 + part; t < rows.limit; t += kSplit) out[t * out_stride] = from_f32<T>(0.f);
    }
    if (p.aggregate && threadIdx.x == 0) store_total(p, w, total);
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 0) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem),
                 "r"(C::kTmemCols));
  }
}

// ------------------------------------------------- bf16 operands as they are

// The same products for bf16 inputs that TMA can take, without the scaling:
// bf16 has fp32's exponents, so q, k and v go from TMA's swizzled tiles
// straight into the products, and what is computed (scores, state, weighted
// values) is split into bf16 parts: hi + lo for the scores and the state
// (2^-17), three parts for the weighted values (2^-25: the state is fp32).
// That costs more products (of 64 x 64 or 64 x 128 rows and columns, 8 for a
// chunk where one part each would take 4) and saves the conversion, which was
// most of the instructions.
//
// Five roles work at once on different steps of neighbouring chunks and meet
// only at mbarriers:
//   outputs group (warps 0-7): its lanes 0..63 weight the scores(c + 1) into P
//     in shared memory; all of them form outputs(c)
//   state group (warps 8-15): weighted values(c + 1), in the layout of v's
//     tile; state(c) and its parts
//   (in the aggregate pass the outputs group weights the values, two chunks
//   ahead, and the state group only adds up the states)
//   warp 16: the products O1(c) = S^T q^T and O2(c) = v^T P^T
//   warp 17: dS(c);   warp 18: scores(c);   warp 19: loads and decays
// A product of 128 x 64 x 16 occupies the tensor core for 32 clocks and its
// warp for about 70, so one warp issuing all of a chunk's 44 was the longest
// chain; three of them are not. Loops are rolled and waits short where they
// can be: the roles' code competes for the instruction caches (unrolled
// products and long waits made the whole kernel a fifth slower).
//
// Measured on one B200: 2.6 us a chunk for heads of 128 x 128 (HBM alone 1.5;
// in step, with scaled fp16 parts, 5.3), 2.3 for 64 x 64. The longest chain is
// the state group's: values, dS, state, parts; the warps issue in 55% of the
// clocks and the tensor core is busy 33%. 8x2048 rows of 40 heads 261 us
// (227 where the next call's first CTAs fill the last wave).
template <int DKP_, int DVP_>
struct DirectCfg {
  // two tiles of q, which the scores and O1 read, and three of k and v
  static constexpr int DKP = DKP_, DVP = DVP_, kStagesQ = 2, kStages = 3;
  static constexpr int kTileQ = DKP / 64 * kSlab, kTileV = DVP / 64 * kSlab;
  static constexpr int kStage = kTileQ + kTileV;  // k, v
  static constexpr int kOffKV = kStagesQ * kTileQ;
  // the weighted values' three parts, two buffers of P's two parts (with DVP =
  // 64 the products' 128 rows of A read one slab past a tile, into what follows)
  static constexpr int kOffW = kOffKV + kStages * kStage, kOffP = kOffW + 3 * kTileV;
  static constexpr int kOffSmall = kOffP + 4 * kSlab;
  // Part `pr` of the weighted values' buffer `buf`. The aggregate pass has a
  // second one, in place of q's tiles and P.
  __host__ __device__ static constexpr int values(int buf, int pr) {
    return buf == 0 ? kOffW + pr * kTileV
           : (pr + 1) * kTileV <= kOffKV ? pr * kTileV : kOffP + (pr - kOffKV / kTileV) * kTileV;
  }
  static constexpr int kColS = 0, kColAcc = DKP, kColO1 = kColAcc + 64, kColO2 = kColO1 + 64;
  static constexpr int kColD = kColO2 + 64, kTmemCols = kColD + DKP <= 256 ? 256 : 512;
  static_assert(kColD + DKP <= kTmemCols, "tensor memory");
};

// Waiters may lag a phase behind only where the barrier is a ring.
struct __align__(16) DirectSmall {
  DecayWeights dec[8];          // of chunks c - 5 .. c + 2
  uint64_t q_full[2], full[3];  // q's tile, k's and v's have landed
  uint64_t decays[8];           // a chunk's decays are there
  uint64_t scores;              // products are done: the scores;
  uint64_t o1[2], out[4], ds[4];  // O1; O1 and O2; dS (rings: the loading warp lags)
  uint64_t p_ready[2], v_ready[2];  // P, the weighted values are there (of either buffer)
  uint64_t o_read, ds_read[2];  // O1 and O2, dS have been read
  uint64_t s_ready;             // the state's parts are in tensor memory
  uint32_t tmem;
  int gave_up;                  // a wait ran out: everyone leaves
};

__device__ __forceinline__ void arrive(uint64_t* bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
}

__device__ __forceinline__ uint32_t pack_bf16(float a, float b) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// (a, b) as a pair of bf16 and what is left of them.
__device__ __forceinline__ uint32_t take_bf16(float2& x) {
  const uint32_t h = pack_bf16(x.x, x.y);
  x = __fadd2_rn(x, make_float2(-__uint_as_float(h << 16), -__uint_as_float(h & 0xffff0000u)));
  return h;
}

template <int DKP, int DVP>
__global__ void __launch_bounds__(640, 1)
    prompt_direct_kernel(const __grid_constant__ Maps maps, const __grid_constant__ Params p) {
  using C = DirectCfg<DKP, DVP>;
  using T = __nv_bfloat16;
  constexpr int kStages = C::kStages;
  constexpr int kSCols = DKP / 2, kTok = kChunk / 2;  // a thread's state columns, rows
  constexpr uint32_t kBf16 = (1u << 7) | (1u << 10);  // A and B bf16 in the instruction descriptor
  extern __shared__ uint8_t smem_raw[];
  uint8_t* sm = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  DirectSmall& s = *reinterpret_cast<DirectSmall*>(sm + C::kOffSmall);
  const mamba_linear_attention_args& a = p.a;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int quarter = warp & 3, part = (warp >> 2) & 1;

  const Work w(p);
  const int row = quarter * 32 + lane, d = w.d0 + row;
  const bool d_ok = d < (int)a.dv && row < DVP;

  if (threadIdx.x == 0) {
    for (int i = 0; i < kStages; ++i) mamba_scan::mbar_init(&s.full[i], 1);
    for (int i = 0; i < C::kStagesQ; ++i) mamba_scan::mbar_init(&s.q_full[i], 1);
    for (int i = 0; i < 8; ++i) mamba_scan::mbar_init(&s.decays[i], 32);
    mamba_scan::mbar_init(&s.scores, 1);
    for (int i = 0; i < 2; ++i) mamba_scan::mbar_init(&s.o1[i], 1);
    for (int i = 0; i < 4; ++i) {
      mamba_scan::mbar_init(&s.out[i], 1);
      mamba_scan::mbar_init(&s.ds[i], 1);
    }
    for (int i = 0; i < 2; ++i) mamba_scan::mbar_init(&s.p_ready[i], 128);
    for (int i = 0; i < 2; ++i) mamba_scan::mbar_init(&s.v_ready[i], 256);
    mamba_scan::mbar_init(&s.o_read, 256);
    for (int i = 0; i < 2; ++i) mamba_scan::mbar_init(&s.ds_read[i], 256);
    mamba_scan::mbar_init(&s.s_ready, 256);
    s.gave_up = 0;
    mamba_scan::fence_mbarrier_init();
  }
  if (warp == 0) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                     smem_u32(&s.tmem)),
                 "r"(C::kTmemCols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = __shfl_sync(0xffffffffu, s.tmem, 0);
  mamba_scan::pdl_trigger();  // (as in prompt_kernel)
  if (w.tail >= 0 || p.n_tail == 0) mamba_scan::pdl_wait();

  const Rows rows(p, w);
  const int row0 = rows.begin, row1 = rows.end, n_chunks = rows.chunks();
  const uint32_t lane_base = tmem + ((uint32_t)(quarter * 32) << 16);
  const bool emits = !p.aggregate;
  auto wait = [&](uint64_t* bar, int phase) {
    return wait_or_leave(bar, (uint32_t)phase & 1u, &s.gave_up);
  };
  auto landed = [&](int c) { return wait(&s.full[c % kStages], c / kStages); };
  auto q_landed = [&](int c) { return wait(&s.q_full[c & 1], c >> 1); };

  // weighted values: decays to the chunk's end, three parts, 16 bytes (8
  // values of a row) at a time at the places of v's own tile, by 256 threads
  auto weigh_values = [&](int c, int me, int buf) -> bool {
    const int n = min(kChunk, row1 - row0 - c * kChunk);
    const DecayWeights& dec = s.dec[c & 7];
    if (!wait(&s.decays[c & 7], c >> 3) || !landed(c)) return false;
    uint8_t* stage = sm + C::kOffKV + c % kStages * C::kStage;  // k, v
    if (n < kChunk && a.lengths) {
      // rows past the length are in the tiles: products with 0 weights must
      // not meet NaN. (A thread clears the values that it reads below.)
      constexpr int kWords = (C::kTileQ + C::kTileV) / 16;
      for (int i = me; i < kWords; i += 256)
        if (i / 8 % 64 >= n)
          reinterpret_cast<uint4*>(stage)[i] = make_uint4(0, 0, 0, 0);
    }
    uint8_t *dst0 = sm + C::values(buf, 0), *dst1 = sm + C::values(buf, 1),
            *dst2 = sm + C::values(buf, 2);
#pragma unroll 1
    for (int i = me; i < C::kTileV / 16; i += 256) {
      const uint4 v16 = *reinterpret_cast<const uint4*>(stage + C::kTileQ + i * 16);
      const float wj = dec.to_end[i / 8 % 64];
      const uint32_t in[4] = {v16.x, v16.y, v16.z, v16.w};
      uint32_t part0[4], part1[4], part2[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        float2 y = __fmul2_rn(make_float2(__uint_as_float(in[e] << 16),
                                          __uint_as_float(in[e] & 0xffff0000u)),
                              make_float2(wj, wj));
        part0[e] = take_bf16(y);
        part1[e] = take_bf16(y);
        part2[e] = pack_bf16(y.x, y.y);
      }
      *reinterpret_cast<uint4*>(dst0 + i * 16) = make_uint4(part0[0], part0[1], part0[2], part0[3]);
      *reinterpret_cast<uint4*>(dst1 + i * 16) = make_uint4(part1[0], part1[1], part1[2], part1[3]);
      *reinterpret_cast<uint4*>(dst2 + i * 16) = make_uint4(part2[0], part2[1], part2[2], part2[3]);
    }
    mamba_scan::fence_proxy_async_smem();
    arrive(&s.v_ready[c & 1]);
    return true;
  };

  // Registers: the state group's 64 columns of S need more than a third of
  // 96 x 640; 256 x (72 + 136) + 128 x 56 = 60416 of the launch's 61440.
  if (warp >= 16) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 56;");
    const uint32_t leader = elect_one(), base = smem_u32(sm);
    auto all = [&](bool ok) { return __all_sync(0xffffffffu, ok) != 0; };
    // (Rolled loops: unrolled, each product's few instructions were fetched
    // from far away once per chunk.)
    if (warp == 16 && emits) {
      for (int c = 0; c < n_chunks; ++c) {
        const uint32_t qt = base + (uint32_t)((c & 1) * C::kTileQ);
        const uint32_t vt = base + C::kOffKV + (uint32_t)(c % kStages * C::kStage) + C::kTileQ;
        if (!all(q_landed(c)) || !all(landed(c))) break;
        if (c > 0 && !all(wait(&s.o_read, c - 1))) break;
        if (!all(wait(&s.s_ready, c))) break;
        tc_fence_after();
        uint32_t acc = 0;
#pragma unroll 1
        for (int pr = 1; pr >= 0; --pr) {  // lo, hi
          uint32_t ac = tmem + C::kColS + pr * (DKP / 2), bd = desc_k(qt);
#pragma unroll 1
          for (int kk = 0; kk < DKP / 16; ++kk) {
            mma_ts(leader, tmem + C::kColO1, ac, bd, idesc(64, false, false) | kBf16, acc);
            ac += 8;
            bd += (kk & 3) == 3 ? (kSlab - 96) >> 4 : 2;  // 16 columns on
            acc = 1;
          }
        }
        mma_commit(leader, &s.o1[c & 1]);
        if (!all(wait(&s.p_ready[c & 1], c >> 1))) break;
        // (v's rows past the length have to be cleared by then)
        if (a.lengths && c + 1 == n_chunks && !all(wait(&s.v_ready[c & 1], c >> 1))) break;
        tc_fence_after();
        acc = 0;
#pragma unroll 1
        for (int pr = 1; pr >= 0; --pr) {  // lo, hi
          uint32_t ad = desc_mn(vt), bd = desc_k(base + C::kOffP + (2 * (c & 1) + pr) * kSlab);
#pragma unroll 1
          for (int kk = 0; kk < kChunk / 16; ++kk) {
            mma_ss(leader, tmem + C::kColO2, ad, bd, idesc(64, true, false) | kBf16, acc);
            ad += 128;
            bd += 2;
            acc = 1;
          }
        }
        mma_commit(leader, &s.out[c & 3]);
      }
    } else if (warp == 17) {
      for (int c = 0; c < n_chunks; ++c) {
        const uint32_t kt = base + C::kOffKV + (uint32_t)(c % kStages * C::kStage);
        if (!all(landed(c))) break;
        // (the aggregate pass has two buffers of dS and of the values)
        const int back = emits ? 1 : 2, buf = emits ? 0 : c & 1;
        if (c >= back && !all(wait(&s.ds_read[(c - back) & 1], (c - back) >> 1))) break;
        if (!all(wait(&s.v_ready[c & 1], c >> 1))) break;
        tc_fence_after();
        uint32_t acc = 0;
#pragma unroll 1
        for (int pr = 2; pr >= 0; --pr) {  // smallest part first
          uint32_t ad = desc_mn(base + C::values(buf, pr)), bd = desc_mn(kt);
#pragma unroll 1
          for (int kk = 0; kk < kChunk / 16; ++kk) {
            mma_ss(leader, tmem + (buf ? C::kColAcc : C::kColD), ad, bd,
                   idesc(DKP, true, true) | kBf16, acc);
            ad += 128;
            bd += 128;
            acc = 1;
          }
        }
        mma_commit(leader, &s.ds[c & 3]);
      }
    } else if (warp == 18 && emits) {
      for (int c = 0; c < n_chunks; ++c) {
        const uint32_t qt = base + (uint32_t)((c & 1) * C::kTileQ);
        const uint32_t kt = base + C::kOffKV + (uint32_t)(c % kStages * C::kStage);
        if (!all(q_landed(c)) || !all(landed(c))) break;
        // the last scores have been read
        if (c > 0 && !all(wait(&s.p_ready[(c - 1) & 1], (c - 1) >> 1))) break;
        tc_fence_after();
        uint32_t ad = desc_k(qt), bd = desc_k(kt), acc = 0;
#pragma unroll 1
        for (int kk = 0; kk < DKP / 16; ++kk) {
          mma_ss(leader, tmem + C::kColAcc, ad, bd, idesc(64, false, false) | kBf16, acc);
          const uint32_t step = (kk & 3) == 3 ? (kSlab - 96) >> 4 : 2;
          ad += step;
          bd += step;
          acc = 1;
        }
        mma_commit(leader, &s.scores);
      }
    } else if (warp == 19) {
      const float* decay = a.log_decay + w.b * a.decay_stride[0] + w.h * a.decay_stride[2];
      auto load_q = [&](int c) {
        uint64_t* bar = &s.q_full[c & 1];
        mamba_scan::mbar_arrive_expect_tx(bar, C::kTileQ);
#pragma unroll
        for (int i = 0; i < DKP / 64; ++i)
          tma_load_4d(sm + (c & 1) * C::kTileQ + i * kSlab, &maps.q, bar, i * 64, w.g,
                      row0 + c * kChunk, w.b);
      };
      auto load_kv = [&](int c) {
        uint8_t* dst = sm + C::kOffKV + c % kStages * C::kStage;
        uint64_t* bar = &s.full[c % kStages];
        const int t = row0 + c * kChunk;
        mamba_scan::mbar_arrive_expect_tx(bar, C::kStage);
#pragma unroll
        for (int i = 0; i < DKP / 64; ++i)
          tma_load_4d(dst + i * kSlab, &maps.k, bar, i * 64, w.g, t, w.b);
#pragma unroll
        for (int i = 0; i < DVP / 64; ++i)
          tma_load_4d(dst + C::kTileQ + i * kSlab, &maps.v, bar, w.d0 + i * 64, w.h, t, w.b);
      };
      if (lane == 0) {
        if (emits)
          for (int c = 0; c < min(2, n_chunks); ++c) load_q(c);
        for (int c = 0; c < min(kStages, n_chunks); ++c) load_kv(c);
      }
      __syncwarp();
      // Step c: the decays of chunk c + 2, into a buffer that chunk c - 6 has
      // left (whoever reads its decays is done with them before dS of c - 4);
      // then, as chunk c's products are done, the loads of q for chunk c + 2
      // and of k and v for c + 3. No wait here may come after its barrier's
      // next phase: O1(c + 2) and P(c + 2) need q's load of step c, after the
      // waits for O1(c) and P(c); dS(c + 2) and the outputs of c + 2 need
      // nothing after the waits for those of c, so they have rings of four
      // (dS(c + 4) and the outputs of c + 4 need the decays of step c + 2).
      int q_loads = emits ? min(2, n_chunks) : 0, kv_loads = min(kStages, n_chunks);
      bool ok = true;
      auto fetch_decays = [&](int c) {
        const int t = row0 + c * kChunk;
        return c < n_chunks ? load_decays(decay, a.decay_stride[1], t, min(kChunk, row1 - t))
                            : make_float2(0.f, 0.f);
      };
      float2 g = fetch_decays(0);  // (fetched a step before they are summed)
      for (int c = -2; c < n_chunks; ++c) {
        if (c + 2 < n_chunks) {
          const float2 next = fetch_decays(c + 3);
          scan_decays(s.dec[(c + 2) & 7], g);
          arrive(&s.decays[(c + 2) & 7]);
          g = next;
        }
        if (c < 0 || c + 1 == n_chunks) continue;
        if (emits && c + 2 < n_chunks) {
          // q's readers are O1 and the scores, which P follows
          if (!(ok = all(wait(&s.o1[c & 1], c >> 1)))) break;
          if (!(ok = all(wait(&s.p_ready[c & 1], c >> 1)))) break;
          if (lane == 0) load_q(c + 2);
          __syncwarp();
          ++q_loads;
        }
        if (!(ok = all(wait(&s.ds[c & 3], c >> 2)))) break;
        if (emits && !(ok = all(wait(&s.out[c & 3], c >> 2)))) break;
        if (c + kStages < n_chunks) {
          if (lane == 0) load_kv(c + kStages);
          __syncwarp();
          ++kv_loads;
        }
      }
      // if all left early: loads in flight have to land before the memory goes
      if (!ok && lane == 0) {
        for (int c = max(0, q_loads - 2); c < q_loads; ++c)
          mamba_scan::mbar_wait(&s.q_full[c & 1], (uint32_t)(c >> 1) & 1u, &g_error);
        for (int c = max(0, kv_loads - kStages); c < kv_loads; ++c)
          mamba_scan::mbar_wait(&s.full[c % kStages], (uint32_t)(c / kStages) & 1u, &g_error);
      }
    }
    __syncwarp();
  } else if (warp >= 8) {
    // ---------------------------------------------------------- state group
    asm volatile("setmaxnreg.inc.sync.aligned.u32 136;");
    float2 S[kSCols / 2];
    load_state<DKP>(reinterpret_cast<float(&)[kSCols]>(S), p, w, part * kSCols, row, d_ok);
    auto store_state_parts = [&]() {
#pragma unroll
      for (int i0 = 0; i0 < kSCols / 2; i0 += 8) {
        uint32_t hi[8], lo[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          float2 x = S[i0 + i];
          hi[i] = take_bf16(x);
          lo[i] = pack_bf16(x.x, x.y);
        }
        const uint32_t col = (uint32_t)(C::kColS + part * kSCols / 2 + i0);
        tmem_st8(lane_base + col, hi);
        tmem_st8(lane_base + col + DKP / 2, lo);
      }
      tmem_wait_st();
      tc_fence_before();
      arrive(&s.s_ready);
    };
    int64_t total = 0;  // log2 decay of the rows so far
    const int me = (int)threadIdx.x - 256;
    bool ok = n_chunks > 0 && (!emits || weigh_values(0, me, 0));
    if (ok && emits) store_state_parts();
    for (int c = 0; ok && c < n_chunks; ++c) {
      if (!wait(&s.decays[c & 7], c >> 3)) break;
      const float gamma = s.dec[c & 7].from_start[kChunk - 1];
      total += s.dec[c & 7].total;
      if (!wait(&s.ds[c & 3], c >> 2)) break;
      // the values' buffer is free: the next chunk's go first, so that its dS
      // is formed while this one's is worked into the state
      if (emits && c + 1 < n_chunks && !weigh_values(c + 1, me, 0)) break;
      const uint32_t dS = lane_base + (uint32_t)((!emits && (c & 1) ? C::kColAcc : C::kColD) + part * kSCols);
      tc_fence_after();
      const float2 gamma2 = make_float2(gamma, gamma);
#pragma unroll
      for (int i0 = 0; i0 < kSCols; i0 += 16) {
        float x[16];
        tmem_ld16(dS + (uint32_t)i0, x);
        tmem_wait_ld();
#pragma unroll
        for (int i = 0; i < 8; ++i)
          S[i0 / 2 + i] = __ffma2_rn(gamma2, S[i0 / 2 + i], make_float2(x[2 * i], x[2 * i + 1]));
      }
      tc_fence_before();
      arrive(&s.ds_read[c & 1]);
      if (c + 1 < n_chunks && emits) {
        if (!wait(&s.o1[c & 1], c >> 1)) break;  // the parts before these have been used
        tc_fence_after();
        store_state_parts();
      }
    }
    store_state<DKP>(reinterpret_cast<float(&)[kSCols]>(S), p, w, part * kSCols, row, d_ok);
    if (!emits && threadIdx.x == 256) store_total(p, w, total);
  } else {
    // -------------------------------------------------------- outputs group
    asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
    const int64_t out_stride = a.heads * a.dv;
    T* out = static_cast<T*>(a.out) + ((int64_t)w.b * a.seqlen * a.heads + w.h) * a.dv + d;

    // weighted scores: lanes 0..63 hold the rows
    auto weigh_scores = [&](int c) -> bool {
      const DecayWeights& dec = s.dec[c & 7];
      if (!wait(&s.decays[c & 7], c >> 3)) return false;
      const float2 Gr = dec.gg[row];
      if (!wait(&s.scores, c)) return false;
      tc_fence_after();
      uint8_t* P = sm + C::kOffP + 2 * (c & 1) * kSlab + row * 128;
#pragma unroll 1
      for (int j0 = 0; j0 < kTok; j0 += 16) {
        const int jb = part * kTok + j0;
        uint32_t hi[8], lo[8];
        if (jb > quarter * 32 + 31) {  // above the diagonal for the whole warp
#pragma unroll
          for (int i = 0; i < 8; ++i) hi[i] = lo[i] = 0;
        } else {
          float x[16];
          tmem_ld16(lane_base + (uint32_t)(C::kColAcc + jb), x);
          tmem_wait_ld();
#pragma unroll
          for (int i = 0; i < 16; i += 2) {
            const float4 gg = *reinterpret_cast<const float4*>(&dec.gg[jb + i]);
            x[i] *= mamba_scan::ex2_approx((Gr.x - gg.x) + (Gr.y - gg.y));
            x[i + 1] *= mamba_scan::ex2_approx((Gr.x - gg.z) + (Gr.y - gg.w));
          }
          if (jb + 15 > quarter * 32) {  // the diagonal's blocks
#pragma unroll
            for (int i = 0; i < 16; ++i) x[i] = jb + i <= row ? x[i] : 0.f;
          }
          const float2 sc = make_float2(a.scale, a.scale);
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            float2 y = __fmul2_rn(make_float2(x[2 * i], x[2 * i + 1]), sc);
            hi[i] = take_bf16(y);
            lo[i] = pack_bf16(y.x, y.y);
          }
        }
#pragma unroll
        for (int hlf = 0; hlf < 2; ++hlf) {
          const int off = ((jb / 8 + hlf) ^ (row & 7)) << 4;
          *reinterpret_cast<uint4*>(P + off) =
              make_uint4(hi[4 * hlf], hi[4 * hlf + 1], hi[4 * hlf + 2], hi[4 * hlf + 3]);
          *reinterpret_cast<uint4*>(P + kSlab + off) =
              make_uint4(lo[4 * hlf], lo[4 * hlf + 1], lo[4 * hlf + 2], lo[4 * hlf + 3]);
        }
      }
      mamba_scan::fence_proxy_async_smem();
      tc_fence_before();
      arrive(&s.p_ready[c & 1]);
      return true;
    };

    auto outputs = [&](int c) -> bool {
      const int t0 = row0 + c * kChunk, n = min(kChunk, row1 - t0);
      const DecayWeights& dec = s.dec[c & 7];
      if (!wait(&s.out[c & 3], c >> 2)) return false;
      tc_fence_after();
      T* o = out + (t0 + part * kTok) * out_stride;
#pragma unroll 1
      for (int j0 = 0; j0 < kTok; j0 += 16) {
        const int jb = part * kTok + j0;
        float x[16], y[16];
        tmem_ld16(lane_base + (uint32_t)(C::kColO1 + jb), x);
        tmem_ld16(lane_base + (uint32_t)(C::kColO2 + jb), y);
        tmem_wait_ld();
#pragma unroll
        for (int i = 0; i < 16; i += 4) {
          const float4 f = *reinterpret_cast<const float4*>(&dec.from_start[jb + i]);
          x[i] = fmaf(x[i], a.scale * f.x, y[i]);
          x[i + 1] = fmaf(x[i + 1], a.scale * f.y, y[i + 1]);
          x[i + 2] = fmaf(x[i + 2], a.scale * f.z, y[i + 2]);
          x[i + 3] = fmaf(x[i + 3], a.scale * f.w, y[i + 3]);
        }
        if (j0 + 16 == kTok) {  // (the last use of this chunk's decays, too)
          tc_fence_before();
          arrive(&s.o_read);
        }
        if (d_ok) {
          if (n == kChunk) {
#pragma unroll
            for (int i = 0; i < 16; ++i, o += out_stride) *o = __float2bfloat16_rn(x[i]);
          } else {
#pragma unroll
            for (int i = 0; i < 16; ++i, o += out_stride)
              if (jb + i < n) *o = __float2bfloat16_rn(x[i]);
          }
        }
      }
      return true;
    };

    if (!emits) {
      for (int c = 0; c < n_chunks; ++c) {
        // the values' buffer was used two chunks ago
        if (c >= 2 && !wait(&s.ds[(c - 2) & 3], (c - 2) >> 2)) break;
        if (!weigh_values(c, (int)threadIdx.x, c & 1)) break;
      }
    } else if (quarter >= 2) {
      for (int c = 0; c < n_chunks; ++c)
        if (!outputs(c)) break;
    } else if (n_chunks > 0 && weigh_scores(0)) {
      // the next chunk's scores while this one's second product runs
      for (int c = 0; c < n_chunks; ++c) {
        if (c + 1 < n_chunks && !weigh_scores(c + 1)) break;
        if (!outputs(c)) break;
      }
    }
    if (emits && d_ok)  // padded rows
      for (int t = row1 + part; t < rows.limit; t += 2) out[t * out_stride] = __float2bfloat16_rn(0.f);
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 0) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem),
                 "r"(C::kTmemCols));
  }
}

// Joins the segments of the tail units: the state entering segment s + 1
// replaces the end state (from zero) of segment s. One thread per element of
// a unit's state; the segments' values are loaded ahead of the chain.
__global__ void __launch_bounds__(256) carry_kernel(const __grid_constant__ Params p, int dkp) {
  mamba_scan::pdl_trigger();
  mamba_scan::pdl_wait();
  const mamba_linear_attention_args& a = p.a;
  const int per_unit = dkp * kLanes / 256;
  const int tail = (int)blockIdx.x / per_unit;
  const int e = ((int)blockIdx.x % per_unit) * 256 + (int)threadIdx.x;
  const int col = e / kLanes, row = e % kLanes, n = p.n_seg - 1;
  const int unit = p.n_full + tail, tile = unit % p.tiles, bh = unit / p.tiles;
  const int d = tile * kLanes + row;
  float x = 0.f;
  if (a.h0 && col < a.dk && d < a.dv)
    x = a.h0[((int64_t)bh * p.state_rows + col) * a.dv + d];
  float* ws = p.ws + (int64_t)tail * n * dkp * kLanes + e;
  const int64_t step = (int64_t)dkp * kLanes;
  const float* f = p.ws_decay + tail * n;
  for (int s0 = 0; s0 < n; s0 += 8) {
    float v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = s0 + i < n ? ws[(s0 + i) * step] : 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (s0 + i < n) {
        x = fmaf(f[s0 + i], x, v[i]);
        ws[(s0 + i) * step] = x;
      }
  }
}

// -------------------------------------------------------------------- host

namespace {

struct Plan {
  int64_t n_full = 0, n_tail = 0;
  int n_seg = 1, seg_len = 0;
};

int padded(int64_t d) { return d <= 64 ? 64 : 128; }

// Two CTAs on an SM, when its tensor and shared memory allow it.
template <typename T, int DKP, int DVP> constexpr bool two_ctas() {
  return Cfg<T, DKP, DVP>::kTmemCols == 256 && Cfg<T, DKP, DVP>::kBytes <= 113 * 1024;
}
bool pairs_on_an_sm(int64_t dk, int64_t dv, int32_t dtype) {
  if (dtype == MAMBA_DTYPE_BF16 || padded(dk) == 128) return false;  // (bf16: the direct kernel)
  const bool wide = padded(std::min<int64_t>(dv, kLanes)) == 128;
  if (dtype == MAMBA_DTYPE_F32)
    return wide ? two_ctas<float, 64, 128>() : two_ctas<float, 64, 64>();
  return wide ? two_ctas<__half, 64, 128>() : two_ctas<__half, 64, 64>();
}

// Full waves of units run in one piece; a last partial wave is split into
// segments of whole chunks when that is shorter. Costs in chunks of a CTA that
// has its SM to itself: two CTAs on an SM take 1.55 for one chunk each
// (measured 6.8 against 4.4 us), a CTA's start and end 1.5, the aggregate pass
// half of the emit pass, the split's two more launches and join 2 (4 to 5 of the
// direct kernel's, which are shorter). Against one that counted the two CTAs as
// whole slots and charged 6: 80 heads x 4096 of 128 x 128 bf16 421 -> 179 us,
// fp32 565 -> 411; 24 x 1024 of 64 x 64 bf16 35 -> 25, 5 ragged prompts of 777
// x 20 heads fp16 73 -> 54 (60 since scores and state have two parts there). In
// some cells the other choice is shorter by 4 to 8%: 1x256 rows of 16 heads of
// 64 x 64 fp32 takes 26.8 us against 24.7, 1x768 of 60 heads 78.8 against 75.9.
Plan make_plan(int64_t units, int64_t seqlen, int64_t sms, bool pairs, double fixed) {
  Plan pl;
  pl.n_full = units;
  const int64_t chunks = (seqlen + kChunk - 1) / kChunk, slots = pairs ? 2 * sms : sms;
  const int64_t tail = units % slots;
  if (tail == 0 || chunks < 4) return pl;
  auto waves = [&](int64_t ctas) {
    const int64_t full = ctas / slots, rest = ctas % slots;
    if (!pairs) return (double)(full + (rest > 0));
    return 1.55 * (double)full + (rest == 0 ? 0.0 : rest <= sms ? 1.0 : 1.55);
  };
  double best = ((double)chunks + 1.5) * waves(tail) * 0.95;  // (a split has to be worth it)
  for (int64_t want = 2; want <= std::min<int64_t>(chunks, 256); ++want) {
    const int64_t per = (chunks + want - 1) / want, n = (chunks + per - 1) / per;
    if (n < 2) continue;
    const double cost =
        ((double)per + 1.5) * (waves(tail * n) + 0.5 * waves(tail * (n - 1))) + fixed;
    if (cost < best) {
      best = cost;
      pl.n_full = units - tail;
      pl.n_tail = tail;
      pl.n_seg = (int)n;
      pl.seg_len = (int)per * kChunk;
    }
  }
  return pl;
}

Plan plan_for(int64_t batch, int64_t seqlen, int64_t heads, int64_t dk, int64_t dv,
              int32_t dtype) {
  const int64_t tiles = (dv + kLanes - 1) / kLanes;
  const double fixed = dtype != MAMBA_DTYPE_BF16 || dk > 128 ? 2.0 : dk > 64 ? 5.0 : 4.0;
  return make_plan(batch * heads * tiles, seqlen, sm_count(), pairs_on_an_sm(dk, dv, dtype), fixed);
}

size_t plan_bytes(const Plan& pl, int dkp) {
  if (pl.n_tail == 0) return 0;
  const size_t segs = (size_t)pl.n_tail * (size_t)(pl.n_seg - 1);
  return segs * dkp * kLanes * sizeof(float) + (segs * sizeof(float) + 15) / 16 * 16;
}

PFN_cuTensorMapEncodeTiled_v12000 encode_fn() {
  static PFN_cuTensorMapEncodeTiled_v12000 fn = nullptr;
  static std::once_flag once;
  std::call_once(once, [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) ==
            cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(p);
  });
  return fn;
}

// [batch][rows][heads][width] with strides, boxes of 64 rows x box columns.
// False when TMA cannot take it (alignment, strides).
bool encode(CUtensorMap* m, const void* ptr, int32_t dtype, int64_t width, int64_t heads,
            int64_t rows, int64_t batch, const int64_t* stride, int box, bool swizzle) {
  auto enc = encode_fn();
  if (enc == nullptr || !mamba_lm::aligned16(ptr)) return false;
  const int64_t size = dtype == MAMBA_DTYPE_F32 ? 4 : 2;
  const int64_t n[3] = {heads, rows, batch}, st[3] = {stride[2], stride[1], stride[0]};
  const cuuint64_t dims[4] = {(cuuint64_t)width, (cuuint64_t)heads, (cuuint64_t)rows,
                              (cuuint64_t)batch};
  cuuint64_t bytes[3];
  for (int i = 0; i < 3; ++i) {
    // the stride of a dimension of one element is never used: any valid one
    const int64_t by = n[i] == 1 ? 16 : st[i] * size;
    if (by % 16 != 0 || by <= 0 || by >= (int64_t)1 << 40) return false;
    bytes[i] = (cuuint64_t)by;
  }
  const cuuint32_t bx[4] = {(cuuint32_t)box, 1, kChunk, 1}, es[4] = {1, 1, 1, 1};
  const CUtensorMapDataType t = dtype == MAMBA_DTYPE_F32   ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                                : dtype == MAMBA_DTYPE_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16
                                                           : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
  return enc(m, t, 4, const_cast<void*>(ptr), dims, bytes, bx, es, CU_TENSOR_MAP_INTERLEAVE_NONE,
             swizzle ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_NONE,
             CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
             CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// setmaxnreg.inc waits for registers that the block was launched with: refuse
// to launch a build of a kernel that has fewer than its roles add up to.
cudaError_t registers_suffice(const void* kernel, int threads, int needed) {
  cudaFuncAttributes attr;
  const cudaError_t e = cudaFuncGetAttributes(&attr, kernel);
  if (e != cudaSuccess) return e;
  return attr.numRegs * threads >= needed ? cudaSuccess : cudaErrorInvalidDeviceFunction;
}

// One build of a kernel and its launch shape.
struct Variant {
  void (*kernel)(Maps, Params);
  int threads;
  size_t smem;
  int registers;  // that its roles add up to (0: they keep what they are given)
};

cudaError_t prepare(const Variant& v) {
  if (v.registers > 0) {
    const cudaError_t e =
        registers_suffice(reinterpret_cast<const void*>(v.kernel), v.threads, v.registers);
    if (e != cudaSuccess) return e;
  }
  return cudaFuncSetAttribute(v.kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)v.smem);
}

// The passes of a plan: `few` for grids of at most one CTA per SM, else `many`.
cudaError_t launch_passes(const Variant& few, const Variant& many, Params p, const Maps& maps,
                          int dkp, cudaStream_t st) {
  const int64_t sms = sm_count();
  cudaError_t e;
  if (p.n_tail > 0) {
    const int64_t ctas = (int64_t)p.n_tail * (p.n_seg - 1);
    const Variant& v = ctas <= sms ? few : many;
    if ((e = prepare(v)) != cudaSuccess) return e;
    // The aggregate pass is an ordinary launch: it begins after all earlier
    // work, which the emit pass's whole units rely on.
    p.aggregate = 1;
    v.kernel<<<(unsigned)ctas, v.threads, v.smem, st>>>(maps, p);
    e = cudaGetLastError();
    if (e != cudaSuccess) return e;
    e = mamba_scan::launch_pdl(carry_kernel, dim3((unsigned)(p.n_tail * (dkp * kLanes / 256))),
                               dim3(256), 0, st, p, dkp);
    if (e != cudaSuccess) return e;
    p.aggregate = 0;
  }
  const int64_t ctas = p.n_full + (int64_t)p.n_tail * p.n_seg;
  const Variant& v = ctas <= sms ? few : many;
  if ((e = prepare(v)) != cudaSuccess) return e;
  return mamba_scan::launch_pdl(v.kernel, dim3((unsigned)ctas), dim3((unsigned)v.threads), v.smem,
                                st, maps, p);
}

template <typename T, int DKP, int DVP>
cudaError_t launch(const Params& p, const Maps& maps, cudaStream_t st) {
  using C = Cfg<T, DKP, DVP>;
  // 16 compute warps shorten a chunk for a CTA that has its SM to itself (64 x
  // 128 fp16: 4.4 us against 4.9 with 8); two CTAs of 8 on an SM take 6.8 us
  // for a chunk each. No more CTAs on an SM than its tensor memory serves.
  constexpr bool kTwo = two_ctas<T, DKP, DVP>();
  constexpr size_t alone = std::max<size_t>(C::kBytes, 116 * 1024);
  static_assert(alone <= 227 * 1024, "shared memory");
  const Variant few{prompt_kernel<T, DKP, DVP, 16>, 32 * (16 + issue_warps(16)), alone,
                    512 * 104 + 128 * 64};
  if constexpr (kTwo) {
    const Variant many{prompt_kernel<T, DKP, DVP, 8>, 32 * (8 + issue_warps(8)),
                       std::max<size_t>(C::kBytes, 78 * 1024), 0};
    return launch_passes(few, many, p, maps, DKP, st);
  } else {
    return launch_passes(few, few, p, maps, DKP, st);
  }
}

template <int DKP, int DVP>
cudaError_t launch_direct(const Params& p, const Maps& maps, cudaStream_t st) {
  using C = DirectCfg<DKP, DVP>;
  constexpr size_t smem = std::max<size_t>(C::kOffSmall + sizeof(DirectSmall) + 1024, 116 * 1024);
  static_assert(smem <= 227 * 1024, "shared memory");
  const Variant v{prompt_direct_kernel<DKP, DVP>, 640, smem, 256 * (72 + 136) + 128 * 56};
  return launch_passes(v, v, p, maps, DKP, st);
}

template <typename T>
cudaError_t launch_halves(const Params& p, const Maps& maps, cudaStream_t st) {
  constexpr size_t smem = std::max<size_t>(Cfg<T, 128, 128>::kBytes, 116 * 1024);
  static_assert(smem <= 227 * 1024, "shared memory");
  const Variant v{prompt_kernel<T, 128, 128, 16, true>, 32 * (16 + issue_warps(16)), smem,
                  512 * 104 + 128 * 64};
  return launch_passes(v, v, p, maps, 128, st);
}

template <typename T>
cudaError_t launch_typed(const Params& p, const Maps& maps, int dkp, int dvp, cudaStream_t st) {
  if (p.state_rows > 128) return launch_halves<T>(p, maps, st);
  if (dkp == 128) return launch<T, 128, 128>(p, maps, st);
  if (dvp == 128) return launch<T, 64, 128>(p, maps, st);
  return launch<T, 64, 64>(p, maps, st);
}

}  // namespace

bool mma_takes(int64_t seqlen, int64_t dk, int64_t dv) {
  (void)dv;
  return seqlen > (dk <= 128 ? 16 : 32);
}

bool mma_needs_workspace(int64_t dk, int32_t dtype) { return dk > 128 && dtype != MAMBA_DTYPE_F32; }

size_t mma_workspace_size(int64_t batch, int64_t seqlen, int64_t heads, int64_t dk, int64_t dv,
                          int32_t dtype) {
  const size_t plan = plan_bytes(plan_for(batch, seqlen, heads, dk, dv, dtype), padded(dk));
  if (!mma_needs_workspace(dk, dtype)) return plan;
  const unsigned __int128 acc =
      (unsigned __int128)(batch * heads) * (unsigned __int128)(seqlen * dv) * sizeof(float);
  const size_t most = (size_t)1 << 62;  // (no GPU has as much)
  return plan + (acc > most ? most : (size_t)acc);
}

cudaError_t launch_mma(const mamba_linear_attention_args& a, void* workspace, cudaStream_t st) {
  const int dkp = padded(a.dk);
  // with dk > 64 the kernel's value tile is 128 wide whatever dv is
  const int dvp = dkp == 128 ? 128 : padded(std::min<int64_t>(a.dv, kLanes));
  const bool direct = a.dtype == MAMBA_DTYPE_BF16 && a.dk <= 128;
  Params p;
  std::memset(&p, 0, sizeof p);
  p.a = a;
  p.tiles = (int)((a.dv + kLanes - 1) / kLanes);
  p.state_rows = a.dk;
  p.acc = static_cast<float*>(a.out);  // (fp32)
  Plan pl;
  if (workspace) {
    pl = plan_for(a.batch, a.seqlen, a.heads, a.dk, a.dv, a.dtype);
    const size_t segs = (size_t)pl.n_tail * (size_t)(pl.n_seg - 1);
    p.ws = static_cast<float*>(workspace);
    p.ws_decay = p.ws + segs * dkp * kLanes;
    if (mma_needs_workspace(a.dk, a.dtype))
      p.acc = reinterpret_cast<float*>(static_cast<char*>(workspace) + plan_bytes(pl, dkp));
  } else {
    pl.n_full = a.batch * a.heads * p.tiles;
  }
  p.n_full = (int)pl.n_full;
  p.n_tail = (int)pl.n_tail;
  p.n_seg = pl.n_seg;
  p.seg_len = pl.seg_len;
  Maps maps;
  std::memset(&maps, 0, sizeof maps);
  auto encode_all = [&](int box_k, int box_v, bool swizzle) {
    return encode(&maps.q, p.a.q, a.dtype, p.a.dk, a.groups, a.seqlen, a.batch, a.q_stride, box_k, swizzle) &&
           encode(&maps.k, p.a.k, a.dtype, p.a.dk, a.groups, a.seqlen, a.batch, a.k_stride, box_k, swizzle) &&
           encode(&maps.v, a.v, a.dtype, a.dv, a.heads, a.seqlen, a.batch, a.v_stride, box_v, swizzle);
  };
  if (direct && encode_all(64, 64, true)) {
    if (dkp == 128) return launch_direct<128, 128>(p, maps, st);
    if (dvp == 128) return launch_direct<64, 128>(p, maps, st);
    return launch_direct<64, 64>(p, maps, st);
  }
  const size_t size = a.dtype == MAMBA_DTYPE_F32 ? 4 : 2;
  for (p.half = 0; p.half * 128 < a.dk; ++p.half) {
    const int64_t col = 128 * p.half;
    p.a.q = static_cast<const char*>(a.q) + col * size;
    p.a.k = static_cast<const char*>(a.k) + col * size;
    p.a.dk = std::min<int64_t>(a.dk - col, 128);
    if (a.h0) p.a.h0 = a.h0 + col * a.dv;
    if (a.h_last) p.a.h_last = a.h_last + col * a.dv;
    p.tma = encode_all(dkp, dvp, false);
    const cudaError_t e =
        a.dtype == MAMBA_DTYPE_F32   ? launch_typed<float>(p, maps, dkp, dvp, st)
        : a.dtype == MAMBA_DTYPE_F16 ? launch_typed<__half>(p, maps, dkp, dvp, st)
                                     : launch_typed<__nv_bfloat16>(p, maps, dkp, dvp, st);
    if (e != cudaSuccess) return e;
  }
  return cudaSuccess;
}

int read_and_clear_error() {
  int v = 0;
  if (cudaMemcpyFromSymbol(&v, g_error, sizeof(int)) != cudaSuccess) return -1;
  if (v != 0) {
    const int zero = 0;
    cudaMemcpyToSymbol(g_error, &zero, sizeof(int));
  }
  return v;
}

}  // namespace mamba_la
