// The gated delta rule over prompts on the tensor cores, in chunks of 64 rows
// (include/mamba_lm_ops.h states the operator).
//
// Mathematics. With G_t the running sum of the chunk's log decays (base 2),
// S the state before the chunk and u_t = beta_t (v_t - 2^(g_t) k_t S_{t-1})
// the updates, S_t = 2^G_t S + sum_{s <= t} 2^(G_t - G_s) k_s u_s^T. So
//   (I + A) U = diag(beta) R,   R = V - diag(2^G) K S,
//   A_ts = beta_t 2^(G_t - G_s) k_t k_s  (s < t),
//   out = scale diag(2^G) Q S + P U,   P_ts = scale 2^(G_t - G_s) q_t k_s,
//   S' = 2^G_C S + K^T diag(2^(G_C - G)) U.
// prepare_kernel forms T = (I + A)^-1 diag(beta), P and the rows' factors of
// every chunk at once; chain_kernel carries the state through the chunks: three
// products in a row, K S, T R, then K^T U (and, beside the chain, Q S, P U).
// float32 tensors, and 16-bit ones that TMA cannot take, go here; the others'
// chain is gated_delta_tiles.cu.
//
// The chain in registers. Everything is held transposed, dv along the rows of
// a product: a warp owns 16 columns of the state, S^T (16 x dk) in its
// accumulator registers. An accumulator tile is, pair by pair, also the left
// operand of the next product, so S^T K^T -> R^T -> U^T = R^T T^T -> S^T +=
// U^T K never leaves the warp: no barriers, no shared memory but the right
// operands K, Q, T, P, which all warps of a head read. That is why these are
// warp-level products (mma.sync): float32's third product and two-part k and q
// make no longer chain here, while through tensor memory each step is a trip of its
// own (commit, wait, load, convert, store, fence). For 16-bit tensors, whose K, Q
// and V come by TMA as they are, those trips take less than the warps' products
// (1 x 2048 tokens of 16 heads of 128 x 128: 121 us there, 137 here; 8 x 2048 of 40
// of 64 x 64: 389 and 442, of 128 x 16: 489 and 676; 130 tokens of 16 such
// heads: 33 and 29).
//
// Numbers. All products are fp16 x fp16 with fp32 sums, of operands scaled by
// powers of two (exact) and split where fp16's 11 bits are too few: the state,
// R, U, T and P are hi + lo (22 bits, the lo lo product dropped, 3 * 2^-22),
// as are q and k of float32 tensors; 16-bit q and k are exact in one part.
// Every row of q and k, every chunk's T and P and every column of the state, R
// and U has its own power of two (largest element to 2^14..2^15); the parts'
// smallest step is 2^-24, 2^-38 of that. The inverse is formed in tf32 hi + lo
// from 16 x 16 blocks inverted in fp32. Decays are summed in 64-bit fixed point
// and enter as differences of sums, so that -inf (held at -2^14) leaves nothing
// behind.
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stddef.h>
#include <stdint.h>

#include <algorithm>
#include <type_traits>

#include "gated_delta.cuh"
#include "lm_device.cuh"
#include "scan_device.cuh"
#include "scan_kernels.h"

namespace mamba_gd {

using mamba_lm::from_f32;
using mamba_lm::to_f32;
using mamba_scan::smem_u32;

__device__ int g_error = 0;

// ------------------------------------------------------------ PTX wrappers

__device__ __forceinline__ void mma_f16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0,
                                        uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, "
      "{%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// The same for products of q and k as they are.
template <typename T>
__device__ __forceinline__ void mma_16bit(float (&d)[4], const uint32_t (&a)[4], uint32_t b0,
                                          uint32_t b1) {
  if constexpr (std::is_same<T, __nv_bfloat16>::value)
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, "
        "{%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    mma_f16(d, a, b0, b1);
}

__device__ __forceinline__ void mma_tf32(float (&d)[4], const float (&a)[4], float b0, float b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, "
      "{%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(__float_as_uint(a[0])), "r"(__float_as_uint(a[1])), "r"(__float_as_uint(a[2])),
        "r"(__float_as_uint(a[3])), "r"(__float_as_uint(b0)), "r"(__float_as_uint(b1)));
}

__device__ __forceinline__ void ldmatrix(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldmatrix_trans(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void stmatrix_trans(uint32_t addr, uint32_t a, uint32_t b, uint32_t c,
                                               uint32_t d) {
  asm volatile("stmatrix.sync.aligned.m8n8.x4.trans.shared.b16 [%0], {%1, %2, %3, %4};" ::"r"(addr),
               "r"(a), "r"(b), "r"(c), "r"(d)
               : "memory");
}

// 16 bytes to shared memory, the first `bytes` of them from `src`, then zeros.
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, int bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes)
               : "memory");
}
__device__ __forceinline__ void cp_async_commit() {
  asm volatile("cp.async.commit_group;" ::: "memory");
}
template <int N> __device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// A bounded wait that also ends when another thread's has run out; each try
// may park the warp for up to 2 us.
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

__device__ __forceinline__ float quad_max(float x) {
  x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 1));
  return fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 2));
}

// 2^(whole + rest) for an integer `whole` and |rest| < 1: in one sum an exponent of
// 16, which rows' scales make common, would cut rest off at 2^-20 (float32 outputs
// 7.5e-7 of their norm off in place of 2.5e-7).
__device__ __forceinline__ float exp2_of(float whole, float rest) {
  return mamba_scan::ex2_approx(whole) * mamba_scan::ex2_approx(rest);
}

__device__ __forceinline__ float to_tf32(float x) {
  uint32_t r;
  asm("cvt.rna.tf32.f32 %0, %1;" : "=r"(r) : "f"(x));
  return __uint_as_float(r);
}

// The rows of q or k as products read them: fp16 parts, hi then (fp32) lo, at
// `pitch` bytes (16 past the row, so that eight rows' 16-byte pieces fall into
// different banks). One warp, one row, DKP / 32 elements a lane; the row's
// power of two comes back. fp16 rows keep theirs (exact, scale 1).
template <typename T, int DKP> struct Tile {
  static constexpr int kPer = DKP / 32;
  static constexpr int kRowBytes = DKP * 2 * Parts<T>::n;  // also that of a raw row
  static constexpr int kPitch = kRowBytes + 16;
  static constexpr int kBytes = kChunk * kPitch;
  // what prepare_kernel multiplies: float32 rows' fp16 parts, 16-bit rows themselves
  using Product = typename std::conditional<sizeof(T) == 4, __half, T>::type;

  // A row's kPer elements of this lane, times `scale`, into the row's parts.
  static __device__ __forceinline__ void write(uint8_t* row, const float (&x)[kPer], float scale,
                                               int lane) {
    uint32_t hi[kPer / 2], lo[kPer / 2];
#pragma unroll
    for (int i = 0; i < kPer / 2; ++i)
      split_half2(x[2 * i] * scale, x[2 * i + 1] * scale, hi[i], lo[i]);
    if constexpr (kPer == 4) {
      *reinterpret_cast<uint2*>(row + lane * 8) = make_uint2(hi[0], hi[1]);
      if constexpr (Parts<T>::n == 2)
        *reinterpret_cast<uint2*>(row + DKP * 2 + lane * 8) = make_uint2(lo[0], lo[1]);
    } else {
      *reinterpret_cast<uint32_t*>(row + lane * 4) = hi[0];
      if constexpr (Parts<T>::n == 2) *reinterpret_cast<uint32_t*>(row + DKP * 2 + lane * 4) = lo[0];
    }
  }

  // 32 rows of raw elements, at row0 on, into their parts, in place.
  static __device__ __forceinline__ void convert(uint8_t* tile, const float* scale, int row0,
                                                 int lane) {
    if constexpr (Parts<T>::n == 2) {
      constexpr int kBatch = 4;
#pragma unroll
      for (int r0 = 0; r0 < 32; r0 += kBatch) {
        float x[kBatch][kPer];
        uint8_t* row = tile + (row0 + r0) * kPitch;
#pragma unroll
        for (int i = 0; i < kBatch; ++i) read(x[i], row + i * kPitch + lane * kPer * 4);
        __syncwarp();  // (a part of the row lies over another lane's elements)
#pragma unroll
        for (int i = 0; i < kBatch; ++i)
          write(row + i * kPitch, x[i], scale[row0 + r0 + i], lane);
      }
    } else if constexpr (!std::is_same<T, __half>::value) {
      constexpr int kPieces = kRowBytes / 16, kN = kPieces, kBatch = 4;
#pragma unroll
      for (int i0 = 0; i0 < kN; i0 += kBatch) {
        uint4 w[kBatch];
        float f[kBatch];
#pragma unroll
        for (int i = 0; i < kBatch; ++i) {
          const int at = (i0 + i) * 32 + lane, t = row0 + at / kPieces;
          w[i] = *reinterpret_cast<const uint4*>(tile + t * kPitch + at % kPieces * 16);
          f[i] = scale[t];
        }
#pragma unroll
        for (int i = 0; i < kBatch; ++i) {
          const int at = (i0 + i) * 32 + lane, t = row0 + at / kPieces;
          uint32_t u[4] = {w[i].x, w[i].y, w[i].z, w[i].w};
#pragma unroll
          for (int j = 0; j < 4; ++j)
            u[j] = pack_half2(__uint_as_float(u[j] << 16) * f[i],
                              __uint_as_float(u[j] & 0xffff0000u) * f[i]);
          *reinterpret_cast<uint4*>(tile + t * kPitch + at % kPieces * 16) =
              make_uint4(u[0], u[1], u[2], u[3]);
        }
      }
    }
  }

  // kPer elements as they lie in memory, and as floats.
  using Raw = typename std::conditional<
      kPer * sizeof(T) == 16, uint4,
      typename std::conditional<kPer * sizeof(T) == 8, uint2, uint32_t>::type>::type;
  static __device__ __forceinline__ void widen(float (&x)[kPer], const Raw& raw) {
    const T* h = reinterpret_cast<const T*>(&raw);
#pragma unroll
    for (int i = 0; i < kPer; ++i) x[i] = to_f32(h[i]);
  }
  static __device__ __forceinline__ void read(float (&x)[kPer], const void* p) {
    widen(x, *reinterpret_cast<const Raw*>(p));
  }
};

// ------------------------------------------------------- chunks on their own

template <typename T, int DKP, typename R> struct __align__(128) PrepareSmem {
  static constexpr bool kTiles = std::is_same<R, TileRecord>::value;
  struct Tiles {
    uint8_t k[Tile<T, DKP>::kBytes];
    uint8_t q[Tile<T, DKP>::kBytes];
  };
  struct Solve {  // once the scores are formed
    // blocks of 16 x 16: below the diagonal A's, on it A's, then T's, and T's (i, j)
    // below it in the place of (j, i); then T's tile for the record
    __align__(16) float m[kChunk][kChunk + 4];
    __align__(16) uint8_t p_tile[kTiles ? 2 * kChunk * 128 : 16];  // P's for the record
  };
  union {
    Tiles tile;
    Solve s;
  };
  float2 G[kChunk];  // running log2 decay: floor and the rest
  float beta[kChunk];
  float ek[kChunk], eq[kChunk];  // the rows' exponents
  float p_max[4], t_max[4], u_max[2];
  int bad;           // a NaN among the decays
};

// One block, scaled, as the fragments of Record: two accumulator tiles, columns
// 2 (lane % 4) + {0, 1} and 8 more, of rows lane / 4 and + 8.
__device__ __forceinline__ void split_block(uint4& hi, uint4& lo, float f, const float (&left)[4],
                                            const float (&right)[4]) {
  split_half2(left[0] * f, left[1] * f, hi.x, lo.x);
  split_half2(right[0] * f, right[1] * f, hi.y, lo.y);
  split_half2(left[2] * f, left[3] * f, hi.z, lo.z);
  split_half2(right[2] * f, right[3] * f, hi.w, lo.w);
}

// Rows 16 warp.. of a lower triangle, scaled by f, into a record: accumulator
// tiles x[n] of columns 8 n.., those past the diagonal block not looked at.
__device__ __forceinline__ void store_triangle(uint4 (*dst)[kBlocks][32], int warp, int lane,
                                               float f, const float (&x)[8][4]) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    if (j > warp) break;
    uint4 hi, lo;
    split_block(hi, lo, f, x[2 * j], x[2 * j + 1]);
    dst[0][warp * (warp + 1) / 2 + j][lane] = hi;
    dst[1][warp * (warp + 1) / 2 + j][lane] = lo;
  }
}
// The same into a tile in shared memory, hi then lo, which goes to the record in
// bulk; hi parts cut off to 11 bits (21 of both), zeros past the diagonal block.
__device__ __forceinline__ void store_triangle(uint8_t* tile, int warp, int lane, float f,
                                               const float (&x)[8][4]) {
  const int r = lane >> 2;
  uint8_t* row = tile + (16 * warp + r) * 128 + (lane & 3) * 4;
#pragma unroll
  for (int n = 0; n < 8; ++n) {
    if (n > 2 * warp + 1) break;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      float2 v = __fmul2_rn(make_float2(x[n][2 * i], x[n][2 * i + 1]), make_float2(f, f));
      const float2 h = make_float2(__uint_as_float(__float_as_uint(v.x) & 0xffffe000u),
                                   __uint_as_float(__float_as_uint(v.y) & 0xffffe000u));
      v = __ffma2_rn(h, make_float2(-1.f, -1.f), v);
      uint8_t* at = row + i * 8 * 128 + ((n ^ r) << 4);
      *reinterpret_cast<uint32_t*>(at) = pack_half2(h.x, h.y);
      *reinterpret_cast<uint32_t*>(at + kChunk * 128) = pack_half2(v.x, v.y);
    }
  }
#pragma unroll
  for (int j = 1; j < 4; ++j) {
    if (j <= warp) continue;  // two pieces of 16 rows
    uint8_t* at = tile + (16 * warp + (lane >> 1)) * 128 +
                  (((2 * j + (lane & 1)) ^ ((lane >> 1) & 7)) << 4);
    *reinterpret_cast<uint4*>(at) = make_uint4(0, 0, 0, 0);
    *reinterpret_cast<uint4*>(at + kChunk * 128) = make_uint4(0, 0, 0, 0);
  }
}

__device__ __forceinline__ void bulk_store(void* dst, const void* src, uint32_t bytes) {
  asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;" ::"l"(dst),
               "r"(smem_u32(src)), "r"(bytes)
               : "memory");
  mamba_scan::bulk_commit();
}

// The small fields of either record.
struct Fields {
  float *x_fac, *u_fac, *o_fac, *k_scale, *q_scale, *carry, *t_inv, *p_inv;
};
__device__ __forceinline__ Fields fields(Record& r) {
  return Fields{r.chain.x_fac, r.chain.u_fac,   r.out.o_fac,   r.chain.k_scale,
                r.out.q_scale, &r.chain.carry, &r.chain.t_inv, &r.out.p_inv};
}
__device__ __forceinline__ Fields fields(TileRecord& r) {
  return Fields{r.main.x_fac,   r.main.u_fac,  r.out.o_fac,   r.main.k_scale,
                r.main.q_scale, &r.main.carry, &r.main.t_inv, &r.out.p_inv};
}

// What bounds it: the latency of these steps, instructions at half the issue rate
// and shared memory at 0.55 (5120 chunks of dk = 128 in bf16 104 us, 3.2 TB/s of
// rows and records; at four CTAs on an SM 0.05 more). Its products are small (two of
// 64 x 64 x dk and the inverse's of 16 x 16 blocks), so warps' own.
//
// A CTA of 4 warps = one chunk of one sequence and head. Warp w forms rows 16
// w.. of K K^T and Q K^T (up to the diagonal), weights them, writes P and
// leaves A; then inverts I + A: diagonal blocks by substitution, a lane per
// column, and warp j the blocks below block j of its column, from
//   T_ij = -T_ii sum_{j <= k < i} A_ik T_kj,
// transposed, so that each product's result is the next one's left operand.
template <typename T, int DKP, typename R>
__global__ void __launch_bounds__(128, 5) prepare_kernel(const Params p) {
  constexpr bool kTiles = std::is_same<R, TileRecord>::value;
  using Tl = Tile<T, DKP>;
  constexpr int NP = Parts<T>::n, kPer = Tl::kPer, kPitch = Tl::kPitch;
  extern __shared__ __align__(128) uint8_t smem_raw[];
  PrepareSmem<T, DKP, R>& sm = *reinterpret_cast<PrepareSmem<T, DKP, R>*>(smem_raw);
  // The first launch of a prompt waits for what comes before it. A later one
  // starts beside the chain over the chunks before (its records are another
  // buffer's), and only its last CTA waits, at its end: so it counts as done, and
  // the chain over its chunks may begin, once that chain is.
  mamba_scan::pdl_trigger();
  const bool last_waits = p.c0 > 0 && blockIdx.x == gridDim.x - 1;
  if (p.c0 == 0) mamba_scan::pdl_wait();
  const mamba_gated_delta_args& a = p.a;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int n_chunks = p.c1 - p.c0;
  const int64_t bh = blockIdx.x / (unsigned)n_chunks;
  const int c = p.c0 + (int)(blockIdx.x % (unsigned)n_chunks);
  const int H = (int)a.heads, dk = (int)a.dk;
  const int b = (int)(bh / H), h = (int)(bh % H), g = h / (int)(a.heads / a.groups);
  const int t0 = c * kChunk;
  const int len = min(kChunk, clamped_length(a.lengths, b, (int)a.seqlen) - t0);
  if (len <= 0) {  // chain_kernel does not look at such a chunk
    if (last_waits) mamba_scan::pdl_wait();
    return;
  }
  R& rec = static_cast<R*>(p.records)[bh * n_chunks + (c - p.c0)];
  const Fields f = fields(rec);

  // rows 16 warp.. of k and q
  const T* src[2] = {static_cast<const T*>(a.k) + b * a.k_stride[0] + g * a.k_stride[2] +
                         (int64_t)t0 * a.k_stride[1],
                     static_cast<const T*>(a.q) + b * a.q_stride[0] + g * a.q_stride[2] +
                         (int64_t)t0 * a.q_stride[1]};
  if constexpr (NP == 1) {
    // as they are: the products take 16-bit rows raw
    constexpr int kPieces = DKP / 8, kRows = 128 / kPieces;  // 16-byte pieces; rows at a time
    const int at = threadIdx.x % kPieces * 8, first = threadIdx.x / kPieces;
    const int bytes = min(max(dk - at, 0) * 2, 16);
#pragma unroll
    for (int which = 0; which < 2; ++which) {
      const int64_t stride = which ? a.q_stride[1] : a.k_stride[1];
      uint8_t* tile = which ? sm.tile.q : sm.tile.k;
#pragma unroll
      for (int i = 0; i < kChunk / kRows; ++i) {
        const int t = first + i * kRows;
        const T* row = src[which] + (int64_t)t * stride + at;
        uint8_t* to = tile + t * kPitch + at * 2;
        if (p.qk_vec) {
          const bool there = t < len && bytes > 0;
          cp_async16(smem_u32(to), there ? row : src[which], there ? bytes : 0);
        } else {
          __align__(16) T x[8];
#pragma unroll
          for (int j = 0; j < 8; ++j) x[j] = t < len && at + j < dk ? row[j] : from_f32<T>(0.f);
          *reinterpret_cast<uint4*>(to) = *reinterpret_cast<const uint4*>(x);
        }
      }
    }
    cp_async_commit();
  } else {
    // (loads first, conversions after: a wait for each row's load was most of
    // this kernel, 105 us for 2240 chunks against 67)
    constexpr int kBatch = 8;
    const bool fast = p.qk_vec && dk % kPer == 0;
    const int at = lane * kPer;
    typename Tl::Raw raw[2][kBatch];
    auto fetch = [&](int which, int r0) {
      const int64_t stride = which ? a.q_stride[1] : a.k_stride[1];
  #pragma unroll
      for (int i = 0; i < kBatch; ++i) {
        const int t = warp * 16 + r0 + i;
        raw[which][i] = typename Tl::Raw{};
        if (t < len && at < dk)
          raw[which][i] =
              *reinterpret_cast<const typename Tl::Raw*>(src[which] + (int64_t)t * stride + at);
      }
    };
    if (fast) fetch(0, 0), fetch(1, 0);
  #pragma unroll
    for (int r0 = 0; r0 < 16; r0 += kBatch) {
  #pragma unroll
      for (int which = 0; which < 2; ++which) {
        uint8_t* tile = which ? sm.tile.q : sm.tile.k;
        float* exps = which ? sm.eq : sm.ek;
        float* scales = which ? f.q_scale : f.k_scale;
        int mine = 0;
  #pragma unroll
        for (int i = 0; i < kBatch; ++i) {
          const int t = warp * 16 + r0 + i;
          float x[kPer], m = 0.f;
          if (fast) {
            Tl::widen(x, raw[which][i]);
          } else {
            const int64_t stride = which ? a.q_stride[1] : a.k_stride[1];
  #pragma unroll
            for (int j = 0; j < kPer; ++j)
              x[j] = t < len && at + j < dk ? to_f32(src[which][(int64_t)t * stride + at + j]) : 0.f;
          }
  #pragma unroll
          for (int j = 0; j < kPer; ++j) m = fmaxf(m, fabsf(x[j]));
          const int e =
              scale_exponent(__uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(m))));
          Tl::write(tile + t * kPitch, x, pow2i(e), lane);
          mine = lane == i ? e : mine;
        }
        if (lane < kBatch) {
          exps[warp * 16 + r0 + lane] = (float)mine;
          scales[warp * 16 + r0 + lane] = pow2i(mine);
        }
        if (fast && r0 + kBatch < 16) fetch(which, r0 + kBatch);
      }
    }
  }
  if (warp == 0) {
    // the decays' running sum: lane l has rows 2 l and 2 l + 1
    int64_t sum[2];
    bool bad = false;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int t = 2 * lane + i;
      float gl = 0.f, be = 0.f;
      if (t < len) {
        const int64_t row = t0 + t;
        gl = a.log_decay[b * a.decay_stride[0] + row * a.decay_stride[1] + h * a.decay_stride[2]];
        be = a.beta[b * a.beta_stride[0] + row * a.beta_stride[1] + h * a.beta_stride[2]];
      }
      bad |= gl != gl;
      gl = fminf(fmaxf(gl * 1.4426950408889634f, -16384.f), 16384.f);
      sum[i] = __float2ll_rn(gl * 1099511627776.f);  // 2^40
      sm.beta[t] = be;
    }
    int64_t upto = sum[0] + sum[1];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t other = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += other;
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int64_t G = i == 0 ? upto - sum[1] : upto;
      sm.G[2 * lane + i] = make_float2((float)(int)(G >> 40),
                                       (float)((uint64_t)(G << 24) >> 40) * 5.9604644775390625e-8f);
    }
    const bool any_bad = __any_sync(0xffffffffu, bad);
    if (lane == 0) sm.bad = any_bad;
  }
  if constexpr (NP == 1) cp_async_wait<0>();
  __syncthreads();
  if constexpr (NP == 1) {
    // the powers of two that the chain scales bf16 rows by (fp16 ones stay as they
    // are), a lane a row of k or q: patterns without the sign order like the
    // magnitudes
    const int row = warp * 16 + (lane & 15), which = lane >> 4;
    int e = 0;
    if constexpr (!std::is_same<T, __half>::value) {
      const uint8_t* at = (which ? sm.tile.q : sm.tile.k) + row * kPitch;
      uint32_t m = 0;
#pragma unroll
      for (int i = 0; i < DKP / 8; ++i) {
        const uint4 w = *reinterpret_cast<const uint4*>(at + i * 16);
        m = __vmaxu2(__vmaxu2(m, w.x & 0x7fff7fffu), w.y & 0x7fff7fffu);
        m = __vmaxu2(__vmaxu2(m, w.z & 0x7fff7fffu), w.w & 0x7fff7fffu);
      }
      e = scale_exponent(__uint_as_float(max(m << 16, m & 0xffff0000u)));
    }
    (which ? sm.eq : sm.ek)[row] = (float)e;
    (which ? f.q_scale : f.k_scale)[row] = pow2i(e);
  }

  // products: tile n covers columns s = 8 n.. of rows t = 16 warp..
  float kk[8][4], qk[8][4];
#pragma unroll
  for (int n = 0; n < 8; ++n)
#pragma unroll
    for (int i = 0; i < 4; ++i) kk[n][i] = qk[n][i] = 0.f;
  const uint32_t k_base = smem_u32(sm.tile.k), q_base = smem_u32(sm.tile.q);
  const uint32_t a_at = (uint32_t)((warp * 16 + (lane & 15)) * kPitch + (lane >> 4) * 16);
  const uint32_t b_at = (uint32_t)(((lane & 7) + ((lane >> 4) << 3)) * kPitch + ((lane >> 3) & 1) * 16);
  // (float32: the small products first, as sums are cut off, see triangular())
#pragma unroll 1
  for (int step = 0; step < NP * DKP / 16; ++step) {
    const bool high = NP == 1 || step >= DKP / 16;
    const int ks = step & (DKP / 16 - 1);
    uint32_t ka[NP][4], qa[NP][4];
#pragma unroll
    for (int i = 0; i < NP; ++i) {
      ldmatrix(ka[i], k_base + a_at + ks * 32 + i * DKP * 2);
      ldmatrix(qa[i], q_base + a_at + ks * 32 + i * DKP * 2);
    }
#pragma unroll
    for (int np = 0; np < 4; ++np) {
      if (np > warp) break;
      uint32_t bf[NP][4];
#pragma unroll
      for (int i = 0; i < NP; ++i)
        ldmatrix(bf[i], k_base + b_at + np * 16 * kPitch + ks * 32 + i * DKP * 2);
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        if (high) {
          mma_16bit<typename Tl::Product>(kk[2 * np + i], ka[0], bf[0][2 * i], bf[0][2 * i + 1]);
          mma_16bit<typename Tl::Product>(qk[2 * np + i], qa[0], bf[0][2 * i], bf[0][2 * i + 1]);
        } else if constexpr (NP == 2) {
          mma_f16(kk[2 * np + i], ka[1], bf[0][2 * i], bf[0][2 * i + 1]);
          mma_f16(qk[2 * np + i], qa[1], bf[0][2 * i], bf[0][2 * i + 1]);
          mma_f16(kk[2 * np + i], ka[0], bf[1][2 * i], bf[1][2 * i + 1]);
          mma_f16(qk[2 * np + i], qa[0], bf[1][2 * i], bf[1][2 * i + 1]);
        }
      }
    }
  }
  __syncthreads();  // the tiles give way to A and T
  // weights; row r of this lane's two (t and t + 8). A score's factor is 2 to a
  // difference of sums, floors and the rows' exponents apart from the rest.
  const int r = lane >> 2, cq = 2 * (lane & 3);
  const int t_lo = warp * 16 + r;
  float p_max = 0.f;
  {
    const float2 Gt[2] = {sm.G[t_lo], sm.G[t_lo + 8]};
    const float bt[2] = {sm.beta[t_lo], sm.beta[t_lo + 8]};
    // (the products of 16-bit rows are not scaled)
    constexpr float kScaled = NP == 2 ? 1.f : 0.f;
    const float kt[2] = {Gt[0].x - kScaled * sm.ek[t_lo], Gt[1].x - kScaled * sm.ek[t_lo + 8]};
    const float qt[2] = {Gt[0].x - kScaled * sm.eq[t_lo], Gt[1].x - kScaled * sm.eq[t_lo + 8]};
#pragma unroll
    for (int n = 0; n < 8; ++n) {
      if (n > 2 * warp + 1) break;
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int s = 8 * n + cq + j;
        const float2 Gs = sm.G[s];
        const float from = Gs.x + kScaled * sm.ek[s];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int t = t_lo + 8 * i;
          const float rest = Gt[i].y - Gs.y;
          // (without rows' scales an exponent is small where its weight matters)
          const float wk = NP == 2 ? exp2_of(kt[i] - from, rest)
                                   : mamba_scan::ex2_approx((kt[i] - from) + rest);
          const float wq = NP == 2 ? exp2_of(qt[i] - from, rest) : wk;
          // (a masked weight may be infinite: selected, not multiplied, away)
          float x = bt[i] * (kk[n][2 * i + j] * wk), y = qk[n][2 * i + j] * wq;
          if (n >= 2 * warp) {
            if (s >= t) x = 0.f;
            if (s > t) y = 0.f;
          }
          sm.s.m[t][s] = x;
          qk[n][2 * i + j] = y;
          p_max = fmaxf(p_max, fabsf(y));
        }
      }
    }
  }
  p_max = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(p_max)));
  if (lane == 0) sm.p_max[warp] = p_max;
  if (threadIdx.x < kChunk) {
    const int t = threadIdx.x;
    const float spoil = sm.bad ? __int_as_float(0x7fc00000) : 0.f;
    const float2 G = sm.G[t], last = sm.G[kChunk - 1];
    f.x_fac[t] = exp2_of(G.x - sm.ek[t], G.y) + spoil;
    f.o_fac[t] = exp2_of(G.x - sm.eq[t], G.y) * a.scale + spoil;
    const float u = exp2_of(last.x - (G.x + sm.ek[t]), last.y - G.y);
    f.u_fac[t] = u;
    if constexpr (kTiles) {
      const uint32_t m = __reduce_max_sync(0xffffffffu, __float_as_uint(u));
      if (lane == 0) sm.u_max[warp] = __uint_as_float(m);
    }
    if (t == 0) *f.carry = exp2_of(last.x, last.y) + spoil;
  }
  __syncwarp();  // this warp's rows of A

  // (I + A_ww)^-1, a column per lane (both halves of the warp do the same)
  {
    const int j = lane & 15;
    float x[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      float s = i == j ? 1.f : 0.f;
      const float4* row = reinterpret_cast<const float4*>(&sm.s.m[warp * 16 + i][warp * 16]);
#pragma unroll
      for (int k = 0; k < i; k += 4) {
        const float4 w = row[k / 4];
        s = fmaf(-w.x, x[k], s);
        if (k + 1 < i) s = fmaf(-w.y, x[k + 1], s);
        if (k + 2 < i) s = fmaf(-w.z, x[k + 2], s);
        if (k + 3 < i) s = fmaf(-w.w, x[k + 3], s);
      }
      x[i] = s;
    }
    __syncwarp();
    if (lane < 16)
#pragma unroll
      for (int i = 0; i < 16; ++i) sm.s.m[warp * 16 + i][warp * 16 + j] = x[i];
  }
  __syncthreads();
  {
    const int e = scale_exponent(fmaxf(fmaxf(sm.p_max[0], sm.p_max[1]),
                                       fmaxf(sm.p_max[2], sm.p_max[3])));
    if constexpr (kTiles) store_triangle(sm.s.p_tile, warp, lane, pow2i(e), qk);
    else store_triangle(rec.out.p, warp, lane, pow2i(e), qk);
    if (threadIdx.x == 0) *f.p_inv = pow2i(-e) * a.scale;
  }
  if constexpr (kTiles) {
    if (threadIdx.x < kChunk) {  // (its own value, written above)
      const int field = (int)(__float_as_uint(fmaxf(sm.u_max[0], sm.u_max[1])) >> 23);
      const int e = max(min(126 - field, 126), -126);
      f.u_fac[threadIdx.x] *= pow2i(e);
      if (threadIdx.x == 0) rec.main.u_inv = pow2i(-e);
    }
  }
  // d += a x b, a and d accumulator tiles (16 x 16, two tiles of 8 columns), b
  // the 16 x 16 block at `block`, transposed (its rows are d's columns)
  auto multiply = [&](float (&d)[2][4], const float (&x)[2][4], const float* block) {
#pragma unroll
    for (int kt = 0; kt < 2; ++kt) {
      // (a product's columns may come in any order if b's rows do: column i of
      // the operand is column 2 i of the tile, i + 4 is 2 i + 1)
      float hi[4], lo[4];
      const float v[4] = {x[kt][0], x[kt][2], x[kt][1], x[kt][3]};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        hi[i] = to_tf32(v[i]);
        lo[i] = to_tf32(v[i] - hi[i]);
      }
#pragma unroll
      for (int nt = 0; nt < 2; ++nt) {
        const float2 y = *reinterpret_cast<const float2*>(
            block + (8 * nt + r) * (kChunk + 4) + 8 * kt + cq);
        const float yh0 = to_tf32(y.x), yh1 = to_tf32(y.y);
        mma_tf32(d[nt], lo, yh0, yh1);
        mma_tf32(d[nt], hi, to_tf32(y.x - yh0), to_tf32(y.y - yh1));
        mma_tf32(d[nt], hi, yh0, yh1);
      }
    }
  };
  if (warp < 3) {
    float y[3][2][4];  // T_kj^T of k = warp, warp + 1, warp + 2
#pragma unroll
    for (int n = 0; n < 2; ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        y[0][n][i] = sm.s.m[warp * 16 + 8 * n + cq + (i & 1)][warp * 16 + r + 8 * (i >> 1)];
#pragma unroll
    for (int step = 1; step <= 3; ++step) {
      const int i = warp + step;
      if (i > 3) break;
      float z[2][4] = {}, d[2][4] = {};
#pragma unroll
      for (int k = 0; k < step; ++k) multiply(z, y[k], &sm.s.m[16 * i][16 * (warp + k)]);
      multiply(d, z, &sm.s.m[16 * i][16 * i]);
#pragma unroll
      for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          sm.s.m[16 * warp + 8 * n + cq + (e & 1)][16 * i + r + 8 * (e >> 1)] = -d[n][e];
          if (step < 3) y[step < 3 ? step : 0][n][e] = -d[n][e];
        }
    }
  }
  __syncthreads();
  {
    float x[8][4], m = 0.f;
#pragma unroll
    for (int n = 0; n < 8; ++n) {
      if (n > 2 * warp + 1) break;
      const float2 bs = *reinterpret_cast<const float2*>(&sm.beta[8 * n + cq]);
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const float2 w = *reinterpret_cast<const float2*>(
            &sm.s.m[16 * (n >> 1) + r + 8 * i][16 * warp + 8 * (n & 1) + cq]);
        x[n][2 * i] = w.x * bs.x;
        x[n][2 * i + 1] = w.y * bs.y;
        m = fmaxf(m, fmaxf(fabsf(x[n][2 * i]), fabsf(x[n][2 * i + 1])));
      }
    }
    m = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(m)));
    if (lane == 0) sm.t_max[warp] = m;
    if constexpr (kTiles) mamba_scan::fence_proxy_async_smem();  // (P's tile)
    __syncthreads();
    if constexpr (kTiles) {
      if (threadIdx.x == 0) bulk_store(rec.out.p, sm.s.p_tile, 2 * kChunk * 128);
    }
    const int e = scale_exponent(fmaxf(fmaxf(sm.t_max[0], sm.t_max[1]),
                                       fmaxf(sm.t_max[2], sm.t_max[3])));
    if (threadIdx.x == 0) *f.t_inv = pow2i(-e);
    if constexpr (kTiles) {
      uint8_t* tile = reinterpret_cast<uint8_t*>(sm.s.m);  // (all of it has been read)
      store_triangle(tile, warp, lane, pow2i(e), x);
      mamba_scan::fence_proxy_async_smem();
      __syncthreads();
      if (threadIdx.x == 0) {
        bulk_store(rec.main.t, tile, 2 * kChunk * 128);
        mamba_scan::bulk_wait_all<0>();
      }
    } else {
      store_triangle(rec.chain.t, warp, lane, pow2i(e), x);
    }
  }
  if (last_waits) mamba_scan::pdl_wait();
}

// --------------------------------------------------------- the chain itself

constexpr int kHelpers = 2;  // warps that load and convert, for each of the two

// NW warps of 16 state columns carry the chain, NW form their outputs.
template <typename T, int DKP_, int NW_> struct ChainCfg {
  static constexpr int DKP = DKP_, NW = NW_;
  static constexpr int kThreads = 32 * (2 * NW + 2 * kHelpers);
  static constexpr int kDv = 16 * NW;
  static constexpr int kVPitch = kDv * (int)sizeof(T) + 16;
  // The chain's chunks: one at work, one converted, one on its way, where there
  // is room.
  static constexpr int kStages = sizeof(T) == 4 && DKP * NW == 256 ? 2 : 3;
  struct __align__(16) ChainStage {
    uint8_t k[Tile<T, DKP>::kBytes];
    uint8_t v[kChunk * kVPitch];
    ChainRecord rec;
  };
  struct __align__(16) OutStage {
    uint8_t q[Tile<T, DKP>::kBytes];
    OutRecord rec;
  };
  struct __align__(16) Smem {
    ChainStage chain[kStages];
    OutStage out[2];
    uint8_t o[kChunk * kVPitch];  // outputs on their way
    // what a chain warp hands to its output warp, as left operands: the state
    // before the chunk and U, and what undoes their rows' scales
    uint4 state[NW][DKP / 16][2][32];
    uint4 u[NW][kChunk / 16][2][32];
    float state_inv[NW][16], u_inv[NW][16];
    uint64_t chain_full[kStages], chain_empty[kStages], out_full[2], out_empty[2];
    uint64_t state_full[NW], state_free[NW], u_full[NW], u_free[NW];
    int gave_up;
  };
  static_assert(sizeof(Smem) <= 227 * 1024, "shared memory per CTA");
};

// 32 rows, from row0 on, of kRow bytes (n elements, then zeros) to a tile, rows
// from `len` on as zeros: asynchronously where rows start at 16 bytes, else
// element by element.
template <typename T, int kRow>
__device__ __forceinline__ void load_rows(uint8_t* tile, int pitch, const T* src, int64_t stride,
                                          int n, int len, bool vec, int row0, int lane) {
  constexpr int kPieces = kRow / 16, kStep = 32 / kPieces;  // rows at a time
  static_assert(kPieces <= 32 && 32 % kPieces == 0, "a row is a whole part of a warp's pieces");
  if (vec) {
    const int at = lane % kPieces * 16;
    const int bytes = min(max(n * (int)sizeof(T) - at, 0), 16);
    int t = row0 + lane / kPieces;
    uint32_t to = smem_u32(tile + t * pitch + at);
    const uint8_t* row = reinterpret_cast<const uint8_t*>(src + (int64_t)t * stride) + at;
    const int64_t step = stride * kStep * (int)sizeof(T);
#pragma unroll
    for (int i = 0; i < kPieces; ++i, t += kStep) {
      const bool there = t < len && bytes > 0;
      cp_async16(to + i * kStep * pitch,
                 there ? row + i * step : reinterpret_cast<const uint8_t*>(src), there ? bytes : 0);
    }
  } else {
    constexpr int kElems = kRow / (int)sizeof(T);
    for (int i = lane; i < 32 * kElems; i += 32) {
      const int t = row0 + i / kElems, e = i % kElems;
      T x = from_f32<T>(0.f);
      if (t < len && e < n) x = src[(int64_t)t * stride + e];
      *reinterpret_cast<T*>(tile + t * pitch + e * (int)sizeof(T)) = x;
    }
  }
}

// A record's part, `bytes` of it up to its 64 scales by both helper warps, and
// the scales of its own 32 rows by each.
template <typename R>
__device__ __forceinline__ void load_record(R& to, const R& from, size_t bytes, int helper, int lane) {
  const uint8_t* src = reinterpret_cast<const uint8_t*>(&from);
  const uint32_t dst = smem_u32(&to);
#pragma unroll
  for (int i = 0; i < (int)(sizeof(R) / 16 + 63) / 64; ++i) {
    const int at = ((2 * i + helper) * 32 + lane) * 16;
    if (at < (int)bytes) cp_async16(dst + at, src + at, 16);
  }
  if (lane < 8) {
    const int at = (int)bytes + helper * 128 + lane * 16;
    cp_async16(dst + at, src + at, 16);
  }
}

// The columns' pair i of an accumulator tile: 0 of row lane / 4, 1 of row + 8.
__device__ __forceinline__ float2 pair(const float (&x)[4], int i) {
  return make_float2(x[2 * i], x[2 * i + 1]);
}
__device__ __forceinline__ float2 twice(float x) { return make_float2(x, x); }

// The left operand's parts of 16 columns (a k-step) of a warp's 16 rows, from
// two accumulator tiles scaled by f0 (row lane / 4) and f1 (row + 8).
__device__ __forceinline__ void split_operand(uint32_t (&hi)[4], uint32_t (&lo)[4],
                                              const float (&x)[4], const float (&y)[4], float f0,
                                              float f1) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 v = __fmul2_rn(i < 2 ? pair(x, i) : pair(y, i - 2), twice(i & 1 ? f1 : f0));
    const __half2 h = __floats2half2_rn(v.x, v.y);
    hi[i] = *reinterpret_cast<const uint32_t*>(&h);
    const float2 rest = __ffma2_rn(__half22float2(h), twice(-1.f), v);
    lo[i] = pack_half2(rest.x, rest.y);
  }
}

// The largest |x| of the lane's parts of both rows, two chains each.
template <int N>
__device__ __forceinline__ void lane_largest(const float (&x)[N][4], float& m0, float& m1) {
  float a0 = 0.f, a1 = 0.f, b0 = 0.f, b1 = 0.f;
#pragma unroll
  for (int n = 0; n < N; n += 2) {
    a0 = max3(a0, fabsf(x[n][0]), fabsf(x[n][1]));
    a1 = max3(a1, fabsf(x[n][2]), fabsf(x[n][3]));
    b0 = max3(b0, fabsf(x[n + 1][0]), fabsf(x[n + 1][1]));
    b1 = max3(b1, fabsf(x[n + 1][2]), fabsf(x[n + 1][3]));
  }
  m0 = fmaxf(a0, b0);
  m1 = fmaxf(a1, b1);
}

template <int N>
__device__ __forceinline__ void row_exponents(const float (&x)[N][4], int& e0, int& e1) {
  float m0, m1;
  lane_largest(x, m0, m1);
  e0 = scale_exponent(quad_max(m0));
  e1 = scale_exponent(quad_max(m1));
}

__device__ __forceinline__ uint4 as_uint4(const uint32_t (&x)[4]) {
  return make_uint4(x[0], x[1], x[2], x[3]);
}

// The products below run in steps of 8 to 12 mma.sync, which take the pipe 8
// clocks each, on accumulators that come again after 4 (their latency is 21),
// and a step's right operands are read one step ahead: read where they are
// used, their latency and the accumulators' were more than half of a chunk.

// The tensor cores cut every sum that goes back to an accumulator off towards zero,
// 2^-24 of it on average, and those of a product add up. So where float32 results
// come of it (kApart) the small products, which take a lo part, have accumulators of
// their own that are added at the end (in prepare_kernel they come first): a third of
// the cuts that matter. Outputs of 128 x 128 heads were 9.2e-7 of their norm off and
// are 5.3e-7, of 64 x 64 5.5e-7 and 2.5e-7, for 5 to 10% of the time; in the state's
// update, whose sums are short, it changed nothing.
template <int N>
__device__ __forceinline__ void add(float (&d)[N][4], const float (&x)[N][4]) {
#pragma unroll
  for (int n = 0; n < N; ++n)
#pragma unroll
    for (int i = 0; i < 4; ++i) d[n][i] += x[n][i];
}

// d[2 w], d[2 w + 1] (columns 16 w..) = sum over blocks (w, j) of left x block^T
// of a lower triangle; left(j, hi, lo) gives the left operand's k-step j.
template <bool kApart, typename Left>
__device__ __forceinline__ void triangular(float (&d)[8][4], const uint4 (*m)[kBlocks][32],
                                           int lane, Left&& left) {
  struct Blocks { uint4 h[2], l[2]; };
  // steps: column j of the triangle, rows first and (two) first + 1
  constexpr int kSteps = 6;
  constexpr int kJ[kSteps] = {0, 0, 1, 1, 2, 3}, kFirst[kSteps] = {0, 2, 1, 3, 2, 3};
  constexpr int kCount[kSteps] = {2, 2, 2, 1, 2, 1};
  auto fetch = [&](Blocks& b, int s) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int w = kFirst[s] + i;
      if (i < kCount[s]) {
        b.h[i] = m[0][w * (w + 1) / 2 + kJ[s]][lane];
        b.l[i] = m[1][w * (w + 1) / 2 + kJ[s]][lane];
      }
    }
  };
  float small[kApart ? 8 : 1][4];
#pragma unroll
  for (int n = 0; n < 8; ++n)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      d[n][i] = 0.f;
      if (kApart) small[n][i] = 0.f;
    }
  auto lows = [&](int n) -> float(&)[4] { return kApart ? small[kApart ? n : 0] : d[n]; };
  Blocks b[2];
  fetch(b[0], 0);
#pragma unroll
  for (int s = 0; s < kSteps; ++s) {
    if (s + 1 < kSteps) fetch(b[(s + 1) & 1], s + 1);
    uint32_t hi[4], lo[4];
    left(kJ[s], hi, lo);
    const Blocks& c = b[s & 1];
    const int w = kFirst[s];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      if (i == kCount[s]) break;
      mma_f16(d[2 * (w + i)], hi, c.h[i].x, c.h[i].y);
      mma_f16(d[2 * (w + i) + 1], hi, c.h[i].z, c.h[i].w);
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      if (i == kCount[s]) break;
      mma_f16(lows(2 * (w + i)), lo, c.h[i].x, c.h[i].y);
      mma_f16(lows(2 * (w + i) + 1), lo, c.h[i].z, c.h[i].w);
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      if (i == kCount[s]) break;
      mma_f16(lows(2 * (w + i)), hi, c.l[i].x, c.l[i].y);
      mma_f16(lows(2 * (w + i) + 1), hi, c.l[i].z, c.l[i].w);
    }
  }
  if constexpr (kApart) add(d, small);
}

// x (columns: the 64 rows of a tile) = left x tile^T over DKP, two or (tiles of
// two parts) three products; left(ks, hi, lo) gives the left operand's k-steps.
template <typename T, int DKP, typename Left>
__device__ __forceinline__ void by_rows(float (&x)[8][4], uint32_t tile_at, Left&& left) {
  constexpr int NP = Parts<T>::n, kPitch = Tile<T, DKP>::kPitch, kPart = DKP * 2;
  struct Rows { uint32_t f[NP][2][4]; };  // 32 rows of the tile, one k-step
  auto fetch = [&](Rows& b, int s) {      // step s: k-step s / 2, rows 32 (s % 2)..
#pragma unroll
    for (int i = 0; i < NP; ++i)
#pragma unroll
      for (int q = 0; q < 2; ++q)
        ldmatrix(b.f[i][q], tile_at + ((s & 1) * 2 + q) * 16 * kPitch + (s >> 1) * 32 + i * kPart);
  };
  float small[NP == 2 ? 8 : 1][4];
#pragma unroll
  for (int n = 0; n < 8; ++n)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[n][i] = 0.f;
      if (NP == 2) small[n][i] = 0.f;
    }
  auto lows = [&](int n) -> float(&)[4] { return NP == 2 ? small[NP == 2 ? n : 0] : x[n]; };
  Rows b[2];
  fetch(b[0], 0);
  uint32_t hi[4], lo[4];
#pragma unroll
  for (int s = 0; s < DKP / 8; ++s) {
    if (s + 1 < DKP / 8) fetch(b[(s + 1) & 1], s + 1);
    if (s % 2 == 0) left(s / 2, hi, lo);
    const Rows& c = b[s & 1];
    const int n0 = (s & 1) * 4;
#pragma unroll
    for (int n = 0; n < 4; ++n)
      mma_f16(x[n0 + n], hi, c.f[0][n >> 1][2 * (n & 1)], c.f[0][n >> 1][2 * (n & 1) + 1]);
#pragma unroll
    for (int n = 0; n < 4; ++n)
      mma_f16(lows(n0 + n), lo, c.f[0][n >> 1][2 * (n & 1)], c.f[0][n >> 1][2 * (n & 1) + 1]);
    if constexpr (NP == 2)
#pragma unroll
      for (int n = 0; n < 4; ++n)
        mma_f16(lows(n0 + n), hi, c.f[1][n >> 1][2 * (n & 1)], c.f[1][n >> 1][2 * (n & 1) + 1]);
  }
  if constexpr (NP == 2) add(x, small);
}

// Registers a thread with 12 warps: 168 at launch; the helpers give up what the
// chain takes, 248 + 168 + 88 = 3 x 168.
constexpr int kLaunchRegisters = 168, kChainRegisters = 248, kHelperRegisters = 88;
static_assert(kChainRegisters + kHelperRegisters <= 2 * kLaunchRegisters, "registers");

// A CTA = one sequence, head and tile of 16 NW columns. A chain warp carries 16
// state columns through the chunks (K S, T R, K^T U) and leaves the state and U
// of each chunk, as the left operands they are, to an output warp (Q S, P U):
// the chain is what takes long, one warp's instructions in sequence, and a
// second warp's products fill the tensor pipe meanwhile. Two warps for each of
// the two load the next chunks' rows and records and bring k and q into fp16
// parts, in place.
template <typename T, class C>
__global__ void __launch_bounds__(C::kThreads, 1) chain_kernel(const Params p) {
  constexpr int DKP = C::DKP, NP = Parts<T>::n, NW = C::NW;
  using Tl = Tile<T, DKP>;
  constexpr int kPitch = Tl::kPitch, kVPitch = C::kVPitch, kPart = DKP * 2;
  extern __shared__ __align__(128) uint8_t smem_raw[];
  typename C::Smem& sm = *reinterpret_cast<typename C::Smem*>(smem_raw);
  const mamba_gated_delta_args& a = p.a;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int H = (int)a.heads, dk = (int)a.dk, dv = (int)a.dv, L = (int)a.seqlen;
  const int tile = (int)(blockIdx.x % (unsigned)p.tiles);
  const int64_t bh = blockIdx.x / (unsigned)p.tiles;
  const int b = (int)(bh / H), h = (int)(bh % H), g = h / (int)(a.heads / a.groups);
  const int col0 = tile * C::kDv, cols = min(C::kDv, dv - col0);
  const int workers = (cols + 15) / 16;  // warps with columns
  constexpr int kStages = C::kStages;
  if (threadIdx.x == 0) {
    for (int i = 0; i < kStages; ++i) {
      mamba_scan::mbar_init(&sm.chain_full[i], kHelpers);
      mamba_scan::mbar_init(&sm.chain_empty[i], workers);
    }
    for (int i = 0; i < 2; ++i) {
      mamba_scan::mbar_init(&sm.out_full[i], kHelpers);
      mamba_scan::mbar_init(&sm.out_empty[i], workers);
    }
    for (int w = 0; w < NW; ++w) {
      mamba_scan::mbar_init(&sm.state_full[w], 1);
      mamba_scan::mbar_init(&sm.state_free[w], 1);
      mamba_scan::mbar_init(&sm.u_full[w], 1);
      mamba_scan::mbar_init(&sm.u_free[w], 1);
    }
    sm.gave_up = 0;
    mamba_scan::fence_mbarrier_init();
  }
  __syncthreads();
  // (the next launch, prepare_kernel over later chunks, may start only once
  // everything before this one is done: it writes the records read by then)
  mamba_scan::pdl_wait();
  mamba_scan::pdl_trigger();
  const int len_all = clamped_length(a.lengths, b, L);
  // chunks with rows that count
  const int c_end = min(p.c1, (len_all + kChunk - 1) / kChunk);

  if (warp >= 2 * NW) {
    if constexpr (NW == 4)
      asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kHelperRegisters));
    const int helper = warp & 1, row0 = 32 * helper, n = c_end - p.c0;
    const Record* recs = static_cast<const Record*>(p.records) + bh * (p.c1 - p.c0);
    if (warp < 2 * NW + kHelpers) {  // k, v and T for the chain
      const T* ks = static_cast<const T*>(a.k) + b * a.k_stride[0] + g * a.k_stride[2];
      const T* vs = static_cast<const T*>(a.v) + b * a.v_stride[0] + h * a.v_stride[2] + col0;
      // With three stages a chunk is converted while the next one is on its way.
      constexpr int kLag = kStages - 2;
      for (int i = 0; i < n + kLag; ++i) {
        if (i < n) {
          typename C::ChainStage& st = sm.chain[i % kStages];
          if (i >= kStages && !wait_or_leave(&sm.chain_empty[i % kStages],
                                             (uint32_t)(i / kStages - 1) & 1u, &sm.gave_up))
            break;
          const int t0 = (p.c0 + i) * kChunk, len = len_all - t0;
          load_rows<T, DKP * (int)sizeof(T)>(st.k, kPitch, ks + (int64_t)t0 * a.k_stride[1],
                                             a.k_stride[1], dk, len, p.qk_vec, row0, lane);
          load_rows<T, C::kDv * (int)sizeof(T)>(st.v, kVPitch, vs + (int64_t)t0 * a.v_stride[1],
                                                a.v_stride[1], cols, len, p.v_vec, row0, lane);
          load_record(st.rec, recs[i].chain, offsetof(ChainRecord, k_scale), helper, lane);
        }
        cp_async_commit();
        if (i < kLag) continue;
        cp_async_wait<kLag>();
        __syncwarp();
        typename C::ChainStage& done = sm.chain[(i - kLag) % kStages];
        if constexpr (!std::is_same<T, __half>::value)
          Tl::convert(done.k, done.rec.k_scale, row0, lane);
        __syncwarp();
        if (lane == 0) mbar_arrive(&sm.chain_full[(i - kLag) % kStages]);
      }
    } else {  // q and P for the outputs
      const T* qs = static_cast<const T*>(a.q) + b * a.q_stride[0] + g * a.q_stride[2];
      for (int i = 0; i < n; ++i) {
        typename C::OutStage& st = sm.out[i & 1];
        if (i >= 2 && !wait_or_leave(&sm.out_empty[i & 1], (uint32_t)((i >> 1) - 1) & 1u, &sm.gave_up))
          break;
        const int t0 = (p.c0 + i) * kChunk;
        load_rows<T, DKP * (int)sizeof(T)>(st.q, kPitch, qs + (int64_t)t0 * a.q_stride[1],
                                           a.q_stride[1], dk, len_all - t0, p.qk_vec, row0, lane);
        load_record(st.rec, recs[i].out, offsetof(OutRecord, q_scale), helper, lane);
        cp_async_commit();
        cp_async_wait<0>();
        __syncwarp();
        if constexpr (!std::is_same<T, __half>::value)
          Tl::convert(st.q, st.rec.q_scale, row0, lane);
        __syncwarp();
        if (lane == 0) mbar_arrive(&sm.out_full[i & 1]);
      }
    }
    cp_async_wait<0>();
    return;
  }
  if constexpr (NW == 4) {
    if (warp < NW) asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kChainRegisters));
  }
  const int w = warp % NW;  // the warp's columns: 16 w..
  if (w >= workers) return;
  const int r = lane >> 2, cq = 2 * (lane & 3);
  const int my0 = col0 + w * 16;  // its first dv column
  // right operands, four fragments at a time: rows 0..15 of a tile
  const uint32_t b_at =
      (uint32_t)(((lane & 7) + ((lane >> 4) << 3)) * kPitch + ((lane >> 3) & 1) * 16);
  // the warp's 16 columns of the values' tile: rows (8 + 8), columns (8 + 8)
  const uint32_t v_at =
      (uint32_t)(((lane & 7) + ((lane >> 4) << 3)) * kVPitch + w * 32 + ((lane >> 3) & 1) * 16);

  if (warp < NW) {  // ---------------------------------------------- the chain
    // rows (dv) lane / 4 and + 8, columns (dk) 8 n + 2 (lane % 4) + {0, 1}
    const bool ok0 = my0 + r < dv, ok1 = my0 + r + 8 < dv;
    float S[DKP / 8][4];
    {
      const float* in = p.state_in + bh * dk * dv + my0;
#pragma unroll
      for (int n = 0; n < DKP / 8; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int k = 8 * n + cq + (i & 1);
          const bool ok = (i < 2 ? ok0 : ok1) && k < dk && p.state_in != nullptr;
          S[n][i] = ok ? in[(int64_t)k * dv + r + 8 * (i >> 1)] : 0.f;
        }
    }
    float largest0, largest1;  // of the lane's part of both rows of S
    lane_largest(S, largest0, largest1);
    bool ok = true;
    for (int c = p.c0; c < c_end; ++c) {
      const int i_st = c - p.c0;
      const int slot = i_st % kStages;
      typename C::ChainStage& st = sm.chain[slot];
      const uint32_t before = (uint32_t)(i_st - 1) & 1u;  // (parity of the chunk before's handing over)
      ok = wait_or_leave(&sm.chain_full[slot], (uint32_t)(i_st / kStages) & 1u, &sm.gave_up) &&
           (i_st == 0 || wait_or_leave(&sm.state_free[w], before, &sm.gave_up));
      if (!__all_sync(0xffffffffu, ok)) break;
      const uint32_t k_base = smem_u32(st.k);
      float x[8][4];  // K S, transposed: columns are rows s of the chunk
      int e0 = scale_exponent(quad_max(largest0)), e1 = scale_exponent(quad_max(largest1));
      {
        const float f0 = pow2i(e0), f1 = pow2i(e1);
        by_rows<T, DKP>(x, k_base + b_at, [&](int ks, uint32_t (&hi)[4], uint32_t (&lo)[4]) {
          split_operand(hi, lo, S[2 * ks], S[2 * ks + 1], f0, f1);
          sm.state[w][ks][0][lane] = as_uint4(hi);
          sm.state[w][ks][1][lane] = as_uint4(lo);
        });
      }
      const float s0 = pow2i(-e0), s1 = pow2i(-e1);
      if ((lane & 3) == 0) {
        sm.state_inv[w][r] = s0;
        sm.state_inv[w][r + 8] = s1;
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&sm.state_full[w]);
      // R^T = V^T - (K S)^T
#pragma unroll
      for (int np = 0; np < 4; ++np) {
        float2 v[2][2];
        if constexpr (sizeof(T) == 4) {
          const float* vt = reinterpret_cast<const float*>(st.v) + w * 16 + r;
          constexpr int kW = kVPitch / 4;
#pragma unroll
          for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              const int at = (16 * np + 8 * i + cq) * kW + 8 * j;
              v[i][j] = make_float2(vt[at], vt[at + kW]);
            }
        } else {
          uint32_t raw[4];
          ldmatrix_trans(raw, smem_u32(st.v) + v_at + 16 * np * kVPitch);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const T* e = reinterpret_cast<const T*>(&raw[i]);
            v[i >> 1][i & 1] = make_float2(to_f32(e[0]), to_f32(e[1]));
          }
        }
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int n = 2 * np + i;
          const float2 fac = *reinterpret_cast<const float2*>(&st.rec.x_fac[8 * n + cq]);
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const float2 y = __ffma2_rn(pair(x[n], j), __fmul2_rn(fac, twice(j ? -s1 : -s0)), v[i][j]);
            x[n][2 * j] = y.x;
            x[n][2 * j + 1] = y.y;
          }
        }
      }
      uint32_t hi[4][4], lo[4][4];
      row_exponents(x, e0, e1);
      {
        const float f0 = pow2i(e0), f1 = pow2i(e1);
#pragma unroll
        for (int j = 0; j < 4; ++j) split_operand(hi[j], lo[j], x[2 * j], x[2 * j + 1], f0, f1);
      }
      // U^T, still scaled by T's power of two and R's
      triangular<NP == 2>(x, st.rec.t, lane, [&](int j, uint32_t (&h_)[4], uint32_t (&l_)[4]) {
#pragma unroll
        for (int i = 0; i < 4; ++i) h_[i] = hi[j][i], l_[i] = lo[j][i];
      });
      const float r0 = pow2i(-e0) * st.rec.t_inv, r1 = pow2i(-e1) * st.rec.t_inv;
      int u0, u1;
      row_exponents(x, u0, u1);
      // the state's update takes U weighted by what decays until the chunk's end
      float y[8][4];
#pragma unroll
      for (int n = 0; n < 8; ++n) {
        const float2 fac = *reinterpret_cast<const float2*>(&st.rec.u_fac[8 * n + cq]);
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const float2 v = __fmul2_rn(pair(x[n], j), fac);
          y[n][2 * j] = v.x;
          y[n][2 * j + 1] = v.y;
        }
      }
      row_exponents(y, e0, e1);
      if (i_st > 0) ok = wait_or_leave(&sm.u_free[w], before, &sm.gave_up);
      if (!__all_sync(0xffffffffu, ok)) break;
      {
        const float f0 = pow2i(e0), f1 = pow2i(e1);
#pragma unroll
        for (int j = 0; j < 4; ++j) split_operand(hi[j], lo[j], y[2 * j], y[2 * j + 1], f0, f1);
      }
      // S^T = 2^G_C S^T + (weighted U)^T K, 32 columns (4 accumulators) at a time.
      // Among the first products U itself goes to the output warp.
      const float2 carry = twice(st.rec.carry);
      const float2 d0 = twice(pow2i(-e0) * r0), d1 = twice(pow2i(-e1) * r1);
      const uint32_t kt_at =
          k_base + (uint32_t)(((lane & 7) + (((lane >> 3) & 1) << 3)) * kPitch + (lane >> 4) * 16);
      struct Columns { uint32_t f[NP][2][4]; };  // 16 rows, 32 columns of K
      auto fetch = [&](Columns& k, int s) {      // step s: columns 32 (s / 4).., rows 16 (s % 4)..
#pragma unroll
        for (int i = 0; i < NP; ++i)
#pragma unroll
          for (int m = 0; m < 2; ++m)
            ldmatrix_trans(k.f[i][m], kt_at + (s & 3) * 16 * kPitch + (4 * (s >> 2) + 2 * m) * 16 +
                                          i * kPart);
      };
      Columns kf[2];
      fetch(kf[0], 0);
      float d[4][4];
      largest0 = largest1 = 0.f;
#pragma unroll
      for (int s = 0; s < DKP / 8; ++s) {
        if (s + 1 < DKP / 8) fetch(kf[(s + 1) & 1], s + 1);
        const int j = s & 3, n0 = s & ~3;
        if (j == 0)
#pragma unroll
          for (int m = 0; m < 4; ++m)
#pragma unroll
            for (int i = 0; i < 4; ++i) d[m][i] = 0.f;
        const Columns& k = kf[s & 1];
#pragma unroll
        for (int m = 0; m < 4; ++m)
          mma_f16(d[m], hi[j], k.f[0][m >> 1][2 * (m & 1)], k.f[0][m >> 1][2 * (m & 1) + 1]);
        if (s < 4) {
          uint32_t uh[4], ul[4];
          split_operand(uh, ul, x[2 * j], x[2 * j + 1], pow2i(u0), pow2i(u1));
          sm.u[w][j][0][lane] = as_uint4(uh);
          sm.u[w][j][1][lane] = as_uint4(ul);
        }
#pragma unroll
        for (int m = 0; m < 4; ++m)
          mma_f16(d[m], lo[j], k.f[0][m >> 1][2 * (m & 1)], k.f[0][m >> 1][2 * (m & 1) + 1]);
        if constexpr (NP == 2)
#pragma unroll
          for (int m = 0; m < 4; ++m)
            mma_f16(d[m], hi[j], k.f[1][m >> 1][2 * (m & 1)], k.f[1][m >> 1][2 * (m & 1) + 1]);
        if (s == 3) {
          if ((lane & 3) == 0) {
            sm.u_inv[w][r] = pow2i(-u0) * r0;
            sm.u_inv[w][r + 8] = pow2i(-u1) * r1;
          }
          __syncwarp();
          if (lane == 0) mbar_arrive(&sm.u_full[w]);
        }
        if (j == 3) {
#pragma unroll
          for (int m = 0; m < 4; ++m) {
            float(&to)[4] = S[n0 + m];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              const float2 v =
                  __ffma2_rn(pair(d[m], i), i ? d1 : d0, __fmul2_rn(carry, pair(to, i)));
              to[2 * i] = v.x;
              to[2 * i + 1] = v.y;
            }
            largest0 = max3(largest0, fabsf(to[0]), fabsf(to[1]));
            largest1 = max3(largest1, fabsf(to[2]), fabsf(to[3]));
          }
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&sm.chain_empty[slot]);
    }
    if (!__all_sync(0xffffffffu, ok)) return;
    if (p.state_out != nullptr) {
      float* to = p.state_out + bh * dk * dv + my0;
#pragma unroll
      for (int n = 0; n < DKP / 8; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int k = 8 * n + cq + (i & 1);
          if ((i < 2 ? ok0 : ok1) && k < dk) to[(int64_t)k * dv + r + 8 * (i >> 1)] = S[n][i];
        }
    }
    return;
  }

  // ------------------------------------------------------------- the outputs
  T* out = static_cast<T*>(a.out) + ((int64_t)b * L * H + h) * dv + my0;
  const int my_cols = min(16, dv - my0);
  bool ok = true;
  for (int c = p.c0; c < c_end; ++c) {
    const int i_st = c - p.c0;
    const uint32_t now = (uint32_t)i_st & 1u;
    typename C::OutStage& st = sm.out[i_st & 1];
    ok = wait_or_leave(&sm.out_full[i_st & 1], (uint32_t)(i_st >> 1) & 1u, &sm.gave_up) &&
         wait_or_leave(&sm.state_full[w], now, &sm.gave_up);
    if (!__all_sync(0xffffffffu, ok)) break;
    const uint32_t q_base = smem_u32(st.q);
    float o[8][4];  // Q S, transposed: columns are rows t of the chunk
    by_rows<T, DKP>(o, q_base + b_at, [&](int ks, uint32_t (&hi)[4], uint32_t (&lo)[4]) {
      const uint4 h_ = sm.state[w][ks][0][lane], l_ = sm.state[w][ks][1][lane];
      hi[0] = h_.x, hi[1] = h_.y, hi[2] = h_.z, hi[3] = h_.w;
      lo[0] = l_.x, lo[1] = l_.y, lo[2] = l_.z, lo[3] = l_.w;
    });
    const float s0 = sm.state_inv[w][r], s1 = sm.state_inv[w][r + 8];
    __syncwarp();
    if (lane == 0) mbar_arrive(&sm.state_free[w]);
    // scale 2^G_t Q S
#pragma unroll
    for (int n = 0; n < 8; ++n) {
      const float2 fac = *reinterpret_cast<const float2*>(&st.rec.o_fac[8 * n + cq]);
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const float2 y = __fmul2_rn(pair(o[n], j), __fmul2_rn(fac, twice(j ? s1 : s0)));
        o[n][2 * j] = y.x;
        o[n][2 * j + 1] = y.y;
      }
    }
    ok = wait_or_leave(&sm.u_full[w], now, &sm.gave_up);
    if (!__all_sync(0xffffffffu, ok)) break;
    {
      float d[8][4];
      triangular<NP == 2>(d, st.rec.p, lane, [&](int j, uint32_t (&hi)[4], uint32_t (&lo)[4]) {
        const uint4 h_ = sm.u[w][j][0][lane], l_ = sm.u[w][j][1][lane];
        hi[0] = h_.x, hi[1] = h_.y, hi[2] = h_.z, hi[3] = h_.w;
        lo[0] = l_.x, lo[1] = l_.y, lo[2] = l_.z, lo[3] = l_.w;
      });
      const float p0 = sm.u_inv[w][r] * st.rec.p_inv, p1 = sm.u_inv[w][r + 8] * st.rec.p_inv;
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(&sm.u_free[w]);
        mbar_arrive(&sm.out_empty[i_st & 1]);
      }
#pragma unroll
      for (int n = 0; n < 8; ++n)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const float2 y = __ffma2_rn(pair(d[n], j), twice(j ? p1 : p0), pair(o[n], j));
          o[n][2 * j] = y.x;
          o[n][2 * j + 1] = y.y;
        }
    }
    // outputs, through this warp's columns of a tile of theirs
    const int t0 = c * kChunk, len = min(kChunk, len_all - t0), rows = min(kChunk, L - t0);
    if constexpr (sizeof(T) == 4) {
      float* vt = reinterpret_cast<float*>(sm.o) + w * 16 + r;
      constexpr int kW = kVPitch / 4;
#pragma unroll
      for (int n = 0; n < 8; ++n)
#pragma unroll
        for (int j = 0; j < 4; ++j) vt[(8 * n + cq + (j & 1)) * kW + 8 * (j >> 1)] = o[n][j];
    } else {
#pragma unroll
      for (int np = 0; np < 4; ++np) {
        uint32_t e[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const T two[2] = {from_f32<T>(o[2 * np + (i >> 1)][2 * (i & 1)]),
                            from_f32<T>(o[2 * np + (i >> 1)][2 * (i & 1) + 1])};
          e[i] = *reinterpret_cast<const uint32_t*>(two);
        }
        stmatrix_trans(smem_u32(sm.o) + v_at + 16 * np * kVPitch, e[0], e[1], e[2], e[3]);
      }
    }
    __syncwarp();
    constexpr int kPieces = 16 * (int)sizeof(T) / 16, kPieceElems = 16 / (int)sizeof(T);
    if (p.out_vec && my_cols == 16) {
#pragma unroll
      for (int i = lane; i < kChunk * kPieces; i += 32) {
        const int t = i / kPieces, at = i % kPieces;
        uint4 e = *reinterpret_cast<const uint4*>(sm.o + t * kVPitch + w * 16 * (int)sizeof(T) +
                                                  at * 16);
        if (t >= len) e = make_uint4(0, 0, 0, 0);
        if (t < rows)
          *reinterpret_cast<uint4*>(out + (int64_t)(t0 + t) * H * dv + at * kPieceElems) = e;
      }
    } else {
      for (int i = lane; i < rows * 16; i += 32) {
        const int t = i >> 4, e = i & 15;
        if (e < my_cols)
          out[(int64_t)(t0 + t) * H * dv + e] =
              t < len ? *reinterpret_cast<const T*>(sm.o + t * kVPitch +
                                                    (w * 16 + e) * (int)sizeof(T))
                      : from_f32<T>(0.f);
      }
    }
    __syncwarp();
  }
  if (!__all_sync(0xffffffffu, ok)) return;
  // rows of chunks past the length
  const int from = max(c_end, p.c0) * kChunk, to = min(p.c1 * kChunk, L);
  for (int64_t i = lane; i < (int64_t)max(to - from, 0) * 16; i += 32) {
    const int e = (int)(i & 15);
    if (e < my_cols) out[(from + (i >> 4)) * H * dv + e] = from_f32<T>(0.f);
  }
}

// -------------------------------------------------------------------- host

namespace {

// A long prompt goes through in several launches of both kernels, the states
// between them in the workspace, the records in two buffers in turn: the
// records of the next chunks are made on the SMs that the chain leaves idle.
// A buffer stays within kRecordBytes, or holds one chunk of every sequence and head
// where that is more (10240 chunks of 128 x 128 at once or in two launches take 530 us,
// in three 6% more, in four, whose records the L2 cache could hold, 15%); where it is
// not that which cuts, there are 3 launches (float32: 8) of at least kFewChunks chunks,
// against the 15 us that a launch and its states cost: 16384 tokens of 16 heads take
// 808 us with 3, 3% more with 8 (bf16, 128 x 128), 1085 and 938 (float32, 64 x 64).
constexpr int64_t kRecordBytes = (int64_t)190 << 20, kFewChunks = 24;

struct Plan {
  int64_t chunks, per_launch;
  size_t record_bytes, state_bytes;  // of a buffer; of the states
  bool several() const { return chunks > per_launch; }
};

Plan make_plan(int64_t batch, int64_t seqlen, int64_t heads, int64_t dk, int64_t dv,
               int32_t dtype) {
  Plan pl;
  pl.chunks = (seqlen + kChunk - 1) / kChunk;
  // (16-bit types may take either kind, by their alignment: the larger one's size)
  const int64_t record = dtype == MAMBA_DTYPE_F32 ? (int64_t)sizeof(Record)
      : (int64_t)std::max(sizeof(Record), sizeof(TileRecord));
  const int64_t each = batch * heads * record;
  const int64_t at_most = dtype == MAMBA_DTYPE_F32 ? 8 : 3;
  // (a grid's CTAs count in 31 bits)
  const int64_t most = std::max<int64_t>(
      1, std::min(kRecordBytes / each, (((int64_t)1 << 31) - 1) / (batch * heads)));
  const int64_t launches =
      std::max((pl.chunks + most - 1) / most, std::min(at_most, pl.chunks / kFewChunks));
  pl.per_launch = launches > 1 ? (pl.chunks + launches - 1) / launches : pl.chunks;
  pl.record_bytes = (size_t)(each * pl.per_launch);
  pl.state_bytes = pl.several() ? (size_t)(batch * heads * dk * dv * 4) : 0;
  return pl;
}

template <typename K>
cudaError_t allow_smem(K kernel, size_t bytes) {
  return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
}

template <typename T, int DKP, int NW>
cudaError_t launch_chain(const Params& p0, cudaStream_t st) {
  using C = ChainCfg<T, DKP, NW>;
  Params p = p0;
  p.tiles = (int)((p.a.dv + C::kDv - 1) / C::kDv);
  auto kernel = chain_kernel<T, C>;
  cudaError_t e = allow_smem(kernel, sizeof(typename C::Smem));
  if (e != cudaSuccess) return e;
  if constexpr (NW == 4) {
    // (warps that ask for more registers than the launch has would wait for good)
    cudaFuncAttributes attr;
    e = cudaFuncGetAttributes(&attr, kernel);
    if (e != cudaSuccess) return e;
    if (attr.numRegs < kLaunchRegisters) return cudaErrorLaunchOutOfResources;
  }
  return mamba_scan::launch_pdl(kernel, dim3((unsigned)(p.a.batch * p.a.heads * p.tiles)),
                                dim3(C::kThreads), sizeof(typename C::Smem), st, p);
}

template <typename T, int DKP, typename R>
cudaError_t launch_prepare(const Params& p, cudaStream_t st) {
  auto kernel = prepare_kernel<T, DKP, R>;
  cudaError_t e = allow_smem(kernel, sizeof(PrepareSmem<T, DKP, R>));
  if (e != cudaSuccess) return e;
  // (as many CTAs on an SM as shared memory holds)
  e = cudaFuncSetAttribute(kernel, cudaFuncAttributePreferredSharedMemoryCarveout,
                           cudaSharedmemCarveoutMaxShared);
  if (e != cudaSuccess) return e;
  return mamba_scan::launch_pdl(kernel,
                                dim3((unsigned)(p.a.batch * p.a.heads * (p.c1 - p.c0))), dim3(128),
                                sizeof(PrepareSmem<T, DKP, R>), st, p);
}

template <typename T, int DKP>
cudaError_t launch_slab(const Params& p, const TileMaps* maps, cudaStream_t st) {
  cudaError_t e;
  if constexpr (sizeof(T) == 2) {
    if (maps != nullptr) {
      e = launch_prepare<T, DKP, TileRecord>(p, st);
      return e != cudaSuccess ? e : launch_tiles(*maps, p, st);
    }
  }
  e = launch_prepare<T, DKP, Record>(p, st);
  if (e != cudaSuccess) return e;
  // Tiles of 64 columns, or of 32 where that many CTAs have an SM each (then no
  // two of a CTA's chain and output warps share a scheduler; 1024 tokens of 24 heads
  // of 64 x 64 in float32 88 us, with 64 columns 94; of 192 heads 293 and 258) and
  // for float32 with dk over 64, where no more fit.
  if constexpr (DKP == 128 && sizeof(T) == 4) return launch_chain<T, DKP, 2>(p, st);
  else if (p.a.batch * p.a.heads * ((p.a.dv + 31) / 32) <= mamba_lm::sm_count())
    return launch_chain<T, DKP, 2>(p, st);
  else
    return launch_chain<T, DKP, 4>(p, st);
}

template <typename T>
cudaError_t launch_typed(const mamba_gated_delta_args& a, void* workspace, cudaStream_t st) {
  const Plan pl = make_plan(a.batch, a.seqlen, a.heads, a.dk, a.dv, a.dtype);
  const int64_t per16 = 16 / (int64_t)sizeof(T);
  auto rows16 = [&](const void* base, const int64_t* stride) {
    return mamba_lm::aligned16(base) && stride[0] % per16 == 0 && stride[1] % per16 == 0 &&
           stride[2] % per16 == 0;
  };
  Params p = {};
  p.a = a;
  uint8_t* behind = static_cast<uint8_t*>(workspace) + pl.record_bytes;
  void* buffers[2] = {workspace, behind};
  float* states = reinterpret_cast<float*>(behind + pl.record_bytes);  // (in several launches)
  p.qk_vec = rows16(a.q, a.q_stride) && rows16(a.k, a.k_stride);
  p.v_vec = rows16(a.v, a.v_stride);
  p.out_vec = mamba_lm::aligned16(a.out) && a.dv % per16 == 0;
  TileMaps maps;
  const TileMaps* tiles = tiles_take(a, &maps) ? &maps : nullptr;
  for (int64_t c = 0; c < pl.chunks; c += pl.per_launch) {
    p.records = buffers[c / pl.per_launch & 1];
    p.c0 = (int)c;
    p.c1 = (int)std::min(pl.chunks, c + pl.per_launch);
    p.state_in = c == 0 ? a.h0 : states;
    p.state_out = p.c1 == pl.chunks ? a.h_last : states;
    const cudaError_t e = a.dk <= 64 ? launch_slab<T, 64>(p, tiles, st)
                                     : launch_slab<T, 128>(p, tiles, st);
    if (e != cudaSuccess) return e;
  }
  return cudaSuccess;
}

}  // namespace

// (shorter prompts take no longer token by token, see recurrent_kernel)
bool mma_takes(int64_t seqlen, int64_t dk, int64_t dv, int32_t dtype) {
  return seqlen > (dtype == MAMBA_DTYPE_F32 ? 48 : 16) && dk <= 128 && dv > 0;
}

size_t mma_workspace_size(int64_t batch, int64_t seqlen, int64_t heads, int64_t dk, int64_t dv,
                          int32_t dtype) {
  const Plan pl = make_plan(batch, seqlen, heads, dk, dv, dtype);
  return pl.several() ? 2 * pl.record_bytes + pl.state_bytes : pl.record_bytes;
}

cudaError_t launch_mma(const mamba_gated_delta_args& a, void* workspace, cudaStream_t st) {
  switch (a.dtype) {
    case MAMBA_DTYPE_F32: return launch_typed<float>(a, workspace, st);
    case MAMBA_DTYPE_F16: return launch_typed<__half>(a, workspace, st);
    default: return launch_typed<__nv_bfloat16>(a, workspace, st);
  }
}

int read_and_clear_error() {
  const int tiles = read_and_clear_tiles_error();
  if (tiles != 0) return tiles;
  int v = 0;
  if (cudaMemcpyFromSymbol(&v, g_error, sizeof(int)) != cudaSuccess) return -1;
  if (v != 0) {
    const int zero = 0;
    cudaMemcpyToSymbol(g_error, &zero, sizeof(int));
  }
  return v;
}

}  // namespace mamba_gd
