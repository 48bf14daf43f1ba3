// A language model's loss from its last hidden states, the logits never
// stored, and its gradients (include/mamba_lm_ops.h): what follows the head of
// the models around the scan op (which the reference leaves to the caller,
// benchmarks/profiler.py:18-150) in training and scoring.
//
// Mathematics. z = H W^T (rows x vocab), m_r = max_v z, s_r = sum_v e^(z - m):
//   loss_r = (m_r - z_rt) + log s_r,
//   dz = g_r (e^(z - m) / s - 1_t),  dH = dz W,  dW = dz^T H.
// Four matrix products, three for the gradients, since z is formed again
// rather than kept. All of them run in one tensor-core kernel (tile_kernel)
// that differs in what happens to a finished tile: kStats folds it into (m, s)
// of its rows, a thread per row, kGrad turns it into dz, rounded to the
// operands' 16-bit type, kOut writes or adds it. dz is made and used a piece
// of the vocabulary at a time, so that it stays in the L2 cache.
//
// tile_kernel: a CTA pair computes 256 x 256 tiles (tcgen05.mma.cta_group::2,
// 16-bit operands, fp32 accumulators in tensor memory), tile after tile
// (persistent), a tile's products beside the one before's epilogue on two
// accumulators of 256 columns. Per 64-wide K block a CTA fetches 128 rows of A
// and half of B by TMA, 32 KB, while the tensor cores take 512 clocks, so the
// tile is near both their rate and what an SM fetches from L2.
//
// Sums. The tensor cores cut every sum that goes back to an accumulator off
// towards zero: over 768 columns that put 1.3e-6 of their norm into the losses,
// four times what fp32 additions to nearest do, and three times that with the
// three products of float32. So the accumulators hold a segment of K only, and
// the epilogue's threads add the segments up in their registers: 128 columns
// where fp32 results come of it (the losses), 64 in float32, whose small products
// come first in a segment. 16-bit gradients are rounded to 8 or 11 bits anyway, but
// what is cut grows with K, the number of rows for d_weight (in one accumulation
// 2.2e-4 of it for 33000 rows of one sign, 8.6e-4 for 131072), so theirs are
// segments of 512.
//
// Up to 16 rows go through linear_cross_entropy_few.cu.
//
// Numbers. bf16 and fp16 operands are exact. float32 ones are scaled by a
// power of two (largest finite element to 2^14..2^15) and split into two fp16
// parts (hi hi + hi lo + lo hi: 22 bits, at half the cost of the tensor cores'
// TF32 form); the parts' smallest step is 2^-24, 2^-38 of the largest element.
// Measured. 4096 x 50280 x 768 in bf16: losses 242 us (1.31 PFLOP/s, 0.80 of what
// cuBLAS was measured at), with both gradients 1231 (four products, 1.03 PFLOP/s):
// the statistics' exponentials and segments, then, per piece of 96 MB, three
// launches. 1024 rows in float32: losses 281 us, of which 28 and 44 find the weights'
// power of two and split them (5.5 TB/s) and 165 are products (1.44 PFLOP/s of fp16),
// with gradients 1010. 33 rows of fp16: 30, 3 rounds of tiles for 77 MB of weights.
//
// One power for a matrix, not one for each row: rows of W and H are also what
// the gradients' products add over, where rows' own powers would have to be
// put into dz. dz itself is relative to the largest |gradient|, so at most 1,
// and goes into fp16 parts times 2^14.
#include <cudaTypedefs.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <cstring>
#include <mutex>
#include <string>
#include <type_traits>

#include "../../include/mamba_lm_ops.h"
#include "linear_cross_entropy.h"
#include "lm_device.cuh"
#include "scan_device.cuh"
#include "scan_kernels.h"

namespace mamba_lce {

using mamba_lm::from_f32;
using mamba_lm::to_f32;
using mamba_scan::smem_u32;

constexpr int kTile = 256;         // rows and columns of a pair's tile
constexpr int kHalf = 128;         // a CTA's rows of A and of B
constexpr int kBK = 64;            // K of a stage: 128 bytes, one swizzled row
constexpr int kOperand = kHalf * kBK * 2;  // bytes of a CTA's A or B part of a stage
constexpr int kSlab = 64 * 128;    // MN-major: 64 K rows of 64 columns
constexpr int kBox = 32 * 128;     // a warp's box of a tile on its way out

__device__ int g_error = 0;

enum Mode { kStats = 0, kGrad = 1, kOut = 2 };

constexpr int kWarps = 8;          // of the epilogue: two for each 32 rows
constexpr int kCols = kTile / 2;   // columns of an epilogue warp
constexpr int kThreads = 32 * (kWarps + 2);  // and one that loads, one that multiplies
constexpr int kLoadWarp = kWarps, kMmaWarp = kWarps + 1;

template <int PARTS> struct Cfg {
  static constexpr int kStages = PARTS == 1 ? 5 : 3;
  static constexpr int kBoxes = PARTS == 1 ? 2 : 1;   // of an epilogue warp
  static constexpr int kStageBytes = 2 * PARTS * kOperand;
  struct __align__(1024) Smem {
    uint8_t stage[kStages][kStageBytes];  // A parts, then B parts
    uint8_t box[kWarps][kBoxes][kBox];
    uint64_t full[kStages];   // leader: both CTAs' parts have landed
    uint64_t empty[kStages];  // each CTA: the pair's products have read the stage
    uint64_t acc_full[2];     // each CTA: a segment is in accumulator b
    uint64_t acc_empty[2];    // leader: both CTAs have read accumulator b
    uint32_t tmem;
  };
  static constexpr size_t kSmemBytes = sizeof(Smem) + 1024;
  static_assert(kSmemBytes <= 227 * 1024, "shared memory per CTA");
};

struct Maps {
  CUtensorMap a[2], b[2], out[2];
};

struct TileParams {
  int m_tiles, n_tiles, splits;
  int kblocks;               // of a unit of work: a tile, or a split's share of it
  int total_kblocks;
  int a_k0, b_k0, b_mn0;     // where K starts in A and B, where the tiles start in B
  uint32_t idesc;
  // kStats and kGrad
  int rows, vocab, v0;       // v0: the vocabulary's column of the first tile
  const int64_t* target;
  const uint32_t* a_max;     // float32: bits of the operands' largest elements
  const uint32_t* b_max;
  float2* partial;           // kStats: [half n tile][rows]
  float* target_logit;       // kStats: [rows]
  const float2* stats;       // kGrad
  const float* rel_grad;     // kGrad: grad / largest |grad|, 0 where nothing counts
  // kOut
  int accumulate;            // add to what is there
  int out_rows, out_cols;
  int split_rows;            // rows between the splits' outputs
  int scaled;                // a finished output: times the largest |grad|
  const float* largest;      // the largest |grad|
  void* out;                 // where TMA cannot write
  int64_t out_stride;
};

// ------------------------------------------------------------ PTX wrappers

__device__ __forceinline__ void tc_fence_before() {
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
}
__device__ __forceinline__ void tc_fence_after() {
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
}

__device__ __forceinline__ uint32_t cluster_ctarank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ uint32_t map_to_rank(const void* p, uint32_t rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(smem_u32(p)), "r"(rank));
  return r;
}
__device__ __forceinline__ void cluster_sync_all() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;"
               ::: "memory");
}

// A 2-D TMA load into this CTA, completing on the barrier at shared::cluster
// address `bar` (the pair's leader).
__device__ __forceinline__ void tma_load(uint32_t dst, const CUtensorMap* map, uint32_t bar, int c0,
                                         int c1) {
  asm volatile(
      "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%3, %4}], [%2];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(c0), "r"(c1)
      : "memory");
}
__device__ __forceinline__ void tma_store(const CUtensorMap* map, uint32_t src, int c0, int c1) {
  asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%2, %3}], [%1];" ::"l"(
                   reinterpret_cast<uint64_t>(map)),
               "r"(src), "r"(c0), "r"(c1)
               : "memory");
}
__device__ __forceinline__ void tma_add(const CUtensorMap* map, uint32_t src, int c0, int c1) {
  asm volatile(
      "cp.reduce.async.bulk.tensor.2d.global.shared::cta.add.bulk_group [%0, {%2, %3}], [%1];" ::"l"(
          reinterpret_cast<uint64_t>(map)),
      "r"(src), "r"(c0), "r"(c1)
      : "memory");
}

// Matrix descriptors of tiles in the 128-byte swizzle, as the low word (start
// address >> 4, leading byte offset >> 4 from bit 16) and the high one (stride
// byte offset >> 4, version 1, layout 2). K-major: rows of M or N, groups of 8
// 1024 bytes apart. MN-major: rows of K, the next 64 columns one slab further.
constexpr uint32_t kDescHigh = (1024u >> 4) | (1u << 14) | (2u << 29);
__device__ __forceinline__ uint32_t desc(uint32_t addr, bool mn) {
  return (addr >> 4) | ((mn ? (uint32_t)(kSlab >> 4) : 1u) << 16);
}

__device__ __forceinline__ uint32_t elect_one() {
  uint32_t leader;
  asm volatile(
      "{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}\n"
      : "=r"(leader));
  return leader;
}

__device__ __forceinline__ void mma_pair(uint32_t leader, uint32_t d, uint32_t a, uint32_t b,
                                         uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t.reg .b64 da, db;\n\t"
      "setp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %6, 0;\n\t"
      "mov.b64 da, {%1, %5};\n\tmov.b64 db, {%2, %5};\n\t"
      "@q tcgen05.mma.cta_group::2.kind::f16 [%0], da, db, %3, p;\n\t}\n" ::"r"(d),
      "r"(a), "r"(b), "r"(idesc), "r"(accumulate), "r"(kDescHigh), "r"(leader)
      : "memory");
}
// One arrival on the barrier of either CTA once the products so far are done.
__device__ __forceinline__ void commit_pair(uint32_t leader, uint64_t* bar) {
  asm volatile(
      "{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %2, 0;\n\t"
      "@q tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64"
      " [%0], %1;\n\t}\n" ::"r"(smem_u32(bar)),
      "h"((uint16_t)0x3), "r"(leader)
      : "memory");
}
__device__ __forceinline__ void arrive_cluster(uint32_t bar) {
  asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}

__device__ __forceinline__ void tmem_ld32(uint32_t addr, float (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, "
      "%11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, "
      "%28, %29, %30, %31}, [%32];"
      : "=f"(r[0]), "=f"(r[1]), "=f"(r[2]), "=f"(r[3]), "=f"(r[4]), "=f"(r[5]), "=f"(r[6]),
        "=f"(r[7]), "=f"(r[8]), "=f"(r[9]), "=f"(r[10]), "=f"(r[11]), "=f"(r[12]), "=f"(r[13]),
        "=f"(r[14]), "=f"(r[15]), "=f"(r[16]), "=f"(r[17]), "=f"(r[18]), "=f"(r[19]),
        "=f"(r[20]), "=f"(r[21]), "=f"(r[22]), "=f"(r[23]), "=f"(r[24]), "=f"(r[25]),
        "=f"(r[26]), "=f"(r[27]), "=f"(r[28]), "=f"(r[29]), "=f"(r[30]), "=f"(r[31])
      : "r"(addr));
}
__device__ __forceinline__ void tmem_wait() {
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
}

// ------------------------------------------------------------- small pieces

__device__ __forceinline__ float pow2i(int e) { return __int_as_float((e + 127) << 23); }

// The exponent that brings a matrix's largest element (its bits) to 2^14..2^15.
__device__ __forceinline__ int scale_exponent(uint32_t largest) {
  return largest == 0 ? 0 : min(141 - (int)(largest >> 23), 126);
}
// What undoes it.
__device__ __forceinline__ float undo_scale(const uint32_t* largest) {
  return pow2i(-scale_exponent(*largest));
}

template <typename T> __device__ __forceinline__ uint32_t pack2(float a, float b) {
  T e[2] = {from_f32<T>(a), from_f32<T>(b)};
  return *reinterpret_cast<const uint32_t*>(e);
}

// What dz carries in fp16.
template <typename T16>
__device__ __forceinline__ float dz_scale() {
  return std::is_same<T16, __half>::value ? 16384.f : 1.f;
}

// ------------------------------------------------------------ the epilogues
//
// An epilogue takes a thread's row of a tile, 32 of its warp's 128 columns at a
// time: begin() before the first, chunk(c, v) for columns c.., end().

// One warp's boxes of 32 rows x 128 bytes, in the 128-byte swizzle, out by TMA.
template <int kBoxes> struct BoxWriter {
  uint8_t* box;
  int lane;
  int next = 0;   // the box to fill

  // before the first piece of a box: its last store has read it
  __device__ __forceinline__ void open() const {
    if (lane == 0) mamba_scan::bulk_wait_read<kBoxes - 1>();
    __syncwarp();
  }
  __device__ __forceinline__ void put(int piece, uint4 w) const {
    *reinterpret_cast<uint4*>(box + next * kBox + lane * 128 + ((piece ^ (lane & 7)) << 4)) = w;
  }
  // the same of two boxes of 32 rows x 64 bytes, in the 64-byte swizzle
  __device__ __forceinline__ void put_half(int which, int piece, uint4 w) const {
    *reinterpret_cast<uint4*>(box + next * kBox + which * (kBox / 2) + lane * 64 +
                              ((piece ^ ((lane >> 1) & 3)) << 4)) = w;
  }
  __device__ __forceinline__ void close_halves(const CUtensorMap (&map)[2], int x, int y) {
    mamba_scan::fence_proxy_async_smem();
    __syncwarp();
    if (lane == 0) {
      const uint32_t src = smem_u32(box + next * kBox);
      tma_store(&map[0], src, x, y);
      tma_store(&map[1], src + kBox / 2, x, y);
      mamba_scan::bulk_commit();
    }
    if constexpr (kBoxes == 2) next ^= 1;
  }
  __device__ __forceinline__ void close(const CUtensorMap* map, int x, int y, bool add, bool there) {
    mamba_scan::fence_proxy_async_smem();
    __syncwarp();
    if (lane == 0) {
      const uint32_t src = smem_u32(box + next * kBox);
      if (there) {
        if (add) tma_add(map, src, x, y);
        else tma_store(map, src, x, y);
      }
      mamba_scan::bulk_commit();
    }
    if constexpr (kBoxes == 2) next ^= 1;
  }
};

// A row's running maximum and sum over its warp's columns of a tile of logits.
template <int PARTS> struct StatsEpilogue {
  const TileParams& p;
  int col0, valid, at, row, part;
  bool row_ok;
  float ia, ib, m, s0, s1, zt;

  __device__ __forceinline__ void begin(int n_tile, int half, int row_) {
    row = row_;
    part = 2 * n_tile + half;
    col0 = part * kCols;  // (p.v0 is 0)
    valid = p.vocab - col0;
    row_ok = row < p.rows;
    ia = ib = 1.f;
    if constexpr (PARTS == 2) ia = undo_scale(p.a_max), ib = undo_scale(p.b_max);
    const int64_t t = row_ok ? p.target[row] : -1;
    at = t >= col0 && t < p.vocab ? (int)min(t - col0, (int64_t)kCols) : kCols;
    m = -INFINITY, s0 = s1 = zt = 0.f;
  }
  __device__ __forceinline__ void chunk(int c, float (&v)[32]) {
    if constexpr (PARTS == 2)
#pragma unroll
      for (int j = 0; j < 32; ++j) v[j] = v[j] * ia * ib;
    if (c + 32 > valid) {
#pragma unroll
      for (int j = 0; j < 32; ++j)
        if (c + j >= valid) v[j] = -INFINITY;
    }
    if ((unsigned)(at - c) < 32u) {
#pragma unroll
      for (int j = 0; j < 32; ++j)
        if (c + j == at) zt = v[j];
    }
    float mx[4] = {v[0], v[1], v[2], v[3]};
#pragma unroll
    for (int j = 4; j < 32; ++j) mx[j & 3] = fmaxf(mx[j & 3], v[j]);
    const float top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
    if (top > m) {
      const float f = mamba_scan::ex2_approx((m - top) * kLog2e);
      s0 *= f;
      s1 *= f;
      m = top;
    }
    // ((v - m) rounds less than v log2(e) - m log2(e) where m is large)
    const float from = finite_max(m);
#pragma unroll
    for (int j = 0; j < 32; j += 2) {
      s0 += mamba_scan::ex2_approx((v[j] - from) * kLog2e);
      s1 += mamba_scan::ex2_approx((v[j + 1] - from) * kLog2e);
    }
  }
  __device__ __forceinline__ void end() {
    if (!row_ok) return;
    p.partial[(int64_t)part * p.rows + row] = make_float2(m, s0 + s1);
    if (at < kCols) p.target_logit[row] = zt;
  }
};

// dz of a tile, in the operands' type.
template <int PARTS, typename T16> struct GradEpilogue {
  const TileParams& p;
  const Maps& maps;
  BoxWriter<Cfg<PARTS>::kBoxes>& out;
  int local0, valid, at, row0;
  bool counts;
  float ia, ib, m, minus, f, spoil;

  __device__ __forceinline__ void begin(int n_tile, int half, int row, int row0_) {
    row0 = row0_;
    local0 = n_tile * kTile + half * kCols;
    const int col0 = p.v0 + local0;
    valid = p.vocab - col0;
    const bool row_ok = row < p.rows;
    const int64_t t = row_ok ? p.target[row] : -1;
    counts = row_ok && t >= 0;
    at = t >= col0 && t < p.vocab ? (int)min(t - col0, (int64_t)kCols) : kCols;
    ia = ib = 1.f;
    if constexpr (PARTS == 2) ia = undo_scale(p.a_max), ib = undo_scale(p.b_max);
    const float2 st = counts ? p.stats[row] : make_float2(0.f, 1.f);
    m = st.x;
    minus = (counts ? p.rel_grad[row] : 0.f) * dz_scale<T16>();
    f = minus / st.y;
    // (a target past the vocabulary has no gradient to give: NaN)
    spoil = counts && t >= p.vocab ? __int_as_float(0x7fc00000) : 0.f;
  }
  __device__ __forceinline__ void chunk(int c, float (&v)[32]) {
#pragma unroll
    for (int j = 0; j < 32; ++j) {
      float z = v[j];
      if constexpr (PARTS == 2) z = z * ia * ib;
      v[j] = fmaf(mamba_scan::ex2_approx((z - m) * kLog2e), f, spoil);
    }
    if ((unsigned)(at - c) < 32u) {
#pragma unroll
      for (int j = 0; j < 32; ++j)
        if (c + j == at) v[j] -= minus;
    }
    if (!counts || c + 32 > valid) {
#pragma unroll
      for (int j = 0; j < 32; ++j)
        if (!counts || c + j >= valid) v[j] = 0.f;
    }
    // a box is 64 columns, two chunks, or 32 of hi and 32 of lo
    if constexpr (PARTS == 2) {
      out.open();
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        uint32_t hi[4], lo[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float x = v[8 * q + 2 * i], y = v[8 * q + 2 * i + 1];
          hi[i] = pack2<T16>(x, y);
          const float2 h = __half22float2(*reinterpret_cast<const __half2*>(&hi[i]));
          lo[i] = pack2<T16>(x - h.x, y - h.y);
        }
        out.put_half(0, q, make_uint4(hi[0], hi[1], hi[2], hi[3]));
        out.put_half(1, q, make_uint4(lo[0], lo[1], lo[2], lo[3]));
      }
      out.close_halves(maps.out, local0 + c, row0);
    } else {
      const int first = (c >> 5 & 1) * 4;
      if (first == 0) out.open();
#pragma unroll
      for (int q = 0; q < 4; ++q)
        out.put(first + q, make_uint4(pack2<T16>(v[8 * q], v[8 * q + 1]),
                                      pack2<T16>(v[8 * q + 2], v[8 * q + 3]),
                                      pack2<T16>(v[8 * q + 4], v[8 * q + 5]),
                                      pack2<T16>(v[8 * q + 6], v[8 * q + 7])));
      if (first == 4) out.close(&maps.out[0], local0 + c - 32, row0, false, true);
    }
  }
  __device__ __forceinline__ void end() {}
};

// A tile of an output: fp32 sums of one split (added to those of earlier
// pieces), or a finished one of type TO, scaled.
template <int PARTS, typename T16, typename TO> struct OutEpilogue {
  static constexpr int kPer = 128 / (int)sizeof(TO);  // columns of a box
  const TileParams& p;
  const Maps& maps;
  BoxWriter<Cfg<PARTS>::kBoxes>& out;
  int col0, row, row0, y;
  float f;

  __device__ __forceinline__ void begin(int n_tile, int half, int split, int row_, int row0_) {
    col0 = n_tile * kTile + half * kCols;
    row = row_;
    row0 = row0_;
    y = split * p.split_rows + row0;
    f = 1.f;
    if (p.scaled) {
      f = *p.largest / dz_scale<T16>();
      if constexpr (PARTS == 2) f *= undo_scale(p.b_max);
    }
  }
  __device__ __forceinline__ void chunk(int c, float (&v)[32]) {
    if (col0 + c >= p.out_cols) return;
#pragma unroll
    for (int j = 0; j < 32; ++j) v[j] *= f;
    if (p.out != nullptr) {  // rows that TMA cannot write
      if (row < p.out_rows) {
        TO* to = static_cast<TO*>(p.out) + (int64_t)row * p.out_stride + col0 + c;
#pragma unroll
        for (int j = 0; j < 32; ++j)
          if (col0 + c + j < p.out_cols) to[j] = from_f32<TO>(v[j]);
      }
      return;
    }
    const int in_box = c % kPer;
    if (in_box == 0) out.open();
    if constexpr (sizeof(TO) == 4) {
#pragma unroll
      for (int q = 0; q < 8; ++q)
        out.put(q, make_uint4(__float_as_uint(v[4 * q]), __float_as_uint(v[4 * q + 1]),
                              __float_as_uint(v[4 * q + 2]), __float_as_uint(v[4 * q + 3])));
    } else {
#pragma unroll
      for (int q = 0; q < 4; ++q)
        out.put(in_box / 8 + q,
                make_uint4(pack2<TO>(v[8 * q], v[8 * q + 1]), pack2<TO>(v[8 * q + 2], v[8 * q + 3]),
                           pack2<TO>(v[8 * q + 4], v[8 * q + 5]),
                           pack2<TO>(v[8 * q + 6], v[8 * q + 7])));
    }
    // (the last piece of the columns there are may leave its box half old:
    // TMA does not write past the last column)
    if (in_box + 32 == kPer || col0 + c + 32 >= p.out_cols)
      out.close(&maps.out[0], col0 + c - in_box, y, p.accumulate, row0 < p.out_rows);
  }
  __device__ __forceinline__ void end() {}
};

// ------------------------------------------------------------------ kernel

template <int MODE, int PARTS, typename T16, typename TO, bool A_MN, bool B_MN>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads, 1)
    tile_kernel(const __grid_constant__ Maps maps, const TileParams p) {
  using C = Cfg<PARTS>;
  constexpr int kStages = C::kStages;
  // K blocks of an accumulation (the comment at the top)
  constexpr int kSegment = PARTS == 2 ? 1 : MODE == kStats ? 2 : 8;
  extern __shared__ uint8_t smem_raw[];
  typename C::Smem& sm = *reinterpret_cast<typename C::Smem*>(
      smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u));
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_ctarank();
  const int n_pairs = (int)gridDim.x / 2, pair = (int)blockIdx.x / 2;
  const int tiles = p.m_tiles * p.n_tiles, units = tiles * p.splits;

  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages; ++s) {
      mamba_scan::mbar_init(&sm.full[s], 1);
      mamba_scan::mbar_init(&sm.empty[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mamba_scan::mbar_init(&sm.acc_full[b], 1);
      mamba_scan::mbar_init(&sm.acc_empty[b], 2 * kWarps);
    }
    mamba_scan::fence_mbarrier_init();
  }
  if (warp == 0) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(
                     smem_u32(&sm.tmem))
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  cluster_sync_all();  // both CTAs' barriers are there, the accumulators allocated
  tc_fence_after();
  const uint32_t tmem = sm.tmem;
  mamba_scan::pdl_trigger();
  mamba_scan::pdl_wait();

  // unit u: split, column tile and row tile, rows fastest, so that the pairs at
  // work share B's tiles and each of them is fetched from memory once
  if (warp == kLoadWarp) {
    if (lane == 0) {
      int it = 0;  // stages filled so far
      bool ok = true;
      for (int u = pair; ok && u < units; u += n_pairs) {
        const int split = u / tiles, m = u % tiles % p.m_tiles, n = u % tiles / p.m_tiles;
        const int m0 = m * kTile + (int)rank * kHalf;
        const int n0 = p.b_mn0 + n * kTile + (int)rank * kHalf;
        const int kb0 = split * p.kblocks, kb1 = min(kb0 + p.kblocks, p.total_kblocks);
        for (int kb = kb0; kb < kb1; ++kb, ++it) {
          const int s = it % kStages;
          if (it >= kStages &&
              !mamba_scan::mbar_wait(&sm.empty[s], (uint32_t)(it / kStages - 1) & 1u, &g_error)) {
            ok = false;
            break;
          }
          if (rank == 0) mamba_scan::mbar_arrive_expect_tx(&sm.full[s], 2 * C::kStageBytes);
          const uint32_t bar = map_to_rank(&sm.full[s], 0);
          const uint32_t base = smem_u32(sm.stage[s]);
          const int ka = p.a_k0 + kb * kBK, kbb = p.b_k0 + kb * kBK;
#pragma unroll
          for (int i = 0; i < PARTS; ++i) {
            const uint32_t a = base + i * kOperand, b = base + (PARTS + i) * kOperand;
            if constexpr (A_MN) {
              tma_load(a, &maps.a[i], bar, m0, ka);
              tma_load(a + kSlab, &maps.a[i], bar, m0 + 64, ka);
            } else {
              tma_load(a, &maps.a[i], bar, ka, m0);
            }
            if constexpr (B_MN) {
              tma_load(b, &maps.b[i], bar, n0, kbb);
              tma_load(b + kSlab, &maps.b[i], bar, n0 + 64, kbb);
            } else {
              tma_load(b, &maps.b[i], bar, kbb, n0);
            }
          }
        }
      }
      if (!ok && rank == 0)  // let the copies in flight land before the pair leaves
        for (int i = max(it - kStages, 0); i < it; ++i)
          mamba_scan::mbar_wait(&sm.full[i % kStages], (uint32_t)(i / kStages) & 1u, &g_error,
                                100000000ull);
    }
    __syncwarp();
  } else if (warp == kMmaWarp) {
    if (rank == 0) {
      const uint32_t leader = elect_one();
      int it = 0, seg = 0;  // stages and accumulators used so far
      bool ok = true;
      for (int u = pair; ok && u < units; u += n_pairs) {
        const int kb0 = u / tiles * p.kblocks, kb1 = min(kb0 + p.kblocks, p.total_kblocks);
        for (int kb = kb0; ok && kb < kb1; ++seg) {
          const int b = seg & 1;
          if (seg >= 2 &&
              !mamba_scan::mbar_wait(&sm.acc_empty[b], (uint32_t)((seg >> 1) - 1) & 1u, &g_error)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint32_t acc = tmem + (uint32_t)(b * kTile);
          uint32_t more = 0;
          for (const int end = min(kb + kSegment, kb1); kb < end; ++kb, ++it) {
            const int s = it % kStages;
            if (!mamba_scan::mbar_wait(&sm.full[s], (uint32_t)(it / kStages) & 1u, &g_error)) {
              ok = false;
              break;
            }
            tc_fence_after();
            const uint32_t base = smem_u32(sm.stage[s]);
            constexpr uint32_t ka = A_MN ? 2048 >> 4 : 32 >> 4, kb_ = B_MN ? 2048 >> 4 : 32 >> 4;
            const uint32_t ah = desc(base, A_MN), bh = desc(base + PARTS * kOperand, B_MN);
            if constexpr (PARTS == 2) {  // the small products first
              constexpr uint32_t lo = kOperand >> 4;
#pragma unroll
              for (uint32_t k = 0; k < kBK / 16; ++k) {
                mma_pair(leader, acc, ah + lo + k * ka, bh + k * kb_, p.idesc, more);
                mma_pair(leader, acc, ah + k * ka, bh + lo + k * kb_, p.idesc, 1u);
                more = 1;
              }
            }
#pragma unroll
            for (uint32_t k = 0; k < kBK / 16; ++k) {
              mma_pair(leader, acc, ah + k * ka, bh + k * kb_, p.idesc, more);
              more = 1;
            }
            commit_pair(leader, &sm.empty[s]);
          }
          commit_pair(leader, &sm.acc_full[b]);
        }
      }
    }
    __syncwarp();
  } else {
    BoxWriter<C::kBoxes> box{sm.box[warp][0], lane};
    const int quarter = warp & 3, half = warp >> 2;
    const uint32_t free0 = map_to_rank(&sm.acc_empty[0], 0);
    const uint32_t free1 = map_to_rank(&sm.acc_empty[1], 0);
    const uint32_t mine = tmem + ((uint32_t)(quarter * 32) << 16) + (uint32_t)(half * kCols);
    int seg = 0;
    bool ok = true;
    auto take = [&]() {  // the next accumulator: its address, once it is there
      const int b = seg & 1;
      ok = __all_sync(0xffffffffu, mamba_scan::mbar_wait(&sm.acc_full[b], (uint32_t)(seg >> 1) & 1u,
                                                         &g_error));
      tc_fence_after();
      return mine + (uint32_t)(b * kTile);
    };
    auto release = [&]() {
      tc_fence_before();
      __syncwarp();
      if (lane == 0) arrive_cluster(seg & 1 ? free1 : free0);
      ++seg;
    };
    for (int u = pair; u < units; u += n_pairs) {
      const int split = u / tiles, m = u % tiles % p.m_tiles, n = u % tiles / p.m_tiles;
      const int row0 = m * kTile + (int)rank * kHalf + quarter * 32, row = row0 + lane;
      const int kb0 = split * p.kblocks, kb1 = min(kb0 + p.kblocks, p.total_kblocks);
      float acc[kCols];
#pragma unroll
      for (int j = 0; j < kCols; ++j) acc[j] = 0.f;
#pragma unroll 1
      for (int kb = kb0; kb < kb1; kb += kSegment) {
        const uint32_t from = take();
        if (!ok) break;
#pragma unroll
        for (int c = 0; c < kCols; c += 32) {
          float v[32];
          tmem_ld32(from + (uint32_t)c, v);
          tmem_wait();
#pragma unroll
          for (int j = 0; j < 32; j += 2) {
            const float2 sum = __fadd2_rn(make_float2(acc[c + j], acc[c + j + 1]),
                                          make_float2(v[j], v[j + 1]));
            acc[c + j] = sum.x;
            acc[c + j + 1] = sum.y;
          }
        }
        release();
      }
      if (!ok) break;
      auto finish = [&](auto& epilogue) {
#pragma unroll
        for (int c = 0; c < kCols; c += 32)
          epilogue.chunk(c, *reinterpret_cast<float(*)[32]>(acc + c));
        epilogue.end();
      };
      if constexpr (MODE == kStats) {
        StatsEpilogue<PARTS> epilogue{p};
        epilogue.begin(n, half, row);
        finish(epilogue);
      } else if constexpr (MODE == kGrad) {
        GradEpilogue<PARTS, T16> epilogue{p, maps, box};
        epilogue.begin(n, half, row, row0);
        finish(epilogue);
      } else {
        OutEpilogue<PARTS, T16, TO> epilogue{p, maps, box};
        epilogue.begin(n, half, split, row, row0);
        finish(epilogue);
      }
    }
    if (MODE != kStats && lane == 0) mamba_scan::bulk_wait_all<0>();
    __syncwarp();
  }
  tc_fence_before();
  cluster_sync_all();  // the pair is done with the accumulators and each other's barriers
  if (warp == 0) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
  }
}

// ---------------------------------------------------------- before and after

// The rows' partial (m, s) of all vocabulary tiles -> stats and loss. 8 rows a
// CTA, 32 threads to a row, their loads eight at a time: there may be few rows,
// and one thread's trips through a row's partials were most of a short call.
__global__ void __launch_bounds__(256)
    combine_kernel(const float2* partial, const float* target_logit, const int64_t* target,
                   float* loss, float2* stats, int rows, int n_parts, int64_t vocab) {
  mamba_scan::pdl_trigger();
  mamba_scan::pdl_wait();
  __shared__ float2 part[8][8];
  const int r = threadIdx.x & 7, slice = threadIdx.x >> 3, warp = threadIdx.x >> 5;
  const int row = (int)blockIdx.x * 8 + r;
  float m = -INFINITY, s = 0.f;
  auto merge = [&](float2 o) { merge_sums(m, s, o.x, o.y); };
  if (row < rows) {
    constexpr int kBatch = 8;
    for (int i = slice; i < n_parts; i += 32 * kBatch) {
      float2 o[kBatch];
#pragma unroll
      for (int j = 0; j < kBatch; ++j)
        o[j] = i + 32 * j < n_parts ? partial[(int64_t)(i + 32 * j) * rows + row]
                                    : make_float2(-INFINITY, 0.f);
#pragma unroll
      for (int j = 0; j < kBatch; ++j) merge(o[j]);
    }
  }
#pragma unroll
  for (int d = 8; d < 32; d <<= 1) {
    const float om = __shfl_xor_sync(0xffffffffu, m, d), os = __shfl_xor_sync(0xffffffffu, s, d);
    merge(make_float2(om, os));
  }
  if ((threadIdx.x & 31) < 8) part[warp][r] = make_float2(m, s);
  __syncthreads();
  if (threadIdx.x >= 8 || row >= rows) return;
  for (int i = 1; i < 8; ++i) merge(part[i][r]);
  if (stats) stats[row] = make_float2(m, s);
  const int64_t t = target[row];
  loss[row] = t < 0 ? 0.f
              : t >= vocab ? __int_as_float(0x7fc00000)
                           : (m - target_logit[row]) + logf(s);
}

// grad relative to the largest finite |grad| of the rows that count (an infinite
// one spoils its row, not the others). One CTA.
__global__ void __launch_bounds__(1024)
    grad_kernel(const float* grad, int64_t stride, const int64_t* target, int rows, float* rel,
                float* largest) {
  mamba_scan::pdl_trigger();
  mamba_scan::pdl_wait();
  __shared__ float part[32];
  float m = 0.f;
  for (int r = threadIdx.x; r < rows; r += 1024)
    if (target[r] >= 0) {
      const float g = fabsf(grad[(int64_t)r * stride]);
      if (g <= 3.402823466e38f) m = fmaxf(m, g);
    }
  m = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(m)));
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = m;
  __syncthreads();
  m = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(part[threadIdx.x & 31])));
  if (threadIdx.x == 0) *largest = m;
  for (int r = threadIdx.x; r < rows; r += 1024) {
    const float g = target[r] >= 0 ? grad[(int64_t)r * stride] : 0.f;
    rel[r] = m > 0.f ? g / m : g;  // (all zeros, or NaN)
  }
}

// The largest finite |element| of a float32 matrix, as bits, into `largest`
// (zero before); rows whose target is negative (where there are targets) do
// not count. A warp takes rows one after the other.
__global__ void __launch_bounds__(256)
    largest_kernel(const float* x, int64_t stride, int64_t rows, int width, const int64_t* target,
                   uint32_t* largest) {
  mamba_scan::pdl_trigger();
  mamba_scan::pdl_wait();
  __shared__ uint32_t part[8];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  uint32_t m = 0;
  auto add = [&](float v) {
    const uint32_t u = __float_as_uint(v) & 0x7fffffffu;
    m = max(m, u < 0x7f800000u ? u : 0u);
  };
  for (int64_t row = (int64_t)blockIdx.x * 8 + warp; row < rows; row += (int64_t)gridDim.x * 8) {
    if (target != nullptr && target[row] < 0) continue;
    const float* src = x + row * stride;
    const int whole = (reinterpret_cast<uintptr_t>(src) & 15u) == 0 ? width / 4 * 4 : 0;
    int at = lane * 4;
    for (; at + 3 * 128 < whole; at += 512) {
      float4 w[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) w[i] = *reinterpret_cast<const float4*>(src + at + i * 128);
#pragma unroll
      for (int i = 0; i < 4; ++i) add(w[i].x), add(w[i].y), add(w[i].z), add(w[i].w);
    }
    for (; at < whole; at += 128) {
      const float4 w = *reinterpret_cast<const float4*>(src + at);
      add(w.x), add(w.y), add(w.z), add(w.w);
    }
    for (at = whole + lane; at < width; at += 32) add(src[at]);
  }
  m = __reduce_max_sync(0xffffffffu, m);
  if (lane == 0) part[warp] = m;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int i = 1; i < 8; ++i) m = max(m, part[i]);
    atomicMax(largest, m);
  }
}

// A float32 matrix as two fp16 parts of pitch `ld`, scaled by the power of two
// that its largest element asks for; rows whose target is negative become
// zeros. One warp a row, the last rows first: they are what the L2 cache still
// holds of the search for the largest.
__global__ void __launch_bounds__(256)
    split_kernel(const float* x, int64_t stride, int64_t rows, int width, const int64_t* target,
                 __half* hi, __half* lo, int64_t ld, const uint32_t* largest) {
  mamba_scan::pdl_trigger();
  mamba_scan::pdl_wait();
  const int64_t row = rows - 1 - ((int64_t)blockIdx.x * 8 + (threadIdx.x >> 5));
  const int lane = threadIdx.x & 31;
  if (row < 0) return;
  const float* src = x + row * stride;
  __half* to_hi = hi + row * ld;
  __half* to_lo = lo + row * ld;
  if (target != nullptr && target[row] < 0) {
    for (int at = lane; at < width; at += 32) to_hi[at] = to_lo[at] = __float2half_rn(0.f);
    return;
  }
  const float f = pow2i(scale_exponent(*largest));
  auto put4 = [&](int at, float4 w) {
    const __half2 a = __floats2half2_rn(w.x * f, w.y * f), b = __floats2half2_rn(w.z * f, w.w * f);
    const float2 fa = __half22float2(a), fb = __half22float2(b);
    uint2 h, l;
    h.x = *reinterpret_cast<const uint32_t*>(&a);
    h.y = *reinterpret_cast<const uint32_t*>(&b);
    l.x = pack2<__half>(w.x * f - fa.x, w.y * f - fa.y);
    l.y = pack2<__half>(w.z * f - fb.x, w.w * f - fb.y);
    *reinterpret_cast<uint2*>(to_hi + at) = h;
    *reinterpret_cast<uint2*>(to_lo + at) = l;
  };
  const int whole = (reinterpret_cast<uintptr_t>(src) & 15u) == 0 ? width / 4 * 4 : 0;
  int at = lane * 4;
  for (; at + 3 * 128 < whole; at += 512) {
    float4 w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = *reinterpret_cast<const float4*>(src + at + i * 128);
#pragma unroll
    for (int i = 0; i < 4; ++i) put4(at + i * 128, w[i]);
  }
  for (; at < whole; at += 128) put4(at, *reinterpret_cast<const float4*>(src + at));
  for (at = whole + lane; at < width; at += 32) {
    const float v = src[at] * f;
    const __half h = __float2half_rn(v);
    to_hi[at] = h;
    to_lo[at] = __float2half_rn(v - __half2float(h));
  }
}

// A 16-bit matrix with rows of pitch `ld` (a multiple of 8 elements), rows
// whose target is negative as zeros. One warp a row.
__global__ void __launch_bounds__(256)
    pack_kernel(const uint16_t* x, int64_t stride, int64_t rows, int width, const int64_t* target,
                uint16_t* out, int64_t ld) {
  mamba_scan::pdl_trigger();
  mamba_scan::pdl_wait();
  const int64_t row = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  if (row >= rows) return;
  const uint16_t* src = x + row * stride;
  uint16_t* to = out + row * ld;
  const bool counts = target == nullptr || target[row] >= 0;
  const int whole = (reinterpret_cast<uintptr_t>(src) & 15u) == 0 ? width / 8 * 8 : 0;
  for (int at = lane * 8; at < whole; at += 256) {
    const uint4 w = *reinterpret_cast<const uint4*>(src + at);
    *reinterpret_cast<uint4*>(to + at) = counts ? w : make_uint4(0, 0, 0, 0);
  }
  for (int at = whole + lane; at < width; at += 32) to[at] = counts ? src[at] : (uint16_t)0;
}

// d_hidden = the splits' sums, scaled, in the output's type; 0 where a row does not
// count (its sums are 0 times the weights: NaN where those are not finite). A thread,
// 4 columns.
template <int PARTS, typename T16, typename TO>
__global__ void __launch_bounds__(256)
    hidden_kernel(const float* sums, int splits, int64_t split_stride, int64_t ld, int rows,
                  int width, const int64_t* target, const float* largest, const uint32_t* b_max,
                  TO* out) {
  mamba_scan::pdl_trigger();
  mamba_scan::pdl_wait();
  const int pieces = (width + 3) / 4;
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int64_t row = i / pieces;
  if (row >= rows) return;
  const int col = (int)(i % pieces) * 4;
  float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int k = 0; k < splits; ++k) {
    const float4 w = *reinterpret_cast<const float4*>(sums + k * split_stride + row * ld + col);
    s.x += w.x, s.y += w.y, s.z += w.z, s.w += w.w;
  }
  float f = *largest / dz_scale<T16>();
  if constexpr (PARTS == 2) f *= undo_scale(b_max);
  const bool counts = target[row] >= 0;
  const float v[4] = {s.x * f, s.y * f, s.z * f, s.w * f};
#pragma unroll
  for (int j = 0; j < 4; ++j)
    if (col + j < width) out[row * width + col + j] = from_f32<TO>(counts ? v[j] : 0.f);
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

// -------------------------------------------------------------------- host

namespace {

using Args = mamba_linear_cross_entropy_args;
using GradArgs = mamba_linear_cross_entropy_grad_args;

constexpr int64_t kMaxVocab = (int64_t)1 << 30, kMaxWidth = 65536;
constexpr int64_t kMaxRows = ((int64_t)1 << 31) - 257, kMaxStride = (int64_t)1 << 40;
constexpr int64_t kStatsRows = 32768;      // rows of one pass over the vocabulary
constexpr int64_t kPieceBytes = (int64_t)96 << 20;  // of dz

int64_t up(int64_t n, int64_t m) { return (n + m - 1) / m * m; }
int64_t element_size(int32_t dtype) {
  return dtype == MAMBA_DTYPE_F32 ? 4 : dtype == MAMBA_DTYPE_F16 || dtype == MAMBA_DTYPE_BF16 ? 2 : 0;
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

// A row-major matrix [rows][cols], `ld` elements between rows, in boxes of
// 128 (64) bytes x box_rows, in the swizzle of that width.
bool encode(CUtensorMap* m, const void* p, CUtensorMapDataType type, int64_t size, int64_t rows,
            int64_t cols, int64_t ld, int box_rows, int box_bytes = 128) {
  const cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows};
  const cuuint64_t strides[1] = {(cuuint64_t)(ld * size)};
  const cuuint32_t box[2] = {(cuuint32_t)(box_bytes / size), (cuuint32_t)box_rows};
  const cuuint32_t estr[2] = {1, 1};
  return encode_fn()(m, type, 2, const_cast<void*>(p), dims, strides, box, estr,
                     CU_TENSOR_MAP_INTERLEAVE_NONE,
                     box_bytes == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B,
                     CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                     CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// Where things lie in the workspace: take() hands out 256-byte aligned parts.
struct Layout {
  uint8_t* base;
  size_t at = 0;
  void* take(int64_t bytes) {
    void* p = base + at;
    at += (size_t)up(bytes, 256);
    return p;
  }
};

// An operand as the products take it: one or two 16-bit parts.
struct Operand {
  const void* part[2] = {nullptr, nullptr};
  int64_t ld = 0;
  uint32_t* largest = nullptr;  // float32
  bool prepared = false;  // parts in the workspace, to be filled
};

Operand place(Layout& ws, const void* x, int64_t rows, int64_t width, int64_t stride, int32_t dtype,
              bool copy) {
  Operand o;
  if (dtype == MAMBA_DTYPE_F32) {
    o.ld = up(width, 8);
    o.part[0] = ws.take(rows * o.ld * 2);
    o.part[1] = ws.take(rows * o.ld * 2);
    o.largest = static_cast<uint32_t*>(ws.take(4));
    o.prepared = true;
  } else if (copy || !mamba_lm::aligned16(x) || stride % 8 != 0) {
    o.ld = up(width, 8);
    o.part[0] = ws.take(rows * o.ld * 2);
    o.prepared = true;
  } else {
    o.part[0] = x;
    o.ld = stride;
  }
  return o;
}

cudaError_t prepare(const Operand& o, const void* x, int64_t rows, int64_t width, int64_t stride,
                    const int64_t* target, cudaStream_t st) {
  if (!o.prepared) return cudaSuccess;
  const dim3 grid((unsigned)((rows + 7) / 8)), block(256);
  if (o.largest != nullptr) {
    cudaError_t e = cudaMemsetAsync(o.largest, 0, 4, st);
    if (e != cudaSuccess) return e;
    const unsigned some = (unsigned)std::min<int64_t>((rows + 7) / 8, 8 * mamba_lm::sm_count());
    e = mamba_scan::launch_pdl(largest_kernel, dim3(some), block, 0, st,
                               static_cast<const float*>(x), stride, rows, (int)width, target,
                               o.largest);
    if (e != cudaSuccess) return e;
    return mamba_scan::launch_pdl(split_kernel, grid, block, 0, st, static_cast<const float*>(x),
                                  stride, rows, (int)width, target,
                                  static_cast<__half*>(const_cast<void*>(o.part[0])),
                                  static_cast<__half*>(const_cast<void*>(o.part[1])), o.ld,
                                  static_cast<const uint32_t*>(o.largest));
  }
  return mamba_scan::launch_pdl(pack_kernel, grid, block, 0, st, static_cast<const uint16_t*>(x),
                                stride, rows, (int)width, target,
                                static_cast<uint16_t*>(const_cast<void*>(o.part[0])), o.ld);
}

int pairs() { return std::max(1, mamba_lm::sm_count() / 2); }

uint32_t instruction(bool bf16, bool a_mn, bool b_mn) {
  return (1u << 4) | (bf16 ? (1u << 7) | (1u << 10) : 0u) | ((uint32_t)a_mn << 15) |
         ((uint32_t)b_mn << 16) | ((uint32_t)(kTile >> 3) << 17) | ((uint32_t)(kTile >> 4) << 24);
}

CUtensorMapDataType half_type(int32_t dtype) {
  return dtype == MAMBA_DTYPE_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16
                                   : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
}

// The map of an operand's parts: [rows][width], K-major (128 rows a box) or
// MN-major (64).
bool operand_maps(CUtensorMap* m, const Operand& o, int64_t rows, int64_t width, int32_t dtype,
                  bool mn) {
  for (int i = 0; i < 2; ++i)
    if (o.part[i] && !encode(m + i, o.part[i], half_type(dtype), 2, rows, width, o.ld, mn ? 64 : 128))
      return false;
  return true;
}

template <int MODE, int PARTS, typename T16, typename TO, bool A_MN, bool B_MN>
cudaError_t launch_tiles(const Maps& maps, const TileParams& p, cudaStream_t st) {
  auto kernel = tile_kernel<MODE, PARTS, T16, TO, A_MN, B_MN>;
  const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                             (int)Cfg<PARTS>::kSmemBytes);
  if (e != cudaSuccess) return e;
  const int64_t units = (int64_t)p.m_tiles * p.n_tiles * p.splits;
  return mamba_scan::launch_pdl(kernel, dim3((unsigned)(2 * std::min<int64_t>(pairs(), units))),
                                dim3(kThreads), Cfg<PARTS>::kSmemBytes, st, maps, p);
}

const char* check(const Args& a) {
  if (element_size(a.dtype) == 0) return "unknown dtype";
  if (a.rows < 0 || a.rows > kMaxRows) return "rows must be 0..2^31-257";
  if (a.vocab < 1 || a.vocab > kMaxVocab) return "vocab must be 1..2^30";
  if (a.width < 1 || a.width > kMaxWidth) return "width must be 1..65536";
  if (a.hidden_stride < a.width || a.hidden_stride > kMaxStride || a.weight_stride < a.width ||
      a.weight_stride > kMaxStride)
    return "strides must be width..2^40";
  // (tiles are counted in 31 bits)
  if (((a.rows + kTile - 1) / kTile) * ((a.vocab + kTile - 1) / kTile) >= (int64_t)1 << 30 ||
      ((a.vocab + kTile - 1) / kTile) * ((a.width + kTile - 1) / kTile) >= (int64_t)1 << 30)
    return "rows x vocab is too large";
  return nullptr;
}

struct ForwardPlan {
  Operand h, w;
  float2* partial;
  float* target_logit;
  size_t bytes;
};

ForwardPlan plan_forward(const Args& a, void* workspace) {
  Layout ws{static_cast<uint8_t*>(workspace)};
  ForwardPlan p;
  p.w = place(ws, a.weight, a.vocab, a.width, a.weight_stride, a.dtype, false);
  p.h = place(ws, a.hidden, a.rows, a.width, a.hidden_stride, a.dtype, false);
  const int64_t rows = std::min(a.rows, kStatsRows);
  p.partial = static_cast<float2*>(ws.take((a.vocab + kTile - 1) / kTile * rows * 16));
  p.target_logit = static_cast<float*>(ws.take(rows * 4));
  p.bytes = ws.at;
  return p;
}

template <int PARTS, typename T16>
cudaError_t forward(const Args& a, void* workspace, cudaStream_t st) {
  const ForwardPlan pl = plan_forward(a, workspace);
  cudaError_t e = prepare(pl.w, a.weight, a.vocab, a.width, a.weight_stride, nullptr, st);
  if (e != cudaSuccess) return e;
  e = prepare(pl.h, a.hidden, a.rows, a.width, a.hidden_stride, a.target, st);
  if (e != cudaSuccess) return e;
  Maps maps;
  std::memset(&maps, 0, sizeof(maps));
  if (!operand_maps(maps.a, pl.h, a.rows, a.width, a.dtype, false) ||
      !operand_maps(maps.b, pl.w, a.vocab, a.width, a.dtype, false))
    return cudaErrorInvalidValue;
  for (int64_t r0 = 0; r0 < a.rows; r0 += kStatsRows) {
    const int64_t rows = std::min(kStatsRows, a.rows - r0);
    if (r0 > 0) {  // the map starts at the pass's first row
      Operand h = pl.h;
      for (int i = 0; i < PARTS; ++i)
        h.part[i] = static_cast<const uint8_t*>(h.part[i]) + r0 * h.ld * 2;
      if (!operand_maps(maps.a, h, rows, a.width, a.dtype, false)) return cudaErrorInvalidValue;
    }
    TileParams p = {};
    p.m_tiles = (int)((rows + kTile - 1) / kTile);
    p.n_tiles = (int)((a.vocab + kTile - 1) / kTile);
    p.splits = 1;
    p.kblocks = p.total_kblocks = (int)((a.width + kBK - 1) / kBK);
    p.idesc = instruction(a.dtype == MAMBA_DTYPE_BF16, false, false);
    p.rows = (int)rows;
    p.vocab = (int)a.vocab;
    p.target = a.target + r0;
    p.a_max = pl.h.largest;
    p.b_max = pl.w.largest;
    p.partial = pl.partial;
    p.target_logit = pl.target_logit;
    e = launch_tiles<kStats, PARTS, T16, float, false, false>(maps, p, st);
    if (e != cudaSuccess) return e;
    e = launch_combine(pl.partial, pl.target_logit, p.target, a.loss + r0,
                       a.stats ? a.stats + 2 * r0 : nullptr, (int)rows, 2 * p.n_tiles, a.vocab, st);
    if (e != cudaSuccess) return e;
  }
  return cudaSuccess;
}

// How the gradients are cut: `piece` vocabulary tiles of dz at a time, the
// product over them for d_hidden split `splits` ways.
struct GradPlan {
  Operand h, w;
  int64_t piece, splits, pad_rows, sums_ld;
  void* dz[2];
  float* rel;
  float* largest;
  float* sums;
  size_t bytes;
};

// Rounds of the pairs times what a round's unit costs: its K blocks, and a
// tile's start and end. Vocabulary pieces are as wide as dz may be, or less
// where that leaves fewer pairs idle; d_hidden, which has few tiles, splits K.
void choose(const GradArgs& g, GradPlan* p) {
  const Args& a = g.forward;
  const int64_t P = pairs(), parts = a.dtype == MAMBA_DTYPE_F32 ? 2 : 1;
  const int64_t mt = p->pad_rows / kTile, vt = (a.vocab + kTile - 1) / kTile;
  const int64_t nt = (a.width + kTile - 1) / kTile;
  const int64_t kw = (a.width + kBK - 1) / kBK, kr = (a.rows + kBK - 1) / kBK;
  const int64_t most = std::max<int64_t>(
      1, std::min(vt, kPieceBytes / (p->pad_rows * kTile * 2 * parts)));
  auto rounds = [&](int64_t units, int64_t cost) { return (units + P - 1) / P * cost; };
  constexpr int64_t kOver = 4;  // a tile's own cost, in K blocks
  int64_t best = -1;
  for (int64_t x = most; x >= std::max<int64_t>(1, most / 2); --x) {
    const int64_t pieces = (vt + x - 1) / x;
    int64_t fixed = 0, split_cost = -1, split = 1;
    fixed += rounds(mt * x, kw + kOver);
    if (g.d_weight) fixed += rounds(x * nt, kr + kOver);
    if (g.d_hidden) {
      for (int64_t s = 1; s <= 64 && (s == 1 || x * 4 / s >= 8); ++s) {
        const int64_t c = rounds(mt * nt * s, (x * 4 + s - 1) / s + kOver) + s;
        if (split_cost < 0 || c < split_cost) split_cost = c, split = s;
      }
      fixed += split_cost;
    }
    const int64_t total = pieces * (fixed + 4);
    if (best < 0 || total < best) {
      best = total;
      p->piece = x;
      p->splits = split;
    }
  }
  // (no split is empty)
  const int64_t kb = p->piece * 4, per = (kb + p->splits - 1) / p->splits;
  p->splits = (kb + per - 1) / per;
}

GradPlan plan_grad(const GradArgs& g, void* workspace) {
  const Args& a = g.forward;
  Layout ws{static_cast<uint8_t*>(workspace)};
  GradPlan p;
  p.pad_rows = up(a.rows, kTile);
  choose(g, &p);
  const int parts = a.dtype == MAMBA_DTYPE_F32 ? 2 : 1;
  p.w = place(ws, a.weight, a.vocab, a.width, a.weight_stride, a.dtype, false);
  // (rows that do not count are zeros: 0 x NaN must not come into d_weight)
  p.h = place(ws, a.hidden, a.rows, a.width, a.hidden_stride, a.dtype, true);
  p.dz[0] = p.dz[1] = nullptr;
  for (int i = 0; i < parts; ++i) p.dz[i] = ws.take(p.pad_rows * p.piece * kTile * 2);
  p.rel = static_cast<float*>(ws.take(a.rows * 4));
  p.largest = static_cast<float*>(ws.take(4));
  p.sums_ld = up(a.width, 4);
  p.sums = g.d_hidden ? static_cast<float*>(ws.take(p.splits * p.pad_rows * p.sums_ld * 4)) : nullptr;
  p.bytes = ws.at;
  return p;
}

template <int PARTS, typename T16, typename TO>
cudaError_t backward(const GradArgs& g, void* workspace, cudaStream_t st) {
  const Args& a = g.forward;
  const GradPlan pl = plan_grad(g, workspace);
  const bool bf16 = a.dtype == MAMBA_DTYPE_BF16;
  cudaError_t e = prepare(pl.w, a.weight, a.vocab, a.width, a.weight_stride, nullptr, st);
  if (e != cudaSuccess) return e;
  e = prepare(pl.h, a.hidden, a.rows, a.width, a.hidden_stride, a.target, st);
  if (e != cudaSuccess) return e;
  e = mamba_scan::launch_pdl(grad_kernel, dim3(1), dim3(1024), 0, st, g.grad, g.grad_stride, a.target,
                             (int)a.rows, pl.rel, pl.largest);
  if (e != cudaSuccess) return e;
  const int64_t piece_cols = pl.piece * kTile;
  Operand dz;
  dz.part[0] = pl.dz[0], dz.part[1] = pl.dz[1];
  dz.ld = piece_cols;
  Maps logits, by_hidden, by_weight;  // dz; d_hidden = dz W; d_weight = dz^T H
  std::memset(&logits, 0, sizeof(Maps));
  std::memset(&by_hidden, 0, sizeof(Maps));
  std::memset(&by_weight, 0, sizeof(Maps));
  bool ok = operand_maps(logits.a, pl.h, a.rows, a.width, a.dtype, false) &&
            operand_maps(logits.b, pl.w, a.vocab, a.width, a.dtype, false) &&
            operand_maps(by_hidden.a, dz, pl.pad_rows, piece_cols, a.dtype, false) &&
            operand_maps(by_hidden.b, pl.w, a.vocab, a.width, a.dtype, true) &&
            operand_maps(by_weight.a, dz, pl.pad_rows, piece_cols, a.dtype, true) &&
            operand_maps(by_weight.b, pl.h, a.rows, a.width, a.dtype, true);
  for (int i = 0; i < PARTS; ++i)
    ok = ok && encode(&logits.out[i], pl.dz[i], half_type(a.dtype), 2, pl.pad_rows, piece_cols,
                      piece_cols, 32, PARTS == 2 ? 64 : 128);
  if (g.d_hidden)
    ok = ok && encode(&by_hidden.out[0], pl.sums, CU_TENSOR_MAP_DATA_TYPE_FLOAT32, 4,
                      pl.splits * pl.pad_rows, a.width, pl.sums_ld, 32);
  const bool direct = !mamba_lm::aligned16(g.d_weight) || a.width * (int64_t)sizeof(TO) % 16 != 0;
  if (!ok) return cudaErrorInvalidValue;

  TileParams base = {};
  base.splits = 1;
  base.rows = (int)a.rows;
  base.vocab = (int)a.vocab;
  base.target = a.target;
  base.stats = reinterpret_cast<const float2*>(a.stats);
  base.rel_grad = pl.rel;
  base.largest = pl.largest;
  const int vt = (int)((a.vocab + kTile - 1) / kTile), mt = (int)(pl.pad_rows / kTile);
  const int nt = (int)((a.width + kTile - 1) / kTile);
  for (int v = 0; v < vt; v += (int)pl.piece) {
    const int n = std::min((int)pl.piece, vt - v);  // tiles of this piece
    TileParams p = base;
    p.m_tiles = mt;
    p.n_tiles = n;
    p.kblocks = p.total_kblocks = (int)((a.width + kBK - 1) / kBK);
    p.b_mn0 = p.v0 = v * kTile;
    p.idesc = instruction(bf16, false, false);
    p.a_max = pl.h.largest;
    p.b_max = pl.w.largest;
    e = launch_tiles<kGrad, PARTS, T16, float, false, false>(logits, p, st);
    if (e != cudaSuccess) return e;
    if (g.d_weight) {
      const int64_t rows = std::min<int64_t>((int64_t)n * kTile, a.vocab - (int64_t)v * kTile);
      p = base;
      p.m_tiles = n;
      p.n_tiles = nt;
      p.kblocks = p.total_kblocks = (int)((a.rows + kBK - 1) / kBK);
      p.idesc = instruction(bf16, true, true);
      p.out_rows = (int)rows;
      p.out_cols = (int)a.width;
      p.scaled = 1;
      p.b_max = pl.h.largest;
      TO* to = static_cast<TO*>(g.d_weight) + (int64_t)v * kTile * a.width;
      if (direct) {
        p.out = to;
        p.out_stride = a.width;
      } else if (!encode(&by_weight.out[0], to,
                         sizeof(TO) == 4 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : half_type(a.dtype),
                         sizeof(TO), rows, a.width, a.width, 32)) {
        return cudaErrorInvalidValue;
      }
      e = launch_tiles<kOut, PARTS, T16, TO, true, true>(by_weight, p, st);
      if (e != cudaSuccess) return e;
    }
    if (g.d_hidden) {
      const int64_t kb = pl.piece * 4, per = (kb + pl.splits - 1) / pl.splits;
      p = base;
      p.m_tiles = mt;
      p.n_tiles = nt;
      p.kblocks = (int)per;
      p.total_kblocks = n * 4;
      // (a narrow last piece may leave later splits without work; the first
      // piece, which writes instead of adding, never does)
      p.splits = (int)std::min<int64_t>(pl.splits, (p.total_kblocks + per - 1) / per);
      p.b_k0 = v * kTile;
      p.idesc = instruction(bf16, false, true);
      p.out_rows = (int)pl.pad_rows;
      p.out_cols = (int)a.width;
      p.split_rows = (int)pl.pad_rows;
      p.accumulate = v > 0;
      e = launch_tiles<kOut, PARTS, T16, float, false, true>(by_hidden, p, st);
      if (e != cudaSuccess) return e;
    }
  }
  if (!g.d_hidden) return cudaSuccess;
  const int64_t pieces = a.rows * ((a.width + 3) / 4);
  return mamba_scan::launch_pdl(hidden_kernel<PARTS, T16, TO>, dim3((unsigned)((pieces + 255) / 256)),
                                dim3(256), 0, st, static_cast<const float*>(pl.sums),
                                (int)pl.splits, pl.pad_rows * pl.sums_ld, pl.sums_ld, (int)a.rows,
                                (int)a.width, a.target, static_cast<const float*>(pl.largest),
                                static_cast<const uint32_t*>(pl.w.largest),
                                static_cast<TO*>(g.d_hidden));
}

// The checks that loss and gradients share; `outs` and `ins` are the rest.
int checked(const Args& a, const char* op, bool stats_in, const void* workspace,
            size_t workspace_bytes, size_t need, const mamba_lm::Range* outs, int n_outs,
            const mamba_lm::Range& more) {
  using mamba_lm::Range;
  using mamba_lm::overlap;
  using mamba_lm::range_of;
  using mamba_scan::set_last_error;
  const std::string name = std::string(op) + ": ";
  const int64_t size = element_size(a.dtype);
  if (!mamba_lm::aligned_to(size, {a.hidden, a.weight}) || !mamba_lm::aligned_to(8, {a.target}) ||
      !mamba_lm::aligned_to(4, {a.loss, a.stats}))
    return set_last_error(MAMBA_SCAN_ERR_INVALID_ARGUMENT,
                          name + "an address is not a multiple of its type's size");
  const int64_t one[1] = {1}, zero[1] = {0}, hn[1] = {a.rows}, hs[1] = {a.hidden_stride};
  const int64_t wn[1] = {a.vocab}, wst[1] = {a.weight_stride};
  const Range ws = range_of(workspace, 1, (int64_t)workspace_bytes, one, zero, 1);
  const Range ins[] = {range_of(a.hidden, size, a.width, hn, hs, 1),
                       range_of(a.weight, size, a.width, wn, wst, 1),
                       range_of(a.target, 8, a.rows, one, zero, 1),
                       range_of(stats_in ? a.stats : nullptr, 4, 2 * a.rows, one, zero, 1), more};
  for (const Range& in : ins) {
    if (overlap(ws, in))
      return set_last_error(MAMBA_SCAN_ERR_ALIASING, name + "workspace overlaps an input");
    for (int i = 0; i < n_outs; ++i)
      if (overlap(outs[i], in))
        return set_last_error(MAMBA_SCAN_ERR_ALIASING, name + "an output overlaps an input");
  }
  for (int i = 0; i < n_outs; ++i) {
    if (overlap(outs[i], ws))
      return set_last_error(MAMBA_SCAN_ERR_ALIASING, name + "an output overlaps the workspace");
    for (int j = 0; j < i; ++j)
      if (overlap(outs[i], outs[j]))
        return set_last_error(MAMBA_SCAN_ERR_ALIASING, name + "outputs overlap");
  }
  if (workspace_bytes < need || workspace == nullptr)
    return set_last_error(MAMBA_SCAN_ERR_WORKSPACE, name + "workspace holds " +
                                                        std::to_string(workspace ? workspace_bytes : 0) +
                                                        " bytes; this call needs " +
                                                        std::to_string(need));
  if (!mamba_lm::aligned16(workspace))
    return set_last_error(MAMBA_SCAN_ERR_WORKSPACE, name + "workspace must be 16-byte aligned");
  return MAMBA_SCAN_OK;
}

int finish(cudaError_t e, const char* op) {
  if (e == cudaSuccess) return MAMBA_SCAN_OK;
  return mamba_scan::set_last_error(MAMBA_SCAN_ERR_CUDA,
                                    std::string(op) + ": " + cudaGetErrorString(e));
}

size_t forward_bytes(const Args& a) {
  return few_rows(a, false) ? few_forward_bytes(a) : plan_forward(a, nullptr).bytes;
}
size_t grad_bytes(const GradArgs& g) {
  return few_rows(g.forward, true) ? few_grad_bytes(g) : plan_grad(g, nullptr).bytes;
}

}  // namespace

cudaError_t launch_combine(const float2* partial, const float* target_logit, const int64_t* target,
                           float* loss, float* stats, int rows, int parts, int64_t vocab,
                           cudaStream_t st) {
  return mamba_scan::launch_pdl(combine_kernel, dim3((unsigned)((rows + 7) / 8)), dim3(256), 0, st,
                                partial, target_logit, target, loss, reinterpret_cast<float2*>(stats),
                                rows, parts, vocab);
}

}  // namespace mamba_lce

extern "C" {

size_t mamba_linear_cross_entropy_workspace_size(const mamba_linear_cross_entropy_args* a) {
  if (a == nullptr || mamba_lce::check(*a) || a->rows == 0) return 0;
  return mamba_lce::forward_bytes(*a);
}

int mamba_linear_cross_entropy(const mamba_linear_cross_entropy_args* a, void* workspace,
                               size_t workspace_bytes, void* stream) try {
  using mamba_scan::set_last_error;
  set_last_error(MAMBA_SCAN_OK, "");
  const char* op = "linear_cross_entropy";
  if (a == nullptr) return set_last_error(MAMBA_SCAN_ERR_INVALID_ARGUMENT, "args is NULL");
  if (const char* bad = mamba_lce::check(*a))
    return set_last_error(MAMBA_SCAN_ERR_INVALID_ARGUMENT, std::string(op) + ": " + bad);
  if (a->rows == 0) return MAMBA_SCAN_OK;
  if (!a->hidden || !a->weight || !a->target || !a->loss)
    return set_last_error(MAMBA_SCAN_ERR_INVALID_ARGUMENT,
                          "linear_cross_entropy: hidden, weight, target and loss must be non-NULL");
  const int64_t one[1] = {1}, zero[1] = {0};
  const mamba_lm::Range outs[] = {mamba_lm::range_of(a->loss, 4, a->rows, one, zero, 1),
                                  mamba_lm::range_of(a->stats, 4, 2 * a->rows, one, zero, 1)};
  if (const int rc = mamba_lce::checked(*a, op, false, workspace, workspace_bytes,
                                        mamba_lce::forward_bytes(*a), outs, 2, {}))
    return rc;
  if (a->stats && !mamba_lm::aligned_to(8, {a->stats}))
    return set_last_error(MAMBA_SCAN_ERR_INVALID_ARGUMENT,
                          "linear_cross_entropy: stats must be 8-byte aligned");
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (mamba_lce::few_rows(*a, false))
    return mamba_lce::finish(mamba_lce::few_forward(*a, workspace, st), op);
  if (mamba_lce::encode_fn() == nullptr)
    return set_last_error(MAMBA_SCAN_ERR_CUDA, "cuTensorMapEncodeTiled is not available");
  switch (a->dtype) {
    case MAMBA_DTYPE_F32: return mamba_lce::finish(mamba_lce::forward<2, __half>(*a, workspace, st), op);
    case MAMBA_DTYPE_F16: return mamba_lce::finish(mamba_lce::forward<1, __half>(*a, workspace, st), op);
    default: return mamba_lce::finish(mamba_lce::forward<1, __nv_bfloat16>(*a, workspace, st), op);
  }
} catch (...) {
  return MAMBA_SCAN_ERR_CUDA;
}

size_t mamba_linear_cross_entropy_grad_workspace_size(
    const mamba_linear_cross_entropy_grad_args* g) {
  if (g == nullptr || mamba_lce::check(g->forward) || g->forward.rows == 0) return 0;
  return mamba_lce::grad_bytes(*g);
}

int mamba_linear_cross_entropy_grad(const mamba_linear_cross_entropy_grad_args* g, void* workspace,
                                    size_t workspace_bytes, void* stream) try {
  using mamba_lm::range_of;
  using mamba_scan::set_last_error;
  set_last_error(MAMBA_SCAN_OK, "");
  const char* op = "linear_cross_entropy_grad";
  if (g == nullptr) return set_last_error(MAMBA_SCAN_ERR_INVALID_ARGUMENT, "args is NULL");
  const mamba_linear_cross_entropy_args& a = g->forward;
  if (const char* bad = mamba_lce::check(a))
    return set_last_error(MAMBA_SCAN_ERR_INVALID_ARGUMENT, std::string(op) + ": " + bad);
  if (g->grad_stride < 0 || g->grad_stride > mamba_lce::kMaxStride)
    return set_last_error(MAMBA_SCAN_ERR_INVALID_ARGUMENT,
                          "linear_cross_entropy_grad: grad_stride must be 0..2^40");
  const int64_t size = mamba_lce::element_size(a.dtype);
  if (!mamba_lm::aligned_to(size, {g->d_hidden, g->d_weight}) ||
      !mamba_lm::aligned_to(4, {g->grad}) || !mamba_lm::aligned_to(8, {a.stats}))
    return set_last_error(MAMBA_SCAN_ERR_INVALID_ARGUMENT,
                          "linear_cross_entropy_grad: an address is not a multiple of its type's size");
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (a.rows == 0) {  // nothing adds to d_weight
    if (!g->d_weight) return MAMBA_SCAN_OK;
    return mamba_lce::finish(
        cudaMemsetAsync(g->d_weight, 0, (size_t)(a.vocab * a.width * size), st), op);
  }
  if (!a.hidden || !a.weight || !a.target || !a.stats || !g->grad)
    return set_last_error(
        MAMBA_SCAN_ERR_INVALID_ARGUMENT,
        "linear_cross_entropy_grad: hidden, weight, target, stats and grad must be non-NULL");
  if (!g->d_hidden && !g->d_weight) return MAMBA_SCAN_OK;
  const int64_t n[1] = {a.rows}, gs[1] = {g->grad_stride};
  const int64_t hn[1] = {a.rows}, wn[1] = {a.vocab}, w1[1] = {a.width};
  const mamba_lm::Range outs[] = {range_of(g->d_hidden, size, a.width, hn, w1, 1),
                                  range_of(g->d_weight, size, a.width, wn, w1, 1)};
  if (const int rc = mamba_lce::checked(a, op, true, workspace, workspace_bytes,
                                        mamba_lce::grad_bytes(*g), outs, 2,
                                        range_of(g->grad, 4, 1, n, gs, 1)))
    return rc;
  if (mamba_lce::few_rows(a, true))
    return mamba_lce::finish(mamba_lce::few_backward(*g, workspace, st), op);
  if (mamba_lce::encode_fn() == nullptr)
    return set_last_error(MAMBA_SCAN_ERR_CUDA, "cuTensorMapEncodeTiled is not available");
  switch (a.dtype) {
    case MAMBA_DTYPE_F32:
      return mamba_lce::finish(mamba_lce::backward<2, __half, float>(*g, workspace, st), op);
    case MAMBA_DTYPE_F16:
      return mamba_lce::finish(mamba_lce::backward<1, __half, __half>(*g, workspace, st), op);
    default:
      return mamba_lce::finish(
          mamba_lce::backward<1, __nv_bfloat16, __nv_bfloat16>(*g, workspace, st), op);
  }
} catch (...) {
  return MAMBA_SCAN_ERR_CUDA;
}

}  // extern "C"
