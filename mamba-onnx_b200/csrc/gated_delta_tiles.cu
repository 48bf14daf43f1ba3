// The chain of the gated delta rule's chunks over tensor memory
// (gated_delta_mma.cu states the mathematics and makes the chunks' records), for
// 16-bit tensors that TMA can take.
//
// A CTA = one sequence, head and up to 128 state columns. Everything is held
// transposed, dv on the 128 lanes of tensor memory; 8 warps share the lanes
// (their quarter of them) and the columns, so that a thread has half of a state
// column, in registers in fp32, and of a row of X and U. A chunk:
//   X^T  [dv x 64] = S^T K^T    (S's parts in tensor memory, K in shared memory)
//   U^T  [dv x 64] = R^T T^T    (R = V - weighted X)
//   dS^T [dv x dk] = U''^T K    (U'' = U weighted until the chunk's end)
// in a row, each a product that one warp issues, then its results read, weighted
// and split by the computing warps. What a chunk takes is this chain: of 5300
// clocks with dk = dv = 128 (5800 with all SMs at work) 600 to 850 are each product,
// from its operands' last store to its result's first load, and the rest the
// weighting, comparing and splitting between them (64 x 96: 3900). One sequence of
// 16384 tokens of 16 heads takes 808 us in bf16 (256 chunks of 2.9 us, the next ones'
// prepare_kernel beside them, and three launches' starts), 8 of 2048 of 40 530 us.
// Beside it the tensor cores form O1^T = S^T Q^T and O2^T = U^T P^T, and four
// more warps send these on their way and bring the next chunk's k and q into
// fp16, from what a warp loads by TMA.
// Where mma.sync takes 8 clocks of a scheduler's quarter for each 16 x 8 x 16 (4
// us of an SM for the 128 columns of a chunk), the tensor cores here take a
// quarter of that, and no issue slots.
//
// Tried and left: 16 computing warps (fewer instructions each, one more exchange
// in four: 8% slower), k and q converted and outputs sent by the computing warps in
// the products' shadow (16384 tokens 1140 us), an SM's share of all chunks to a CTA,
// whole heads and two halves (which fills the last round, but what tells the warps
// of the next part costs every chunk 10 to 30%, most of it instructions fetched
// again, since the roles' code no longer fits their cache: 8 x 2048 18% slower).
//
// Numbers as there: fp16 parts hi + lo of operands scaled by powers of two, S, R, U
// and U'' each by its columns' largest elements, which the two threads of a lane
// compare through shared memory. (U and U'' by U's bound, 64 x 2^15 x 2^15 of R's and
// T's scales, would save two of the four exchanges, but what a reset or growing decays
// leave of U may lie so far below the bound that its parts end: after one value 2^20
// times the others, forgotten by a reset, the state was 1e-3 off.)
#include <cudaTypedefs.h>

#include <algorithm>
#include <cstring>
#include <mutex>
#include <type_traits>

#include "gated_delta.cuh"
#include "scan_kernels.h"

namespace mamba_gd {

using mamba_lm::from_f32;
using mamba_lm::to_f32;
using mamba_scan::smem_u32;

namespace {

__device__ int g_tiles_error = 0;

constexpr int kLanes = 128;      // state columns of a CTA: lanes of tensor memory
constexpr int kSlab = 64 * 128;  // 64 rows of 64 16-bit elements, 128-byte swizzle
constexpr int kWarps = 8;        // that compute
constexpr int kParts = kWarps / 4;      // of a lane's columns
constexpr int kRows = kChunk / kParts;  // of a chunk, to a thread
constexpr int kHelpers = 4;      // that convert and send outputs
constexpr int kIssueWarp = kWarps + kHelpers, kLoadWarp = kIssueWarp + 1;
constexpr int kThreads = 32 * (kWarps + kHelpers + 4);  // whole warpgroups
// Registers of a thread at the launch, and then: the computing warpgroups', that
// of the helpers and the last one's (with 128 for all parts of the state were
// spilled: 7600 clocks a chunk of 128 x 128 in place of 6130).
constexpr int kLaunchRegs = 128, kComputeRegs = 176, kHelperRegs = 112, kOtherRegs = 40;
static_assert(kComputeRegs * kWarps + kHelperRegs * kHelpers + kOtherRegs * 4 <=
                  kLaunchRegs * (kWarps + kHelpers + 4),
              "no more than the launch has");

template <int DKP_> struct TilesCfg {
  static constexpr int DKP = DKP_;
  static constexpr int kSlabs = DKP / 64;
  struct __align__(1024) Stage {
    uint8_t k[kSlabs * kSlab];
    uint8_t q[kSlabs * kSlab];
    uint8_t v[2 * kSlab];
    __align__(1024) TileMain rec;
  };
  struct __align__(1024) OutStage {
    TileOut rec;
  };
  struct __align__(1024) Smem {
    Stage stage[2];
    OutStage out[2];
    uint8_t o[2 * kSlab];         // a chunk's outputs on their way
    float largest[2][kParts][kLanes];          // two in turn: between a value's reads and
                                               // the next one in its place is a barrier
    float s_inv[2][kLanes], u_inv[2][kLanes];  // what undoes S's and U's scales, for O1 and O2
    uint64_t full[2], out_full[2];             // loads have landed
    // (two of those that a warp that is behind could else find two phases on)
    uint64_t converted[2];                     // helpers: a stage's k and q are fp16
    // computing warps -> issuing warp: the first halves of their S's parts are
    // there, the others; R's; those of U weighted; U's
    uint64_t s_ready[2], r_ready[2], u_ready[2], uo_ready;
    uint64_t o_read, o_free;                   // helpers: O1 and O2 are read; in `o`
    uint64_t o_sent;                           // loading warp: `o` has left
    uint64_t x_done, u_done, s_done[2], o_done;  // products
    int gave_up;
    uint32_t tmem;
  };
  static constexpr size_t kBytes = sizeof(Smem) + 1024;
  static_assert(kBytes <= 227 * 1024, "shared memory per CTA");
  // tensor memory, 512 columns: S's parts; X, then U; R's parts, then those of U
  // weighted; U's parts; O1; dS, then O2
  static constexpr int kColS = 0, kColX = DKP, kColR = kColX + 64, kColU = kColR + 64;
  static constexpr int kColO1 = kColU + 64, kColD = kColO1 + 64;
  static_assert(kColD + DKP <= 512, "tensor memory");
};

// ------------------------------------------------------------ PTX wrappers

__device__ __forceinline__ void tma_load_4d(uint32_t dst, const CUtensorMap* map, uint64_t* bar,
                                            int c0, int c1, int c2, int c3) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%3, %4, %5, %6}], [%2];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(smem_u32(bar)), "r"(c0), "r"(c1), "r"(c2), "r"(c3)
      : "memory");
}
__device__ __forceinline__ void tma_store_4d(const CUtensorMap* map, uint32_t src, int c0, int c1,
                                             int c2, int c3) {
  asm volatile(
      "cp.async.bulk.tensor.4d.global.shared::cta.bulk_group [%0, {%2, %3, %4, %5}], [%1];" ::"l"(
          reinterpret_cast<uint64_t>(map)),
      "r"(src), "r"(c0), "r"(c1), "r"(c2), "r"(c3)
      : "memory");
}
__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes,
                                          uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
          dst),
      "l"(src), "r"(bytes), "r"(smem_u32(bar))
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

__device__ __forceinline__ void tmem_ld16(uint32_t addr, float* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, "
      "%12, %13, %14, %15}, [%16];"
      : "=f"(r[0]), "=f"(r[1]), "=f"(r[2]), "=f"(r[3]), "=f"(r[4]), "=f"(r[5]), "=f"(r[6]),
        "=f"(r[7]), "=f"(r[8]), "=f"(r[9]), "=f"(r[10]), "=f"(r[11]), "=f"(r[12]), "=f"(r[13]),
        "=f"(r[14]), "=f"(r[15])
      : "r"(addr));
}
template <int N> __device__ __forceinline__ void tmem_ld(uint32_t addr, float (&r)[N]) {
#pragma unroll
  for (int j = 0; j < N; j += 16) tmem_ld16(addr + j, r + j);
}
__device__ __forceinline__ void tmem_st8(uint32_t addr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"r"(addr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
      : "memory");
}

// Matrix descriptors of tiles in the 128-byte swizzle, as the low word and the
// high one (stride byte offset 1024, version 1, layout 2). K-major: the rows are
// M or N. MN-major: the rows are K, the next 64 columns one slab further.
constexpr uint32_t kDescHigh = (1024u >> 4) | (1u << 14) | (2u << 29);
__device__ __forceinline__ uint32_t desc_k(uint32_t addr) { return (addr >> 4) | (1u << 16); }
__device__ __forceinline__ uint32_t desc_mn(uint32_t addr) {
  return (addr >> 4) | ((uint32_t)(kSlab >> 4) << 16);
}
// Instruction descriptor of kind::f16: D fp32, A and B fp16, B MN-major in bit
// 16, N >> 3 in [17,23), M >> 4 in [24,29); M = 128.
__host__ __device__ constexpr uint32_t idesc(int n, bool b_mn) {
  return (1u << 4) | ((uint32_t)b_mn << 16) | ((uint32_t)(n >> 3) << 17) |
         ((uint32_t)(128 >> 4) << 24);
}

__device__ __forceinline__ uint32_t elect_one() {
  uint32_t leader;
  asm volatile(
      "{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}\n"
      : "=r"(leader));
  return leader;
}
// D += A B with A in tensor memory (issued by a converged warp, one lane's
// predicate on the instruction).
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

// A bounded wait that also ends when another thread's has run out (what that means
// for the caller is said once, at the kernel's end: few instructions here, where
// the roles' code competes for the instruction cache). No hint on how long a try may
// park the warp: with one of 2 us a chunk took 3% longer.
__device__ __forceinline__ bool wait_or_leave(uint64_t* bar, uint32_t parity, int* gave_up) {
#pragma unroll 1
  for (int tries = 0; tries < (1 << 22); ++tries) {
    uint32_t done;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}\n"
        : "=r"(done)
        : "r"(smem_u32(bar)), "r"(parity)
        : "memory");
    if (done) return true;
    if (*reinterpret_cast<volatile int*>(gave_up)) return false;
  }
  *reinterpret_cast<volatile int*>(gave_up) = 1;
  return false;
}

// ------------------------------------------------------------- small pieces

// N values times f as fp16 hi and lo, into N / 2 columns of tensor memory each.
// hi is cut off to 11 bits, not rounded: a mask instead of the two conversions
// back from fp16, which run at half rate; lo then has up to 2^-10 of the value
// and both together 21 bits.
template <int N>
__device__ __forceinline__ void store_parts(uint32_t hi_at, uint32_t lo_at, const float* x, float f) {
#pragma unroll
  for (int b = 0; b < N / 16; ++b) {
    uint32_t hi[8], lo[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      float2 v = make_float2(x[16 * b + 2 * i], x[16 * b + 2 * i + 1]);
      v = __fmul2_rn(v, make_float2(f, f));
      const float2 h = make_float2(__uint_as_float(__float_as_uint(v.x) & 0xffffe000u),
                                   __uint_as_float(__float_as_uint(v.y) & 0xffffe000u));
      hi[i] = pack_half2(h.x, h.y);
      v = __ffma2_rn(h, make_float2(-1.f, -1.f), v);
      lo[i] = pack_half2(v.x, v.y);
    }
    tmem_st8(hi_at + 8 * b, hi);
    tmem_st8(lo_at + 8 * b, lo);
  }
}

__device__ __forceinline__ float2 twice(float x) { return make_float2(x, x); }

// N floats at a multiple of 16 bytes.
template <int N> __device__ __forceinline__ void load_floats(float (&x)[N], const float* p) {
#pragma unroll
  for (int j = 0; j < N; j += 4)
    *reinterpret_cast<float4*>(x + j) = *reinterpret_cast<const float4*>(p + j);
}

template <int N> __device__ __forceinline__ float largest_of(const float (&x)[N]) {
  float a = 0.f, b = 0.f;
#pragma unroll
  for (int i = 0; i < N; i += 4) {
    a = max3(a, fabsf(x[i]), fabsf(x[i + 1]));
    b = max3(b, fabsf(x[i + 2]), fabsf(x[i + 3]));
  }
  return fmaxf(a, b);
}

// The products of A's parts and a tile over K = 16 steps, hi hi + lo hi (+ hi lo):
// A's parts `a_part` columns apart, B's `b_part` (>> 4) apart. With kHalf 0 or 1
// the steps whose A is the first or the second half of a computing warp's part.
template <int kSteps, bool kBLow, int kHalf = -1>
__device__ __forceinline__ void products(uint32_t leader, uint32_t d, uint32_t a, uint32_t a_part,
                                         uint32_t b, uint32_t b_step, uint32_t b_slab,
                                         uint32_t b_part, uint32_t desc) {
  constexpr int kOf = kSteps / kParts / 2;  // steps of such a half
  uint32_t more = kHalf == 1;
#pragma unroll
  for (int s = 0; s < kSteps; ++s) {
    if (kHalf >= 0 && s / kOf % 2 != kHalf) continue;
    const uint32_t at = b + (uint32_t)(s / 4) * b_slab + (uint32_t)(s % 4) * b_step;
    mma_ts(leader, d, a + 8 * s, at, desc, more);
    more = 1;
    mma_ts(leader, d, a + a_part + 8 * s, at, desc, 1u);
    if constexpr (kBLow) mma_ts(leader, d, a + 8 * s, at + b_part, desc, 1u);
  }
}

// ------------------------------------------------------------------ kernel

template <typename T, int DKP>
__global__ void __launch_bounds__(kThreads, 1)
    tiles_kernel(const __grid_constant__ TileMaps maps, const Params p) {
  using C = TilesCfg<DKP>;
  constexpr int kS = DKP / kParts;  // state elements of a thread
  extern __shared__ uint8_t smem_raw[];
  typename C::Smem& sm = *reinterpret_cast<typename C::Smem*>(
      smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u));
  const mamba_gated_delta_args& a = p.a;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int H = (int)a.heads, dk = (int)a.dk, dv = (int)a.dv, L = (int)a.seqlen;
  const int tile = (int)(blockIdx.x % (unsigned)p.tiles);
  const int64_t bh = blockIdx.x / (unsigned)p.tiles;
  const int b = (int)(bh / H), h = (int)(bh % H), g = h / (int)(a.heads / a.groups);
  const int col0 = tile * kLanes;
  if (threadIdx.x == 0) {
    for (int s = 0; s < 2; ++s) {
      mamba_scan::mbar_init(&sm.full[s], 1);
      mamba_scan::mbar_init(&sm.out_full[s], 1);
      mamba_scan::mbar_init(&sm.converted[s], kHelpers);
      mamba_scan::mbar_init(&sm.s_done[s], 1);
    }
    for (uint64_t* bar : {&sm.s_ready[0], &sm.s_ready[1], &sm.r_ready[0], &sm.r_ready[1],
                          &sm.u_ready[0], &sm.u_ready[1], &sm.uo_ready})
      mamba_scan::mbar_init(bar, kWarps);
    for (uint64_t* bar : {&sm.o_read, &sm.o_free})
      mamba_scan::mbar_init(bar, kHelpers);
    for (uint64_t* bar : {&sm.x_done, &sm.u_done, &sm.o_done, &sm.o_sent})
      mamba_scan::mbar_init(bar, 1);
    sm.gave_up = 0;
    mamba_scan::fence_mbarrier_init();
  }
  if (warp == kIssueWarp) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(
                     smem_u32(&sm.tmem))
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = sm.tmem;
  // (the next launch, prepare_kernel over later chunks, may start only once
  // everything before this one is done: it writes the records read by then)
  mamba_scan::pdl_wait();
  mamba_scan::pdl_trigger();
  const int len_all = clamped_length(a.lengths, b, L);
  const int c_end = min(p.c1, (len_all + kChunk - 1) / kChunk);
  const int n = max(c_end - p.c0, 0);  // chunks with rows that count
  int* gave_up = &sm.gave_up;

  if (warp >= kWarps + kHelpers) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kOtherRegs));
    if (warp == kLoadWarp && lane == 0) {
      const TileRecord* recs = static_cast<const TileRecord*>(p.records) + bh * (p.c1 - p.c0);
      const bool two = dv - col0 > 64;  // slabs of v with columns
      auto load = [&](int i) {
        if (i >= n) return;
        typename C::Stage& st = sm.stage[i & 1];
        const int t0 = (p.c0 + i) * kChunk;
        uint64_t* bar = &sm.full[i & 1];
        mamba_scan::mbar_arrive_expect_tx(
            bar, 2 * C::kSlabs * kSlab + (two ? 2 : 1) * kSlab + (uint32_t)sizeof(TileMain));
#pragma unroll
        for (int s = 0; s < C::kSlabs; ++s) {
          tma_load_4d(smem_u32(st.k + s * kSlab), &maps.k, bar, 64 * s, g, t0, b);
          tma_load_4d(smem_u32(st.q + s * kSlab), &maps.q, bar, 64 * s, g, t0, b);
        }
        bulk_load(smem_u32(&st.rec), &recs[i].main, (uint32_t)sizeof(TileMain), bar);
        tma_load_4d(smem_u32(st.v), &maps.v, bar, col0, h, t0, b);
        if (two) tma_load_4d(smem_u32(st.v + kSlab), &maps.v, bar, col0 + 64, h, t0, b);
      };
      auto load_out = [&](int i) {
        if (i >= n) return;
        mamba_scan::mbar_arrive_expect_tx(&sm.out_full[i & 1], (uint32_t)sizeof(TileOut));
        bulk_load(smem_u32(&sm.out[i & 1].rec), &recs[i].out, (uint32_t)sizeof(TileOut),
                  &sm.out_full[i & 1]);
      };
      load(0);
      load(1);
      load_out(0);
      load_out(1);
      bool ok = true;
      int i = 0;
      for (; i < n; ++i) {
        // (the state's update is chunk i's last use of k, q, T and their factors)
        if (!(ok = wait_or_leave(&sm.s_done[i & 1], (uint32_t)(i >> 1) & 1u, gave_up))) break;
        load(i + 2);
        if (!(ok = wait_or_leave(&sm.o_free, (uint32_t)i & 1u, gave_up))) break;
        load_out(i + 2);
        if (p.out_vec) {
          const int t0 = (p.c0 + i) * kChunk;
          tma_store_4d(&maps.out, smem_u32(sm.o), col0, h, t0, b);
          if (two) tma_store_4d(&maps.out, smem_u32(sm.o + kSlab), col0 + 64, h, t0, b);
          mamba_scan::bulk_commit();
          mamba_scan::bulk_wait_read<0>();
        }
        mbar_arrive(&sm.o_sent);
      }
      if (!ok)  // let the copies in flight land
        for (int j = i; j < min(i + 3, n); ++j) {
          mamba_scan::mbar_wait(&sm.full[j & 1], (uint32_t)(j >> 1) & 1u, &g_tiles_error, 50000000ull);
          mamba_scan::mbar_wait(&sm.out_full[j & 1], (uint32_t)(j >> 1) & 1u, &g_tiles_error,
                                50000000ull);
        }
      mamba_scan::bulk_wait_all<0>();
    }
    if (warp == kIssueWarp) {
      const uint32_t leader = elect_one();
      constexpr int kSteps = DKP / 16;
      constexpr uint32_t kRow = 32 >> 4, kDeep = 2048 >> 4, kNext = kSlab >> 4;
      auto outputs = [&](int i) {  // O2 of chunk i, in the place of its state's update
        if (!wait_or_leave(&sm.uo_ready, (uint32_t)i & 1u, gave_up) ||
            !wait_or_leave(&sm.out_full[i & 1], (uint32_t)(i >> 1) & 1u, gave_up))
          return false;
        tc_fence_after();
        products<4, true>(leader, tmem + C::kColD, tmem + C::kColU, 32,
                          desc_k(smem_u32(sm.out[i & 1].rec.p[0])), kRow, 0, kNext, idesc(64, false));
        mma_commit(leader, &sm.o_done);
        return true;
      };
      for (int i = 0; i < n; ++i) {
        const uint32_t now = (uint32_t)i & 1u;
        typename C::Stage& st = sm.stage[i & 1];
        if (!wait_or_leave(&sm.converted[i & 1], (uint32_t)(i >> 1) & 1u, gave_up) ||
            !wait_or_leave(&sm.s_ready[0], now, gave_up))
          break;
        tc_fence_after();
        products<kSteps, false, 0>(leader, tmem + C::kColX, tmem + C::kColS, DKP / 2,
                                   desc_k(smem_u32(st.k)), kRow, kNext, 0, idesc(64, false));
        if (!wait_or_leave(&sm.s_ready[1], now, gave_up)) break;
        tc_fence_after();
        products<kSteps, false, 1>(leader, tmem + C::kColX, tmem + C::kColS, DKP / 2,
                                   desc_k(smem_u32(st.k)), kRow, kNext, 0, idesc(64, false));
        mma_commit(leader, &sm.x_done);
        if (i > 0 && !outputs(i - 1)) break;  // (s_ready: the update has been read)
        if (!wait_or_leave(&sm.r_ready[0], now, gave_up)) break;
        tc_fence_after();
        products<4, true, 0>(leader, tmem + C::kColX, tmem + C::kColR, 32,
                             desc_k(smem_u32(st.rec.t[0])), kRow, 0, kNext, idesc(64, false));
        if (!wait_or_leave(&sm.r_ready[1], now, gave_up)) break;
        tc_fence_after();
        products<4, true, 1>(leader, tmem + C::kColX, tmem + C::kColR, 32,
                             desc_k(smem_u32(st.rec.t[0])), kRow, 0, kNext, idesc(64, false));
        mma_commit(leader, &sm.u_done);
        if (i > 0 && !wait_or_leave(&sm.o_read, now ^ 1u, gave_up)) break;
        tc_fence_after();
        products<kSteps, false>(leader, tmem + C::kColO1, tmem + C::kColS, DKP / 2,
                                desc_k(smem_u32(st.q)), kRow, kNext, 0, idesc(64, false));
        if (!wait_or_leave(&sm.u_ready[0], now, gave_up)) break;
        tc_fence_after();
        products<4, false, 0>(leader, tmem + C::kColD, tmem + C::kColR, 32, desc_mn(smem_u32(st.k)),
                              kDeep, 0, 0, idesc(DKP, true));
        if (!wait_or_leave(&sm.u_ready[1], now, gave_up)) break;
        tc_fence_after();
        products<4, false, 1>(leader, tmem + C::kColD, tmem + C::kColR, 32, desc_mn(smem_u32(st.k)),
                              kDeep, 0, 0, idesc(DKP, true));
        mma_commit(leader, &sm.s_done[i & 1]);
      }
      if (n > 0 && wait_or_leave(&sm.s_ready[1], (uint32_t)n & 1u, gave_up)) outputs(n - 1);
    }
    __syncwarp();
  } else if (warp >= kWarps) {  // -------------------- conversions and outputs
    // (like the computing warps these go through every chunk even when a wait has
    // run out, since warps meet at barriers: every later wait then ends at once)
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kHelperRegs));
    const int quarter = warp & 3, at_lane = 32 * quarter + lane, me = threadIdx.x - 32 * kWarps;
    const int col = col0 + at_lane;
    const uint32_t mine = tmem + ((uint32_t)(32 * quarter) << 16);
    // q and k of a stage as the products take them: bf16 rows scaled and as fp16,
    // rows that do not count as zeros
    auto convert = [&](int i) {
      typename C::Stage& st = sm.stage[i & 1];
      wait_or_leave(&sm.full[i & 1], (uint32_t)(i >> 1) & 1u, gave_up);
      const int len = len_all - (p.c0 + i) * kChunk;
      if (!std::is_same<T, __half>::value || len < kChunk) {
        constexpr int kPieces = kSlab / 16 / (32 * kHelpers);  // of a slab, to a thread
#pragma unroll 1  // (the roles' code together is more than the instruction cache holds)
        for (int s = 0; s < kPieces; ++s) {
          const int piece = s * 32 * kHelpers + me, t = piece >> 3;
          const float ks = st.rec.k_scale[t], qs = st.rec.q_scale[t];
#pragma unroll
          for (int slab = 0; slab < 2 * C::kSlabs; ++slab) {
            uint8_t* at = piece * 16 + (slab < C::kSlabs ? st.k + slab * kSlab
                                                         : st.q + (slab - C::kSlabs) * kSlab);
            uint4 w = *reinterpret_cast<const uint4*>(at);
            if constexpr (!std::is_same<T, __half>::value) {
              const float2 f = twice(slab < C::kSlabs ? ks : qs);
              uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
              for (int j = 0; j < 4; ++j) {
                const float2 v = __fmul2_rn(make_float2(__uint_as_float(u[j] << 16),
                                                        __uint_as_float(u[j] & 0xffff0000u)), f);
                u[j] = pack_half2(v.x, v.y);
              }
              w = make_uint4(u[0], u[1], u[2], u[3]);
            }
            if (t >= len) w = make_uint4(0, 0, 0, 0);
            *reinterpret_cast<uint4*>(at) = w;
          }
        }
        mamba_scan::fence_proxy_async_smem();
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&sm.converted[i & 1]);
    };
    T* out = static_cast<T*>(a.out) + ((int64_t)b * L * H + h) * dv + col;
    const int64_t row = (int64_t)H * dv;
    if (n > 0) convert(0);
    for (int i = 0; i < n; ++i) {
      if (i + 1 < n) convert(i + 1);
      // a lane's outputs of chunk i, from O1 and O2: to shared memory, from where
      // they go by TMA, or straight to rows that TMA cannot take
      const TileOut& rec = sm.out[i & 1].rec;
      wait_or_leave(&sm.out_full[i & 1], (uint32_t)(i >> 1) & 1u, gave_up);
      if (i > 0) wait_or_leave(&sm.o_sent, (uint32_t)(i - 1) & 1u, gave_up);
      wait_or_leave(&sm.o_done, (uint32_t)i & 1u, gave_up);
      __syncwarp();
      tc_fence_after();
      const float2 si = twice(sm.s_inv[i & 1][at_lane]), pu = twice(sm.u_inv[i & 1][at_lane] * rec.p_inv);
      const int t0 = (p.c0 + i) * kChunk, len = len_all - t0;
#pragma unroll 1
      for (int j0 = 0; j0 < kChunk; j0 += 32) {
        float o[32], d[32], fac[32];
        tmem_ld(mine + C::kColO1 + j0, o);
        tmem_ld(mine + C::kColD + j0, d);
        load_floats(fac, rec.o_fac + j0);
        tmem_wait_ld();
        if (j0 + 32 == kChunk) {
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&sm.o_read);
        }
#pragma unroll
        for (int j = 0; j < 32; j += 2) {
          const float2 v = __ffma2_rn(make_float2(d[j], d[j + 1]), pu,
                                      __fmul2_rn(make_float2(o[j], o[j + 1]),
                                                 __fmul2_rn(make_float2(fac[j], fac[j + 1]), si)));
          o[j] = v.x;
          o[j + 1] = v.y;
        }
        if (len < kChunk)
#pragma unroll
          for (int j = 0; j < 32; ++j)
            if (j0 + j >= len) o[j] = 0.f;
        if (p.out_vec) {
          T* to = reinterpret_cast<T*>(sm.o + (at_lane >> 6) * kSlab) + j0 * 64 + (at_lane & 63);
#pragma unroll
          for (int j = 0; j < 32; ++j) to[64 * j] = from_f32<T>(o[j]);
        } else if (col < dv) {
          T* to = out + (t0 + j0) * row;
#pragma unroll
          for (int j = 0; j < 32; ++j)
            if (t0 + j0 + j < L) to[j * row] = from_f32<T>(o[j]);
        }
      }
      if (p.out_vec) mamba_scan::fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(&sm.o_free);
    }
    // rows of chunks past the length
    if (col < dv)
      for (int t = (p.c0 + n) * kChunk; t < min(p.c1 * kChunk, L); ++t) out[t * row] = from_f32<T>(0.f);
  } else {  // ------------------------------------------------------- the chain
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kComputeRegs));
    const int quarter = warp & 3, part = warp >> 2, at_lane = 32 * quarter + lane;
    const int col = col0 + at_lane;
    const bool col_ok = col < dv;
    const uint32_t mine = tmem + ((uint32_t)(32 * quarter) << 16);
    float S[kS];  // rows (dk) kS part ..
    {
      const float* in = p.state_in + bh * dk * dv + col;
#pragma unroll
      for (int j = 0; j < kS; ++j) {
        const int k = kS * part + j;
        S[j] = p.state_in != nullptr && col_ok && k < dk ? in[(int64_t)k * dv] : 0.f;
      }
    }
    // the largest of a lane's threads' values, through shared memory: the warps of
    // a quarter meet at a barrier (none of them leaves before the last chunk: once a
    // wait has run out, every later one ends at once)
    auto compare = [&](float m, int which) {
      float(*all)[kLanes] = sm.largest[which];
      all[part][at_lane] = m;
      asm volatile("bar.sync %0, %1;" ::"r"(1 + quarter), "n"(32 * kParts) : "memory");
#pragma unroll
      for (int i = 1; i < kParts; ++i) m = fmaxf(m, all[(part + i) % kParts][at_lane]);
      return m;
    };
    auto arrive = [&](uint64_t* bar) {
      tmem_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(bar);
    };
    auto product = [&](uint64_t* bar, uint32_t parity) {  // is done
      wait_or_leave(bar, parity, gave_up);
      __syncwarp();
      tc_fence_after();
    };
    float largest = compare(largest_of(S), 0);
    for (int i = 0; i < n; ++i) {
      const uint32_t now = (uint32_t)i & 1u;
      typename C::Stage& st = sm.stage[i & 1];
      const TileMain& rec = st.rec;
      const int e = scale_exponent(largest);
      const float s_inv = pow2i(-e);
      if (part == 0) sm.s_inv[now][at_lane] = s_inv;
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const uint32_t to = mine + C::kColS + kS / 2 * part + kS / 4 * half;
        store_parts<kS / 2>(to, to + DKP / 2, S + kS / 2 * half, pow2i(e));
        arrive(&sm.s_ready[half]);
      }
      // R = V - weighted X, this thread's rows
      const int len = len_all - (p.c0 + i) * kChunk - kRows * part;
      float x[kRows], v[kRows], fac[kRows];
      wait_or_leave(&sm.full[now], (uint32_t)(i >> 1) & 1u, gave_up);
      load_floats(fac, rec.x_fac + kRows * part);
      {
        const uint8_t* at = st.v + (at_lane >> 6) * kSlab + kRows * part * 128 + (at_lane & 7) * 2;
        const int piece = (at_lane & 63) >> 3;
#pragma unroll
        for (int j = 0; j < kRows; ++j)
          v[j] = to_f32(*reinterpret_cast<const T*>(at + j * 128 + ((piece ^ (j & 7)) << 4)));
      }
      product(&sm.x_done, now);
      tmem_ld(mine + C::kColX + kRows * part, x);
      tmem_wait_ld();
#pragma unroll
      for (int j = 0; j < kRows; j += 2) {
        const float2 r = __ffma2_rn(make_float2(x[j], x[j + 1]),
                                    __fmul2_rn(make_float2(fac[j], fac[j + 1]), twice(-s_inv)),
                                    make_float2(v[j], v[j + 1]));
        x[j] = r.x;
        x[j + 1] = r.y;
      }
      if (len < kRows)  // rows that do not count, whatever they hold
#pragma unroll
        for (int j = 0; j < kRows; ++j)
          if (j >= len) x[j] = 0.f;
      const int er = scale_exponent(compare(largest_of(x), 1));
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const uint32_t to = mine + C::kColR + kRows / 2 * part + kRows / 4 * half;
        store_parts<kRows / 2>(to, to + 32, x + kRows / 2 * half, pow2i(er));
        arrive(&sm.r_ready[half]);
      }
      load_floats(fac, rec.u_fac + kRows * part);
      const float r_inv = pow2i(-er) * rec.t_inv, w_inv = rec.u_inv, carry = rec.carry;
      product(&sm.u_done, now);
      tmem_ld(mine + C::kColX + kRows * part, x);
      tmem_wait_ld();
      // U weighted by what decays until the chunk's end, for the state's update;
      // and U, for the outputs, whose product comes after the next chunk's X
#pragma unroll
      for (int j = 0; j < kRows; j += 2) {
        const float2 w = __fmul2_rn(make_float2(x[j], x[j + 1]), make_float2(fac[j], fac[j + 1]));
        v[j] = w.x, v[j + 1] = w.y;
      }
      const int ew = scale_exponent(compare(largest_of(v), 0));
      const float d_inv = pow2i(-ew) * r_inv * w_inv;
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const uint32_t to = mine + C::kColR + kRows / 2 * part + kRows / 4 * half;
        store_parts<kRows / 2>(to, to + 32, v + kRows / 2 * half, pow2i(ew));
        arrive(&sm.u_ready[half]);
      }
      const int eu = scale_exponent(compare(largest_of(x), 1));
      if (part == 0) sm.u_inv[now][at_lane] = pow2i(-eu) * r_inv;
      store_parts<kRows>(mine + C::kColU + kRows / 2 * part,
                         mine + C::kColU + 32 + kRows / 2 * part, x, pow2i(eu));
      arrive(&sm.uo_ready);
      product(&sm.s_done[i & 1], (uint32_t)(i >> 1) & 1u);
      float d[kS];
      tmem_ld(mine + C::kColD + kS * part, d);
      tmem_wait_ld();
#pragma unroll
      for (int j = 0; j < kS; j += 2) {
        const float2 w = __ffma2_rn(make_float2(d[j], d[j + 1]), twice(d_inv),
                                    __fmul2_rn(twice(carry), make_float2(S[j], S[j + 1])));
        S[j] = w.x;
        S[j + 1] = w.y;
      }
      tc_fence_before();
      largest = compare(largest_of(S), 0);
    }
    if (n > 0) arrive(&sm.s_ready[1]);  // (the last update has been read)
    if (p.state_out != nullptr && col_ok) {
      float* to = p.state_out + bh * dk * dv + col;
#pragma unroll
      for (int j = 0; j < kS; ++j) {
        const int k = kS * part + j;
        if (k < dk) to[(int64_t)k * dv] = S[j];
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (threadIdx.x == 0 && sm.gave_up)
    atomicExch(&g_tiles_error, 6);  // MAMBA_SCAN_ERR_DEVICE_TIMEOUT
  if (warp == kIssueWarp) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
  }
}

// -------------------------------------------------------------------- host

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

// [batch][rows][heads][width] with strides, boxes of 64 rows x 64 columns.
// False when TMA cannot take it (alignment, strides).
bool encode(CUtensorMap* m, const void* ptr, int32_t dtype, int64_t width, int64_t heads,
            int64_t rows, int64_t batch, const int64_t* stride, bool swizzle = true) {
  auto enc = encode_fn();
  if (enc == nullptr || !mamba_lm::aligned16(ptr)) return false;
  const int64_t n[3] = {heads, rows, batch}, st[3] = {stride[2], stride[1], stride[0]};
  const cuuint64_t dims[4] = {(cuuint64_t)width, (cuuint64_t)heads, (cuuint64_t)rows,
                              (cuuint64_t)batch};
  cuuint64_t bytes[3];
  for (int i = 0; i < 3; ++i) {
    // the stride of a dimension of one element is never used: any valid one
    const int64_t by = n[i] == 1 ? 16 : st[i] * 2;
    if (by % 16 != 0 || by <= 0 || by >= (int64_t)1 << 40) return false;
    bytes[i] = (cuuint64_t)by;
  }
  const cuuint32_t box[4] = {64, 1, kChunk, 1}, es[4] = {1, 1, 1, 1};
  return enc(m, dtype == MAMBA_DTYPE_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16
                                         : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16,
             4, const_cast<void*>(ptr), dims, bytes, box, es, CU_TENSOR_MAP_INTERLEAVE_NONE,
             swizzle ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_NONE,
             CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
             CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <typename T, int DKP>
cudaError_t launch_typed(const TileMaps& maps, const Params& p, cudaStream_t st) {
  auto kernel = tiles_kernel<T, DKP>;
  cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                       (int)TilesCfg<DKP>::kBytes);
  if (e != cudaSuccess) return e;
  // (warps that ask for more registers than the launch has would wait for good)
  cudaFuncAttributes attr;
  e = cudaFuncGetAttributes(&attr, kernel);
  if (e != cudaSuccess) return e;
  if (attr.numRegs < kLaunchRegs) return cudaErrorLaunchOutOfResources;
  return mamba_scan::launch_pdl(kernel, dim3((unsigned)(p.a.batch * p.a.heads * p.tiles)),
                                dim3(kThreads), TilesCfg<DKP>::kBytes, st, maps, p);
}

}  // namespace

bool tiles_take(const mamba_gated_delta_args& a, TileMaps* maps) {
  if (a.dtype == MAMBA_DTYPE_F32) return false;
  std::memset(maps, 0, sizeof(*maps));
  const int64_t out_stride[3] = {a.seqlen * a.heads * a.dv, a.heads * a.dv, a.dv};
  maps->out_taken = encode(&maps->out, a.out, a.dtype, a.dv, a.heads, a.seqlen, a.batch, out_stride,
                           false);
  return encode(&maps->q, a.q, a.dtype, a.dk, a.groups, a.seqlen, a.batch, a.q_stride) &&
         encode(&maps->k, a.k, a.dtype, a.dk, a.groups, a.seqlen, a.batch, a.k_stride) &&
         encode(&maps->v, a.v, a.dtype, a.dv, a.heads, a.seqlen, a.batch, a.v_stride);
}

cudaError_t launch_tiles(const TileMaps& maps, const Params& p0, cudaStream_t st) {
  Params p = p0;
  p.tiles = (int)((p.a.dv + kLanes - 1) / kLanes);
  p.out_vec = maps.out_taken;
  if (p.a.dtype == MAMBA_DTYPE_F16)
    return p.a.dk <= 64 ? launch_typed<__half, 64>(maps, p, st)
                        : launch_typed<__half, 128>(maps, p, st);
  return p.a.dk <= 64 ? launch_typed<__nv_bfloat16, 64>(maps, p, st)
                      : launch_typed<__nv_bfloat16, 128>(maps, p, st);
}

int read_and_clear_tiles_error() {
  int v = 0;
  if (cudaMemcpyFromSymbol(&v, g_tiles_error, sizeof(int)) != cudaSuccess) return -1;
  if (v != 0) {
    const int zero = 0;
    cudaMemcpyToSymbol(g_tiles_error, &zero, sizeof(int));
  }
  return v;
}

}  // namespace mamba_gd
