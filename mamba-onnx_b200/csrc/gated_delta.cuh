// What the kernels of the gated delta rule over prompts share: the records of
// chunks that prepare_kernel leaves (gated_delta_mma.cu) to the two chain
// kernels (there, and gated_delta_tiles.cu), and small device pieces.
#pragma once

#include <cuda.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "gated_delta.h"
#include "lm_device.cuh"
#include "scan_device.cuh"

namespace mamba_gd {

constexpr int kChunk = 64;
constexpr int kBlocks = 10;  // 16 x 16 blocks of a lower triangle of 64 rows

// What prepare_kernel leaves of a chunk. T and P as the right operands' own
// fragments: block (w, j) holds rows 16 w.. and columns 16 j.., for each lane
// 16 bytes: rows 16w + lane/4 (x, y) and + 8 (z, w), columns 16 j + 2
// (lane % 4) + {0, 1} (x, z) and + 8 (y, w).
struct __align__(16) ChainRecord {  // what the chain reads
  uint4 t[2][kBlocks][32];  // hi, lo
  float x_fac[kChunk];      // of K S's rows:     2^(G_s - e(k_s))
  float u_fac[kChunk];      // of U's rows:       2^(G_C - G_s - e(k_s))
  float carry;              // 2^G_C
  float t_inv;              // 2^-e(T)
  float pad[2];
  float k_scale[kChunk];    // 2^e(k_t), for the rows' conversion
};
struct __align__(16) OutRecord {    // what the outputs read
  uint4 p[2][kBlocks][32];
  float o_fac[kChunk];      // of Q S's rows:     scale 2^(G_t - e(q_t))
  float p_inv;              // scale 2^-e(P)
  float pad[3];
  float q_scale[kChunk];
};
struct __align__(16) Record {
  ChainRecord chain;
  OutRecord out;
};
static_assert(sizeof(ChainRecord) % 16 == 0 && sizeof(OutRecord) % 16 == 0,
              "copied 16 bytes at a time");

// The same for the kernel that keeps the state in tensor memory: T and P as whole
// tiles of 64 rows of 128 bytes in the 128-byte swizzle, hi then lo, and U's
// factors brought to at most 1.
struct __align__(16) TileMain {
  uint8_t t[2][kChunk * 128];
  float x_fac[kChunk], u_fac[kChunk];
  float k_scale[kChunk], q_scale[kChunk];
  float carry, t_inv;
  float u_inv;              // what undoes u_fac's scale
  float pad;
};
struct __align__(16) TileOut {
  uint8_t p[2][kChunk * 128];
  float o_fac[kChunk];
  float p_inv;
  float pad[3];
};
struct __align__(16) TileRecord {
  TileMain main;
  TileOut out;
};
static_assert(sizeof(TileMain) % 16 == 0 && sizeof(TileOut) % 16 == 0, "copied in bulk");

template <typename T> struct Parts { static constexpr int n = 1; };
template <> struct Parts<float> { static constexpr int n = 2; };

struct Params {
  mamba_gated_delta_args a;
  void* records;           // [sequence and head][chunk - c0] of Record or TileRecord
  const float* state_in;   // NULL: zeros
  float* state_out;        // NULL: not written
  int c0, c1;              // chunks of this launch
  int tiles;               // dv tiles of a head
  int qk_vec;              // rows of q and k start at 16 bytes
  int v_vec, out_vec;
};

// The exponent e with |x| 2^e in [2^14, 2^15) for the largest |x| of a row (at
// most 126: rows of tiny values stay finite).
__device__ __forceinline__ int scale_exponent(float largest) {
  return min(141 - (int)(__float_as_uint(largest) >> 23), 126);
}
__device__ __forceinline__ float pow2i(int e) { return __int_as_float((e + 127) << 23); }

__device__ __forceinline__ uint32_t pack_half2(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// A pair as fp16 hi + lo, each to nearest.
__device__ __forceinline__ void split_half2(float x, float y, uint32_t& hi, uint32_t& lo) {
  const __half2 h = __floats2half2_rn(x, y);
  const float2 f = __half22float2(h);
  hi = *reinterpret_cast<const uint32_t*>(&h);
  lo = pack_half2(x - f.x, y - f.y);
}

__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

__device__ __forceinline__ int clamped_length(const int32_t* lengths, int b, int seqlen) {
  if (lengths == nullptr) return seqlen;
  const int n = lengths[b];
  return n < 0 ? 0 : (n > seqlen ? seqlen : n);
}

__device__ __forceinline__ void mbar_arrive(uint64_t* bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(mamba_scan::smem_u32(bar)) : "memory");
}

// The chain over tensor memory (gated_delta_tiles.cu): q, k and v of 16-bit
// types by TMA, and the outputs where it can write them.
struct TileMaps {
  CUtensorMap q, k, v, out;
  int out_taken;
};
// Whether it takes this call; fills the maps then.
bool tiles_take(const mamba_gated_delta_args& a, TileMaps* maps);
// Enqueues it over chunks p.c0 .. p.c1, whose TileRecords are in p.records.
cudaError_t launch_tiles(const TileMaps& maps, const Params& p, cudaStream_t st);
int read_and_clear_tiles_error();

}  // namespace mamba_gd
