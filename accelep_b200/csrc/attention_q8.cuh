// What the attention kernels over the int8 key/value cache share: their
// arguments, the exact fp16 form of int8 elements, and fp16 pairs of fp32
// queries and weights.
#pragma once

#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "accel_b200.h"
#include "common.cuh"
#include "q8_cache.cuh"

namespace accel_b200 {

constexpr float kSlack = 4.f;  // how far (in powers of two) a score may pass the softmax reference before it moves
constexpr float kBias = 10.f;  // weights are 2^(score - reference + kBias)
constexpr float kLog2e = 1.4426950408889634f;

struct AttnArgs {
  const float* q;
  int64_t q_ld;
  accel_b200_q8_cache cache;
  RaggedRows rows;         // prefill: rows by sequence
  const int32_t* row_seq;  // single rows: slot (null: the row's number) and position
  const int32_t* row_pos;
  int32_t single_rows;     // how many of them
  int32_t sequences;       // prefill: sequences of `rows`
  int32_t by_sequence;     // tiles of one sequence after the other, not the latest of all sequences first
  int32_t heads;
  int32_t group;        // heads per kv head
  int32_t block_shift;  // tokens per scale block, as a power of two
  int32_t window;
  int32_t sinks;
  float scale;
  float* out;
  int64_t out_ld;
  int32_t* status;
  int32_t* counters;  // splits through the workspace: arrivals by vector group, then the CTAs' states
  float* parts;
  accel_b200_l2_prefetch prefetch;  // single rows: ranges for L2, and whether blocks are read before the wait
};

__device__ __forceinline__ float Exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Bytes 0 and 1 (kHi: 2 and 3) of w, each an int8 plus 128, as two fp16
// numbers: 0x6400 | byte is 1024 + byte, less 1152.
template <bool kHi>
__device__ __forceinline__ uint32_t Halves(uint32_t w) {
  const uint32_t x = __byte_perm(w, 0x64646464u, kHi ? 0x4342 : 0x4140);
  const uint32_t k1152 = 0x64806480u;
  const __half2 y = __hsub2(*reinterpret_cast<const __half2*>(&x), *reinterpret_cast<const __half2*>(&k1152));
  return *reinterpret_cast<const uint32_t*>(&y);
}

// (x, y) as fp16 pairs hi + lo, each off by at most 2^-22 of its value.
__device__ __forceinline__ void SplitPair(float x, float y, uint32_t* hi, uint32_t* lo) {
  const __half2 h = __floats2half2_rn(x, y);
  const float2 f = __half22float2(h);
  const __half2 l = __floats2half2_rn(x - f.x, y - f.y);
  *hi = *reinterpret_cast<const uint32_t*>(&h);
  *lo = *reinterpret_cast<const uint32_t*>(&l);
}

// Rows and heads of query vectors v0, v0 + 1, ... (row x head, `group` heads a
// row). 64-bit divisions cost a hundred instructions each, so there is one, and
// none where v0 fits 32 bits.
struct Vectors {
  int64_t row0;
  uint32_t head0, group;
  __device__ __forceinline__ Vectors(int64_t v0, int32_t heads_per_row) : group(static_cast<uint32_t>(heads_per_row)) {
    row0 = v0 <= 0xffffffffll ? static_cast<int64_t>(static_cast<uint32_t>(v0) / group) : v0 / group;
    head0 = static_cast<uint32_t>(v0 - row0 * group);
  }
  // Row behind row0 of vector v0 + i.
  __device__ __forceinline__ uint32_t Down(int i) const { return (head0 + static_cast<uint32_t>(i)) / group; }
  __device__ __forceinline__ uint32_t Head(int i, uint32_t down) const {
    return head0 + static_cast<uint32_t>(i) - down * group;
  }
};

// First position that a window ending at pos covers.
__device__ __forceinline__ int NearOf(int pos, int window) { return window > 0 ? max(0, pos - window + 1) : 0; }

// Prefill attention on the tcgen05 tensor cores, kTileVectors query vectors per
// SM (attention_q8_tiles.cu).
constexpr int kTileVectors = 256;

// How a call would run there: the bytes of workspace that it takes, and estimates
// by which the kernel is chosen and shared walks are prepared, of the waves of
// CTAs and the 128-token steps of a whole walk. The device alone knows counts and
// positions: sequences shorter than the cache's context take fewer steps, and a
// tile's walk through a window a few more (its own rows, and partly seen tiles at
// the ends of window and sinks). Results do not depend on them.
struct TilesPlan {
  bool split;  // the last wave's walks are shared by several CTAs
  double waves;
  int64_t steps;
  size_t workspace;
};
TilesPlan PlanTilesQ8(const accel_b200_q8_cache& c, int32_t batch, int32_t max_rows, int32_t heads, int32_t window,
                      int32_t sinks);
int LaunchTilesQ8(const AttnArgs& a, const TilesPlan& plan, int32_t max_rows, cudaStream_t stream);

}  // namespace accel_b200
