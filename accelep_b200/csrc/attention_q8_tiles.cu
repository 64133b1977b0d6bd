// Attention of many query rows over the int8 key/value cache on the 5th-
// generation tensor cores (include/accel_b200.h, accel_b200_attention_prefill_q8).
//
// One CTA takes consecutive query vectors (row x head, the heads of one kv head)
// of one sequence, one or two halves of 128, and walks the 128-token tiles that
// any of them sees. Keys and values become fp16 exactly; queries and weights
// are sums of two fp16 numbers (22 bits), the second parts' products summed
// first, so results are fp32 results. Per tile and half:
//
//   S = Qlo K^T + Qhi K^T      128 x 128 x D, operands in shared memory
//   online softmax             one or two threads per vector, S read from TMEM
//   P, lo and hi parts         written over S in TMEM
//   O = Plo V + Phi V          128 x D x 128, A operand from TMEM
//   registers += vscale * O    fp32, rounded to nearest
//
// O is read out per tile, not summed over the context in TMEM: the tensor
// core's running sum rounds towards zero, which drifts over a long context, and
// the value scale and the softmax reference change from tile to tile. Scales
// of the tile's blocks are folded into the weights relative to the largest.
//
// Roles: the first warps are the softmax (while one half, or the SM's other CTA,
// computes, the tensor core works for this one); four turn the int8 tiles that
// TMA brings into fp16 operands with the 128-byte swizzle; one thread of the
// next issues every MMA.
//
// Measured (in a captured graph; called one by one 528 and 63): 2 sequences of 2047
// and fewer rows behind 14000 tokens, 32 heads over 8 kv heads of 128, window 4096:
// 487 us, 490 TFLOP/s of scores and values (twice that in fp16 products). A half's chain (weights 2600 cycles, its four products
// 2800, maximum 900, read-out 500) and the other's overlap to 7000 cycles a tile,
// of which the tensor core works 5600: an M = 128, N = 128, K = 16 product takes
// 102 cycles with A in shared memory, 72 from TMEM. 32 sequences of 512 rows, 9
// heads over 3 of 64: 63 us, by issue slots (55% of them used) and the first and
// last steps of short walks (13000 of a four-tile CTA's 39000 cycles). What brought
// it there, on the first of these: one elected thread instead of lane 0 issuing
// (1617 -> 1250 us), values freed in front of the next scores and four converter
// warps (-> 806), chunk loops kept rolled so that their code stays in the
// instruction cache (-> 632); on the second: one half per CTA (80 -> 76), no 64-bit
// divisions in any role and the first loads ahead of the set-up (-> 69), the longest
// walks first (-> 63). ptxas reports spills (72 to 172 bytes of stores).
//
// Every wait is bounded. A role whose wait runs out notes it and stops, and with
// it stop, each at the end of a wait of its own, the roles that wait for its
// work: a CTA ends after a few wait limits, gives NaN and ORs
// ACCEL_B200_STATUS_COPY_TIMEOUT.
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>

#include <atomic>
#include <string>
#include <type_traits>

#include "accel_b200.h"
#include "attention_q8.cuh"
#include "common.cuh"
#include "q8_cache.cuh"
#include "tcgen05.cuh"
#include "tensor_map.cuh"

namespace accel_b200 {
namespace {

constexpr int kHalf = 128;         // vectors of a half: TMEM lanes
constexpr int kTile = 128;         // tokens per tile
constexpr int kConverters = 4;     // warps
constexpr int kChunk = 32;         // tokens whose scores a thread holds at a time: one scale block at most
constexpr int kChunks = kTile / kChunk;
constexpr int kMostShares = 8;      // CTAs that a walk is split over at most
constexpr uint64_t kLevelsUpTo = 64 << 20;  // bytes of keys and values up to which L2 holds what a wave reads
constexpr int kLeastShare = 4;      // tiles that each of them gets at least (it costs about two to begin and end)
constexpr float kMostLift = 6.f;    // scales of a tile further apart than 2^6 are applied one by one
constexpr int kPanel = 128 * 128;  // bytes of 128 rows x 64 fp16, the swizzle's row length

template <int D>
struct Tiles {
  // Threads that share a vector, each with half of a tile's tokens and half of
  // the dimensions: two where the sums of 64 dimensions leave the registers
  // for it (one is left waiting for its own instructions most of the time).
  static constexpr int kParts = D == 64 ? 2 : 1;
  // Halves of a CTA and CTAs of an SM: 256 vectors in all. Two CTAs, where shared
  // memory and TMEM allow, hide each other's first and last steps; two halves
  // share one conversion of the keys and values.
  static constexpr int kHalves = D == 64 ? 1 : 2, kCtas = 2 / kHalves;
  static_assert(kHalves * kCtas * kHalf == kTileVectors, "");
  static constexpr int kSoftWarps = 4 * kParts * kHalves, kMmaWarp = kSoftWarps + kConverters;
  static constexpr int kThreads = (kSoftWarps + 8) * 32;  // whole warpgroups
  // Registers of the softmax threads and of the others from their start on: in
  // all no more than the launch gives out (a multiple of 8 each). With 8 more or
  // fewer for the others calls take 1 to 4% longer.
  static constexpr int kLaunch = 65536 / (kThreads * kCtas) / 8 * 8;
  static constexpr int kLess = D == 64 ? 32 : 48, kMore = kLaunch + (kLaunch - kLess) * 256 / (kSoftWarps * 32);
  static_assert(kMore % 8 == 0 && kSoftWarps * 32 * kMore + 256 * kLess <= kThreads * kLaunch, "");
  static constexpr int kPanels = D / 64;
  static constexpr int kOperand = kPanels * kPanel;     // a 128 x D fp16 operand
  static constexpr int kQ = 0;                          // [half][hi, lo]
  static constexpr int kK = kQ + 2 * kHalves * kOperand;
  static constexpr int kV = kK + kOperand;
  static constexpr int kRaw = kV + kOperand;            // int8 tiles as they come: keys, values
  static constexpr int kRawBytes = kTile * D;
  static constexpr int kBars = kRaw + 2 * kRawBytes;
  static constexpr int kShared = kBars + 256;           // float [half][vector] and [2][half][part][vector]
  static constexpr int kBytes = kShared + (kParts > 1 ? (1 + 2 * kParts) * kHalves * 128 * 4 : 0);
  static constexpr int kAlign = 1024;
  static_assert((kBytes + kAlign + 1024) * kCtas <= 228 * 1024, "shared memory of an SM");
  static constexpr int kSlots = kSms * kCtas;                          // CTAs of a wave
  static constexpr int kStateFloats = kHalves * kHalf * (D + 2);       // a split walk's: sums, references, weights
  // TMEM columns: scores (then weights) and weighted values of the halves.
  static constexpr uint32_t kScores = 0, kOut = kHalves * kTile, kTmemCols = 512 / kCtas;
  static_assert(kOut + kHalves * D <= kTmemCols, "TMEM of an SM");
};

struct Bars {
  uint64_t raw_full[2];       // TMA -> converters (keys, values)
  uint64_t full[2];           // converters -> MMA: fp16 keys, values
  uint64_t empty[2];          // MMA -> converters
  uint64_t queries[2];        // softmax -> MMA, by half
  uint64_t scores[2];         // MMA -> softmax
  uint64_t weights[2];        // softmax -> MMA
  uint64_t out[2];            // MMA -> softmax
  uint64_t drain;             // after a failure
  uint32_t tmem;
  int32_t failed;
  int32_t apart[2];           // the half's tile sums each chunk's values on its own
};
static_assert(sizeof(Bars) <= 256, "");

// What a range of vectors sees.
struct Range {
  int pos_lo, pos_hi, near_lo, near_hi;
};

// Vectors lo .. hi behind those that `v` begins with, whose first is at pos0.
__device__ __forceinline__ Range RangeOf(const Vectors& v, int lo, int hi, int pos0, int window) {
  Range r;
  r.pos_lo = lo == 0 ? pos0 : pos0 + static_cast<int>(v.Down(lo));
  r.pos_hi = pos0 + static_cast<int>(v.Down(hi));
  r.near_lo = NearOf(r.pos_lo, window);
  r.near_hi = NearOf(r.pos_hi, window);
  return r;
}

// Whether any (all) vectors of the range see any (all) of tokens t .. t + n - 1.
__device__ __forceinline__ bool SeesSome(const Range& r, int t, int n, int sinks) {
  return t <= r.pos_hi && (t + n > r.near_lo || t < sinks);
}
__device__ __forceinline__ bool SeesAll(const Range& r, int t, int n, int sinks) {
  return t + n - 1 <= r.pos_lo && (t >= r.near_hi || t + n <= sinks);
}

// Registers of a warpgroup's threads from here on.
template <int kRegs>
__device__ __forceinline__ void RegsUp() {
  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegs));
}
template <int kRegs>
__device__ __forceinline__ void RegsDown() {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegs));
}

// Two fp32 numbers in a register pair, and sm_100's paired arithmetic on them:
// one issue slot for both.
using Pair = unsigned long long;
__device__ __forceinline__ Pair MakePair(float x, float y) {
  Pair p;
  asm("mov.b64 %0, {%1, %2};" : "=l"(p) : "f"(x), "f"(y));
  return p;
}
__device__ __forceinline__ float2 Split2(Pair p) {
  float2 v;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(v.x), "=f"(v.y) : "l"(p));
  return v;
}
__device__ __forceinline__ Pair Fma2(Pair a, Pair b, Pair c) {
  Pair d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
__device__ __forceinline__ Pair Mul2(Pair a, Pair b) {
  Pair d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ Pair Add2(Pair a, Pair b) {
  Pair d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ float Max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

// Barrier `id` of `threads` threads; whether any of them passed true. What ends
// one warp's loop (a wait that ran out) goes through here, so that warps that
// meet at a barrier leave their loops together.
__device__ __forceinline__ bool MeetAny(int id, int threads, bool any) {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.u32 p, %1, 0;\n\t"
      "barrier.cta.red.or.pred q, %2, %3, p;\n\t"
      "selp.u32 %0, 1, 0, q;\n\t}"
      : "=r"(r)
      : "r"(any ? 1u : 0u), "r"(id), "r"(threads)
      : "memory");
  return r != 0;
}

// Grid (kv head, sequence, tile of kHalves * 128 vectors from the latest on): the
// longest walks of all sequences start first, so that the last to start are short
// (70 -> 62 us at 32 x 512 rows, against sequence after sequence). Where the calls'
// keys and values are more than L2 holds, sequence after sequence, grid (kv head,
// tile, sequence): CTAs that run together then read the same (5015 against 5452 us
// for 8 x 1000 rows behind 30000 tokens, 8 kv heads of 128). Tiles past the grid's
// 65535 go with x.
constexpr int64_t kGridTiles = 65535;
//
// kSplit: a flat grid over the tiles of at most 32 sequences, in the same orders (the
// counting costs nothing that was measured). Those that fill whole waves of the SMs
// go a CTA each; the walks of the rest are dealt to several CTAs, so that the last
// wave is as short as it has room to be, and the last CTA of a tile to arrive merges
// their states in order. (480 tiles, 3.2 waves, of walks of 33: 559 -> 488 us.)
template <int D, bool kSplit>
__global__ void __launch_bounds__(Tiles<D>::kThreads, Tiles<D>::kCtas)
    AttnTilesQ8Kernel(const __grid_constant__ CUtensorMap tk, const __grid_constant__ CUtensorMap tv, const AttnArgs a) {
  using L = Tiles<D>;
  extern __shared__ char smem_raw[];
  char* smem = smem_raw + ((L::kAlign - (SmemAddr(smem_raw) & (L::kAlign - 1))) & (L::kAlign - 1));
  Bars& bars = *reinterpret_cast<Bars*>(smem + L::kBars);
  const int tid = threadIdx.x, lane = tid & 31, warp = __shfl_sync(kFull, tid >> 5, 0);
  const accel_b200_q8_cache& c = a.cache;
  const int G = a.group;
  constexpr int kVectors = L::kHalves * kHalf;
  int g = blockIdx.x, b = a.by_sequence ? blockIdx.z : blockIdx.y;
  int64_t from_end = a.by_sequence ? blockIdx.y : blockIdx.z;
  int share = 0, shares = 1;  // this CTA's part of the tile's walk
  int split_tile = 0, state0 = 0;  // the tile's counter and first state
  PdlWait();
  Run run;
  if constexpr (kSplit) {
    // Lane r counts the tiles of sequence r. In front of level d (the tiles that
    // are d-th from the end of their sequences) are min(tiles, d) of each.
    run = lane < a.sequences ? RunOf(a.rows, lane, c.context, blockIdx.x == 0 && warp == 0, a.status) : Run{0, 0, 0};
    const int own = static_cast<int>((static_cast<int64_t>(run.count) * G + kVectors - 1) / kVectors);
    const int items = __reduce_add_sync(kFull, own) * c.kv_heads, whole = items / L::kSlots * L::kSlots;
    int item = blockIdx.x;
    if (item >= whole && items > whole) {
      shares = min(kMostShares, L::kSlots / (items - whole));
      split_tile = (item - whole) / shares;
      share = item - whole - split_tile * shares;
      state0 = split_tile * shares;
      item = whole + split_tile;
    }
    if (item >= items) {
      PdlTrigger();
      return;
    }
    const int pair = item / c.kv_heads;
    g = item - pair * c.kv_heads;
    // Tiles of keys that the call sees, of a kv head.
    const int64_t upto = static_cast<int64_t>(run.pos0) + run.count;
    const int64_t seen = a.window > 0 ? Min64(upto, static_cast<int64_t>(a.window) + a.sinks + run.count) : upto;
    const uint32_t key_tiles = __reduce_add_sync(kFull, static_cast<uint32_t>(run.count > 0 ? seen / kTile + 1 : 0));
    if (static_cast<uint64_t>(key_tiles) * c.kv_heads * (2 * kTile * D) > kLevelsUpTo) {
      int end = own;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int other = __shfl_up_sync(kFull, end, o);
        if (lane >= o) end += other;
      }
      b = __ffs(__ballot_sync(kFull, end > pair)) - 1;
      from_end = pair - __shfl_sync(kFull, end - own, b);
    } else {
      int level = 0, next = __reduce_max_sync(kFull, own), before = 0;  // before: tiles in front of `level`
      while (next - level > 1) {
        const int mid = (level + next) / 2, count = __reduce_add_sync(kFull, min(own, mid));
        if (count <= pair) {
          level = mid;
          before = count;
        } else {
          next = mid;
        }
      }
      from_end = level;
      const uint32_t at_level = __ballot_sync(kFull, own > level);
      b = __ffs(__ballot_sync(kFull, own > level && __popc(at_level & ((1u << lane) - 1u)) == pair - before)) - 1;
    }
    run = Run{__shfl_sync(kFull, run.first, b), __shfl_sync(kFull, run.count, b), __shfl_sync(kFull, run.pos0, b)};
  } else {
    run = RunOf(a.rows, b, c.context, g == 0 && from_end == 0 && tid == 0, a.status);
    if (gridDim.x > c.kv_heads) {
      from_end += g / c.kv_heads * kGridTiles;
      g %= c.kv_heads;
    }
  }
  const int64_t vectors = static_cast<int64_t>(run.count) * G;
  const int64_t tiles = (vectors + kVectors - 1) / kVectors;
  const int64_t v0 = (tiles - 1 - from_end) * kVectors;
  if (v0 < 0) {
    PdlTrigger();
    return;
  }
  // Every role passes here once, the softmax with its queries' loads in flight.
  const auto set_up = [&] {
    TcFenceBeforeSync();
    __syncthreads();
    TcFenceAfterSync();
    PdlTrigger();
    return bars.tmem;
  };

  // The tiles: those of the sinks before the windows, then the windows.
  const Vectors place(v0, G);
  const int last = static_cast<int>(Min64(kVectors, vectors - v0)) - 1;
  const int pos_of_v0 = run.pos0 + static_cast<int>(place.row0);
  const Range all = RangeOf(place, 0, last, pos_of_v0, a.window);
  const int tile0 = all.near_lo / kTile;
  const int sink_tiles = static_cast<int>(Min64((static_cast<int64_t>(a.sinks) + kTile - 1) / kTile, tile0));
  int n = sink_tiles + all.pos_hi / kTile - tile0 + 1, j0 = 0;
  if (kSplit && shares > 1) {
    shares = min(shares, max(1, n / kLeastShare));  // the same for all CTAs of the tile
    if (share >= shares) {
      PdlTrigger();
      return;
    }
    j0 = n * share / shares;
    n = n * (share + 1) / shares - j0;
  }
  const auto token_of = [&](int j) {
    j += j0;
    return (j < sink_tiles ? j : tile0 + (j - sink_tiles)) * kTile;
  };
  const bool second = L::kHalves > 1 && kHalf <= last;
  // Half w's vectors, and whether they see any of tile j.
  const auto half_range = [&](int w) {
    if (L::kHalves == 1) return all;
    const int lo = min(w * kHalf, last);
    return RangeOf(place, lo, min(lo + kHalf - 1, last), pos_of_v0, a.window);
  };
  const auto needed = [&](const Range& range, int w, int j) {
    return (w == 0 || second) && SeesSome(range, token_of(j), kTile, a.sinks);
  };
  volatile int32_t* failed = &bars.failed;
  // A bounded wait; false where it ran out, which the CTA reports as it ends.
  const auto wait = [&](uint64_t* bar, uint32_t parity) {
    if (MbarWaitSleep(bar, parity)) return true;
    *failed = 1;
    return false;
  };

  if (warp < L::kSoftWarps) {
    // ------------------------------------------------------------- softmax
    RegsUp<L::kMore>();
    constexpr int kParts = L::kParts;
    const int w = warp / (4 * kParts), part = (warp >> 2) % kParts;  // half, and which tokens and dimensions of it
    const int quad = warp & 3, r = quad * 32 + lane;                  // vector of the half: its TMEM lane
    const Range range = half_range(w);
    const int my_vector = w * kHalf + r;
    const bool mine = my_vector <= last;
    // Row (behind the first vector's) and head of this lane's vector, for itself
    // and, by shuffle, for lanes that move its row.
    const uint32_t my_down = place.Down(my_vector);
    const uint32_t my_place = my_down << 16 | place.Head(my_vector, my_down);
    const int my_pos = mine ? pos_of_v0 + static_cast<int>(my_down) : range.pos_hi;
    const int my_near = NearOf(my_pos, a.window);
    const uint32_t lanes = static_cast<uint32_t>(quad * 32) << 16;
    constexpr int kOwnChunks = kChunks / kParts, kDims = D / kParts;
    // What the threads of a vector tell each other, over a barrier of their two warps.
    float* factors = reinterpret_cast<float*>(smem + L::kShared) + w * kHalf;
    float* tops = reinterpret_cast<float*>(smem + L::kShared) + (L::kHalves + w * kParts) * kHalf;
    const auto meet = [&](bool bad) { return MeetAny(2 + w * 4 + quad, kParts * 32, bad); };
    const float* ksp = c.k_scale + b * c.scale_seq_stride + g * c.scale_head_stride;
    const float* vsp = c.v_scale + b * c.scale_seq_stride + g * c.scale_head_stride;
    // Scales of a tile's chunks, one per lane: keys' in lanes 0 .. 3, values' in
    // 4 .. 7; of chunks that nobody sees 0 and -1. They load a tile ahead.
    const auto next_needed = [&](int j) {
      while (j < n && !needed(range, w, j)) ++j;
      return j;
    };
    const auto load_scales = [&](int j) {
      const int t = (j < n ? token_of(j) : 0) + (lane & 3) * kChunk;
      const bool value = (lane & 4) != 0;
      if (j >= n || lane >= 2 * kChunks || !SeesSome(range, t, kChunk, a.sinks)) return value ? -1.f : 0.f;
      return (value ? vsp : ksp)[t >> a.block_shift];
    };
    int j = next_needed(0);
    float scales = load_scales(j);
    // The queries as two fp16 parts of q * 2^e, their largest element at 2^13.
    // Four lanes load a vector, a warp 8 at a time.
    float factor = 0.f;
    uint32_t tmem;
    {
      constexpr int kLoads = D / 16;  // 16-byte pieces of a vector per lane
      constexpr int kBatches = 4 / kParts;
      char* dst = smem + L::kQ + w * 2 * L::kOperand;
      constexpr int kTogether = D == 64 ? kBatches : 2;  // as many as registers hold
      float4 x[kTogether][kLoads];
      const auto load = [&](int b0) {
#pragma unroll
        for (int i = 0; i < kTogether; ++i) {
          const int row = (part * kBatches + b0 + i) * 8 + (lane >> 2);  // of the quad
          const uint32_t at = __shfl_sync(kFull, my_place, row);
          const float* q = a.q + (run.first + place.row0 + (at >> 16)) * a.q_ld +
                           static_cast<int64_t>(g * G + (at & 0xffffu)) * D + (lane & 3) * 4;
          const bool some = w * kHalf + quad * 32 + row <= last;
#pragma unroll
          for (int k = 0; k < kLoads; ++k) {
            x[i][k] = some ? *reinterpret_cast<const float4*>(q + 16 * k) : make_float4(0.f, 0.f, 0.f, 0.f);
          }
        }
      };
      load(0);
      tmem = set_up();
#pragma unroll 1
      for (int b0 = 0; b0 < kBatches; b0 += kTogether) {
        if (b0 > 0) load(b0);
#pragma unroll
        for (int i = 0; i < kTogether; ++i) {
          const int batch = part * kBatches + b0 + i, row = quad * 32 + batch * 8 + (lane >> 2);
          uint32_t amax = 0;
#pragma unroll
          for (int k = 0; k < kLoads; ++k) {
            amax = max(max(amax, __float_as_uint(x[i][k].x) & 0x7fffffffu), __float_as_uint(x[i][k].y) & 0x7fffffffu);
            amax = max(max(amax, __float_as_uint(x[i][k].z) & 0x7fffffffu), __float_as_uint(x[i][k].w) & 0x7fffffffu);
          }
          amax = max(amax, __shfl_xor_sync(kFull, amax, 1));
          amax = max(amax, __shfl_xor_sync(kFull, amax, 2));
          const int e = min(13 + 127 - static_cast<int>(amax >> 23), 126);
          const float up = __uint_as_float(static_cast<uint32_t>(127 + e) << 23);
          const float down = __uint_as_float(static_cast<uint32_t>(127 - e) << 23) * (a.scale * kLog2e);
          if (kParts == 1) {
            const float theirs = __shfl_sync(kFull, down, (lane & 7) * 4);
            if ((lane >> 3) == batch) factor = theirs;
          } else if ((lane & 3) == 0) {
            factors[row] = down;
          }
#pragma unroll
          for (int k = 0; k < kLoads; ++k) {
            uint2 hi, lo;
            SplitPair(x[i][k].x * up, x[i][k].y * up, &hi.x, &lo.x);
            SplitPair(x[i][k].z * up, x[i][k].w * up, &hi.y, &lo.y);
            // Elements 16 k + 4 (lane % 4) on: half a 16-byte piece.
            const int piece = 2 * (k % 4) + ((lane & 3) >> 1);
            char* p = dst + (k / 4) * kPanel + row * 128 + ((piece ^ (row & 7)) << 4) + (lane & 1) * 8;
            *reinterpret_cast<uint2*>(p) = hi;
            *reinterpret_cast<uint2*>(p + L::kOperand) = lo;
          }
        }
      }
      FenceProxyAsyncSmem();
      __syncwarp();
      if (lane == 0) MbarArrive(&bars.queries[w]);
      if (kParts > 1) {
        meet(false);
        factor = factors[r];
      }
    }

    const uint32_t my_scores = tmem + lanes + L::kScores + w * kTile;
    const uint32_t my_out = tmem + lanes + L::kOut + w * D + part * kDims;
    float m = -INFINITY, l = 0.f, v_ref = 0.f;
    Pair o[kDims / 2];  // weighted values of dimensions 2 d and 2 d + 1 of this part
#pragma unroll
    for (int d = 0; d < kDims / 2; ++d) o[d] = 0;
    // registers += v_ref * the last tile's weighted values.
    const auto take_out = [&] {
      const Pair ref2 = MakePair(v_ref, v_ref);
#pragma unroll
      for (int d = 0; d < kDims; d += 16) {
        uint32_t x[16];
        TmemLoad16Raw(my_out + d, x);
        TmemWaitLoads(x);
#pragma unroll
        for (int i = 0; i < 16; i += 2) {
          o[(d + i) / 2] = Fma2(ref2, MakePair(__uint_as_float(x[i]), __uint_as_float(x[i + 1])), o[(d + i) / 2]);
        }
      }
    };
    // The tile's scores: their maximum, and then the weights in their place.
    // Chunks in a loop that is not unrolled: the code of a tile stays small
    // (every CTA fetches it anew). kWhole: every vector of the half sees all of
    // the tile; else bit i of a chunk's mask says whether it sees token i.
    const auto pick = [](const float (&x)[kChunks], int k) {
      return k < 2 ? (k == 0 ? x[0] : x[1]) : (k == 2 ? x[2] : x[3]);
    };
    const auto mask_of = [&](int t) {
      const auto below = [](int n) { return n <= 0 ? 0u : n >= 32 ? ~0u : (1u << n) - 1u; };  // bits 0 .. n - 1
      return below(my_pos + 1 - t) & (~below(my_near - t) | below(a.sinks - t));
    };
    const auto maximum = [&](auto whole, int t0, const float (&ks)[kChunks]) {
      constexpr bool kWhole = decltype(whole)::value;
      float top = -INFINITY;
#pragma unroll 1
      for (int i0 = 0; i0 < kOwnChunks; ++i0) {
        const int k = i0 * kParts + part;
        if (!kWhole && !SeesSome(range, t0 + k * kChunk, kChunk, a.sinks)) continue;
        uint32_t x[32];
        TmemLoad32Raw(my_scores + k * kChunk, x);
        const uint32_t mask = kWhole ? ~0u : mask_of(t0 + k * kChunk);
        TmemWaitLoads(x);
        float mx = -INFINITY;
#pragma unroll
        for (int i = 0; i < 32; i += 2) {
          const float x0 = kWhole || (mask >> i & 1u) != 0 ? __uint_as_float(x[i]) : -INFINITY;
          const float x1 = kWhole || (mask >> (i + 1) & 1u) != 0 ? __uint_as_float(x[i + 1]) : -INFINITY;
          mx = Max3(mx, x0, x1);
        }
        // A chunk with no visible token stays at -inf (its scale may be 0).
        if (kWhole || mx != -INFINITY) top = fmaxf(top, mx * (factor * pick(ks, k)));
      }
      return top;
    };
    const auto weigh = [&](auto whole, int t0, const float (&ks)[kChunks], const float (&lift)[kChunks], float ref) {
      constexpr bool kWhole = decltype(whole)::value;
#pragma unroll 1
      for (int i0 = 0; i0 < kOwnChunks; ++i0) {
        const int k = i0 * kParts + part;
        if (!kWhole && !SeesSome(range, t0 + k * kChunk, kChunk, a.sinks)) {
          const uint32_t none[16] = {};
          TmemStore16Raw(my_scores + k * kChunk, none);
          TmemStore16Raw(my_scores + k * kChunk + 16, none);
          continue;
        }
        const float f = factor * pick(ks, k), up = pick(lift, k), shift = ref - up;
        const uint32_t mask = kWhole ? ~0u : mask_of(t0 + k * kChunk);
        const Pair f2 = MakePair(f, f), shift2 = MakePair(-shift, -shift), minus2 = MakePair(-1.f, -1.f);
        Pair sum2 = 0;
        // 16 tokens at a time: an MMA step's 8 columns of hi and 8 of lo.
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          uint32_t x[16], y[16];
          TmemLoad16Raw(my_scores + k * kChunk + 16 * h, x);
          TmemWaitLoads(x);
#pragma unroll
          for (int i = 0; i < 16; i += 2) {
            const float2 e =
                Split2(Fma2(MakePair(__uint_as_float(x[i]), __uint_as_float(x[i + 1])), f2, shift2));
            float2 p = make_float2(Exp2(e.x), Exp2(e.y));
            if (!kWhole) {
              p.x = (mask >> (16 * h + i) & 1u) != 0 ? p.x : 0.f;
              p.y = (mask >> (16 * h + i + 1) & 1u) != 0 ? p.y : 0.f;
            }
            const Pair p2 = MakePair(p.x, p.y);
            sum2 = Add2(sum2, p2);
            const __half2 hi = __floats2half2_rn(p.x, p.y);
            const float2 back = __half22float2(hi);
            const float2 rest = Split2(Fma2(MakePair(back.x, back.y), minus2, p2));
            const __half2 lo = __floats2half2_rn(rest.x, rest.y);
            y[i / 2] = *reinterpret_cast<const uint32_t*>(&hi);
            y[8 + i / 2] = *reinterpret_cast<const uint32_t*>(&lo);
          }
          TmemStore16Raw(my_scores + k * kChunk + 16 * h, y);
        }
        const float2 sums = Split2(sum2);
        const float sum = sums.x + sums.y;
        l = fmaf(sum, Exp2(-up), l);
      }
    };
    int taken = 0, outs = 0;  // tiles whose scores, and MMA groups whose values, were taken
    bool pending = false;     // weighted values of the last tile are still to be taken
    bool ok = true;
    while (j < n && ok) {
      const int t0 = token_of(j), next = next_needed(j + 1);
      // Weights carry their chunk's value scale relative to the tile's largest,
      // as a shift of the exponent, and the sum of weights takes it out again.
      // Where scales are so far apart that the smaller ones' weights would lose
      // bits, each chunk is summed on its own; and where the largest is 0 or below
      // 2^-128, whose reciprocal is infinite.
      const bool value = (lane & 4) != 0;
      float v_now = value ? fmaxf(scales, 0.f) : 0.f;
      v_now = fmaxf(v_now, __shfl_xor_sync(kFull, v_now, 1));
      v_now = fmaxf(v_now, __shfl_xor_sync(kFull, v_now, 2));
      const float up = value && scales != -1.f ? __log2f(scales * (1.f / v_now)) : 0.f;
      const bool apart = (__ballot_sync(kFull, !(fabsf(up) <= kMostLift)) & 0xf0u) != 0;  // lanes 4 .. 7
      const float mine_up = value ? (apart ? 0.f : up) : scales;
      v_now = __shfl_sync(kFull, v_now, kChunks);
      float ks[kChunks], lift[kChunks];
#pragma unroll
      for (int k = 0; k < kChunks; ++k) {
        ks[k] = __shfl_sync(kFull, mine_up, k);
        lift[k] = __shfl_sync(kFull, mine_up, kChunks + k);
      }
      scales = load_scales(next);
      if (pending) {
        // The last tile's weighted values, while the tensor core sums this one's scores.
        ok = __all_sync(kFull, wait(&bars.out[w], outs & 1));
        if (ok) {
          TcFenceAfterSync();
          take_out();
          ++outs;
        }
      }
      v_ref = v_now;
      const bool whole = SeesAll(range, t0, kTile, a.sinks);
      ok = ok && __all_sync(kFull, wait(&bars.scores[w], taken & 1));
      float top = -INFINITY;
      if (ok) {
        TcFenceAfterSync();
        top = whole ? maximum(std::true_type{}, t0, ks) : maximum(std::false_type{}, t0, ks);
      }
      if (kParts > 1) {
        // Every other tile's exchange has its own place: the last one may still be read.
        float* t = tops + (taken & 1) * L::kHalves * kParts * kHalf;
        t[part * kHalf + r] = top;
        ok = !meet(!ok);
        top = fmaxf(top, t[(part ^ 1) * kHalf + r]);
      }
      if (!ok) break;
      if (__any_sync(kFull, top > m + kSlack)) {
        const float now = fmaxf(m, top);
        const float corr = now == -INFINITY ? 1.f : Exp2(m - now);
        m = now;
        l *= corr;
        const Pair corr2 = MakePair(corr, corr);
#pragma unroll
        for (int d = 0; d < kDims / 2; ++d) o[d] = Mul2(o[d], corr2);
      }
      const float ref = (m == -INFINITY ? 0.f : m) - kBias;
      if (whole) {
        weigh(std::true_type{}, t0, ks, lift, ref);
      } else {
        weigh(std::false_type{}, t0, ks, lift, ref);
      }
      TmemWaitStores();
      const auto tell = [&] {
        TcFenceBeforeSync();
        __syncwarp();
        if (lane == 0) MbarArrive(&bars.weights[w]);
      };
      if (lane == 0) bars.apart[w] = apart ? 1 : 0;  // the same of all four warps
      tell();
      ++taken;
      pending = !apart;
      if (apart) {
#pragma unroll 1
        for (int k = 0; k < kChunks && ok; ++k) {
          const bool seen = SeesSome(range, t0 + k * kChunk, kChunk, a.sinks);
          v_ref = seen ? vsp[(t0 + k * kChunk) >> a.block_shift] : 0.f;
          ok = __all_sync(kFull, wait(&bars.out[w], outs & 1));
          if (!ok) break;
          TcFenceAfterSync();
          take_out();
          ++outs;
          if (k + 1 < kChunks) tell();
        }
        if (kParts > 1) ok = !meet(!ok);
      }
      j = next;
    }
    if (ok && pending) {
      ok = __all_sync(kFull, wait(&bars.out[w], outs & 1));
      if (ok) {
        TcFenceAfterSync();
        take_out();
      }
    }
    if (!ok) l = __int_as_float(0x7fc00000);
    if (kParts > 1) {
      // The sum of all of the tokens' weights.
      float* t = tops + (taken & 1) * L::kHalves * kParts * kHalf;
      t[part * kHalf + r] = l;
      meet(false);
      l += t[(part ^ 1) * kHalf + r];
    }
    // Out through the bytes of the half's queries, which nothing reads any more:
    // a thread's row in, then whole rows out.
    {
      constexpr int kRowBytes = kDims * 4, kPieces = kRowBytes / 16;
      static_assert(32 * kRowBytes * 4 * kParts == 2 * L::kOperand, "");
      char* mine_rows = smem + L::kQ + w * 2 * L::kOperand + (part * 4 + quad) * 32 * kRowBytes;
      const bool partial = kSplit && shares > 1;
      const float inv = partial ? 1.f : 1.f / l;
      const Pair inv2 = MakePair(inv, inv);
#pragma unroll
      for (int k = 0; k < kPieces; ++k) {
        const float2 x = Split2(Mul2(o[2 * k], inv2)), y = Split2(Mul2(o[2 * k + 1], inv2));
        *reinterpret_cast<float4*>(mine_rows + lane * kRowBytes + ((k ^ (lane & 7)) << 4)) =
            make_float4(x.x, x.y, y.x, y.y);
      }
      __syncwarp();
      constexpr int kRows = 32 / kPieces;  // rows that the warp's lanes cover
      float* out = a.out + (run.first + place.row0) * a.out_ld + static_cast<int64_t>(g) * G * D + part * kDims;
      float* state = a.parts + static_cast<int64_t>(state0 + share) * L::kStateFloats;
#pragma unroll 8
      for (int i0 = 0; i0 < 32; i0 += kRows) {
        const int i = i0 + lane / kPieces, piece = lane % kPieces;
        const uint32_t at = __shfl_sync(kFull, my_place, i);
        if (w * kHalf + quad * 32 + i <= last) {
          float* to = partial ? state + (w * kHalf + quad * 32 + i) * D + part * kDims
                              : out + static_cast<int64_t>(at >> 16) * a.out_ld + (at & 0xffffu) * D;
          *reinterpret_cast<float4*>(to + piece * 4) =
              *reinterpret_cast<const float4*>(mine_rows + i * kRowBytes + ((piece ^ (i & 7)) << 4));
        }
      }
      if (partial) {
        if (part == 0) {
          state[kVectors * D + my_vector] = m;
          state[kVectors * (D + 1) + my_vector] = l;
        }
        constexpr int kThreads = L::kSoftWarps * 32, kMergeBarrier = 10;
        MeetAny(kMergeBarrier, kThreads, false);
        bool merges = false;
        if (tid == 0) {
          __threadfence();  // the barrier put the CTA's stores before it
          merges = atomicAdd(a.counters + split_tile, 1) == shares - 1;
          if (merges) a.counters[split_tile] = 0;
          __threadfence();
        }
        if (MeetAny(kMergeBarrier, kThreads, merges)) {
          const float* states = a.parts + static_cast<int64_t>(state0) * L::kStateFloats;
          for (int e = tid; e < (last + 1) * (D / 4); e += kThreads) {
            const int v = e / (D / 4), d = e % (D / 4) * 4;
            float pm[kMostShares], pl[kMostShares], mx = -INFINITY, sum = 0.f;
            float4 po[kMostShares], acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int p = 0; p < kMostShares; ++p) {
              if (p < shares) {
                const float* s = states + static_cast<int64_t>(p) * L::kStateFloats;
                pm[p] = __ldcg(s + kVectors * D + v);
                pl[p] = __ldcg(s + kVectors * (D + 1) + v);
                po[p] = __ldcg(reinterpret_cast<const float4*>(s + v * D + d));
                mx = fmaxf(mx, pm[p]);
              }
            }
#pragma unroll
            for (int p = 0; p < kMostShares; ++p) {
              if (p < shares) {
                // A share that saw nothing of a vector has reference -inf and sums of
                // 0; one of NaN scores has that reference too, and sums that stay.
                const float f = pm[p] == -INFINITY ? 1.f : Exp2(pm[p] - mx);
                sum = fmaf(pl[p], f, sum);
                acc.x = fmaf(po[p].x, f, acc.x);
                acc.y = fmaf(po[p].y, f, acc.y);
                acc.z = fmaf(po[p].z, f, acc.z);
                acc.w = fmaf(po[p].w, f, acc.w);
              }
            }
            const uint32_t down = place.Down(v), head = place.Head(v, down);
            *reinterpret_cast<float4*>(a.out + (run.first + place.row0 + down) * a.out_ld +
                                       static_cast<int64_t>(g * G + head) * D + d) =
                make_float4(acc.x / sum, acc.y / sum, acc.z / sum, acc.w / sum);
          }
        }
      }
    }
  } else if (warp < L::kMmaWarp) {
    // ---------------------------------------------------------- int8 -> fp16
    RegsDown<L::kLess>();
    const int ct = tid - L::kSoftWarps * 32;
    const int plane_row = static_cast<int>((b * c.seq_stride + g * c.head_stride) / D);
    const auto fetch = [&](int plane, int j) {
      MbarArriveExpectTx(&bars.raw_full[plane], L::kRawBytes);
      TmaLoad2D(smem + L::kRaw + plane * L::kRawBytes, plane == 0 ? &tk : &tv, 0, plane_row + token_of(j),
                &bars.raw_full[plane]);
    };
    // The first tiles come while the other roles set up.
    if (ct == 0) {
      for (int i = 0; i < 2; ++i) {
        MbarInit(&bars.raw_full[i], 1);
        MbarInit(&bars.full[i], kConverters);
        MbarInit(&bars.empty[i], 1);
        MbarInit(&bars.queries[i], 4 * L::kParts);
        MbarInit(&bars.scores[i], 1);
        MbarInit(&bars.weights[i], 4 * L::kParts);
        MbarInit(&bars.out[i], 1);
      }
      MbarInit(&bars.drain, 1);
      bars.failed = 0;
      FenceBarrierInit();
      fetch(0, 0);
      fetch(1, 0);
    }
    set_up();
    bool ok = true;
    int fetched[2] = {0, 0};  // tiles read of each plane; the next is in flight
    for (int j = 0; j < n && ok; ++j) {
#pragma unroll 1
      for (int plane = 0; plane < 2; ++plane) {
        if (!ok) break;  // all converters together
        ok = wait(&bars.raw_full[plane], j & 1) && wait(&bars.empty[plane], (j & 1) ^ 1);
        const char* src = smem + L::kRaw + plane * L::kRawBytes;
        char* dst = smem + (plane == 0 ? L::kK : L::kV);
        // 8 elements at a time. The threads are whole multiples of 8 rows, so a
        // thread's swizzle and piece stay the same from row to row.
        constexpr int kPieces = D / 8, kStep = kConverters * 32 / kPieces;  // pieces of a row, rows per pass
        static_assert(kStep % 8 == 0, "");
        constexpr int kBatch = 8;  // pieces a thread has in flight
        const int row0 = ct / kPieces, piece = ct % kPieces;
        src += ct * 8;
        dst += (piece / 8) * kPanel + row0 * 128 + (((piece % 8) ^ (row0 & 7)) << 4);
#pragma unroll 1
        for (int r = 0; r < kTile; r += kBatch * kStep, src += kBatch * kStep * D, dst += kBatch * kStep * 128) {
          uint2 x[kBatch];
#pragma unroll
          for (int k = 0; k < kBatch; ++k) x[k] = *reinterpret_cast<const uint2*>(src + k * kStep * D);
#pragma unroll
          for (int k = 0; k < kBatch; ++k) {
            const uint32_t u = x[k].x ^ 0x80808080u, v = x[k].y ^ 0x80808080u;
            *reinterpret_cast<uint4*>(dst + k * kStep * 128) =
                make_uint4(Halves<false>(u), Halves<true>(u), Halves<false>(v), Halves<true>(v));
          }
        }
        FenceProxyAsyncSmem();
        __syncwarp();
        if (lane == 0) MbarArrive(&bars.full[plane]);
        // Every converter has read the int8 tile: its bytes take the next one.
        // One whose wait ran out takes all of them out of the loop together.
        ok = !MeetAny(1, kConverters * 32, !ok);
        if (ct == 0 && ok && j + 1 < n) fetch(plane, j + 1);
        if (ok) ++fetched[plane];
      }
    }
    // After a failure: the copies still in flight land first (bounded).
    if (!ok && ct == 0) {
      for (int plane = 0; plane < 2; ++plane) MbarWait(&bars.raw_full[plane], min(fetched[plane], n - 1) & 1);
    }
  } else {
    // ------------------------------------------------------------------ MMA
    RegsDown<L::kLess>();
    // TMEM is taken behind the wait for the previous kernel, and the next kernel
    // is let in behind that: neither can hold the columns the other waits for.
    // (The softmax's registers wait for this warpgroup's, so those went first.)
    if (warp == L::kMmaWarp) TmemAlloc(&bars.tmem, L::kTmemCols);
    const uint32_t tmem = set_up();
    if (warp == L::kMmaWarp && ElectOne()) {
      constexpr uint32_t kQkDesc = InstrDescF16(kTile, false), kPvDesc = InstrDescF16(D, true);
      const uint32_t q_at = SmemAddr(smem + L::kQ), k_at = SmemAddr(smem + L::kK), v_at = SmemAddr(smem + L::kV);
      const auto scores = [&](int w) {
        // The small parts' products first: fewer roundings at full size.
#pragma unroll 1
        for (int part = 1; part >= 0; --part) {
          const uint32_t qa = q_at + (w * 2 + part) * L::kOperand;
#pragma unroll
          for (int s = 0; s < D / 16; ++s) {
            const uint32_t at = (s / 4) * kPanel + (s % 4) * 32;  // 16 elements along the swizzled row
            MmaF16(tmem + L::kScores + w * kTile, SmemDescSw128(qa + at, 16, 1024), SmemDescSw128(k_at + at, 16, 1024),
                   kQkDesc, part == 0 || s > 0);
          }
        }
        MmaCommit(&bars.scores[w]);
      };
      // Weighted values of tokens 16 s0 .. 16 (s0 + kSteps) - 1 of the tile.
      const auto values = [&](int w, int s0, auto steps) {
        constexpr int kSteps = decltype(steps)::value;
#pragma unroll 1
        for (int part = 1; part >= 0; --part) {
          // A step: 16 tokens, 8 columns of weights, 16 rows of values.
          const uint32_t pa = tmem + L::kScores + w * kTile + part * 8 + s0 * 16;
          const uint32_t vb = v_at + s0 * 2048;
#pragma unroll
          for (int s = 0; s < kSteps; ++s) {
            MmaF16FromTmem(tmem + L::kOut + w * D, pa + s * 16, SmemDescSw128(vb + s * 2048, kPanel, 1024), kPvDesc,
                           part == 0 || s > 0);
          }
        }
        MmaCommit(&bars.out[w]);
      };
      const Range range0 = half_range(0), range1 = half_range(1);
      int done[2] = {0, 0};  // weights taken from each half
      bool ok = true;
      // Scores of tile j for half w, once the half's queries and the keys are there.
      const auto next_scores = [&](int w, int j) {
        if (!ok || !needed(w == 0 ? range0 : range1, w, j)) return;
        ok = wait(&bars.queries[w], 0) && wait(&bars.full[0], j & 1);
        if (!ok) return;
        TcFenceAfterSync();
        scores(w);
      };
      next_scores(0, 0);
      if (L::kHalves > 1) next_scores(1, 0);
      if (ok) MmaCommit(&bars.empty[0]);
      for (int j = 0; j < n && ok; ++j) {
#pragma unroll
        for (int w = 0; w < L::kHalves; ++w) {
          if (ok && needed(w == 0 ? range0 : range1, w, j)) {
            ok = wait(&bars.weights[w], done[w] & 1) && wait(&bars.full[1], j & 1);
            if (!ok) continue;
            ++done[w];
            TcFenceAfterSync();
            if (*reinterpret_cast<volatile int32_t*>(&bars.apart[w]) == 0) {
              values(w, 0, std::integral_constant<int, kTile / 16>{});
            } else {
              for (int k = 0; k < kChunks && ok; ++k) {
                if (k > 0) {
                  ok = wait(&bars.weights[w], done[w] & 1);
                  if (!ok) break;
                  ++done[w];
                  TcFenceAfterSync();
                }
                values(w, k * (kChunk / 16), std::integral_constant<int, kChunk / 16>{});
              }
            }
          }
          // The values are free before the next scores are.
          if (ok && w == L::kHalves - 1) MmaCommit(&bars.empty[1]);
          if (j + 1 < n) next_scores(w, j + 1);
        }
        if (!ok) break;
        if (j + 1 < n) MmaCommit(&bars.empty[0]);
      }
      if (!ok) {
        // After a failure: what was issued ends before the TMEM is freed (bounded).
        MmaCommit(&bars.drain);
        MbarWait(&bars.drain, 0);
      }
    }
    __syncwarp();
  }
  TcFenceBeforeSync();
  __syncthreads();
  if (*failed != 0 && tid == 0) {
    if (a.status != nullptr) atomicOr(a.status, ACCEL_B200_STATUS_COPY_TIMEOUT);
  }
  if (warp == L::kMmaWarp) TmemDealloc(bars.tmem, L::kTmemCols);
}

// Tiles that a call has at most, by its largest number of rows.
template <int D>
int64_t MostTiles(const accel_b200_q8_cache& c, int64_t max_rows, int32_t heads) {
  return CeilDiv(max_rows * (heads / c.kv_heads), Tiles<D>::kHalves * kHalf);
}

// The last wave's walks are split in calls of few waves and of walks long enough,
// and of 32 sequences at most (a lane counts each; more of them go a CTA per tile).
template <int D>
TilesPlan Plan(const accel_b200_q8_cache& c, int32_t batch, int32_t max_rows, int32_t heads, int32_t window,
               int32_t sinks) {
  constexpr int64_t kSlots = Tiles<D>::kSlots;
  static_assert(kSlots <= kMaxCounters, "a counter per split tile");
  TilesPlan p{};
  const int64_t seen = window > 0 ? Min64(c.context, static_cast<int64_t>(window) + sinks) : c.context;
  const int64_t items = batch * c.kv_heads * MostTiles<D>(c, max_rows, heads), rest = items % kSlots;
  p.steps = CeilDiv(seen, kTile);
  p.split = batch <= 32 && p.steps >= 2 * kLeastShare && items <= 16 * kSlots;
  p.waves = static_cast<double>(items / kSlots);
  if (rest > 0) {
    const int64_t shares = p.split ? Min64(Min64(kMostShares, kSlots / rest), p.steps / kLeastShare) : 1;
    p.waves += 1. / static_cast<double>(shares);
  }
  if (p.split) p.workspace = kCounterRegion + static_cast<size_t>(kSlots) * Tiles<D>::kStateFloats * sizeof(float);
  return p;
}

template <int D, bool kSplit>
int Launch(const AttnArgs& a, int32_t max_rows, cudaStream_t stream) {
  constexpr int kSmem = Tiles<D>::kBytes + Tiles<D>::kAlign;
  // The roles trade the registers that the launch gives out; were they fewer
  // than the split adds up to, the role that takes more would wait for good.
  // Asked for until there is an answer: a device that cannot give one now may later.
  static std::atomic<int> regs{0};
  cudaError_t err = cudaSuccess;
  if (regs.load(std::memory_order_relaxed) == 0) {
    cudaFuncAttributes f{};
    err = cudaFuncGetAttributes(&f, AttnTilesQ8Kernel<D, kSplit>);
    if (err != cudaSuccess) return CheckLaunchEx(err, "attention_prefill_q8");
    regs.store(f.numRegs, std::memory_order_relaxed);
  }
  if (regs.load(std::memory_order_relaxed) != Tiles<D>::kLaunch) {
    return SetError(ACCEL_B200_ECUDA, "attention_prefill_q8: the kernel's registers do not fit its split");
  }
  err = cudaFuncSetAttribute(AttnTilesQ8Kernel<D, kSplit>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem);
  if (err != cudaSuccess) return CheckLaunchEx(err, "attention_prefill_q8");
  const uint64_t plane_rows = static_cast<uint64_t>(PlaneRows(a.cache));
  CUtensorMap tk{}, tv{};
  if (!Encode2D(&tk, CU_TENSOR_MAP_DATA_TYPE_UINT8, a.cache.k, D, plane_rows, D, D, kTile, CU_TENSOR_MAP_SWIZZLE_NONE) ||
      !Encode2D(&tv, CU_TENSOR_MAP_DATA_TYPE_UINT8, a.cache.v, D, plane_rows, D, D, kTile, CU_TENSOR_MAP_SWIZZLE_NONE)) {
    return SetError(ACCEL_B200_EINVAL, "attention_prefill_q8: cache tensor map rejected");
  }
  const int64_t tiles = MostTiles<D>(a.cache, max_rows, a.heads), kv = a.cache.kv_heads;
  const unsigned x = static_cast<unsigned>(CeilDiv(tiles, kGridTiles) * kv), y = static_cast<unsigned>(a.sequences),
                 z = static_cast<unsigned>(Min64(tiles, kGridTiles));
  const dim3 grid = kSplit ? dim3(static_cast<unsigned>(a.sequences * kv * tiles + Tiles<D>::kSlots))
                           : a.by_sequence ? dim3(x, z, y) : dim3(x, y, z);
  return CheckLaunchEx(
      LaunchK(AttnTilesQ8Kernel<D, kSplit>, grid, dim3(Tiles<D>::kThreads), kSmem, stream, 1u, 1u, tk, tv, a),
      "attention_prefill_q8");
}

template <int D>
int LaunchFor(AttnArgs a, const TilesPlan& plan, int32_t max_rows, cudaStream_t stream) {
  if (plan.split) return Launch<D, true>(a, max_rows, stream);
  const int64_t rows = a.window > 0 ? static_cast<int64_t>(a.window) + a.sinks + max_rows : a.cache.context;
  const int64_t bytes = Min64(a.cache.context, rows) * (2 * D) * a.cache.kv_heads;  // of a sequence
  a.by_sequence = bytes > static_cast<int64_t>(kLevelsUpTo) / a.sequences;
  return Launch<D, false>(a, max_rows, stream);
}

}  // namespace

TilesPlan PlanTilesQ8(const accel_b200_q8_cache& c, int32_t batch, int32_t max_rows, int32_t heads, int32_t window,
                      int32_t sinks) {
  return c.head_dim == 64 ? Plan<64>(c, batch, max_rows, heads, window, sinks)
                          : Plan<128>(c, batch, max_rows, heads, window, sinks);
}

int LaunchTilesQ8(const AttnArgs& a, const TilesPlan& plan, int32_t max_rows, cudaStream_t stream) {
  return a.cache.head_dim == 64 ? LaunchFor<64>(a, plan, max_rows, stream) : LaunchFor<128>(a, plan, max_rows, stream);
}

}  // namespace accel_b200
