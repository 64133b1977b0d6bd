// Attention of many query rows over the int8 key/value cache on the 5th-
// generation tensor cores (include/accel_b200.h, accel_b200_attention_prefill_q8).
//
// One CTA takes 256 consecutive query vectors (row x head, the heads of one kv
// head) of one sequence and walks the 128-token tiles that any of them sees.
// Keys and values become fp16 exactly; queries and weights are sums of two fp16
// numbers (22 bits), the second parts' products summed first, so results are
// fp32 results. Per tile and half (128 vectors):
//
//   S = Qlo K^T + Qhi K^T      128 x 128 x D, operands in shared memory
//   online softmax             one thread per vector, S read from TMEM
//   P, lo and hi parts         written over S in TMEM
//   O = Plo V + Phi V          128 x D x 128, A operand from TMEM
//   registers += vscale * O    fp32, rounded to nearest
//
// O is read out per tile, not summed over the context in TMEM: the tensor
// core's running sum rounds towards zero, which drifts over a long context, and
// the value scale and the softmax reference change from tile to tile. Scales
// of the tile's blocks are folded into the weights relative to the largest.
//
// Roles: warps 0..3 and 4..7 the softmax of the two halves (while one half
// computes, the tensor core works for the other); warps 8..11 turn the int8
// tiles that TMA brings into fp16 operands with the 128-byte swizzle; one
// thread of warp 12 issues every MMA. Bound by the tensor core at 128
// dimensions (two fp16 products in place of one) and by the softmax's issue
// slots at 64.
//
// Every wait is bounded; one that runs out sets a flag that ends every role,
// gives NaN and ORs ACCEL_B200_STATUS_COPY_TIMEOUT.
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>

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

constexpr int kThreads = 512;
constexpr int kHalf = 128;         // vectors of a half: TMEM lanes
constexpr int kTile = 128;         // tokens per tile
constexpr int kConverters = 4;     // warps
constexpr int kMmaWarp = 8 + kConverters;
constexpr int kChunk = 32;         // tokens whose scores a thread holds at a time: one scale block at most
constexpr int kChunks = kTile / kChunk;
constexpr uint32_t kTmemCols = 512;
constexpr float kMostLift = 6.f;    // scales of a tile further apart than 2^6 are applied one by one
constexpr int kPanel = 128 * 128;  // bytes of 128 rows x 64 fp16, the swizzle's row length

template <int D>
struct Tiles {
  static constexpr int kPanels = D / 64;
  static constexpr int kOperand = kPanels * kPanel;     // a 128 x D fp16 operand
  static constexpr int kStages = D == 64 ? 2 : 1;       // fp16 key and value tiles
  static constexpr int kQ = 0;                          // [half][hi, lo]
  static constexpr int kK = kQ + 4 * kOperand;
  static constexpr int kV = kK + kStages * kOperand;
  static constexpr int kRaw = kV + kStages * kOperand;  // int8 tiles as they come: keys, values
  static constexpr int kRawBytes = kTile * D;
  static constexpr int kBars = kRaw + 2 * kRawBytes;
  static constexpr int kBytes = kBars + 256;
  static constexpr int kAlign = 1024;
  static_assert(kBytes + kAlign <= 227 * 1024, "shared memory of a CTA");
  // TMEM columns: scores (then weights) and weighted values of the halves.
  static constexpr uint32_t kScores = 0, kOut = 2 * kTile;
  static_assert(kOut + 2 * D <= kTmemCols, "TMEM of an SM");
};

struct Bars {
  uint64_t raw_full[2];       // TMA -> converters (keys, values)
  uint64_t full[2][2];        // converters -> MMA: fp16 keys, values by stage
  uint64_t empty[2][2];       // MMA -> converters
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

__device__ __forceinline__ Range RangeOf(int64_t v_lo, int64_t v_hi, int G, int pos0, int window) {
  Range r;
  r.pos_lo = pos0 + static_cast<int>(v_lo / G);
  r.pos_hi = pos0 + static_cast<int>(v_hi / G);
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

// Registers of a warpgroup's threads from here on. 512 threads start with 128
// each; the two softmax groups, whose threads hold D sums and a run of scores,
// take what the other two give: 256 * kMore + 256 * kLess = 512 * 128.
constexpr int kMore = 208, kLess = 48;
static_assert(kMore + kLess == 2 * 128, "");
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

// Barrier of the converter warps; whether any thread passed true.
__device__ __forceinline__ bool ConvertersAny(bool any) {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.u32 p, %1, 0;\n\t"
      "barrier.cta.red.or.pred q, 1, %2, p;\n\t"
      "selp.u32 %0, 1, 0, q;\n\t}"
      : "=r"(r)
      : "r"(any ? 1u : 0u), "n"(kConverters * 32)
      : "memory");
  return r != 0;
}

// Grid (256-vector tile, kv head, sequence).
template <int D>
__global__ void __launch_bounds__(kThreads, 1)
    AttnTilesQ8Kernel(const __grid_constant__ CUtensorMap tk, const __grid_constant__ CUtensorMap tv, const AttnArgs a) {
  using L = Tiles<D>;
  extern __shared__ char smem_raw[];
  char* smem = smem_raw + ((L::kAlign - (SmemAddr(smem_raw) & (L::kAlign - 1))) & (L::kAlign - 1));
  Bars& bars = *reinterpret_cast<Bars*>(smem + L::kBars);
  const int tid = threadIdx.x, lane = tid & 31, warp = __shfl_sync(kFull, tid >> 5, 0);
  const accel_b200_q8_cache& c = a.cache;
  const int G = a.heads / c.kv_heads, g = blockIdx.y, b = blockIdx.z;
  PdlWait();
  const Run run = RunOf(a.rows, b, c.context, blockIdx.x == 0 && g == 0 && tid == 0, a.status);
  const int64_t vectors = static_cast<int64_t>(run.count) * G;
  // Latest rows (the longest walks) first.
  const int64_t tiles = (vectors + 2 * kHalf - 1) / (2 * kHalf);
  const int64_t v0 = (tiles - 1 - static_cast<int64_t>(blockIdx.x)) * (2 * kHalf);
  if (v0 < 0) {
    PdlTrigger();
    return;
  }
  if (tid == 0) {
    for (int i = 0; i < 2; ++i) {
      MbarInit(&bars.raw_full[i], 1);
      for (int s = 0; s < 2; ++s) {
        MbarInit(&bars.full[i][s], kConverters);
        MbarInit(&bars.empty[i][s], 1);
      }
      MbarInit(&bars.queries[i], 4);
      MbarInit(&bars.scores[i], 1);
      MbarInit(&bars.weights[i], 4);
      MbarInit(&bars.out[i], 1);
    }
    MbarInit(&bars.drain, 1);
    bars.failed = 0;
    FenceBarrierInit();
  }
  // TMEM is taken behind the wait for the previous kernel, and the next kernel
  // is let in behind that: neither can hold the columns the other waits for.
  if (warp == kMmaWarp) TmemAlloc(&bars.tmem, kTmemCols);
  TcFenceBeforeSync();
  __syncthreads();
  TcFenceAfterSync();
  PdlTrigger();
  const uint32_t tmem = bars.tmem;

  // The tiles: those of the sinks before the windows, then the windows.
  const int64_t v_last = Min64(v0 + 2 * kHalf, vectors) - 1;
  const Range all = RangeOf(v0, v_last, G, run.pos0, a.window);
  const int tile0 = all.near_lo / kTile;
  const int sink_tiles = static_cast<int>(Min64((static_cast<int64_t>(a.sinks) + kTile - 1) / kTile, tile0));
  const int n = sink_tiles + all.pos_hi / kTile - tile0 + 1;
  const auto token_of = [&](int j) { return (j < sink_tiles ? j : tile0 + (j - sink_tiles)) * kTile; };
  const bool second = v0 + kHalf < vectors;
  // Half w's vectors, and whether they see any of tile j.
  const auto half_range = [&](int w) {
    const int64_t lo = Min64(v0 + w * kHalf, v_last);
    return RangeOf(lo, Min64(lo + kHalf - 1, v_last), G, run.pos0, a.window);
  };
  const auto needed = [&](const Range& range, int w, int j) {
    return (w == 0 || second) && SeesSome(range, token_of(j), kTile, a.sinks);
  };
  volatile int32_t* failed = &bars.failed;
  // A bounded wait; false, and every role's cue to stop, once any ran out.
  const auto wait = [&](uint64_t* bar, uint32_t parity) {
    if (MbarWaitSleep(bar, parity)) return true;
    *failed = 1;
    return false;
  };

  if (warp < 8) {
    // ------------------------------------------------------------- softmax
    RegsUp<kMore>();
    const int w = warp >> 2, r = (warp & 3) * 32 + lane;  // half, vector of the half
    const Range range = half_range(w);
    const int64_t v = v0 + w * kHalf + r;
    const bool mine = v < vectors;
    const int my_pos = mine ? run.pos0 + static_cast<int>(v / G) : range.pos_hi;
    const int my_near = NearOf(my_pos, a.window);
    const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const uint32_t my_scores = tmem + lanes + L::kScores + w * kTile, my_out = tmem + lanes + L::kOut + w * D;
    // The queries as two fp16 parts of q * 2^e, their largest element at 2^13.
    // The warp loads its 32 vectors one after another, a vector over its lanes.
    float factor = 0.f;
    {
      constexpr int kPer = D / 32;  // elements of a vector per lane
      const int64_t vw = v0 + w * kHalf + (warp & 3) * 32;
      char* dst = smem + L::kQ + w * 2 * L::kOperand;
      const int at0 = (kPer * lane / 64) * kPanel, piece = (kPer * lane % 64) / 8, in = kPer * lane % 8 * 2;
      constexpr int kBatch = D == 64 ? 32 : 16;  // vectors whose loads are in flight together
      int64_t row_at = vw / G;
      int head_at = static_cast<int>(vw - row_at * G);
#pragma unroll 1
      for (int i0 = 0; i0 < 32; i0 += kBatch) {
        float x[kBatch][kPer];
#pragma unroll
        for (int i = 0; i < kBatch; ++i) {
          const float* q = a.q + (run.first + row_at) * a.q_ld + (g * G + head_at) * D + kPer * lane;
          const bool some = vw + i0 + i < vectors;
          if (++head_at == G) {
            head_at = 0;
            ++row_at;
          }
          if constexpr (D == 128) {
            *reinterpret_cast<float4*>(x[i]) =
                some ? *reinterpret_cast<const float4*>(q) : make_float4(0.f, 0.f, 0.f, 0.f);
          } else {
            *reinterpret_cast<float2*>(x[i]) = some ? *reinterpret_cast<const float2*>(q) : make_float2(0.f, 0.f);
          }
        }
#pragma unroll
        for (int i = 0; i < kBatch; ++i) {
          uint32_t amax = 0;
#pragma unroll
          for (int k = 0; k < kPer; ++k) amax = max(amax, __float_as_uint(x[i][k]) & 0x7fffffffu);
          amax = __reduce_max_sync(kFull, amax);
          const int e = min(13 + 127 - static_cast<int>(amax >> 23), 126);
          const float up = __uint_as_float(static_cast<uint32_t>(127 + e) << 23);
          if (lane == i0 + i) factor = __uint_as_float(static_cast<uint32_t>(127 - e) << 23) * (a.scale * kLog2e);
          uint32_t hi[kPer / 2], lo[kPer / 2];
#pragma unroll
          for (int k = 0; k < kPer; k += 2) SplitPair(x[i][k] * up, x[i][k + 1] * up, &hi[k / 2], &lo[k / 2]);
          const int row = (warp & 3) * 32 + i0 + i;
          char* p = dst + at0 + row * 128 + ((piece ^ (row & 7)) << 4) + in;
          if constexpr (D == 128) {
            *reinterpret_cast<uint2*>(p) = make_uint2(hi[0], hi[kPer / 2 - 1]);
            *reinterpret_cast<uint2*>(p + L::kOperand) = make_uint2(lo[0], lo[kPer / 2 - 1]);
          } else {
            *reinterpret_cast<uint32_t*>(p) = hi[0];
            *reinterpret_cast<uint32_t*>(p + L::kOperand) = lo[0];
          }
        }
      }
      FenceProxyAsyncSmem();
      __syncwarp();
      if (lane == 0) MbarArrive(&bars.queries[w]);
    }

    float m = -INFINITY, l = 0.f, v_ref = 0.f;
    Pair o[D / 2];  // weighted values of dimensions 2 d and 2 d + 1
#pragma unroll
    for (int d = 0; d < D / 2; ++d) o[d] = 0;
    const float* ksp = c.k_scale + b * c.scale_seq_stride + g * c.scale_head_stride;
    const float* vsp = c.v_scale + b * c.scale_seq_stride + g * c.scale_head_stride;
    // registers += v_ref * the last tile's weighted values.
    const auto take_out = [&] {
      const Pair ref2 = MakePair(v_ref, v_ref);
#pragma unroll
      for (int d = 0; d < D; d += 16) {
        uint32_t x[16];
        TmemLoad16Raw(my_out + d, x);
        TmemWaitLoads();
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
      for (int k = 0; k < kChunks; ++k) {
        uint32_t x[32];
        TmemLoad32Raw(my_scores + k * kChunk, x);
        const uint32_t mask = kWhole ? ~0u : mask_of(t0 + k * kChunk);
        TmemWaitLoads();
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
      for (int k = 0; k < kChunks; ++k) {
        const float f = factor * pick(ks, k), up = pick(lift, k), shift = ref - up;
        const uint32_t mask = kWhole ? ~0u : mask_of(t0 + k * kChunk);
        const Pair f2 = MakePair(f, f), shift2 = MakePair(-shift, -shift), minus2 = MakePair(-1.f, -1.f);
        Pair sum2 = 0;
        // 16 tokens at a time: an MMA step's 8 columns of hi and 8 of lo.
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          uint32_t x[16], y[16];
          TmemLoad16Raw(my_scores + k * kChunk + 16 * h, x);
          TmemWaitLoads();
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
    for (int j = 0; j < n && ok; ++j) {
      if (!needed(range, w, j)) continue;
      const int t0 = token_of(j);
      // Scales of the tile's chunks. Weights carry their chunk's value scale
      // relative to the tile's largest, as a shift of the exponent, and the sum
      // of weights takes it out again. Where scales are so far apart that the
      // smaller ones' weights would lose bits, each chunk is summed on its own.
      float ks[kChunks], lift[kChunks], v_now = 0.f;
      bool apart = false;
#pragma unroll
      for (int k = 0; k < kChunks; ++k) {
        const bool seen = SeesSome(range, t0 + k * kChunk, kChunk, a.sinks);
        ks[k] = seen ? ksp[(t0 + k * kChunk) / c.block] : 0.f;
        lift[k] = seen ? vsp[(t0 + k * kChunk) / c.block] : -1.f;
        v_now = fmaxf(v_now, lift[k]);
      }
      const float v_inv = 1.f / v_now;
#pragma unroll
      for (int k = 0; k < kChunks; ++k) {
        lift[k] = lift[k] == -1.f ? 0.f : __log2f(lift[k] * v_inv);
        apart = apart || !(lift[k] >= -kMostLift);
      }
      if (apart) {
#pragma unroll
        for (int k = 0; k < kChunks; ++k) lift[k] = 0.f;
      }
      if (pending) {
        // The last tile's weighted values, while the tensor core sums this one's scores.
        ok = __all_sync(kFull, wait(&bars.out[w], outs & 1));
        if (!ok) break;
        TcFenceAfterSync();
        take_out();
        ++outs;
      }
      v_ref = v_now;
      const bool whole = SeesAll(range, t0, kTile, a.sinks);
      ok = __all_sync(kFull, wait(&bars.scores[w], taken & 1));
      if (!ok) break;
      TcFenceAfterSync();
      const float top = whole ? maximum(std::true_type{}, t0, ks) : maximum(std::false_type{}, t0, ks);
      if (__any_sync(kFull, top > m + kSlack)) {
        const float now = fmaxf(m, top);
        const float corr = now == -INFINITY ? 1.f : Exp2(m - now);
        m = now;
        l *= corr;
        const Pair corr2 = MakePair(corr, corr);
#pragma unroll
        for (int d = 0; d < D / 2; ++d) o[d] = Mul2(o[d], corr2);
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
          v_ref = seen ? vsp[(t0 + k * kChunk) / c.block] : 0.f;
          ok = __all_sync(kFull, wait(&bars.out[w], outs & 1));
          if (!ok) break;
          TcFenceAfterSync();
          take_out();
          ++outs;
          if (k + 1 < kChunks) tell();
        }
      }
    }
    if (ok && pending) {
      ok = __all_sync(kFull, wait(&bars.out[w], outs & 1));
      if (ok) {
        TcFenceAfterSync();
        take_out();
      }
    }
    if (!ok) l = __int_as_float(0x7fc00000);
    if (mine) {
      float* dst = a.out + (run.first + v / G) * a.out_ld + static_cast<int64_t>(g * G + v % G) * D;
#pragma unroll
      for (int d = 0; d < D; d += 4) {
        const float2 x = Split2(o[d / 2]), y = Split2(o[d / 2 + 1]);
        *reinterpret_cast<float4*>(dst + d) = make_float4(x.x / l, x.y / l, y.x / l, y.y / l);
      }
    }
  } else if (warp < 8 + kConverters) {
    // ---------------------------------------------------------- int8 -> fp16
    RegsDown<kLess>();
    const int ct = tid - 256;
    const int plane_row = static_cast<int>((b * c.seq_stride + g * c.head_stride) / D);
    const auto fetch = [&](int plane, int j) {
      MbarArriveExpectTx(&bars.raw_full[plane], L::kRawBytes);
      TmaLoad2D(smem + L::kRaw + plane * L::kRawBytes, plane == 0 ? &tk : &tv, 0, plane_row + token_of(j),
                &bars.raw_full[plane]);
    };
    if (ct == 0) {
      fetch(0, 0);
      fetch(1, 0);
    }
    bool ok = true;
    int fetched[2] = {0, 0};  // tiles read of each plane; the next is in flight
    for (int j = 0; j < n && ok; ++j) {
      const int stage = j % L::kStages;
      const uint32_t lap = static_cast<uint32_t>(j / L::kStages) & 1;
#pragma unroll 1
      for (int plane = 0; plane < 2; ++plane) {
        if (!ok) break;  // all converters together
        ok = wait(&bars.raw_full[plane], j & 1) && wait(&bars.empty[plane][stage], lap ^ 1);
        const char* src = smem + L::kRaw + plane * L::kRawBytes;
        char* dst = smem + (plane == 0 ? L::kK : L::kV) + stage * L::kOperand;
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
        if (lane == 0) MbarArrive(&bars.full[plane][stage]);
        // Every converter has read the int8 tile: its bytes take the next one.
        // One whose wait ran out takes all of them out of the loop together.
        ok = !ConvertersAny(!ok);
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
    RegsDown<kLess>();
    if (warp == kMmaWarp && ElectOne()) {
      constexpr uint32_t kQkDesc = InstrDescF16(kTile, false), kPvDesc = InstrDescF16(D, true);
      const uint32_t q_at = SmemAddr(smem + L::kQ), k_at = SmemAddr(smem + L::kK), v_at = SmemAddr(smem + L::kV);
      const auto scores = [&](int w, int stage) {
        // The small parts' products first: fewer roundings at full size.
#pragma unroll 1
        for (int part = 1; part >= 0; --part) {
          const uint32_t qa = q_at + (w * 2 + part) * L::kOperand, kb = k_at + stage * L::kOperand;
#pragma unroll
          for (int s = 0; s < D / 16; ++s) {
            const uint32_t at = (s / 4) * kPanel + (s % 4) * 32;  // 16 elements along the swizzled row
            MmaF16(tmem + L::kScores + w * kTile, SmemDescSw128(qa + at, 16, 1024), SmemDescSw128(kb + at, 16, 1024),
                   kQkDesc, part == 0 || s > 0);
          }
        }
        MmaCommit(&bars.scores[w]);
      };
      // Weighted values of tokens 16 s0 .. 16 (s0 + kSteps) - 1 of the tile.
      const auto values = [&](int w, int stage, int s0, auto steps) {
        constexpr int kSteps = decltype(steps)::value;
#pragma unroll 1
        for (int part = 1; part >= 0; --part) {
          // A step: 16 tokens, 8 columns of weights, 16 rows of values.
          const uint32_t pa = tmem + L::kScores + w * kTile + part * 8 + s0 * 16;
          const uint32_t vb = v_at + stage * L::kOperand + s0 * 2048;
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
        ok = wait(&bars.queries[w], 0) && wait(&bars.full[0][j % L::kStages], (j / L::kStages) & 1);
        if (!ok) return;
        TcFenceAfterSync();
        scores(w, j % L::kStages);
      };
      next_scores(0, 0);
      next_scores(1, 0);
      if (ok) MmaCommit(&bars.empty[0][0]);
      for (int j = 0; j < n && ok; ++j) {
#pragma unroll
        for (int w = 0; w < 2; ++w) {
          if (ok && needed(w == 0 ? range0 : range1, w, j)) {
            ok = wait(&bars.weights[w], done[w] & 1) && wait(&bars.full[1][j % L::kStages], (j / L::kStages) & 1);
            if (!ok) continue;
            ++done[w];
            TcFenceAfterSync();
            if (*reinterpret_cast<volatile int32_t*>(&bars.apart[w]) == 0) {
              values(w, j % L::kStages, 0, std::integral_constant<int, kTile / 16>{});
            } else {
              for (int k = 0; k < kChunks && ok; ++k) {
                if (k > 0) {
                  ok = wait(&bars.weights[w], done[w] & 1);
                  if (!ok) break;
                  ++done[w];
                  TcFenceAfterSync();
                }
                values(w, j % L::kStages, k * (kChunk / 16), std::integral_constant<int, kChunk / 16>{});
              }
            }
          }
          // The values are free before the next scores are.
          if (ok && w == 1) MmaCommit(&bars.empty[1][j % L::kStages]);
          if (j + 1 < n) next_scores(w, j + 1);
        }
        if (!ok) break;
        if (j + 1 < n) MmaCommit(&bars.empty[0][(j + 1) % L::kStages]);
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
  if (warp == kMmaWarp) TmemDealloc(tmem, kTmemCols);
}

template <int D>
int Launch(const AttnArgs& a, int32_t batch, int32_t max_rows, cudaStream_t stream) {
  constexpr int kSmem = Tiles<D>::kBytes + Tiles<D>::kAlign;
  const cudaError_t err =
      cudaFuncSetAttribute(AttnTilesQ8Kernel<D>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem);
  if (err != cudaSuccess) return CheckLaunchEx(err, "attention_prefill_q8");
  const uint64_t plane_rows = static_cast<uint64_t>(PlaneRows(a.cache));
  CUtensorMap tk{}, tv{};
  if (!Encode2D(&tk, CU_TENSOR_MAP_DATA_TYPE_UINT8, a.cache.k, D, plane_rows, D, D, kTile, CU_TENSOR_MAP_SWIZZLE_NONE) ||
      !Encode2D(&tv, CU_TENSOR_MAP_DATA_TYPE_UINT8, a.cache.v, D, plane_rows, D, D, kTile, CU_TENSOR_MAP_SWIZZLE_NONE)) {
    return SetError(ACCEL_B200_EINVAL, "attention_prefill_q8: cache tensor map rejected");
  }
  const int64_t vectors = static_cast<int64_t>(max_rows) * (a.heads / a.cache.kv_heads);
  const dim3 grid(static_cast<unsigned>(CeilDiv(vectors, 2 * kHalf)), static_cast<unsigned>(a.cache.kv_heads),
                  static_cast<unsigned>(batch));
  return CheckLaunchEx(LaunchK(AttnTilesQ8Kernel<D>, grid, dim3(kThreads), kSmem, stream, 1u, 1u, tk, tv, a),
                       "attention_prefill_q8");
}

}  // namespace

int LaunchTilesQ8(const AttnArgs& a, int32_t batch, int32_t max_rows, cudaStream_t stream) {
  return a.cache.head_dim == 64 ? Launch<64>(a, batch, max_rows, stream) : Launch<128>(a, batch, max_rows, stream);
}

}  // namespace accel_b200
