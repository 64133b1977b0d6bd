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
// computes, the tensor core works for the other); warps 8..10 turn the int8
// tiles that TMA brings into fp16 operands with the 128-byte swizzle; one
// thread of warp 11 issues every MMA. Bound by the tensor core at 128
// dimensions (two fp16 products in place of one) and by the softmax's issue
// slots at 64.
//
// Every wait is bounded; one that runs out sets a flag that ends every role,
// gives NaN and ORs ACCEL_B200_STATUS_COPY_TIMEOUT.
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>

#include <string>

#include "accel_b200.h"
#include "attention_q8.cuh"
#include "common.cuh"
#include "q8_cache.cuh"
#include "tcgen05.cuh"
#include "tensor_map.cuh"

namespace accel_b200 {
namespace {

constexpr int kThreads = 384;
constexpr int kHalf = 128;         // vectors of a half: TMEM lanes
constexpr int kTile = 128;         // tokens per tile
constexpr int kConverters = 3;     // warps
constexpr int kChunk = 32;         // tokens whose scores a thread holds at a time: one scale block at most
constexpr int kChunks = kTile / kChunk;
constexpr uint32_t kTmemCols = 512;
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
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
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
  if (warp == 11) TmemAlloc(&bars.tmem, kTmemCols);
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
  const Range half_range[2] = {RangeOf(v0, Min64(v0 + kHalf - 1, v_last), G, run.pos0, a.window),
                               RangeOf(second ? v0 + kHalf : v_last, v_last, G, run.pos0, a.window)};
  const auto needed = [&](int w, int j) {
    return (w == 0 || second) && SeesSome(half_range[w], token_of(j), kTile, a.sinks);
  };
  volatile int32_t* failed = &bars.failed;
  // A bounded wait; false, and every role's cue to stop, once any ran out.
  const auto wait = [&](uint64_t* bar, uint32_t parity) {
    if (MbarWait(bar, parity)) return true;
    *failed = 1;
    return false;
  };

  if (warp < 8) {
    // ------------------------------------------------------------- softmax
    const int w = warp >> 2, r = (warp & 3) * 32 + lane;  // half, vector of the half
    const Range& range = half_range[w];
    const int64_t v = v0 + w * kHalf + r;
    const bool mine = v < vectors;
    const int my_pos = mine ? run.pos0 + static_cast<int>(v / G) : range.pos_hi;
    const int my_near = NearOf(my_pos, a.window);
    const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const uint32_t my_scores = tmem + lanes + L::kScores + w * kTile, my_out = tmem + lanes + L::kOut + w * D;
    float factor;
    {
      // The query as two fp16 parts of q * 2^e, its largest element at 2^13.
      const float* q = a.q + (run.first + (mine ? v / G : 0)) * a.q_ld + static_cast<int64_t>(g * G + (mine ? v % G : 0)) * D;
      uint32_t amax = 0;
#pragma unroll 8
      for (int d = 0; d < D; d += 4) {
        const float4 x = mine ? *reinterpret_cast<const float4*>(q + d) : make_float4(0.f, 0.f, 0.f, 0.f);
        amax = max(max(amax, __float_as_uint(x.x) & 0x7fffffffu), __float_as_uint(x.y) & 0x7fffffffu);
        amax = max(max(amax, __float_as_uint(x.z) & 0x7fffffffu), __float_as_uint(x.w) & 0x7fffffffu);
      }
      const int e = min(13 + 127 - static_cast<int>(amax >> 23), 126);
      const float up = __uint_as_float(static_cast<uint32_t>(127 + e) << 23);
      factor = __uint_as_float(static_cast<uint32_t>(127 - e) << 23) * (a.scale * kLog2e);
      char* dst = smem + L::kQ + w * 2 * L::kOperand + r * 128;
#pragma unroll 2
      for (int d = 0; d < D; d += 8) {
        uint4 hi = make_uint4(0, 0, 0, 0), lo = hi;
        if (mine) {
          const float4 x = *reinterpret_cast<const float4*>(q + d), y = *reinterpret_cast<const float4*>(q + d + 4);
          SplitPair(x.x * up, x.y * up, &hi.x, &lo.x);
          SplitPair(x.z * up, x.w * up, &hi.y, &lo.y);
          SplitPair(y.x * up, y.y * up, &hi.z, &lo.z);
          SplitPair(y.z * up, y.w * up, &hi.w, &lo.w);
        }
        const int at = (d / 64) * kPanel + ((((d % 64) / 8) ^ (r & 7)) << 4);
        *reinterpret_cast<uint4*>(dst + at) = hi;
        *reinterpret_cast<uint4*>(dst + L::kOperand + at) = lo;
      }
      FenceProxyAsyncSmem();
      __syncwarp();
      if (lane == 0) MbarArrive(&bars.queries[w]);
    }

    float m = -INFINITY, l = 0.f, v_ref = 0.f, o[D];
#pragma unroll
    for (int d = 0; d < D; ++d) o[d] = 0.f;
    const float* ksp = c.k_scale + b * c.scale_seq_stride + g * c.scale_head_stride;
    const float* vsp = c.v_scale + b * c.scale_seq_stride + g * c.scale_head_stride;
    // registers += v_ref * the last tile's weighted values.
    const auto take_out = [&] {
#pragma unroll
      for (int d = 0; d < D; d += 16) {
        uint32_t x[16];
        TmemLoad16Raw(my_out + d, x);
        TmemWaitLoads();
#pragma unroll
        for (int i = 0; i < 16; ++i) o[d + i] = fmaf(v_ref, __uint_as_float(x[i]), o[d + i]);
      }
    };
    int taken = 0;  // tiles this half has gone through
    bool ok = true;
    for (int j = 0; j < n && ok; ++j) {
      if (!needed(w, j)) continue;
      const int t0 = token_of(j);
      // Scales of the tile's chunks; one that nobody sees has weight 0 whatever
      // its scale says.
      float ks[kChunks], vs[kChunks], v_now = 0.f;
#pragma unroll
      for (int k = 0; k < kChunks; ++k) {
        const bool seen = SeesSome(range, t0 + k * kChunk, kChunk, a.sinks);
        ks[k] = seen ? ksp[(t0 + k * kChunk) / c.block] : 0.f;
        vs[k] = seen ? vsp[(t0 + k * kChunk) / c.block] : 0.f;
        v_now = fmaxf(v_now, vs[k]);
      }
      const bool whole = SeesAll(range, t0, kTile, a.sinks);
      ok = __all_sync(kFull, wait(&bars.scores[w], taken & 1));
      if (!ok) break;
      TcFenceAfterSync();
      const auto hidden = [&](int t) { return t > my_pos || (t < my_near && t >= a.sinks); };
      float top = -INFINITY;
#pragma unroll
      for (int k = 0; k < kChunks; ++k) {
        uint32_t x[32];
        TmemLoad32Raw(my_scores + k * kChunk, x);
        TmemWaitLoads();
        float mx = -INFINITY;
        if (whole) {
#pragma unroll
          for (int i = 0; i < 32; ++i) mx = fmaxf(mx, __uint_as_float(x[i]));
        } else {
#pragma unroll
          for (int i = 0; i < 32; ++i) mx = fmaxf(mx, hidden(t0 + k * kChunk + i) ? -INFINITY : __uint_as_float(x[i]));
        }
        // A chunk with no visible token stays at -inf (its scale may be 0).
        if (mx != -INFINITY) top = fmaxf(top, mx * (factor * ks[k]));
      }
      const bool moves = __any_sync(kFull, top > m + kSlack);
      const float now = moves ? fmaxf(m, top) : m;
      if (taken > 0) {
        ok = __all_sync(kFull, wait(&bars.out[w], (taken - 1) & 1));
        if (!ok) break;
        TcFenceAfterSync();
        take_out();
      }
      if (moves) {
        const float corr = now == -INFINITY ? 1.f : Exp2(m - now);
        m = now;
        l *= corr;
#pragma unroll
        for (int d = 0; d < D; ++d) o[d] *= corr;
      }
      v_ref = v_now;
      const float ref = (m == -INFINITY ? 0.f : m) - kBias;
      const float v_inv = v_now > 0.f ? 1.f / v_now : 0.f;
      // Weights, 16 tokens at a time: an MMA step's 8 columns of hi and 8 of lo.
#pragma unroll
      for (int k = 0; k < kTile / 16; ++k) {
        const float f = factor * ks[k / 2], scale = vs[k / 2];
        const float ratio = scale == v_now ? 1.f : scale * v_inv;
        uint32_t x[16], y[16];
        TmemLoad16Raw(my_scores + 16 * k, x);
        TmemWaitLoads();
#pragma unroll
        for (int i = 0; i < 16; i += 2) {
          float p0 = Exp2(fmaf(__uint_as_float(x[i]), f, -ref)), p1 = Exp2(fmaf(__uint_as_float(x[i + 1]), f, -ref));
          if (!whole) {
            p0 = hidden(t0 + 16 * k + i) ? 0.f : p0;
            p1 = hidden(t0 + 16 * k + i + 1) ? 0.f : p1;
          }
          l += p0 + p1;
          SplitPair(p0 * ratio, p1 * ratio, &y[i / 2], &y[8 + i / 2]);
        }
        TmemStore16Raw(my_scores + 16 * k, y);
      }
      TmemWaitStores();
      TcFenceBeforeSync();
      __syncwarp();
      if (lane == 0) MbarArrive(&bars.weights[w]);
      ++taken;
    }
    if (ok && taken > 0) {
      ok = __all_sync(kFull, wait(&bars.out[w], (taken - 1) & 1));
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
        *reinterpret_cast<float4*>(dst + d) = make_float4(o[d] / l, o[d + 1] / l, o[d + 2] / l, o[d + 3] / l);
      }
    }
  } else if (warp < 8 + kConverters) {
    // ---------------------------------------------------------- int8 -> fp16
    const int ct = tid - 256;
    const int row0 = static_cast<int>((b * c.seq_stride + g * c.head_stride) / D);
    const auto fetch = [&](int plane, int j) {
      MbarArriveExpectTx(&bars.raw_full[plane], L::kRawBytes);
      TmaLoad2D(smem + L::kRaw + plane * L::kRawBytes, plane == 0 ? &tk : &tv, 0, row0 + token_of(j),
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
        constexpr int kPieces = D / 8;  // 8-element pieces of a row
#pragma unroll 4
        for (int i = ct; i < kTile * kPieces; i += kConverters * 32) {
          uint2 x = *reinterpret_cast<const uint2*>(src + i * 8);
          x.x ^= 0x80808080u;
          x.y ^= 0x80808080u;
          const int row = i / kPieces, piece = i % kPieces;
          *reinterpret_cast<uint4*>(dst + (piece / 8) * kPanel + row * 128 + (((piece % 8) ^ (row & 7)) << 4)) =
              make_uint4(Halves<false>(x.x), Halves<true>(x.x), Halves<false>(x.y), Halves<true>(x.y));
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
    if (lane == 0) {
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
      const auto values = [&](int w, int stage) {
#pragma unroll 1
        for (int part = 1; part >= 0; --part) {
          const uint32_t pa = tmem + L::kScores + w * kTile + part * 8, vb = v_at + stage * L::kOperand;
#pragma unroll
          for (int s = 0; s < kTile / 16; ++s) {
            // Step s: 16 tokens, 8 columns of weights, 16 rows of values.
            MmaF16FromTmem(tmem + L::kOut + w * D, pa + s * 16,
                           SmemDescSw128(vb + s * 2048, kPanel, 1024), kPvDesc, part == 0 || s > 0);
          }
        }
        MmaCommit(&bars.out[w]);
      };
      int done[2] = {0, 0};  // weights taken from each half
      bool ok = true;
      // Scores of tile j for half w, once the half's queries and the keys are there.
      const auto next_scores = [&](int w, int j) {
        if (!ok || !needed(w, j)) return;
        ok = wait(&bars.queries[w], 0) && wait(&bars.full[0][j % L::kStages], (j / L::kStages) & 1);
        if (!ok) return;
        TcFenceAfterSync();
        scores(w, j % L::kStages);
      };
      next_scores(0, 0);
      next_scores(1, 0);
      if (ok) MmaCommit(&bars.empty[0][0]);
      for (int j = 0; j < n && ok; ++j) {
        for (int w = 0; w < 2 && ok; ++w) {
          if (needed(w, j)) {
            ok = wait(&bars.weights[w], done[w] & 1) && wait(&bars.full[1][j % L::kStages], (j / L::kStages) & 1);
            if (!ok) break;
            ++done[w];
            TcFenceAfterSync();
            values(w, j % L::kStages);
          }
          if (j + 1 < n) next_scores(w, j + 1);
        }
        if (!ok) break;
        MmaCommit(&bars.empty[1][j % L::kStages]);
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
  if (warp == 11) TmemDealloc(tmem, kTmemCols);
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
