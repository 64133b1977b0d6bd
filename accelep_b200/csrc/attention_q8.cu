// Attention over the int8 key/value cache (include/accel_b200.h, "int8 key/value
// cache"), causal, with an optional sliding window and first tokens (sinks)
// that stay visible: of single rows and of many rows per sequence.
//
// Scores and weighted values run on the tensor cores (mma.sync m16n8k16, fp16
// operands, fp32 sums) without giving up fp32 results: an int8 key or value is
// an exact fp16 number, and a query or a weight is the sum of two fp16 numbers
// (22 bits), whose products with it are exact in fp32. The two parts of 8
// vectors (query rows x heads that share a kv head) are the 16 rows of one
// MMA operand. (The 128-row tiles of attention_q8_tiles.cu would stand almost
// empty here: a decoded row brings heads / kv_heads vectors, 3 to 8 in common
// models.) Queries are scaled by a power of two to 2^13 and weights to about
// 2^10, so their second parts stay far above fp16's smallest step.
//
// Work split. A warp owns 8 vectors and walks units of 32 tokens, which TMA
// brings into the warp's own queue in shared memory; no barrier but the copy's
// own in the loop. Which lane stands for which dimension or token of a sum is
// free to choose, and is chosen so that a lane's share of an MMA operand is a
// run of bytes, the shared-memory reads have no bank conflicts under TMA's
// swizzle, and the scores' register layout is the weights' operand layout.
// Units are dealt to all warps of the S CTAs of a vector group in turn. Each
// unit's weighted values are summed on their own and added, times the unit's
// value scale, to fp32 registers (the tensor core's running sum rounds towards
// zero, which would drift over a long context). Bound by HBM on long sequences:
// 4 of 40001 to 65536 tokens, 8 kv heads of 128, take 77 us, 5.6 TB/s with inputs
// that no cache holds, in a captured graph (87 called one by one). Before the split by lengths it took 88 us, with loads to
// registers 128 and with per-lane cp.async 132: an SM keeps too few of those in
// flight. Short calls are a chain of latencies, so what needs no division has none.
//
// Online softmax in base 2 against a reference that moves only when a score
// passes it by more than kSlack (a vote; no weight above 2^(kBias + kSlack)).
// The warps' states merge in shared memory, the CTAs' through distributed
// shared memory when they are one cluster (S <= 8), else through the
// workspace by the last CTA to arrive; always in index order, so the result
// does not depend on scheduling.
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>

#include "accel_b200.h"
#include "attention_q8.cuh"
#include "cluster.cuh"
#include "common.cuh"
#include "l2_prefetch.cuh"
#include "q8_cache.cuh"
#include "tensor_map.cuh"

namespace accel_b200 {
namespace {

constexpr int kThreads = 128;
constexpr int kWarps = kThreads / 32;
constexpr int kUnit = 32;      // tokens per step of a warp
constexpr int kVec = 8;        // query vectors of a CTA
constexpr int kMaxCluster = 8; // CTAs whose states merge through distributed shared memory
constexpr int64_t kBalanceFrom = 16384;  // tokens from which single rows take CTAs by their lengths
constexpr int kWarpUnits = 2;  // units a warp gets at least before the tokens are split further
template <int D>
constexpr int kResident = D == 64 ? 3 : 2;  // CTAs per SM

__device__ __forceinline__ void Mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// Shared memory: each warp's own queue of kStages units (32 key rows, then 32
// value rows, as TMA writes them with the swizzle of their row length), the
// barriers behind them, and after the loop, in the queues' bytes, the warps'
// states. The swizzle is computed from address bits up to 1024.
template <int D>
struct Queue {
  static constexpr int kStages = D == 64 ? 3 : 2;
  static constexpr int kPlaneBytes = kUnit * D;
  static constexpr int kUnitBytes = 2 * kPlaneBytes;
  static constexpr int kWarpBytes = kStages * kUnitBytes;
  static constexpr int kBarriers = kWarps * kWarpBytes;
  static constexpr int kBytes = kBarriers + kWarps * kStages * 8;
  static constexpr int kAlign = 1024;
};

// The softmax state of a CTA: reference, sum and weighted values of its vectors.
template <int D>
struct alignas(16) State {
  float m[kVec], l[kVec];
  float o[kVec][D];
};

// Units of 32 tokens of which some are seen: those of the sinks that lie before
// the unit of `near`, then from that on to the unit of pos.
struct Units {
  int near, sinks, count;
};
__device__ __forceinline__ Units UnitsOf(int near, int pos, int sinks) {
  Units u;
  u.near = near / kUnit;
  u.sinks = static_cast<int>(Min64((static_cast<int64_t>(sinks) + kUnit - 1) / kUnit, u.near));
  u.count = u.sinks + pos / kUnit - u.near + 1;
  return u;
}

// The sizes (in units) that a CTA of a balanced launch may have: 32, evenly
// spread from the even share to twice that.
constexpr int BalancedSize(int even, int i) { return even + (even * i + 30) / 31; }
static_assert(BalancedSize(8, 0) == 8 && BalancedSize(8, 31) == 16 && BalancedSize(33, 31) == 66 &&
                  BalancedSize(1 << 25, 0) == 1 << 25 && BalancedSize(1 << 25, 31) == 1 << 26,
              "from the even share to exactly twice that, without overflow");

// What a launch's rows are: single rows or runs of a sequence's rows, in grid
// (split, kv head x vector group, row or sequence); or single rows, at most 32,
// over a flat grid whose CTAs go to the rows by how much each row sees.
enum class Rows { kSingle, kRuns, kBalanced };

template <int D, Rows kRows>
__global__ void __launch_bounds__(kThreads, kResident<D>) AttnVectorsQ8Kernel(
    const __grid_constant__ CUtensorMap tk, const __grid_constant__ CUtensorMap tv, const AttnArgs a) {
  constexpr int kKw = D / 16;      // 32-bit words of a lane's share of a key row
  constexpr int kTiles = D / 8;    // 8-dimension tiles of the output
  constexpr int kVw = D / 32;      // words of a lane's share of a value row
  using Qu = Queue<D>;
  extern __shared__ char smem_raw[];
  char* smem = smem_raw + ((Qu::kAlign - (SmemAddr(smem_raw) & (Qu::kAlign - 1))) & (Qu::kAlign - 1));
  static_assert(sizeof(State<D>) * (kWarps + 1) <= Qu::kBarriers, "the states fit the queues' bytes");
  State<D>* warp_state = reinterpret_cast<State<D>*>(smem);
  State<D>& cta_state = warp_state[kWarps];
  __shared__ bool last;
  PdlTrigger();
  // With CACHE_BEFORE_WAIT everything but the queries and the rows' own blocks
  // is as the kernels before the previous one left it, and those have completed.
  const bool early = kRows != Rows::kRuns && (a.prefetch.flags & ACCEL_B200_ATTN_CACHE_BEFORE_WAIT) != 0;
  if (kRows != Rows::kRuns && threadIdx.x == 0 && a.prefetch.count > 0) PrefetchShare(a.prefetch);
  if (!early) PdlWait();
  const accel_b200_q8_cache& c = a.cache;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, gid = lane >> 2, tig = lane & 3;
  constexpr bool kRuns = kRows == Rows::kRuns;
  const int G = a.group;
  int S = static_cast<int>(gridDim.x), split = static_cast<int>(blockIdx.x), pair = static_cast<int>(blockIdx.y);
  int64_t z = blockIdx.z;
  if constexpr (kRows == Rows::kBalanced) {
    // Lane r counts row r's units (rows that are not attended: none). CTAs of
    // q units each, q the least of 32 sizes, from an even share of all units to
    // twice that, whose CTAs do not exceed the grid: rows get ceil(units / q).
    const int pairs = c.kv_heads * ((G + kVec - 1) / kVec), T = static_cast<int>(gridDim.x);
    int mine_units = 0;
    if (lane < a.single_rows) {
      const int pos = a.row_pos[lane];
      const int64_t slot = a.row_seq != nullptr ? a.row_seq[lane] : lane;
      if (pos >= 0 && (pos >= c.context || slot < 0 || slot >= c.slots)) {
        if (blockIdx.x == 0 && warp == 0 && a.status != nullptr) atomicOr(a.status, ACCEL_B200_STATUS_BAD_POSITION);
      } else if (pos >= 0) {
        mine_units = UnitsOf(NearOf(pos, a.window), pos, a.sinks).count;
      }
    }
    int64_t total = mine_units;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(kFull, total, o);
    const int even = static_cast<int>(Max64(kWarps * kWarpUnits, (total * pairs + T - 1) / T));
    const int size = BalancedSize(even, lane);
    int64_t ctas = 0;
    for (int r = 0; r < a.single_rows; ++r) ctas += (__shfl_sync(kFull, mine_units, r) + size - 1) / size;
    // (Lane 31's size, twice the even share, always fits: it needs T / 2 CTAs
    // and less than one more for each row and pair, of which there are T / 2 at most.)
    const int q = __shfl_sync(kFull, size, __ffs(__ballot_sync(kFull, ctas * pairs <= T)) - 1);
    const int share = (mine_units + q - 1) / q;  // CTAs per pair of row `lane`
    int end = share * pairs;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int before = __shfl_up_sync(kFull, end, o);
      if (lane >= o) end += before;
    }
    const int row = __ffs(__ballot_sync(kFull, end > static_cast<int>(blockIdx.x))) - 1;
    if (row < 0) {
      if (early) PdlWait();  // no CTA leaves in front of the previous kernel's end
      return;
    }
    S = __shfl_sync(kFull, share, row);
    const int local = static_cast<int>(blockIdx.x) - (__shfl_sync(kFull, end, row) - S * pairs);
    pair = local / S;
    split = local % S;
    z = row;
  }
  const int g = pair % c.kv_heads, group = pair / c.kv_heads;
  const bool reports = split == 0 && pair == 0 && tid == 0;

  // The rows: `count` from `first` at positions pos0 + i of `slot`. A single
  // row's query does not wait for its position.
  float x[kKw][4];
  const auto load_query = [&](int64_t row, int head, bool some) {
    const float* q = a.q + row * a.q_ld + static_cast<int64_t>(g * G + head) * D + tig * 16;
#pragma unroll
    for (int j = 0; j < kKw; ++j) {
      *reinterpret_cast<float4*>(x[j]) = some ? *reinterpret_cast<const float4*>(q + (j / 4) * 64 + (j % 4) * 4)
                                              : make_float4(0.f, 0.f, 0.f, 0.f);
    }
  };
  if (!kRuns && !early) load_query(z, group * kVec + gid, group * kVec + gid < G);
  int64_t first, slot;
  int count, pos0;
  if (kRuns) {
    slot = z;
    const Run run = RunOf(a.rows, static_cast<int>(slot), c.context, reports, a.status);
    first = run.first;
    count = run.count;
    pos0 = run.pos0;
  } else {
    first = z;
    pos0 = a.row_pos[first];
    slot = a.row_seq != nullptr ? a.row_seq[first] : first;
    count = pos0 >= 0 ? 1 : 0;
    if (count > 0 && (pos0 >= c.context || slot < 0 || slot >= c.slots)) {
      if (reports && a.status != nullptr) atomicOr(a.status, ACCEL_B200_STATUS_BAD_POSITION);
      count = 0;
    }
  }
  // Vectors v0 .. v0 + 7 of the run's count * G (row v / G, head v % G). A
  // whole cluster leaves here or none of it.
  const int64_t v0 = static_cast<int64_t>(group) * kVec, vectors = static_cast<int64_t>(count) * G;
  if (v0 >= vectors) {
    if (early) PdlWait();
    return;
  }
  // (A single row's vectors are its heads.)
  const Vectors place(kRuns ? v0 : 0, G);
  const int top_vec = static_cast<int>(Min64(kVec, vectors - v0)) - 1;
  const int row_lo = kRuns ? static_cast<int>(place.row0) : 0;
  const int row_hi = kRuns ? row_lo + static_cast<int>(place.Down(top_vec)) : 0;
  const bool mine = gid <= top_vec;
  const uint32_t my_down = kRuns ? place.Down(gid) : 0;
  const int my_row = mine && kRuns ? row_lo + static_cast<int>(my_down) : row_hi;
  const int my_pos = pos0 + my_row, my_near = NearOf(my_pos, a.window);
  const int pos_lo = pos0 + row_lo, pos_hi = pos0 + row_hi;
  const int near_lo = NearOf(pos_lo, a.window), near_hi = NearOf(pos_hi, a.window);

  // Units that some vector sees: sinks before the windows, then the windows.
  const Units seen = UnitsOf(near_lo, pos_hi, a.sinks);
  const int unit0 = seen.near, sink_units = seen.sinks, units = seen.count;
  const int step = S * kWarps;

  const float* ksp = c.k_scale + slot * c.scale_seq_stride + g * c.scale_head_stride;
  const float* vsp = c.v_scale + slot * c.scale_seq_stride + g * c.scale_head_stride;
  const int unit_shift = a.block_shift - 5;  // units per scale block
  static_assert(kUnit == 32, "");
  const int plane_row = static_cast<int>((slot * c.seq_stride + g * c.head_stride) / D);

  // One lane of the warp copies its units; rows behind the context are of the
  // next run or zeros, and hidden.
  const auto unit_of = [&](int u) { return u < sink_units ? u : unit0 + (u - sink_units); };
  char* queue = smem + warp * Qu::kWarpBytes;
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + Qu::kBarriers) + warp * Qu::kStages;
  const auto issue = [&](int u, int stage) {
    if (lane == 0 && u < units) {
      const int row = plane_row + unit_of(u) * kUnit;
      char* dst = queue + stage * Qu::kUnitBytes;
      MbarArriveExpectTx(&full[stage], Qu::kUnitBytes);
      TmaLoad2D(dst, &tk, 0, row, &full[stage]);
      TmaLoad2D(dst + Qu::kPlaneBytes, &tv, 0, row, &full[stage]);
    }
  };
  if (lane == 0) {
    for (int i = 0; i < Qu::kStages; ++i) MbarInit(&full[i], 1);
    FenceBarrierInit();
  }
  int u = split * kWarps + warp;
  // Units in front of the row's own block do not wait for the previous kernel.
  const int settled = early ? pos_lo >> a.block_shift << a.block_shift : 0;
  const auto settles = [&](int i) { return u + i * step < units && unit_of(u + i * step) * kUnit < settled; };
  if (early) {
#pragma unroll
    for (int i = 0; i < Qu::kStages - 1; ++i) {
      if (settles(i)) issue(u + i * step, i);
    }
    PdlWait();
    load_query(z, group * kVec + gid, group * kVec + gid < G);
  }
#pragma unroll
  for (int i = 0; i < Qu::kStages - 1; ++i) {
    if (!early || !settles(i)) issue(u + i * step, i);
  }

  // Which token, and which dimensions, a lane's place in an MMA operand stands
  // for is free, as long as keys and queries, and weights and values, agree. It
  // is chosen so that a lane's share is a run of bytes and each shared-memory
  // phase of 8 (or 16) lanes covers all banks under the swizzle: column gid of
  // a score tile is token (gid / 2) + 4 (gid % 2), its low bit flipped for odd
  // gid; tig's share of a key row is the 16-byte pieces tig and tig + 4; gid's
  // share of a value row is 16-byte piece gid / 2 + 4 (gid % 2), or for 64
  // dimensions the 8-byte half gid % 2 of piece 2 ((gid / 2) % 2) + gid / 4.
  const auto token_of = [](int n) { return ((n >> 1) + 4 * (n & 1)) ^ (n & 1); };
  const auto dim_of = [](int n) {
    return D == 128 ? 16 * ((n >> 1) + 4 * (n & 1)) : 16 * (2 * ((n >> 1) & 1) + (n >> 2)) + 8 * (n & 1);
  };
  const auto piece_at = [](int row, int byte) {  // offset of a byte of a row under the swizzle
    return row * D + (byte ^ ((D == 128 ? row & 7 : (row >> 1) & 3) << 4));
  };
  const int key_at0 = piece_at(token_of(gid), 16 * tig), key_at1 = piece_at(token_of(gid), 64 % D + 16 * tig);
  const int value_at0 = piece_at(token_of(2 * tig), dim_of(gid)), value_at1 = piece_at(token_of(2 * tig + 1), dim_of(gid));

  // This lane's share of its query vector, as the two fp16 parts of q * 2^e.
  uint32_t qa[kKw][4];
  float factor;  // raw sums to scores in base 2 (without the key scale)
  {
    uint32_t amax = 0;
    if (kRuns) load_query(first + my_row, static_cast<int>(place.Head(gid, my_down)), mine);
#pragma unroll
    for (int j = 0; j < kKw; ++j) {
#pragma unroll
      for (int k = 0; k < 4; ++k) amax = max(amax, __float_as_uint(x[j][k]) & 0x7fffffffu);
    }
    amax = max(amax, __shfl_xor_sync(kFull, amax, 1));
    amax = max(amax, __shfl_xor_sync(kFull, amax, 2));
    const int e = min(13 + 127 - static_cast<int>(amax >> 23), 126);  // the largest to 2^13 .. 2^14
    const float up = __uint_as_float(static_cast<uint32_t>(127 + e) << 23);
    factor = __uint_as_float(static_cast<uint32_t>(127 - e) << 23) * (a.scale * kLog2e);
#pragma unroll
    for (int j = 0; j < kKw; ++j) {
      SplitPair(x[j][0] * up, x[j][1] * up, &qa[j][0], &qa[j][1]);
      SplitPair(x[j][2] * up, x[j][3] * up, &qa[j][2], &qa[j][3]);
    }
  }

  float m = -INFINITY, l = 0.f, o[kTiles][2];
#pragma unroll
  for (int i = 0; i < kTiles; ++i) o[i][0] = o[i][1] = 0.f;

  int stage = 0;
  uint32_t parity = 0;
  bool ok = true;
  for (; u < units; u += step) {
    const int t0 = unit_of(u) * kUnit;
    const float ks = ksp[unit_of(u) >> unit_shift], vs = vsp[unit_of(u) >> unit_shift];
    // The stage behind the last one read is free: every lane has read it.
    __syncwarp();
    issue(u + (Qu::kStages - 1) * step, stage == 0 ? Qu::kStages - 1 : stage - 1);
    ok = __all_sync(kFull, MbarWait(&full[stage], parity));
    if (!ok) break;
    const char* keys = queue + stage * Qu::kUnitBytes;
    const char* values = keys + Qu::kPlaneBytes;
    if (++stage == Qu::kStages) {
      stage = 0;
      parity ^= 1;
    }
    // Scores: tile i's columns 2 tig and 2 tig + 1 of vector gid.
    float s[4][2];
    {
      const float f = factor * ks;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float acc[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = 0; w < D / 64; ++w) {
          const uint4 x = *reinterpret_cast<const uint4*>(keys + i * 8 * D + (w == 0 ? key_at0 : key_at1));
          const uint32_t k4[4] = {x.x ^ 0x80808080u, x.y ^ 0x80808080u, x.z ^ 0x80808080u, x.w ^ 0x80808080u};
#pragma unroll
          for (int j = 0; j < 4; ++j) Mma16816(acc, qa[4 * w + j], Halves<false>(k4[j]), Halves<true>(k4[j]));
        }
        s[i][0] = (acc[0] + acc[2]) * f;
        s[i][1] = (acc[1] + acc[3]) * f;
      }
    }
    // A unit that not every vector sees whole.
    if (t0 + kUnit - 1 > pos_lo || (t0 < near_hi && t0 + kUnit > a.sinks)) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const int t = t0 + 8 * i + token_of(2 * tig + k);
          if (t > my_pos || (t < my_near && t >= a.sinks)) s[i][k] = -INFINITY;
        }
      }
    }
    float top = fmaxf(s[0][0], s[0][1]);
#pragma unroll
    for (int i = 1; i < 4; ++i) top = fmaxf(top, fmaxf(s[i][0], s[i][1]));
    if (__any_sync(kFull, top > m + kSlack)) {
      top = fmaxf(top, __shfl_xor_sync(kFull, top, 1));
      top = fmaxf(top, __shfl_xor_sync(kFull, top, 2));
      const float now = fmaxf(m, top);
      const float corr = now == -INFINITY ? 1.f : Exp2(m - now);
      m = now;
      l *= corr;
#pragma unroll
      for (int i = 0; i < kTiles; ++i) {
        o[i][0] *= corr;
        o[i][1] *= corr;
      }
    }
    // Weights, in the layout of an MMA operand. A vector that has seen nothing
    // yet has scores of -inf alone.
    const float ref = (m == -INFINITY ? 0.f : m) - kBias;
    uint32_t pa[2][4];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const float p0 = Exp2(s[2 * h][0] - ref), p1 = Exp2(s[2 * h][1] - ref);
      const float p2 = Exp2(s[2 * h + 1][0] - ref), p3 = Exp2(s[2 * h + 1][1] - ref);
      l += (p0 + p1) + (p2 + p3);
      SplitPair(p0, p1, &pa[h][0], &pa[h][1]);
      SplitPair(p2, p3, &pa[h][2], &pa[h][3]);
    }
    // Weighted values, four dimensions of this lane's run at a time.
    // Row 4 h + 2 t + k of vw: column 2 tig + k of score tile 2 h + t.
    uint32_t vw[8][kVw];
#pragma unroll
    for (int r = 0; r < 8; ++r) {
      const char* p = values + (r >> 1) * 8 * D + ((r & 1) == 0 ? value_at0 : value_at1);
      if (D == 64) {
        const uint2 x = *reinterpret_cast<const uint2*>(p);
        vw[r][0] = x.x ^ 0x80808080u;
        vw[r][1] = x.y ^ 0x80808080u;
      } else {
        const uint4 x = *reinterpret_cast<const uint4*>(p);
        vw[r][0] = x.x ^ 0x80808080u;
        vw[r][1] = x.y ^ 0x80808080u;
        vw[r][kVw - 2] = x.z ^ 0x80808080u;
        vw[r][kVw - 1] = x.w ^ 0x80808080u;
      }
    }
#pragma unroll
    for (int w = 0; w < kVw; ++w) {
      float acc[4][4];
#pragma unroll
      for (int k = 0; k < 4; ++k)
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[k][i] = 0.f;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        uint32_t x[2], y[2];  // tile 2 h + r's two tokens: dimensions 0 and 1, 2 and 3
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const uint32_t w0 = vw[4 * h + 2 * r][w], w1 = vw[4 * h + 2 * r + 1][w];
          x[r] = __byte_perm(w0, w1, 0x5140);
          y[r] = __byte_perm(w0, w1, 0x7362);
        }
        Mma16816(acc[0], pa[h], Halves<false>(x[0]), Halves<false>(x[1]));
        Mma16816(acc[1], pa[h], Halves<true>(x[0]), Halves<true>(x[1]));
        Mma16816(acc[2], pa[h], Halves<false>(y[0]), Halves<false>(y[1]));
        Mma16816(acc[3], pa[h], Halves<true>(y[0]), Halves<true>(y[1]));
      }
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        o[4 * w + k][0] = fmaf(vs, acc[k][0] + acc[k][2], o[4 * w + k][0]);
        o[4 * w + k][1] = fmaf(vs, acc[k][1] + acc[k][3], o[4 * w + k][1]);
      }
    }
  }
  if (!ok) {
    // A copy did not land: say so, give NaN, and let the copies still in
    // flight land before the bytes are used again (bounded waits).
    if (lane == 0 && a.status != nullptr) atomicOr(a.status, ACCEL_B200_STATUS_COPY_TIMEOUT);
    l = __int_as_float(0x7fc00000);
    for (int i = 0; i < Qu::kStages && u < units; ++i, u += step) {
      MbarWait(&full[stage], parity);
      if (++stage == Qu::kStages) {
        stage = 0;
        parity ^= 1;
      }
    }
  }
  __syncthreads();  // the queues' bytes become the states'

  // The warps' states to one, in order. Lane (gid, tig) holds dimensions
  // dim_of(2 tig + k) + i of vector gid.
  l += __shfl_xor_sync(kFull, l, 1);
  l += __shfl_xor_sync(kFull, l, 2);
  State<D>& ws = warp_state[warp];
#pragma unroll
  for (int k = 0; k < 2; ++k) {
#pragma unroll
    for (int i = 0; i < kTiles; i += 4) {
      *reinterpret_cast<float4*>(&ws.o[gid][dim_of(2 * tig + k) + i]) =
          make_float4(o[i][k], o[i + 1][k], o[i + 2][k], o[i + 3][k]);
    }
  }
  if (tig == 0) {
    ws.m[gid] = m;
    ws.l[gid] = l;
  }
  __syncthreads();
  // Element e of the CTA's vectors, four at a time.
  const auto store = [&](int e, float sum, float4 acc) {
    const int v = e / D;
    if (v <= top_vec) {
      const uint32_t down = kRuns ? place.Down(v) : 0, head = kRuns ? place.Head(v, down) : group * kVec + v;
      *reinterpret_cast<float4*>(a.out + (first + row_lo + down) * a.out_ld + static_cast<int64_t>(g * G + head) * D + e % D) =
          make_float4(acc.x / sum, acc.y / sum, acc.z / sum, acc.w / sum);
    }
  };
  // acc += f * x. A state that saw nothing (reference -inf) counts for nothing
  // with factor 1; one of NaN scores has reference -inf too, and a NaN sum
  // that must survive.
  const auto factor_of = [](float m_part, float m_all) { return m_part == -INFINITY ? 1.f : Exp2(m_part - m_all); };
  const auto add4 = [](float4* acc, float f, const float4& x) {
    acc->x = fmaf(x.x, f, acc->x);
    acc->y = fmaf(x.y, f, acc->y);
    acc->z = fmaf(x.z, f, acc->z);
    acc->w = fmaf(x.w, f, acc->w);
  };
#pragma unroll
  for (int e = 4 * tid; e < kVec * D; e += 4 * kThreads) {
    const int vec = e / D, d = e % D;
    float pm[kWarps], mx = -INFINITY, sum = 0.f;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      pm[w] = warp_state[w].m[vec];
      mx = fmaxf(mx, pm[w]);
    }
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const float f = factor_of(pm[w], mx);
      sum = fmaf(warp_state[w].l[vec], f, sum);
      add4(&acc, f, *reinterpret_cast<const float4*>(&warp_state[w].o[vec][d]));
    }
    if (S == 1) {
      store(e, sum, acc);
    } else {
      *reinterpret_cast<float4*>(&cta_state.o[vec][d]) = acc;
      if (d == 0) {
        cta_state.m[vec] = mx;
        cta_state.l[vec] = sum;
      }
    }
  }
  if (S == 1) return;

  if (kRows != Rows::kBalanced && S <= kMaxCluster) {
    ClusterSync();  // every CTA's state is there
    // CTA `split` merges every S-th group of 4 elements, all peers' loads in flight.
    for (int e = 4 * (split + S * tid); e < kVec * D; e += 4 * S * kThreads) {
      const int vec = e / D, d = e % D;
      float pm[kMaxCluster], pl[kMaxCluster], mx = -INFINITY, sum = 0.f;
      float4 po[kMaxCluster], acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int p = 0; p < kMaxCluster; ++p) {
        if (p < S) {
          pm[p] = LoadPeer(&cta_state.m[vec], static_cast<uint32_t>(p));
          pl[p] = LoadPeer(&cta_state.l[vec], static_cast<uint32_t>(p));
          po[p] = LoadPeer4(&cta_state.o[vec][d], static_cast<uint32_t>(p));
          mx = fmaxf(mx, pm[p]);
        }
      }
#pragma unroll
      for (int p = 0; p < kMaxCluster; ++p) {
        if (p < S) {
          const float f = factor_of(pm[p], mx);
          sum = fmaf(pl[p], f, sum);
          add4(&acc, f, po[p]);
        }
      }
      store(e, sum, acc);
    }
    ClusterSync();  // no CTA leaves while a peer may still read its state
    return;
  }

  // Through the workspace: a state per CTA, those of a group side by side; the
  // group's last CTA to arrive merges them.
  constexpr int kFloats = sizeof(State<D>) / 4;
  const bool flat = kRows == Rows::kBalanced;
  const int64_t at = flat ? static_cast<int64_t>(z) * c.kv_heads * ((G + kVec - 1) / kVec) + pair
                          : blockIdx.y + static_cast<int64_t>(gridDim.y) * blockIdx.z;
  const int64_t part0 = flat ? static_cast<int64_t>(blockIdx.x) - split : at * S;
  __syncthreads();
  float* part = a.parts + (part0 + split) * kFloats;
  for (int e = tid; e < kFloats / 4; e += kThreads) {
    reinterpret_cast<float4*>(part)[e] = reinterpret_cast<const float4*>(&cta_state)[e];
  }
  __syncthreads();
  if (tid == 0) {
    __threadfence();  // the barrier put the CTA's stores before it
    last = atomicAdd(a.counters + at, 1) == S - 1;
    if (last) a.counters[at] = 0;
    __threadfence();
  }
  __syncthreads();
  if (!last) return;
  const float* parts = a.parts + part0 * kFloats;
#pragma unroll
  for (int e = 4 * tid; e < kVec * D; e += 4 * kThreads) {
    const int vec = e / D;
    float mx = -INFINITY, sum = 0.f;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int p0 = 0; p0 < S; p0 += 8) {
      // Eight CTAs' loads in flight, then their states in order.
      float pm[8], pl[8];
      float4 po[8];
#pragma unroll
      for (int p = 0; p < 8; ++p) {
        const float* part_p = parts + static_cast<int64_t>(min(p0 + p, S - 1)) * kFloats;
        pm[p] = __ldcg(part_p + vec);
        pl[p] = __ldcg(part_p + kVec + vec);
        po[p] = __ldcg(reinterpret_cast<const float4*>(part_p + 2 * kVec + e));
      }
      float now = mx;
#pragma unroll
      for (int p = 0; p < 8; ++p) now = fmaxf(now, pm[p]);
      const float corr = factor_of(mx, now);
      sum *= corr;
      acc = make_float4(acc.x * corr, acc.y * corr, acc.z * corr, acc.w * corr);
      mx = now;
#pragma unroll
      for (int p = 0; p < 8; ++p) {
        if (p0 + p < S) {
          const float f = factor_of(pm[p], mx);
          sum = fmaf(pl[p], f, sum);
          add4(&acc, f, po[p]);
        }
      }
    }
    store(e, sum, acc);
  }
}

// How the vector groups of a call split the tokens they see.
struct Split {
  int64_t groups;  // grid y * z
  int vec_groups;  // per (sequence or row, kv head)
  int s;
  int balanced;    // CTAs of a balanced launch (0: none)
  size_t workspace;
};

Split SplitFor(const accel_b200_q8_cache& c, int64_t runs, int64_t rows_per_run, int32_t heads, int32_t window,
               int32_t sinks, bool single) {
  Split p{};
  p.vec_groups = static_cast<int>(CeilDiv(rows_per_run * (heads / c.kv_heads), kVec));
  p.groups = runs * c.kv_heads * p.vec_groups;
  // As many splits as fill the CTAs that are resident at once (a second wave
  // costs more than it balances), while a warp gets kWarpUnits units.
  const int64_t resident = kSms * (c.head_dim == 64 ? kResident<64> : kResident<128>);
  const int64_t seen = window > 0 ? Min64(c.context, static_cast<int64_t>(window) + sinks + rows_per_run) : c.context;
  const int64_t most = CeilDiv(CeilDiv(seen, kUnit), kWarps * kWarpUnits);
  const int64_t s = Max64(1, Min64(resident / Max64(1, p.groups), most));
  static_assert(kSms * kResident<64> <= kMaxCounters && kSms * kResident<128> <= kMaxCounters,
                "a counter per group: where they are split there are no more than resident CTAs");
  p.s = static_cast<int>(s);
  // Single rows of few, long sequences take CTAs by their own lengths, where the
  // grid has room for a CTA more per row and pair. (Measured with 8 kv heads
  // of 128: 16 sequences of 2048..16384 tokens 91 -> 61 us, of 4096..32768 178
  // -> 127; where all have the same length the states' way through the
  // workspace instead of the cluster costs 3 us of 51 to 97. A lane counts a row,
  // and a CTA serves one row and pair: beyond either limit the longest row's CTA
  // sets the time, 18 sequences of 2048..16384 tokens 78 us, 19 of them 142.)
  const bool few = single && runs <= 32 && p.groups <= resident / 2;
  if (few && (s > kMaxCluster || seen >= kBalanceFrom)) p.balanced = static_cast<int>(resident);
  if (s > kMaxCluster || p.balanced > 0) {
    const size_t state = static_cast<size_t>(2 * kVec + kVec * c.head_dim) * sizeof(float);
    p.workspace = kCounterRegion + static_cast<size_t>(resident) * state;
  }
  return p;
}

// Arrivals, then the CTAs' states.
void SetWorkspace(AttnArgs* a, void* workspace) {
  a->counters = static_cast<int32_t*>(workspace);
  a->parts = reinterpret_cast<float*>(static_cast<char*>(workspace) + kCounterRegion);
}

template <int D, Rows kRows>
int LaunchVectors(AttnArgs a, const Split& p, int64_t runs, void* workspace, cudaStream_t stream, const char* what) {
  if (p.workspace > 0) SetWorkspace(&a, workspace);
  a.single_rows = static_cast<int32_t>(runs);
  const dim3 grid = kRows == Rows::kBalanced
                        ? dim3(static_cast<unsigned>(p.balanced))
                        : dim3(static_cast<unsigned>(p.s), static_cast<unsigned>(a.cache.kv_heads * p.vec_groups),
                               static_cast<unsigned>(runs));
  const unsigned cluster = kRows != Rows::kBalanced && p.s <= kMaxCluster ? static_cast<unsigned>(p.s) : 1u;
  constexpr int kSmem = Queue<D>::kBytes + Queue<D>::kAlign;
  const cudaError_t err = cudaFuncSetAttribute(AttnVectorsQ8Kernel<D, kRows>,
                                               cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem);
  if (err != cudaSuccess) return CheckLaunchEx(err, what);
  const CUtensorMapSwizzle swizzle = D == 64 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_128B;
  const uint64_t plane_rows = static_cast<uint64_t>(PlaneRows(a.cache));
  CUtensorMap tk{}, tv{};
  if (!Encode2D(&tk, CU_TENSOR_MAP_DATA_TYPE_UINT8, a.cache.k, D, plane_rows, D, D, kUnit, swizzle) ||
      !Encode2D(&tv, CU_TENSOR_MAP_DATA_TYPE_UINT8, a.cache.v, D, plane_rows, D, D, kUnit, swizzle)) {
    return SetError(ACCEL_B200_EINVAL, std::string(what) + ": cache tensor map rejected");
  }
  return CheckLaunchEx(
      LaunchK(AttnVectorsQ8Kernel<D, kRows>, grid, dim3(kThreads), kSmem, stream, cluster, 1u, tk, tv, a), what);
}

int CheckWorkspace(size_t need, const void* workspace, size_t bytes, const std::string& what) {
  if (need == 0) return ACCEL_B200_OK;
  if (workspace == nullptr || bytes < need) return SetError(ACCEL_B200_EINVAL, what + ": workspace too small");
  if (reinterpret_cast<uintptr_t>(workspace) % 16 != 0) {
    return SetError(ACCEL_B200_EINVAL, what + ": the workspace must be 16-byte aligned");
  }
  return ACCEL_B200_OK;
}

// Whether a prefill takes the tiles of attention_q8_tiles.cu. Both kernels' times
// go by the tokens that rows see. A wave of tile CTAs (256 vectors per SM) walks
// 128 of them in about 2.4 us (3.0 at 128 dimensions), and where the last wave's
// walks are split, merging takes 20 us (37). The groups of 8 vectors here share
// the whole GPU at about 1700 (1100) of their units of 32 tokens per us. So tiles are
// faster from 900 groups per wave, or where walks are split from 900 per part of a
// wave and 9000 / steps for the merge.
// (Measured, tiles and groups. 3 kv heads of 64, 12 heads, behind 16000 tokens: 4
// sequences of 16 rows 42 and 32 us, of 32 rows 51 and 65, 32 of 16 rows 147 and 214;
// behind 5000: 4 of 32 rows 26 and 19, of 64 rows 30 and 43. 8 kv heads of 128, 32
// heads, behind 16000: 1 of 32 rows 42 and 33, of 64 rows 90 and 142, 32 of 8 rows 681
// and 451, of 16 rows 711 and 735; behind 300, unsplit: 32 of 8 rows 35 and 42. All of
// them in caches that they fill: the plan goes by the context, so that 64 rows behind
// 300 tokens of 16384 take tiles, 23 us, whose walks are then too short to be shared,
// where in a cache of 2048 the groups take 7.)
constexpr double kTileGroups = 900, kSplitGroupSteps = 9000;
bool TakesTiles(const accel_b200_q8_cache& c, int64_t batch, int64_t max_rows, int32_t heads, const TilesPlan& plan) {
  const int64_t groups = batch * c.kv_heads * CeilDiv(max_rows * (heads / c.kv_heads), kVec);
  double least = kTileGroups * ceil(plan.waves);
  if (plan.split) least = fmin(least, kTileGroups * plan.waves + kSplitGroupSteps / static_cast<double>(plan.steps));
  return static_cast<double>(groups) > least;
}

AttnArgs ArgsOf(const float* q, int64_t q_ld, const accel_b200_q8_cache* cache, const RaggedRows& rows,
                const int32_t* row_seq, const int32_t* row_pos, int32_t heads, int32_t window, int32_t sinks,
                float* out, int64_t out_ld, int32_t* status) {
  AttnArgs a{};
  a.q = q;
  a.q_ld = q_ld;
  a.cache = *cache;
  a.rows = rows;
  a.row_seq = row_seq;
  a.row_pos = row_pos;
  a.heads = heads;
  a.group = heads / cache->kv_heads;
  a.block_shift = cache->block == 32 ? 5 : cache->block == 64 ? 6 : 7;
  a.window = window;
  a.sinks = sinks;
  a.scale = 1.f / sqrtf(static_cast<float>(cache->head_dim));
  a.out = out;
  a.out_ld = out_ld;
  a.status = status;
  return a;
}

// Whether sizes are those of a prefill call that has something to do.
bool PrefillSizes(const accel_b200_q8_cache* cache, int32_t batch, int32_t max_rows, int32_t heads, int32_t window,
                  int32_t sinks, const char* what) {
  return CheckQ8Cache(cache, what) == ACCEL_B200_OK && batch > 0 && max_rows > 0 && heads > 0 &&
         heads % cache->kv_heads == 0 && window >= 0 && sinks >= 0;
}

int CheckAttention(const float* q, int64_t q_ld, const accel_b200_q8_cache* cache, int32_t heads, int32_t window,
                   int32_t sinks, const float* out, int64_t out_ld, int64_t rows, const std::string& what) {
  const int rc = CheckQ8Cache(cache, what.c_str());
  if (rc != ACCEL_B200_OK) return rc;
  if (heads <= 0 || heads % cache->kv_heads != 0 || window < 0 || sinks < 0 || q == nullptr || out == nullptr) {
    return SetError(ACCEL_B200_EINVAL, what + ": bad arguments");
  }
  const int64_t width = static_cast<int64_t>(heads) * cache->head_dim;
  if (q_ld < width || out_ld < width) return SetError(ACCEL_B200_EINVAL, what + ": row strides too small");
  if (q_ld % 4 != 0 || out_ld % 4 != 0 || (reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(out)) % 16 != 0) {
    return SetError(ACCEL_B200_EINVAL, what + ": rows must be 16-byte aligned");
  }
  if (!RowsApart(q, q_ld, width, out, out_ld, width, rows)) {
    return SetError(ACCEL_B200_EINVAL, what + ": out overlaps q otherwise than in place");
  }
  if (heads > 65535) return SetError(ACCEL_B200_EINVAL, what + ": more than 65535 heads");
  return ACCEL_B200_OK;
}

}  // namespace
}  // namespace accel_b200

using namespace accel_b200;

extern "C" {

ACCEL_B200_API size_t accel_b200_attention_decode_q8_workspace(const accel_b200_q8_cache* cache, int64_t rows,
                                                               int32_t heads, int32_t window, int32_t sinks) {
  if (CheckQ8Cache(cache, "attention_decode_q8_workspace") != ACCEL_B200_OK || rows <= 0 || heads <= 0 ||
      heads % cache->kv_heads != 0 || window < 0 || sinks < 0) {
    return 0;
  }
  return SplitFor(*cache, rows, 1, heads, window, sinks, true).workspace;
}

ACCEL_B200_API int accel_b200_attention_decode_q8_prefetch(const float* q, int64_t q_ld, const accel_b200_q8_cache* cache,
                                                  const int32_t* row_seq, const int32_t* row_pos, int64_t rows,
                                                  int32_t heads, int32_t window, int32_t sinks, float* out,
                                                  int64_t out_ld, void* workspace, size_t workspace_bytes,
                                                  int32_t* status, const accel_b200_l2_prefetch* prefetch,
                                                  void* stream) {
  int rc = CheckAttention(q, q_ld, cache, heads, window, sinks, out, out_ld, rows, "attention_decode_q8");
  if (rc != ACCEL_B200_OK) return rc;
  if (rows < 0 || row_pos == nullptr) return SetError(ACCEL_B200_EINVAL, "attention_decode_q8: bad arguments");
  if (row_seq == nullptr && rows > cache->slots) {
    return SetError(ACCEL_B200_EINVAL, "attention_decode_q8: more rows than cache slots");
  }
  if (rows == 0) return ClearError();
  if (rows > 65535) return SetError(ACCEL_B200_EINVAL, "attention_decode_q8: more than 65535 rows");
  if (prefetch != nullptr) {
    rc = CheckPrefetch(*prefetch, "attention_decode_q8");
    if (rc != ACCEL_B200_OK) return rc;
  }
  const Split p = SplitFor(*cache, rows, 1, heads, window, sinks, true);
  if (static_cast<int64_t>(cache->kv_heads) * p.vec_groups > 65535) {
    return SetError(ACCEL_B200_EINVAL, "attention_decode_q8: grid too large");
  }
  rc = CheckWorkspace(p.workspace, workspace, workspace_bytes, "attention_decode_q8");
  if (rc != ACCEL_B200_OK) return rc;
  AttnArgs a = ArgsOf(q, q_ld, cache, RaggedRows{}, row_seq, row_pos, heads, window, sinks, out, out_ld, status);
  if (prefetch != nullptr) a.prefetch = *prefetch;
  const char* what = "attention_decode_q8";
  cudaStream_t st = AsStream(stream);
  if (p.balanced > 0) {
    return cache->head_dim == 64 ? LaunchVectors<64, Rows::kBalanced>(a, p, rows, workspace, st, what)
                                 : LaunchVectors<128, Rows::kBalanced>(a, p, rows, workspace, st, what);
  }
  return cache->head_dim == 64 ? LaunchVectors<64, Rows::kSingle>(a, p, rows, workspace, st, what)
                               : LaunchVectors<128, Rows::kSingle>(a, p, rows, workspace, st, what);
}

ACCEL_B200_API int accel_b200_attention_decode_q8(const float* q, int64_t q_ld, const accel_b200_q8_cache* cache,
                                                  const int32_t* row_seq, const int32_t* row_pos, int64_t rows,
                                                  int32_t heads, int32_t window, int32_t sinks, float* out,
                                                  int64_t out_ld, void* workspace, size_t workspace_bytes,
                                                  int32_t* status, void* stream) {
  return accel_b200_attention_decode_q8_prefetch(q, q_ld, cache, row_seq, row_pos, rows, heads, window, sinks, out,
                                                 out_ld, workspace, workspace_bytes, status, nullptr, stream);
}

ACCEL_B200_API size_t accel_b200_attention_prefill_q8_workspace(const accel_b200_q8_cache* cache, int32_t batch,
                                                                int32_t max_rows, int32_t heads, int32_t window,
                                                                int32_t sinks) {
  if (!PrefillSizes(cache, batch, max_rows, heads, window, sinks, "attention_prefill_q8_workspace")) return 0;
  max_rows = static_cast<int32_t>(Min64(max_rows, cache->context));
  const TilesPlan tiles = PlanTilesQ8(*cache, batch, max_rows, heads, window, sinks);
  if (TakesTiles(*cache, batch, max_rows, heads, tiles)) return tiles.workspace;
  return SplitFor(*cache, batch, max_rows, heads, window, sinks, false).workspace;
}

ACCEL_B200_API int accel_b200_attention_prefill_q8_tiles(const accel_b200_q8_cache* cache, int32_t batch,
                                                         int32_t max_rows, int32_t heads, int32_t window,
                                                         int32_t sinks) {
  if (!PrefillSizes(cache, batch, max_rows, heads, window, sinks, "attention_prefill_q8_tiles")) return 0;
  max_rows = static_cast<int32_t>(Min64(max_rows, cache->context));
  return TakesTiles(*cache, batch, max_rows, heads, PlanTilesQ8(*cache, batch, max_rows, heads, window, sinks)) ? 1 : 0;
}

ACCEL_B200_API int accel_b200_attention_prefill_q8(const float* q, int64_t q_ld, const accel_b200_q8_cache* cache,
                                                   const int32_t* first, const int32_t* count, const int32_t* pos0,
                                                   int32_t batch, int32_t max_rows, int64_t rows, int32_t heads,
                                                   int32_t window, int32_t sinks, float* out, int64_t out_ld,
                                                   void* workspace, size_t workspace_bytes, int32_t* status,
                                                   void* stream) {
  int rc = CheckAttention(q, q_ld, cache, heads, window, sinks, out, out_ld, rows, "attention_prefill_q8");
  if (rc != ACCEL_B200_OK) return rc;
  if (rows < 0 || batch < 0 || max_rows < 0 || first == nullptr || count == nullptr || pos0 == nullptr) {
    return SetError(ACCEL_B200_EINVAL, "attention_prefill_q8: bad arguments");
  }
  if (batch > cache->slots) return SetError(ACCEL_B200_EINVAL, "attention_prefill_q8: more sequences than cache slots");
  if (rows == 0 || batch == 0 || max_rows == 0) return ClearError();
  if (batch > 65535) return SetError(ACCEL_B200_EINVAL, "attention_prefill_q8: more than 65535 sequences");
  max_rows = static_cast<int32_t>(Min64(max_rows, cache->context));  // a longer run does not fit
  AttnArgs a = ArgsOf(q, q_ld, cache, RaggedRows{first, count, pos0, max_rows, rows}, nullptr, nullptr, heads, window,
                      sinks, out, out_ld, status);
  a.sequences = batch;
  const TilesPlan tiles = PlanTilesQ8(*cache, batch, max_rows, heads, window, sinks);
  if (TakesTiles(*cache, batch, max_rows, heads, tiles)) {
    rc = CheckWorkspace(tiles.workspace, workspace, workspace_bytes, "attention_prefill_q8");
    if (rc != ACCEL_B200_OK) return rc;
    if (tiles.workspace > 0) SetWorkspace(&a, workspace);
    return LaunchTilesQ8(a, tiles, max_rows, AsStream(stream));
  }
  const Split p = SplitFor(*cache, batch, max_rows, heads, window, sinks, false);
  if (static_cast<int64_t>(cache->kv_heads) * p.vec_groups > 65535) {
    return SetError(ACCEL_B200_EINVAL, "attention_prefill_q8: grid too large");
  }
  rc = CheckWorkspace(p.workspace, workspace, workspace_bytes, "attention_prefill_q8");
  if (rc != ACCEL_B200_OK) return rc;
  const char* what = "attention_prefill_q8";
  cudaStream_t st = AsStream(stream);
  return cache->head_dim == 64 ? LaunchVectors<64, Rows::kRuns>(a, p, batch, workspace, st, what)
                               : LaunchVectors<128, Rows::kRuns>(a, p, batch, workspace, st, what);
}

}  // extern "C"
