// Writing the int8 key/value cache (RoPE, quantising, append) and reading rows
// back (include/accel_b200.h, "int8 key/value cache").
//
// Write. One CTA owns one (sequence, block of tokens, plane) of a call, where a
// plane is the keys or the values of one kv head; it holds all of the block's
// new rows in registers (at most 128 rows of 128 floats over 256 threads), so
// the rows are read once: load and rotate, largest magnitude over the CTA,
// scale, quantise, store. Because the CTA also owns the block's scale and the
// rows the block already holds, growing the scale needs no atomics and the
// result does not depend on scheduling. Query heads are rotated by CTAs of
// their own in the same grid. Bound by HBM at prompt sizes (4 bytes in per
// element, 1 out for keys and values, 4 out for queries), by launch and one
// memory round trip at decode sizes.
//
// Read. One CTA owns 64 rows of one plane; a thread turns 4 bytes into one
// 16-byte store, so loads and stores of a warp are contiguous. Bound by the
// fp32 stores.
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>

#include "accel_b200.h"
#include "common.cuh"
#include "q8_cache.cuh"

namespace accel_b200 {
namespace {

constexpr int kThreads = 256;
constexpr int kReadRows = 64;

struct AppendArgs {
  const float* qkv;
  int64_t qkv_ld;
  accel_b200_q8_cache cache;
  RaggedRows rows;
  int32_t heads;
  const float* cos_t;
  const float* sin_t;
  float* q_out;
  int64_t q_ld;
  int32_t* status;
};

// The least power of two s >= 2^-126 with amax <= 127 * s, from the bits of a
// finite amax >= 0: amax = 1.m * 2^e needs 2^(e - 6) up to 1.m = 127 / 64
// (mantissa 0x7e0000) and 2^(e - 5) above.
__device__ __forceinline__ float ScaleFor(uint32_t amax_bits) {
  int e = static_cast<int>(amax_bits >> 23) - 6 + ((amax_bits & 0x7fffffu) > 0x7e0000u ? 1 : 0);
  e = max(e, 1);
  return __uint_as_float(static_cast<uint32_t>(e) << 23);
}

// rint(x / s) clamped to the int8 range, NaN to 0. For a power of two s with a
// normal reciprocal, x * inv is the same quotient.
__device__ __forceinline__ int32_t Quantise(float x, float s, float inv, bool exact_inv) {
  const float y = exact_inv ? __fmul_rn(x, inv) : __fdiv_rn(x, s);
  return x != x ? 0 : __float2int_rn(fminf(fmaxf(y, -127.f), 127.f));
}

__device__ __forceinline__ uint32_t Pack4(int32_t a, int32_t b, int32_t c, int32_t d) {
  return (static_cast<uint32_t>(a) & 0xffu) | (static_cast<uint32_t>(b) & 0xffu) << 8 |
         (static_cast<uint32_t>(c) & 0xffu) << 16 | static_cast<uint32_t>(d) << 24;
}

// The bytes of `w`, scaled by `ratio` and rounded again.
__device__ __forceinline__ uint32_t Rescale4(uint32_t w, float ratio) {
  int32_t q[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float x = static_cast<float>(static_cast<int8_t>(w >> (8 * i)));
    q[i] = __float2int_rn(fminf(fmaxf(__fmul_rn(x, ratio), -127.f), 127.f));
  }
  return Pack4(q[0], q[1], q[2], q[3]);
}

// IT: how many items (4 + 4 elements of a row, one of each half) a thread may
// hold. Grid (block of the sequence, plane or query head, sequence).
template <int D, int IT>
__global__ void __launch_bounds__(kThreads) RopeAppendQ8Kernel(AppendArgs a) {
  constexpr int kHalf = D / 2;
  constexpr int kPerRow = D / 8;  // items of a row
  __shared__ uint32_t red[kThreads / 32];
  // The next kernel starts only behind this wait, so that every kernel before
  // this one has completed by then (the decode attention reads the blocks that
  // this one leaves alone meanwhile).
  PdlWait();
  PdlTrigger();
  const accel_b200_q8_cache& c = a.cache;
  const int b = blockIdx.z, y = blockIdx.y;
  const Run run = RunOf(a.rows, b, c.context, blockIdx.x == 0 && y == 0 && threadIdx.x == 0, a.status);
  if (run.count == 0) return;
  const int64_t j = run.pos0 / c.block + static_cast<int64_t>(blockIdx.x);  // block of the slot
  const int64_t base = j * c.block;
  const int64_t lo = Max64(base, run.pos0);
  const int n = static_cast<int>(Min64(base + c.block, static_cast<int64_t>(run.pos0) + run.count) - lo);
  if (n <= 0) return;
  const bool is_q = y >= 2 * c.kv_heads, is_k = y < c.kv_heads;
  const int g = is_k ? y : y - c.kv_heads;
  // Column of the head in a qkv row: q | k | v.
  const int64_t col = static_cast<int64_t>(is_q ? y - 2 * c.kv_heads : is_k ? a.heads + y : a.heads + y) * D;
  const int64_t row0 = run.first + (lo - run.pos0);

  // All items' loads in flight, then the rotation.
  float4 x0[IT], x1[IT];
#pragma unroll
  for (int i = 0; i < IT; ++i) {
    const int item = threadIdx.x + i * blockDim.x;
    const int r = item / kPerRow, d = item % kPerRow * 4;
    if (r < n) {
      const float* p = a.qkv + (row0 + r) * a.qkv_ld + col + d;
      x0[i] = *reinterpret_cast<const float4*>(p);
      x1[i] = *reinterpret_cast<const float4*>(p + kHalf);
    } else {
      x0[i] = x1[i] = make_float4(0.f, 0.f, 0.f, 0.f);
    }
  }
  if (is_q || is_k) {
#pragma unroll
    for (int i = 0; i < IT; ++i) {
      const int item = threadIdx.x + i * blockDim.x;
      const int r = item / kPerRow, d = item % kPerRow * 4;
      if (r < n) {
        const int64_t at = (lo + r) * D + d;
        float cs[8], sn[8];
        *reinterpret_cast<float4*>(cs) = __ldg(reinterpret_cast<const float4*>(a.cos_t + at));
        *reinterpret_cast<float4*>(cs + 4) = __ldg(reinterpret_cast<const float4*>(a.cos_t + at + kHalf));
        *reinterpret_cast<float4*>(sn) = __ldg(reinterpret_cast<const float4*>(a.sin_t + at));
        *reinterpret_cast<float4*>(sn + 4) = __ldg(reinterpret_cast<const float4*>(a.sin_t + at + kHalf));
        float* lo4 = reinterpret_cast<float*>(&x0[i]);
        float* hi4 = reinterpret_cast<float*>(&x1[i]);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          float u, v;
          RopePair(lo4[k], hi4[k], cs, sn, k, 4, &u, &v);
          lo4[k] = u;
          hi4[k] = v;
        }
        if (is_q) {
          float* p = a.q_out + (row0 + r) * a.q_ld + col + d;
          *reinterpret_cast<float4*>(p) = x0[i];
          *reinterpret_cast<float4*>(p + kHalf) = x1[i];
        }
      }
    }
  }
  if (is_q) return;

  // Largest finite magnitude (positive floats order as their bits).
  uint32_t amax = 0;
  bool odd = false;
#pragma unroll
  for (int i = 0; i < IT; ++i) {
    const float e[8] = {x0[i].x, x0[i].y, x0[i].z, x0[i].w, x1[i].x, x1[i].y, x1[i].z, x1[i].w};
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const uint32_t bits = __float_as_uint(e[k]) & 0x7fffffffu;
      if (bits < 0x7f800000u) {
        amax = max(amax, bits);
      } else {
        odd = true;
      }
    }
  }
  if (odd && a.status != nullptr) atomicOr(a.status, ACCEL_B200_STATUS_NONFINITE);
  int8_t* plane = (is_k ? c.k : c.v) + b * c.seq_stride + g * c.head_stride;
  float* scale = (is_k ? c.k_scale : c.v_scale) + b * c.scale_seq_stride + g * c.scale_head_stride + j;
  const int old_rows = static_cast<int>(lo - base);
  const float was = old_rows > 0 ? *scale : 0.f;  // every thread reads it before the barrier, thread 0 writes behind it
  amax = __reduce_max_sync(kFull, amax);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = amax;
  __syncthreads();
  for (int w = 0; w < static_cast<int>(blockDim.x >> 5); ++w) amax = max(amax, red[w]);

  const bool held = old_rows > 0 && was > 0.f && was < INFINITY;
  const bool keep = held && __fmul_rn(127.f, was) >= __uint_as_float(amax);
  const float s = keep ? was : ScaleFor(amax);
  if (threadIdx.x == 0 && !keep) *scale = s;
  if (old_rows > 0 && !keep) {
    const float ratio = held ? __fdiv_rn(was, s) : 0.f;
    uint4* p = reinterpret_cast<uint4*>(plane + base * D);
    for (int i = threadIdx.x; i < old_rows * (D / 16); i += blockDim.x) {
      uint4 w = p[i];
      w.x = Rescale4(w.x, ratio);
      w.y = Rescale4(w.y, ratio);
      w.z = Rescale4(w.z, ratio);
      w.w = Rescale4(w.w, ratio);
      p[i] = w;
    }
  }
  const float inv = __fdiv_rn(1.f, s);
  const bool exact_inv = (__float_as_uint(s) & 0x7fffffu) == 0 && __float_as_uint(s) >= 0x00800000u;
#pragma unroll
  for (int i = 0; i < IT; ++i) {
    const int item = threadIdx.x + i * blockDim.x;
    const int r = item / kPerRow, d = item % kPerRow * 4;
    if (r < n) {
      int8_t* p = plane + (lo + r) * D + d;
      *reinterpret_cast<uint32_t*>(p) =
          Pack4(Quantise(x0[i].x, s, inv, exact_inv), Quantise(x0[i].y, s, inv, exact_inv),
                Quantise(x0[i].z, s, inv, exact_inv), Quantise(x0[i].w, s, inv, exact_inv));
      *reinterpret_cast<uint32_t*>(p + kHalf) =
          Pack4(Quantise(x1[i].x, s, inv, exact_inv), Quantise(x1[i].y, s, inv, exact_inv),
                Quantise(x1[i].z, s, inv, exact_inv), Quantise(x1[i].w, s, inv, exact_inv));
    }
  }
}

struct ReadArgs {
  accel_b200_q8_cache cache;
  RaggedRows rows;
  float* k_out;
  float* v_out;
  int64_t out_ld;
  int32_t* status;
};

// Grid (64-row tile of the sequence, plane, sequence).
template <int D>
__global__ void __launch_bounds__(kThreads) CacheRowsQ8Kernel(ReadArgs a) {
  constexpr int kPerRow = D / 4;  // 4-element items of a row
  PdlTrigger();
  PdlWait();
  const accel_b200_q8_cache& c = a.cache;
  const int b = blockIdx.z, y = blockIdx.y;
  const Run run = RunOf(a.rows, b, c.context, blockIdx.x == 0 && y == 0 && threadIdx.x == 0, a.status);
  const int r0 = static_cast<int>(blockIdx.x) * kReadRows;
  const int n = min(kReadRows, run.count - r0);  // tiles behind the sequence: none
  const bool is_k = y < c.kv_heads;
  float* out = is_k ? a.k_out : a.v_out;
  if (n <= 0 || out == nullptr) return;
  const int g = is_k ? y : y - c.kv_heads;
  const int64_t t0 = static_cast<int64_t>(run.pos0) + r0;
  const int8_t* plane = (is_k ? c.k : c.v) + b * c.seq_stride + g * c.head_stride + t0 * D;
  const float* scale = (is_k ? c.k_scale : c.v_scale) + b * c.scale_seq_stride + g * c.scale_head_stride;
  out += (run.first + r0) * a.out_ld + static_cast<int64_t>(g) * D;
  constexpr int kIt = kReadRows * kPerRow / kThreads;
  uint32_t w[kIt];
  float s[kIt];
#pragma unroll
  for (int i = 0; i < kIt; ++i) {
    const int item = threadIdx.x + i * kThreads, r = item / kPerRow;
    if (r < n) {
      w[i] = *reinterpret_cast<const uint32_t*>(plane + item * 4);
      s[i] = scale[(t0 + r) / c.block];
    }
  }
#pragma unroll
  for (int i = 0; i < kIt; ++i) {
    const int item = threadIdx.x + i * kThreads, r = item / kPerRow, d = item % kPerRow * 4;
    if (r < n) {
      float4 v;
      v.x = __fmul_rn(static_cast<float>(static_cast<int8_t>(w[i])), s[i]);
      v.y = __fmul_rn(static_cast<float>(static_cast<int8_t>(w[i] >> 8)), s[i]);
      v.z = __fmul_rn(static_cast<float>(static_cast<int8_t>(w[i] >> 16)), s[i]);
      v.w = __fmul_rn(static_cast<float>(static_cast<int8_t>(w[i] >> 24)), s[i]);
      *reinterpret_cast<float4*>(out + r * a.out_ld + d) = v;
    }
  }
}

template <int D>
int LaunchAppend(const AppendArgs& a, int32_t batch, cudaStream_t stream) {
  const int32_t most = static_cast<int32_t>(Min64(a.cache.block, a.rows.max_rows));  // new rows of a block
  const int items = most * (D / 8);
  const int threads = items >= kThreads ? kThreads : static_cast<int>(CeilDiv(items, 32)) * 32;
  // Blocks that max_rows rows can touch, wherever in a block they begin.
  const int64_t blocks = CeilDiv(static_cast<int64_t>(a.rows.max_rows) - 1, a.cache.block) + 1;
  const dim3 grid(static_cast<unsigned>(blocks), static_cast<unsigned>(2 * a.cache.kv_heads + a.heads),
                  static_cast<unsigned>(batch));
  const int it = static_cast<int>(CeilDiv(items, threads));
  auto launch = [&](auto kernel) {
    return CheckLaunchEx(LaunchK(kernel, grid, dim3(threads), 0, stream, 1u, 1u, a), "rope_append_q8");
  };
  if (it <= 1) return launch(RopeAppendQ8Kernel<D, 1>);
  if (it <= 2) return launch(RopeAppendQ8Kernel<D, 2>);
  if (it <= 4) return launch(RopeAppendQ8Kernel<D, 4>);
  return launch(RopeAppendQ8Kernel<D, D / 16>);
}

}  // namespace
}  // namespace accel_b200

using namespace accel_b200;

extern "C" {

ACCEL_B200_API int accel_b200_rope_append_q8(const float* qkv, int64_t qkv_ld, int64_t rows,
                                             const accel_b200_q8_cache* cache, const int32_t* first,
                                             const int32_t* count, const int32_t* pos0, int32_t batch,
                                             int32_t max_rows, int32_t heads, const float* cos_table,
                                             const float* sin_table, float* q_out, int64_t q_ld, int32_t* status,
                                             void* stream) {
  const int rc = CheckQ8Cache(cache, "rope_append_q8");
  if (rc != ACCEL_B200_OK) return rc;
  if (rows < 0 || batch < 0 || max_rows < 0 || heads <= 0 || heads % cache->kv_heads != 0 || qkv == nullptr ||
      q_out == nullptr || first == nullptr || count == nullptr || pos0 == nullptr || cos_table == nullptr ||
      sin_table == nullptr) {
    return SetError(ACCEL_B200_EINVAL, "rope_append_q8: bad arguments");
  }
  if (batch > cache->slots) return SetError(ACCEL_B200_EINVAL, "rope_append_q8: more sequences than cache slots");
  const int64_t width = (static_cast<int64_t>(heads) + 2 * static_cast<int64_t>(cache->kv_heads));
  if (qkv_ld < width * cache->head_dim || q_ld < static_cast<int64_t>(heads) * cache->head_dim) {
    return SetError(ACCEL_B200_EINVAL, "rope_append_q8: row strides too small");
  }
  if (qkv_ld % 4 != 0 || q_ld % 4 != 0 ||
      (reinterpret_cast<uintptr_t>(qkv) | reinterpret_cast<uintptr_t>(q_out) | reinterpret_cast<uintptr_t>(cos_table) |
       reinterpret_cast<uintptr_t>(sin_table)) % 16 != 0) {
    return SetError(ACCEL_B200_EINVAL, "rope_append_q8: rows must be 16-byte aligned");
  }
  if (!RowsApart(qkv, qkv_ld, width * cache->head_dim, q_out, q_ld, static_cast<int64_t>(heads) * cache->head_dim, rows)) {
    return SetError(ACCEL_B200_EINVAL, "rope_append_q8: q_out overlaps qkv otherwise than in place");
  }
  if (batch == 0 || max_rows == 0 || rows == 0) return ClearError();
  if (batch > 65535 || width > 65535) return SetError(ACCEL_B200_EINVAL, "rope_append_q8: grid too large");
  max_rows = static_cast<int32_t>(Min64(max_rows, cache->context));  // a longer run does not fit
  const AppendArgs a{qkv,       qkv_ld,    *cache, RaggedRows{first, count, pos0, max_rows, rows}, heads,
                     cos_table, sin_table, q_out,  q_ld,                                           status};
  if (cache->head_dim == 64) return LaunchAppend<64>(a, batch, AsStream(stream));
  return LaunchAppend<128>(a, batch, AsStream(stream));
}

ACCEL_B200_API int accel_b200_cache_rows_q8(const accel_b200_q8_cache* cache, const int32_t* first,
                                            const int32_t* count, const int32_t* pos0, int32_t batch,
                                            int32_t max_rows, float* k_out, float* v_out, int64_t out_ld,
                                            int64_t rows, int32_t* status, void* stream) {
  const int rc = CheckQ8Cache(cache, "cache_rows_q8");
  if (rc != ACCEL_B200_OK) return rc;
  if (rows < 0 || batch < 0 || max_rows < 0 || first == nullptr || count == nullptr || pos0 == nullptr) {
    return SetError(ACCEL_B200_EINVAL, "cache_rows_q8: bad arguments");
  }
  if (batch > cache->slots) return SetError(ACCEL_B200_EINVAL, "cache_rows_q8: more sequences than cache slots");
  if (out_ld < static_cast<int64_t>(cache->kv_heads) * cache->head_dim) {
    return SetError(ACCEL_B200_EINVAL, "cache_rows_q8: row stride too small");
  }
  if (out_ld % 4 != 0 || (reinterpret_cast<uintptr_t>(k_out) | reinterpret_cast<uintptr_t>(v_out)) % 16 != 0) {
    return SetError(ACCEL_B200_EINVAL, "cache_rows_q8: rows must be 16-byte aligned");
  }
  if (k_out != nullptr && v_out != nullptr &&
      (k_out == v_out || !RowsApart(k_out, out_ld, static_cast<int64_t>(cache->kv_heads) * cache->head_dim, v_out, out_ld,
                                    static_cast<int64_t>(cache->kv_heads) * cache->head_dim, rows))) {
    return SetError(ACCEL_B200_EINVAL, "cache_rows_q8: k_out overlaps v_out");
  }
  if (batch == 0 || max_rows == 0 || rows == 0 || (k_out == nullptr && v_out == nullptr)) return ClearError();
  if (batch > 65535 || cache->kv_heads > 32767) return SetError(ACCEL_B200_EINVAL, "cache_rows_q8: grid too large");
  max_rows = static_cast<int32_t>(Min64(max_rows, cache->context));  // a longer run does not fit
  const ReadArgs a{*cache, RaggedRows{first, count, pos0, max_rows, rows}, k_out, v_out, out_ld, status};
  const dim3 grid(static_cast<unsigned>(CeilDiv(max_rows, kReadRows)), static_cast<unsigned>(2 * cache->kv_heads),
                  static_cast<unsigned>(batch));
  auto launch = [&](auto kernel) {
    return CheckLaunchEx(LaunchK(kernel, grid, dim3(kThreads), 0, AsStream(stream), 1u, 1u, a), "cache_rows_q8");
  };
  return cache->head_dim == 64 ? launch(CacheRowsQ8Kernel<64>) : launch(CacheRowsQ8Kernel<128>);
}

}  // extern "C"
