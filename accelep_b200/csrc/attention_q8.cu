// Attention over the int8 key/value cache (include/accel_b200.h, "int8 key/value
// cache"), causal, with an optional sliding window and first tokens (sinks)
// that stay visible: of single rows and of many rows per sequence.
//
// The row at position p sees [0, min(sinks, first)) and [first, p], where
// first = max(0, p - window + 1), or 0 without a window. One CTA takes one
// row and query head; each warp walks every fourth visible position with an
// online softmax (running maximum, sum and weighted values in fp32), and the
// warps' states are merged once.
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>

#include "accel_b200.h"
#include "common.cuh"
#include "q8_cache.cuh"

namespace accel_b200 {
namespace {

constexpr int kThreads = 128;
constexpr int kWarps = kThreads / 32;

struct AttnArgs {
  const float* q;
  int64_t q_ld;
  accel_b200_q8_cache cache;
  RaggedRows rows;         // prefill: rows by sequence
  const int32_t* row_seq;  // single rows: slot (null: the row's number) and position
  const int32_t* row_pos;
  int32_t heads;
  int32_t window;
  int32_t sinks;
  float scale;
  float* out;
  int64_t out_ld;
  int32_t* status;
};

template <int D>
__device__ void AttendRow(const AttnArgs& a, int64_t row, int64_t slot, int64_t pos, int h) {
  constexpr int kE = D / 32;  // elements of a row per lane
  const accel_b200_q8_cache& c = a.cache;
  __shared__ float sm[kWarps], sl[kWarps], so[kWarps][D];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int g = h / (a.heads / c.kv_heads);
  const int8_t* kp = c.k + slot * c.seq_stride + g * c.head_stride;
  const int8_t* vp = c.v + slot * c.seq_stride + g * c.head_stride;
  const float* ks = c.k_scale + slot * c.scale_seq_stride + g * c.scale_head_stride;
  const float* vs = c.v_scale + slot * c.scale_seq_stride + g * c.scale_head_stride;
  float q[kE], o[kE], m = -INFINITY, l = 0.f;
#pragma unroll
  for (int e = 0; e < kE; ++e) {
    q[e] = a.q[row * a.q_ld + static_cast<int64_t>(h) * D + lane * kE + e];
    o[e] = 0.f;
  }
  const int64_t near = a.window > 0 ? Max64(0, pos + 1 - a.window) : 0;
  const int64_t sinks = Min64(a.sinks, near), seen = sinks + pos + 1 - near;
  for (int64_t i = warp; i < seen; i += kWarps) {
    const int64_t t = i < sinks ? i : near + (i - sinks);
    float s = 0.f;
#pragma unroll
    for (int e = 0; e < kE; ++e) s = fmaf(q[e], static_cast<float>(kp[t * D + lane * kE + e]), s);
    s = WarpSum(s) * (a.scale * ks[t / c.block]);
    const float mx = fmaxf(m, s);
    const float corr = expf(m - mx), p = expf(s - mx);
    m = mx;
    l = l * corr + p;
    const float pv = p * vs[t / c.block];
#pragma unroll
    for (int e = 0; e < kE; ++e) o[e] = fmaf(pv, static_cast<float>(vp[t * D + lane * kE + e]), o[e] * corr);
  }
#pragma unroll
  for (int e = 0; e < kE; ++e) so[warp][lane * kE + e] = o[e];
  if (lane == 0) {
    sm[warp] = m;
    sl[warp] = l;
  }
  __syncthreads();
  if (threadIdx.x < D) {
    float mx = -INFINITY, sum = 0.f, acc = 0.f;
    for (int w = 0; w < kWarps; ++w) mx = fmaxf(mx, sm[w]);
    for (int w = 0; w < kWarps; ++w) {
      if (sm[w] == -INFINITY) continue;
      const float f = expf(sm[w] - mx);
      sum = fmaf(sl[w], f, sum);
      acc = fmaf(so[w][threadIdx.x], f, acc);
    }
    a.out[row * a.out_ld + static_cast<int64_t>(h) * D + threadIdx.x] = acc / sum;
  }
}

// Grid (row, head).
template <int D>
__global__ void __launch_bounds__(kThreads) AttnDecodeQ8Kernel(AttnArgs a) {
  PdlTrigger();
  PdlWait();
  const int64_t r = blockIdx.x;
  const int64_t pos = a.row_pos[r];
  if (pos < 0) return;
  const int64_t slot = a.row_seq != nullptr ? a.row_seq[r] : r;
  if (pos >= a.cache.context || slot < 0 || slot >= a.cache.slots) {
    if (blockIdx.y == 0 && threadIdx.x == 0 && a.status != nullptr) {
      atomicOr(a.status, ACCEL_B200_STATUS_BAD_POSITION);
    }
    return;
  }
  AttendRow<D>(a, r, slot, pos, blockIdx.y);
}

// Grid (row of the sequence, head, sequence).
template <int D>
__global__ void __launch_bounds__(kThreads) AttnPrefillQ8Kernel(AttnArgs a) {
  PdlTrigger();
  PdlWait();
  const int b = blockIdx.z;
  const Run run = RunOf(a.rows, b, a.cache.context, blockIdx.x == 0 && blockIdx.y == 0 && threadIdx.x == 0, a.status);
  const int i = blockIdx.x;
  if (i >= run.count) return;
  AttendRow<D>(a, run.first + i, b, static_cast<int64_t>(run.pos0) + i, blockIdx.y);
}

int CheckAttention(const float* q, int64_t q_ld, const accel_b200_q8_cache* cache, int32_t heads, int32_t window,
                   int32_t sinks, const float* out, int64_t out_ld, const std::string& what) {
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
  if (heads > 65535) return SetError(ACCEL_B200_EINVAL, what + ": more than 65535 heads");
  return ACCEL_B200_OK;
}

}  // namespace
}  // namespace accel_b200

using namespace accel_b200;

extern "C" {

ACCEL_B200_API size_t accel_b200_attention_decode_q8_workspace(const accel_b200_q8_cache* cache, int64_t rows,
                                                               int32_t heads, int32_t window, int32_t sinks) {
  (void)cache, (void)rows, (void)heads, (void)window, (void)sinks;
  return 0;
}

ACCEL_B200_API int accel_b200_attention_decode_q8(const float* q, int64_t q_ld, const accel_b200_q8_cache* cache,
                                                  const int32_t* row_seq, const int32_t* row_pos, int64_t rows,
                                                  int32_t heads, int32_t window, int32_t sinks, float* out,
                                                  int64_t out_ld, void* workspace, size_t workspace_bytes,
                                                  int32_t* status, void* stream) {
  (void)workspace, (void)workspace_bytes;
  const int rc = CheckAttention(q, q_ld, cache, heads, window, sinks, out, out_ld, "attention_decode_q8");
  if (rc != ACCEL_B200_OK) return rc;
  if (rows < 0 || row_pos == nullptr) return SetError(ACCEL_B200_EINVAL, "attention_decode_q8: bad arguments");
  if (row_seq == nullptr && rows > cache->slots) {
    return SetError(ACCEL_B200_EINVAL, "attention_decode_q8: more rows than cache slots");
  }
  if (rows == 0) return ClearError();
  if (rows > 65535) return SetError(ACCEL_B200_EINVAL, "attention_decode_q8: more than 65535 rows");
  const AttnArgs a{q,      q_ld,  *cache, RaggedRows{}, row_seq, row_pos, heads,
                   window, sinks, 1.f / sqrtf(static_cast<float>(cache->head_dim)), out, out_ld, status};
  const dim3 grid(static_cast<unsigned>(rows), static_cast<unsigned>(heads));
  auto launch = [&](auto kernel) {
    return CheckLaunchEx(LaunchK(kernel, grid, dim3(kThreads), 0, AsStream(stream), 1u, 1u, a), "attention_decode_q8");
  };
  return cache->head_dim == 64 ? launch(AttnDecodeQ8Kernel<64>) : launch(AttnDecodeQ8Kernel<128>);
}

ACCEL_B200_API size_t accel_b200_attention_prefill_q8_workspace(const accel_b200_q8_cache* cache, int32_t batch,
                                                                int32_t max_rows, int32_t heads, int32_t window,
                                                                int32_t sinks) {
  (void)cache, (void)batch, (void)max_rows, (void)heads, (void)window, (void)sinks;
  return 0;
}

ACCEL_B200_API int accel_b200_attention_prefill_q8(const float* q, int64_t q_ld, const accel_b200_q8_cache* cache,
                                                   const int32_t* first, const int32_t* count, const int32_t* pos0,
                                                   int32_t batch, int32_t max_rows, int64_t rows, int32_t heads,
                                                   int32_t window, int32_t sinks, float* out, int64_t out_ld,
                                                   void* workspace, size_t workspace_bytes, int32_t* status,
                                                   void* stream) {
  (void)workspace, (void)workspace_bytes;
  const int rc = CheckAttention(q, q_ld, cache, heads, window, sinks, out, out_ld, "attention_prefill_q8");
  if (rc != ACCEL_B200_OK) return rc;
  if (rows < 0 || batch < 0 || max_rows < 0 || first == nullptr || count == nullptr || pos0 == nullptr) {
    return SetError(ACCEL_B200_EINVAL, "attention_prefill_q8: bad arguments");
  }
  if (batch > cache->slots) return SetError(ACCEL_B200_EINVAL, "attention_prefill_q8: more sequences than cache slots");
  if (rows == 0 || batch == 0 || max_rows == 0) return ClearError();
  if (batch > 65535) return SetError(ACCEL_B200_EINVAL, "attention_prefill_q8: more than 65535 sequences");
  max_rows = static_cast<int32_t>(Min64(max_rows, cache->context));  // a longer run does not fit
  const AttnArgs a{q,      q_ld,  *cache, RaggedRows{first, count, pos0, max_rows, rows}, nullptr, nullptr, heads,
                   window, sinks, 1.f / sqrtf(static_cast<float>(cache->head_dim)), out, out_ld, status};
  const dim3 grid(static_cast<unsigned>(max_rows), static_cast<unsigned>(heads), static_cast<unsigned>(batch));
  auto launch = [&](auto kernel) {
    return CheckLaunchEx(LaunchK(kernel, grid, dim3(kThreads), 0, AsStream(stream), 1u, 1u, a), "attention_prefill_q8");
  };
  return cache->head_dim == 64 ? launch(AttnPrefillQ8Kernel<64>) : launch(AttnPrefillQ8Kernel<128>);
}

}  // extern "C"
