// The int8 key/value cache (accel_b200_q8_cache): host checks of its layout and
// of the ragged row lists that name its sequences, and the device side of both.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

#include <string>
#include <utility>

#include "accel_b200.h"
#include "common.cuh"

namespace accel_b200 {

// Whether n0 runs at stride s0 and, inside them, n1 runs at stride s1 of
// `inner` elements each do not overlap, in either order.
inline bool Disjoint(int64_t n0, int64_t s0, int64_t n1, int64_t s1, int64_t inner) {
  if (n1 <= 1) return n0 <= 1 || s0 >= inner;
  if (n0 <= 1) return s1 >= inner;
  return (s1 >= inner && s0 / n1 >= s1) || (s0 >= inner && s1 / n0 >= s0);
}

// Whether row buffers a (`wa` floats of each row, stride lda) and b may both be
// used when b is written: they do not touch, are the same rows, or are other
// columns of rows of the same stride.
inline bool RowsApart(const float* a, int64_t lda, int64_t wa, const float* b, int64_t ldb, int64_t wb, int64_t rows) {
  if (rows <= 0) return true;
  const intptr_t a0 = reinterpret_cast<intptr_t>(a), b0 = reinterpret_cast<intptr_t>(b);
  const intptr_t a1 = a0 + ((rows - 1) * lda + wa) * 4, b1 = b0 + ((rows - 1) * ldb + wb) * 4;
  if (a1 <= b0 || b1 <= a0) return true;
  if (rows > 1 && lda != ldb) return false;
  const int64_t delta = (b0 - a0) / 4;  // 16-byte aligned rows
  if (delta == 0) return true;
  return delta > 0 ? delta >= wa && (rows == 1 || delta + wb <= lda) : -delta >= wb && (rows == 1 || wa - delta <= lda);
}

// Whether runs of one layout touch runs of another like it (Disjoint in itself)
// that lies `delta` elements behind. A run of the other reaches a run of the
// first only next to where the strides put it: two candidates per level.
inline bool Touch(int64_t delta, int64_t n0, int64_t s0, int64_t n1, int64_t s1, int64_t inner) {
  if (n0 <= 1 || (n1 > 1 && s1 > s0)) {  // the wider stride first; a stride of one run counts for nothing
    std::swap(n0, n1);
    std::swap(s0, s1);
  }
  const auto steps = [](int64_t d, int64_t n, int64_t s) { return n <= 1 ? 0 : d / s - (d % s < 0 ? 1 : 0); };
  for (int i = 0; i < 2; ++i) {
    const int64_t i0 = steps(delta, n0, s0) + i;
    if (i0 <= -n0 || i0 >= n0) continue;
    const int64_t rest = delta - (i0 != 0 ? i0 * s0 : 0);
    for (int j = 0; j < 2; ++j) {
      const int64_t i1 = steps(rest, n1, s1) + j;
      if (i1 <= -n1 || i1 >= n1) continue;
      const int64_t off = rest - (i1 != 0 ? i1 * s1 : 0);
      if (off > -inner && off < inner) return true;
    }
  }
  return false;
}

constexpr int64_t kMostRows = (int64_t{1} << 31) - 256;  // of a plane: row numbers are 32-bit in its tensor map

// Rows of head_dim bytes from the first of a plane to behind its last run; row
// t of (slot s, head g) is (s * seq_stride + g * head_stride) / head_dim + t.
// Above kMostRows: some number above it.
inline int64_t PlaneRows(const accel_b200_q8_cache& c) {
  const auto span = [&](int64_t n, int64_t stride) {
    if (n <= 1) return int64_t{0};
    return stride / c.head_dim > kMostRows / (n - 1) ? kMostRows : (n - 1) * (stride / c.head_dim);
  };
  return span(c.slots, c.seq_stride) + span(c.kv_heads, c.head_stride) + c.context;
}

// ACCEL_B200_OK, or EINVAL with a message that begins with `what`.
inline int CheckQ8Cache(const accel_b200_q8_cache* c, const char* what) {
  const std::string w(what);
  if (c == nullptr || c->k == nullptr || c->v == nullptr || c->k_scale == nullptr || c->v_scale == nullptr) {
    return SetError(ACCEL_B200_EINVAL, w + ": the cache has a null plane");
  }
  if (c->head_dim != 64 && c->head_dim != 128) {
    return SetError(ACCEL_B200_EINVAL, w + ": head_dim must be 64 or 128");
  }
  if (c->block != 32 && c->block != 64 && c->block != 128) {
    return SetError(ACCEL_B200_EINVAL, w + ": block must be 32, 64 or 128 tokens");
  }
  if (c->slots <= 0 || c->kv_heads <= 0 || c->context <= 0) {
    return SetError(ACCEL_B200_EINVAL, w + ": the cache has no slots, heads or context");
  }
  if (c->context > (1 << 30)) return SetError(ACCEL_B200_EINVAL, w + ": more than 2^30 positions");
  if ((reinterpret_cast<uintptr_t>(c->k) | reinterpret_cast<uintptr_t>(c->v)) % 16 != 0 || c->seq_stride % c->head_dim != 0 ||
      c->head_stride % c->head_dim != 0) {
    return SetError(ACCEL_B200_EINVAL, w + ": the planes must be 16-byte aligned, their strides whole rows");
  }
  if ((reinterpret_cast<uintptr_t>(c->k_scale) | reinterpret_cast<uintptr_t>(c->v_scale)) % 4 != 0) {
    return SetError(ACCEL_B200_EINVAL, w + ": cache scales must be 4-byte aligned");
  }
  const int64_t run = static_cast<int64_t>(c->context) * c->head_dim;
  const int64_t blocks = CeilDiv(c->context, c->block);
  if (!Disjoint(c->slots, c->seq_stride, c->kv_heads, c->head_stride, run) ||
      !Disjoint(c->slots, c->scale_seq_stride, c->kv_heads, c->scale_head_stride, blocks)) {
    return SetError(ACCEL_B200_EINVAL, w + ": cache strides do not hold the context");
  }
  const int64_t scales = reinterpret_cast<intptr_t>(c->v_scale) / 4 - reinterpret_cast<intptr_t>(c->k_scale) / 4;
  if (Touch(c->v - c->k, c->slots, c->seq_stride, c->kv_heads, c->head_stride, run) ||
      Touch(scales, c->slots, c->scale_seq_stride, c->kv_heads, c->scale_head_stride, blocks)) {
    return SetError(ACCEL_B200_EINVAL, w + ": keys and values overlap");
  }
  if (PlaneRows(*c) > kMostRows) return SetError(ACCEL_B200_EINVAL, w + ": more than 2^31 cache rows");
  return ACCEL_B200_OK;
}

// The rows of one sequence of a ragged list: sequence b owns `count` rows from
// `first` at positions pos0 + i. count 0: nothing to do, or not in bounds.
struct RaggedRows {
  const int32_t* first;
  const int32_t* count;
  const int32_t* pos0;
  int32_t max_rows;
  int64_t rows;  // rows of the buffers that first / count index
};

struct Run {
  int64_t first;
  int32_t count;
  int32_t pos0;
};

// Sequence b's rows, all inside the buffers and the cache. One that does not
// fit is empty here and, if `report`, noted in *status.
__device__ __forceinline__ Run RunOf(const RaggedRows& r, int b, int32_t context, bool report, int32_t* status) {
  Run run{r.first[b], r.count[b], r.pos0[b]};
  if (run.pos0 < 0 || run.count <= 0) return Run{0, 0, 0};
  if (run.count > r.max_rows || run.first < 0 || run.first + run.count > r.rows ||
      static_cast<int64_t>(run.pos0) + run.count > context) {
    if (report && status != nullptr) atomicOr(status, ACCEL_B200_STATUS_BAD_POSITION);
    return Run{0, 0, 0};
  }
  return run;
}

}  // namespace accel_b200
