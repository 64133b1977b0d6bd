// Ranges that an attention kernel brings into L2 for later kernels
// (accel_b200_l2_prefetch): the host's check and the device's share.
#pragma once

#include <stdint.h>

#include <string>

#include "accel_b200.h"
#include "common.cuh"
#include "tma.cuh"

namespace accel_b200 {

inline int CheckPrefetch(const accel_b200_l2_prefetch& prefetch, const char* what) {
  if (prefetch.count < 0 || prefetch.count > 4 || (prefetch.flags & ~ACCEL_B200_ATTN_CACHE_BEFORE_WAIT) != 0) {
    return SetError(ACCEL_B200_EINVAL, std::string(what) + ": bad prefetch");
  }
  for (int i = 0; i < prefetch.count; ++i) {
    if (prefetch.bytes[i] < 0 || (prefetch.bytes[i] > 0 && prefetch.ptr[i] == nullptr) ||
        reinterpret_cast<uintptr_t>(prefetch.ptr[i]) % 16 != 0) {
      return SetError(ACCEL_B200_EINVAL, std::string(what) + ": prefetch ranges must be 16-byte aligned");
    }
  }
  return ACCEL_B200_OK;
}

constexpr int64_t kPrefetchChunk = 32 * 1024;  // bytes per L2 prefetch instruction

// This CTA's share of the prefetch ranges: chunk c of the ranges' 32 KiB
// chunks goes to CTA c mod (CTAs).
__device__ __forceinline__ void PrefetchShare(const accel_b200_l2_prefetch& pf) {
  const int64_t cta = blockIdx.x + static_cast<int64_t>(gridDim.x) * (blockIdx.y + static_cast<int64_t>(gridDim.y) *
                                                                                       blockIdx.z);
  const int64_t ctas = static_cast<int64_t>(gridDim.x) * gridDim.y * gridDim.z;
  for (int i = 0; i < pf.count && i < 4; ++i) {
    const char* base = static_cast<const char*>(pf.ptr[i]);
    for (int64_t off = cta * kPrefetchChunk; off < pf.bytes[i]; off += ctas * kPrefetchChunk) {
      const uint32_t n = static_cast<uint32_t>(Min64(kPrefetchChunk, pf.bytes[i] - off)) & ~15u;
      if (n > 0) PrefetchL2(base + off, n);
    }
  }
}

}  // namespace accel_b200
