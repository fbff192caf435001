// Shared by the kernels over the block-scaled 8-bit KV cache: e4m3 rows
// [num_blocks, block_size, Hk, 128] and one fp32 scale per (scale_block tokens, head),
// [num_blocks, block_size / scale_block, Hk].  A cache value stands for e4m3 * scale.
#pragma once

#include "hl_common.cuh"

namespace hl {

constexpr int kBlockHeadDim = 128;
constexpr uint32_t kMinScaleExp = 127 - 100;  // 2^-100, biased: the smallest scale written

// The smallest power of two s with amax / s <= 448 = 1.75 * 2^8, at least 2^-100 (amax finite, >= 0).
// Powers of two make x / s, and the rescaling of rows already in the cache, exact in fp32.
__device__ __forceinline__ float scale_for(float amax) {
  const uint32_t u = __float_as_uint(amax);
  const int e = int(u >> 23) - 8 + ((u & 0x7fffffu) > 0x600000u ? 1 : 0);
  return __uint_as_float(uint32_t(max(e, int(kMinScaleExp))) << 23);
}

// The smallest power of two >= x (x positive and finite; at most 2^126).  A scale this store wrote
// is one already; a caller's own scale is rounded up to one when a row is added to its group.
__device__ __forceinline__ float ceil_pow2(float x) {
  const uint32_t u = __float_as_uint(x);
  const uint32_t e = (u >> 23) + ((u & 0x7fffffu) ? 1u : 0u);
  return __uint_as_float(min(max(e, 1u), 253u) << 23);
}

}  // namespace hl
