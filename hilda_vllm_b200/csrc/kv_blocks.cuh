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

}  // namespace hl
