// 8-bit floating point (e4m3) conversions shared by the quantiser and the product.
#pragma once

#include <stdint.h>

namespace b200 {

constexpr float kFp8Max = 448.0f;                 // largest e4m3 value
constexpr float kFp8Flush = 7.8886090522101181e-31f;  // 2^-100: a smaller peak counts as zero

// Four 32-bit values to e4m3, nearest-even, the first in the lowest byte.
__device__ __forceinline__ uint32_t pack_e4m3x4(float a, float b, float c, float d) {
  uint16_t lo, hi;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(lo) : "f"(b), "f"(a));
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(hi) : "f"(d), "f"(c));
  return static_cast<uint32_t>(lo) | (static_cast<uint32_t>(hi) << 16);
}

}  // namespace b200
