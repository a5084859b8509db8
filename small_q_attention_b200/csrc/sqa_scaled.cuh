// sqa_scaled.cuh -- the block-scaled e4m3 cache: one fp32 scale per page (16 tokens)
// and KV head, K and V apart; a cached value stands for scale * e4m3.
#pragma once

#include "sqa_internal.h"
#include "sqa_ptx.cuh"

namespace sqa {

// The scale of a page whose largest finite magnitude is amax: the smallest power
// of two with amax <= 448 * scale, 2^-100 at least (an all-zero page: any scale
// would do, and the smallest one never limits what is appended later).  Powers of
// two, because e4m3 keeps its relative precision over its exponent range: an exact
// amax / 448 would gain nothing, while a page whose scale grows only moves its old
// values' exponents, so they are not rounded a second time (unless they fall below
// e4m3's smallest normal value).
__device__ __forceinline__ float page_scale(float amax) {
  const uint32_t u = __float_as_uint(amax);  // amax >= 0 and finite
  // amax = m * 2^e with m in [0.5, 1) and 448 = 0.875 * 2^9
  const int e = (int)(u >> 23) - 126 - 9 + ((u & 0x7fffffu) > 0x600000u ? 1 : 0);
  return __uint_as_float((uint32_t)(max(e, -100) + 127) << 23);
}

// |x| where it is finite, else 0 (infinities and NaN do not size a scale).
__device__ __forceinline__ float finite_abs(float x) {
  const float a = fabsf(x);
  return a <= 3.402823466e38f ? a : 0.f;
}

__device__ __forceinline__ float warp_max(float v) {
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, off));
  return v;
}

// Two packed e4m3 (low 16 bits) -> two fp16, exact; and back, to nearest even and saturating.
__device__ __forceinline__ __half2 half2_of_e4m3x2(uint32_t v) {
  uint32_t r;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"((uint16_t)v));
  return *reinterpret_cast<const __half2*>(&r);
}
__device__ __forceinline__ uint32_t e4m3x2_of_half2(__half2 h) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f16x2 %0, %1;" : "=h"(r) : "r"(*reinterpret_cast<const uint32_t*>(&h)));
  return r;
}
__device__ __forceinline__ uint32_t e4m3x2_of_floats(float lo, float hi) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
  return r;
}

// Four floats -> four e4m3 (round to nearest even, saturating, NaN kept), first in the low byte.
__device__ __forceinline__ uint32_t pack_e4m3x4(float a, float b, float c, float d) {
  return pack_e4m3x2(a, b) | (pack_e4m3x2(c, d) << 16);
}

}  // namespace sqa
