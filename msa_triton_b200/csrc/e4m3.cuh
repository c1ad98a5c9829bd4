// e4m3 values with one float32 scale per page and head (the 8-bit KV cache): a code c of
// a page with scale s stands for c * s. The append writes power-of-two scales (the
// smallest s with amax <= 448 s): e4m3 is a floating format, so a power of two costs no
// precision, and moving a page to a larger scale is exact for every code that stays a
// normal number. Readers take any positive scale.
#pragma once

#include <cuda_fp8.h>

#include "common.cuh"

namespace msa {
namespace e4m3 {

// The smallest power of two s >= 2^-126 with amax <= 448 s = 0.875 * 2^9 s (amax finite).
__device__ __forceinline__ float scale_for(float amax) {
  const uint32_t b = __float_as_uint(amax);
  const int e = (int)(b >> 23) - 135 + ((b & 0x7fffffu) > 0x600000u);  // biased exponent of amax - 126 - 9
  return __uint_as_float((uint32_t)(max(e, -126) + 127) << 23);
}

__device__ __forceinline__ bool finite(float x) { return fabsf(x) <= 3.402823466e38f; }

// Two values that lie within the scale (or are NaN) to two codes, the first in the low byte.
__device__ __forceinline__ uint32_t encode2(float a, float b) {
  uint16_t c;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %2, %1;" : "=h"(c) : "f"(a), "f"(b));
  return c;
}

// Four values / scale to four codes, nearest even; what is not finite becomes the NaN code.
__device__ __forceinline__ uint32_t encode4(float a, float b, float c, float d, float inv_scale) {
  const float nan = __int_as_float(0x7fc00000);
  const float2 lo = make_float2(finite(a) ? a * inv_scale : nan, finite(b) ? b * inv_scale : nan);
  const float2 hi = make_float2(finite(c) ? c * inv_scale : nan, finite(d) ? d * inv_scale : nan);
  return (uint32_t)__nv_cvt_float2_to_fp8x2(lo, __NV_SATFINITE, __NV_E4M3) |
         ((uint32_t)__nv_cvt_float2_to_fp8x2(hi, __NV_SATFINITE, __NV_E4M3) << 16);
}

__device__ __forceinline__ uint8_t encode1(float x, float inv_scale) {
  return __nv_cvt_float_to_fp8(finite(x) ? x * inv_scale : __int_as_float(0x7fc00000), __NV_SATFINITE, __NV_E4M3);
}

__device__ __forceinline__ float decode1(uint8_t c) {
  return __half2float(__half(__nv_cvt_fp8_to_halfraw(c, __NV_E4M3)));
}

// Four codes to two pairs of halves (low bytes first): exact, e4m3's range lies inside fp16's.
__device__ __forceinline__ void decode4(uint32_t w, uint32_t& lo, uint32_t& hi) {
  asm("{\n\t.reg .b16 x, y;\n\tmov.b32 {x, y}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, x;\n\tcvt.rn.f16x2.e4m3x2 %1, y;\n\t}"
      : "=r"(lo), "=r"(hi)
      : "r"(w));
}

// Four codes moved to another scale (ratio = old / new).
__device__ __forceinline__ uint32_t rescale4(uint32_t w, float ratio) {
  uint32_t lo, hi;
  decode4(w, lo, hi);
  const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&lo));
  const float2 b = __half22float2(*reinterpret_cast<const __half2*>(&hi));
  return encode4(a.x, a.y, b.x, b.y, ratio);
}

}  // namespace e4m3
}  // namespace msa
