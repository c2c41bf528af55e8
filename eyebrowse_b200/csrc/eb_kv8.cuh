// eb_kv8.cuh -- the 8-bit KV cache's number formats: codes in E4M3 or E5M2 and
// power-of-two block scales.
#pragma once

#include <cuda_fp8.h>

#include "eb_common.cuh"
#include "eb_kernels.cuh"

namespace eb {

constexpr int kKv8MinExp = -64;  // no scale is below 2^-64

// Nearest code of x, ties to even; infinities become the largest value, a
// NaN the NaN code.
__device__ __forceinline__ uint8_t f8_encode(float x, bool e5m2) {
  return (uint8_t)__nv_cvt_float_to_fp8(x, __NV_SATFINITE, e5m2 ? __NV_E5M2 : __NV_E4M3);
}
__device__ __forceinline__ float f8_decode(uint8_t c, bool e5m2) {
  return __half2float(__half(__nv_cvt_fp8_to_halfraw(c, e5m2 ? __NV_E5M2 : __NV_E4M3)));
}

// Largest magnitude that counts for a block's scale: finite values only.
__device__ __forceinline__ float f8_amax(float m, float x) {
  const float a = fabsf(x);  // fmaxf passes a NaN over
  return fmaxf(m, a <= 3.402823466e38f ? a : 0.f);
}

// The smallest power of two (2^-64 at least) with amax <= largest * scale. The
// largest value is 1.75 * 2^8 (E4M3) or 1.75 * 2^15 (E5M2), so the exponent
// follows from amax's own and from whether its significand passes 1.75.
__device__ __forceinline__ float f8_need_scale(float amax, bool e5m2) {
  const uint32_t b = __float_as_uint(amax);
  const int e = (int)(b >> 23) - 127 - (e5m2 ? 15 : 8) + ((b & 0x7fffffu) > 0x600000u ? 1 : 0);
  return __uint_as_float((uint32_t)(max(e, kKv8MinExp) + 127) << 23);
}

}  // namespace eb
