// eb_kv8.cuh -- the 8-bit KV cache's number formats: codes in E4M3 or E5M2 and
// power-of-two block scales.
#pragma once

#include <cuda_fp8.h>

#include <type_traits>

#include "eb_common.cuh"
#include "eb_kernels.cuh"
#include "eb_rowops.cuh"

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

template <int E, bool E5M2>
__device__ __forceinline__ void f8_store(uint8_t* p, const float (&v)[E], float inv) {
  uint32_t w[(E + 3) / 4] = {};
#pragma unroll
  for (int e = 0; e < E; e += 2)
    w[e / 4] |= (uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(v[e] * inv, v[e + 1] * inv),
                                                   __NV_SATFINITE, E5M2 ? __NV_E5M2 : __NV_E4M3)
                << (8 * (e & 3));
  if constexpr (E == 2) *reinterpret_cast<uint16_t*>(p) = (uint16_t)w[0];
  else if constexpr (E == 4) *reinterpret_cast<uint32_t*>(p) = w[0];
  else *reinterpret_cast<uint2*>(p) = make_uint2(w[0], w[1]);
}

// E neighbouring elements at a multiple of their size: one or two loads.
template <typename T, int E>
struct RawRow {
  static constexpr int W = E * (int)sizeof(T) / 4;
  uint32_t w[W];
  __device__ __forceinline__ void load(const T* p) {
    if constexpr (W == 1) {
      w[0] = *reinterpret_cast<const uint32_t*>(p);
    } else if constexpr (W == 2) {
      const uint2 u = *reinterpret_cast<const uint2*>(p);
      w[0] = u.x;
      w[1] = u.y;
    } else {
#pragma unroll
      for (int i = 0; i < W; i += 4) {
        const uint4 u = *reinterpret_cast<const uint4*>(reinterpret_cast<const uint32_t*>(p) + i);
        w[i] = u.x;
        w[i + 1] = u.y;
        w[i + 2] = u.z;
        w[i + 3] = u.w;
      }
    }
  }
  __device__ __forceinline__ void f32(float (&f)[E]) const {
    const T* e = reinterpret_cast<const T*>(w);
#pragma unroll
    for (int i = 0; i < E; i++) f[i] = Elem<T>::to_f32(e[i]);
  }
};

// A decode step's new K (which = 0) or V (1) row of one KV head, appended by two
// warps (w = 0, 1, barrier id `bar`) with kv8_write's arithmetic; returns when
// both warps' writes are done.
template <int E>
__device__ __forceinline__ void kv8_append(const Kv8DecodeArgs& a, int which, int b, int kvh, int pos,
                                           int w, int lane, int bar) {
  constexpr int HD = 32 * E;
  const void* src = which ? a.v_new : a.k_new;
  const float* norm = which ? a.v_norm_w : a.k_norm_w;
  const bool turn = !which && a.cos_t;
  const int blk = pos / a.block, before = pos - blk * a.block;
  float* scale = const_cast<float*>(which ? a.v_scale : a.k_scale) + b * a.scale_bstride + (int64_t)blk * a.hkv + kvh;
  const float old = before > 0 ? __ldcg(scale) : 0.f;
  float v[E];
  const int64_t at = b * a.kv_bstride + (int64_t)kvh * HD + lane * E;
  if (a.kv_aligned) {
    ld_row<E>(src, at, a.dtype_q, v);
  } else {
#pragma unroll
    for (int e = 0; e < E; e++) v[e] = ld_any(src, at + e, a.dtype_q);
  }
  warp_kv_row<E>(v, norm, a.eps, turn ? a.cos_t + (int64_t)pos * (HD / 2) : nullptr,
                 turn ? a.sin_t + (int64_t)pos * (HD / 2) : nullptr, lane);
  float amax = 0.f;
#pragma unroll
  for (int e = 0; e < E; e++) amax = f8_amax(amax, v[e]);
  float s = f8_need_scale(warp_max(amax), a.e5m2);
  const bool grown = before > 0 && fmaxf(s, old) != old;
  if (before > 0) s = fmaxf(s, old);
  const float inv = 1.0f / s, ratio = old / s;
  const int64_t stride = (int64_t)a.hkv * HD;
  uint8_t* first = static_cast<uint8_t*>(const_cast<void*>(which ? a.vcache : a.kcache)) + b * a.cache_bstride +
                   (int64_t)blk * a.block * stride + (int64_t)kvh * HD + lane * E;
  named_bar_and(bar, 64, true);  // both warps have read the old scale
  auto store = [&](auto e5m2) {
    constexpr bool E5M2 = decltype(e5m2)::value;
    if (grown)
      for (int r = w; r < before; r += 2) {
        float f[E];
#pragma unroll
        for (int e = 0; e < E; e++) f[e] = f8_decode(first[r * stride + e], E5M2);
        f8_store<E, E5M2>(first + r * stride, f, ratio);
      }
    if (w == 0) f8_store<E, E5M2>(first + before * stride, v, inv);
  };
  if (a.e5m2) store(std::true_type{});
  else store(std::false_type{});
  if (w == 0 && lane == 0) *scale = s;
}

}  // namespace eb
