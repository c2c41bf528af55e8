// eb_w4.cu -- projections with 4-bit weights and group scales (eb_linear_w4)
// and the host functions that lay the weights out.
//
//   y[r, o] = sum_g s[g, o] * sum_{i in g} (code[o, i] - z[g, o]) * x[r, i]
#include <math.h>
#include <string.h>

#include <algorithm>

#include "eb_common.cuh"
#include "eb_kernels.cuh"
#include "eb_rowops.cuh"

namespace eb {

// One warp per output row and up to 8 rows of x: lane l takes word l % 16 of
// every second block of 128 inputs (8 codes, all of one group).
__global__ void __launch_bounds__(256) linear_w4_kernel(W4Args a) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t o = (int64_t)blockIdx.x * 8 + warp;
  if (o >= a.out_f) return;
  const int64_t m0 = (int64_t)blockIdx.y * 8;
  const int mr = (int)min((int64_t)8, a.m - m0);
  const int64_t blocks = (a.in_f + 127) / 128;
  const uint32_t* row = reinterpret_cast<const uint32_t*>(a.q) + o * blocks * 16;
  float acc[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  const int word = lane & 15, c = word >> 2, i = word & 3;
  for (int64_t b = lane >> 4; b < blocks; b += 2) {
    const int64_t k0 = b * 128 + 32 * i + 8 * c;
    if (k0 >= a.in_f) continue;
    const uint32_t w = row[b * 16 + word];
    const int64_t g = k0 / a.group;
    const float s = ld_any(a.scale, g * a.out_f + o, a.dtype_scale);
    const int z = a.zero ? a.zero[g * a.out_f + o] : 8;
    for (int r = 0; r < mr; r++) {
      float dot = 0.f;
      for (int n = 0; n < 8 && k0 + n < a.in_f; n++)
        dot = fmaf((float)((int)((w >> (4 * n)) & 15u) - z),
                   ld_any(a.x, (m0 + r) * a.x_stride + k0 + n, a.dtype_x), dot);
      acc[r] = fmaf(s, dot, acc[r]);
    }
  }
  for (int r = 0; r < mr; r++) {
    const float v = warp_sum(acc[r]);
    if (lane == 0) st_any(a.y, (m0 + r) * a.y_stride + o, a.dtype_y, v);
  }
}

size_t linear_w4_workspace_bytes(int64_t, int64_t, int64_t) { return 0; }

cudaError_t launch_linear_w4(const W4Args& a, cudaStream_t st) {
  dim3 grid((unsigned)((a.out_f + 7) / 8), (unsigned)((a.m + 7) / 8));
  linear_w4_kernel<<<grid, 256, 0, st>>>(a);
  return cudaGetLastError();
}

// ---------------------------------------------------------------- host layout
// Byte of a packed row that holds input k, and the shift of its nibble.
static inline int64_t w4_byte(int64_t k) {
  const int64_t in = k & 127;
  return (k >> 7) * 64 + ((in & 31) >> 3) * 16 + (in >> 5) * 4 + ((in & 7) >> 1);
}
static inline void w4_put(uint8_t* row, int64_t k, int code) {
  row[w4_byte(k)] |= (uint8_t)(code << (4 * (k & 1)));
}

int w4_pack_host(const uint8_t* codes, int64_t in_f, int64_t out_f, uint8_t* q) {
  const int64_t stride = (in_f + 127) / 128 * 64;
  for (int64_t j = 0; j < in_f * out_f; j++)
    if (codes[j] > 15) return EB_ERR_INVALID_ARGUMENT;
  memset(q, 0, (size_t)(stride * out_f));
  for (int64_t o = 0; o < out_f; o++)
    for (int64_t k = 0; k < in_f; k++) w4_put(q + o * stride, k, codes[o * in_f + k]);
  return EB_OK;
}

// Nearest value of the scale type; false if it is past the type's range.
static bool store_scale(double s, int dtype, uint16_t* bits, double* value) {
  if (dtype == kF16) {
    const __half h = __double2half(s);
    memcpy(bits, &h, 2);
    *value = (double)__half2float(h);
  } else {
    const __nv_bfloat16 h = __double2bfloat16(s);
    memcpy(bits, &h, 2);
    *value = (double)__bfloat162float(h);
  }
  return std::isfinite(*value);
}

int w4_quantize_host(const float* w, int64_t in_f, int64_t out_f, int group, int dtype_scale,
                     uint8_t* q, uint16_t* scale, uint8_t* zero) {
  const int64_t stride = (in_f + 127) / 128 * 64;
  memset(q, 0, (size_t)(stride * out_f));
  const int64_t groups = (in_f + group - 1) / group;
  for (int64_t o = 0; o < out_f; o++)
    for (int64_t g = 0; g < groups; g++) {
      const int64_t k0 = g * group, k1 = std::min(in_f, k0 + group);
      float lo = 0.f, hi = 0.f;
      for (int64_t k = k0; k < k1; k++) {
        const float v = w[o * in_f + k];
        if (!std::isfinite(v)) return EB_ERR_INVALID_ARGUMENT;
        lo = std::min(lo, v);
        hi = std::max(hi, v);
      }
      const double span = zero ? ((double)hi - (double)lo) / 15.0
                               : std::max((double)hi, -(double)lo) / 7.0;
      double s;
      if (!store_scale(span, dtype_scale, &scale[g * out_f + o], &s)) return EB_ERR_INVALID_ARGUMENT;
      int z = 8;
      if (zero) {
        z = s > 0 ? (int)std::min(15.0, nearbyint(-(double)lo / s)) : 0;
        zero[g * out_f + o] = (uint8_t)z;
      }
      for (int64_t k = k0; k < k1; k++) {
        const double t = s > 0 ? nearbyint((double)w[o * in_f + k] / s) : 0.0;
        w4_put(q + o * stride, k, (int)std::min(15.0, std::max(0.0, t + z)));
      }
    }
  return EB_OK;
}

}  // namespace eb
