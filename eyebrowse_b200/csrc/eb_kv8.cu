// eb_kv8.cu -- the 8-bit KV cache: rows in (prompt pieces and decode steps) and
// decode attention for any head_dim.
//
// A block of `block` rows of one KV head shares a power-of-two scale for K and
// one for V. A write finds the largest magnitude of its rows in a block, takes
// the larger of the scale that needs and the block's own, and rounds: the new
// rows once, the block's earlier rows again where the scale grew.
#include <type_traits>

#include "eb_kv8.cuh"
#include "eb_rowops.cuh"

namespace eb {

// Sums of R values over the warp, R at once: each exchange with a lane 16, 8, ..
// away halves the number of sums a lane carries, so that at the end 32 / R
// neighbouring lanes hold one of them. Adds the same pairs as warp_sum.
template <int R>
__device__ __forceinline__ float warp_sums(float (&s)[R], int lane) {
  int off = 16;
#pragma unroll
  for (int r = R / 2; r >= 1; r >>= 1, off >>= 1)
#pragma unroll
    for (int k = 0; k < r; k++) {
      const bool up = lane & off;
      const float give = up ? s[k] : s[k + r], keep = up ? s[k + r] : s[k];
      s[k] = keep + __shfl_xor_sync(0xffffffffu, give, off);
    }
#pragma unroll
  for (; off; off >>= 1) s[0] += __shfl_xor_sync(0xffffffffu, s[0], off);
  return s[0];
}

// One CTA per (block of rows, KV head, K or V of a sequence).
//
// kv8_write_rows_kernel (head_dim 64, 128, 256) keeps the rows in registers
// between finding their largest value and rounding them: a warp holds R rows,
// E = head_dim / 32 neighbouring values of each per lane, all loaded before the
// first is used, so every byte is read once and written once. 8192 rows of 8
// heads of 128 in bf16 (50 MB) take 19.4 us of which HBM needs 8. What bounds it
// is the latency of that one round of loads, so the registers are held to 64 a
// thread (with 76, three CTAs of 256 threads an SM instead of four, 25 us), and
// the issue slots: addresses in 32 bits from a base, the norm's sums, roots and
// quotients of eight rows at once.
// kv8_write_kernel (any other head_dim, or rows and tables that do not start at
// multiples of 16 bytes) stages them as f32 in shared memory: 57 us there. (With
// both kinds of loads in the first kernel the second were issued as well, under
// a predicate: 27 us instead of 25.)
// CTAs of the same rows (K and V, every head) are neighbours: together they
// read and write whole rows.
template <typename T, int E, int R>
__global__ void __launch_bounds__(R >= 8 ? 512 : 1024, R >= 8 ? 2 : 1) kv8_write_rows_kernel(Kv8WriteArgs a) {
  constexpr int HD = 32 * E;
  __shared__ float warp_max_[32];
  const unsigned at_block = (blockIdx.x >> 1) / (unsigned)a.hkv;
  const int which = blockIdx.x & 1, head = (int)((blockIdx.x >> 1) - at_block * a.hkv), b = blockIdx.y;
  const int shift = 31 - __clz(a.block);  // a power of two
  const int warps = blockDim.x >> 5, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  int64_t start = a.start;
  if (a.positions) {
    const int p = a.positions[b];
    if (p < 0 || p > a.max_pos) return;  // an empty slot of the batch
    start = p;
  }
  const int64_t end = start + a.count;
  const int64_t blk = (start >> shift) + at_block;
  const int64_t lo = max(start, blk << shift), hi = min(end, (blk + 1) << shift);
  const int n = (int)(hi - lo);
  float* scale = (which ? a.v_scale : a.k_scale) + b * a.scale_bstride + blk * a.hkv + head;
  const int before = (int)(lo - (blk << shift));  // rows of the block in front of the new ones
  const float old = before > 0 ? *scale : 0.f;

  // row r of the block: 32-bit products, 64-bit sums
  const T* src = static_cast<const T*>(which ? a.v : a.k) + b * a.kv_bstride + (lo - start) * a.kv_stride +
                 head * HD + lane * E;
  const int src_stride = (int)a.kv_stride;
  const float* w = which ? a.v_norm_w : a.k_norm_w;
  const bool turn = !which && a.cos_t;
  // all loads first (a row past the end reads the last one again)
  RawRow<T, E> raw[R];
#pragma unroll
  for (int i = 0; i < R; i++)
    raw[i].load(src + (int64_t)min(i * warps + warp, n - 1) * src_stride);
  RawRow<float, E> wr;
  if (w) wr.load(w + lane * E);
  float v[R][E], amax = 0.f;
#pragma unroll
  for (int i = 0; i < R; i++) raw[i].f32(v[i]);
  if (w) {
    float ss[R], g[E];
    wr.f32(g);
#pragma unroll
    for (int i = 0; i < R; i++) {
      ss[i] = 0.f;
#pragma unroll
      for (int e = 0; e < E; e++) ss[i] = __fadd_rn(ss[i], __fmul_rn(v[i][e], v[i][e]));
    }
    // one root and one quotient for R rows
    const float own = 1.0f / sqrtf(warp_sums<R>(ss, lane) / (float)HD + a.eps);
#pragma unroll
    for (int i = 0; i < R; i++) {
      const float inv = __shfl_sync(0xffffffffu, own, i * (32 / R));
#pragma unroll
      for (int e = 0; e < E; e++) v[i][e] = __fmul_rn(__fmul_rn(v[i][e], inv), g[e]);
    }
  }
  if (turn) {
    RawRow<float, E> tc[R], ts[R];
    const float sign = lane < 16 ? -1.f : 1.f;
    const float* cos_t = a.cos_t + lo * (HD / 2) + (lane & 15) * E;
    const float* sin_t = a.sin_t + lo * (HD / 2) + (lane & 15) * E;
#pragma unroll
    for (int i = 0; i < R; i++) {
      const int at = min(i * warps + warp, n - 1) * (HD / 2);
      tc[i].load(cos_t + at);
      ts[i].load(sin_t + at);
    }
#pragma unroll
    for (int i = 0; i < R; i++) {
      float c[E], sn[E];
      tc[i].f32(c);
      ts[i].f32(sn);
#pragma unroll
      for (int e = 0; e < E; e++) {
        const float other = __shfl_xor_sync(0xffffffffu, v[i][e], 16);
        const float q = __fmul_rn(other, sn[e]), p = __fmul_rn(v[i][e], c[e]);
        v[i][e] = __fmaf_rn(q, sign, p);  // p -+ q: the product with 1 is exact
      }
    }
  }
#pragma unroll
  for (int i = 0; i < R; i++)
#pragma unroll
    for (int e = 0; e < E; e++) amax = fmaxf(amax, fabsf(v[i][e]));
  if (amax > 3.402823466e38f) {  // an infinity: again, without it
    amax = 0.f;
#pragma unroll
    for (int i = 0; i < R; i++)
#pragma unroll
      for (int e = 0; e < E; e++) amax = f8_amax(amax, v[i][e]);
  }
  // (floats that are not negative are in the order of their bits)
  amax = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(amax)));
  if (lane == 0) warp_max_[warp] = amax;
  __syncthreads();  // and every thread has read the old scale
  amax = __uint_as_float(__reduce_max_sync(0xffffffffu, lane < warps ? __float_as_uint(warp_max_[lane]) : 0u));

  const int stride = a.hkv * HD;
  float s = f8_need_scale(amax, a.e5m2);
  const bool grown = before > 0 && fmaxf(s, old) != old;
  if (before > 0) s = fmaxf(s, old);
  const float inv = 1.0f / s;
  uint8_t* first = static_cast<uint8_t*>(which ? a.vcache : a.kcache) + b * a.cache_bstride +
                   (blk << shift) * stride + head * HD + lane * E;
  auto store = [&](auto e5m2) {
    constexpr bool E5M2 = decltype(e5m2)::value;
    if (grown) {  // the block's earlier rows, rounded again
      const float ratio = old / s;
      for (int r = warp; r < before; r += warps) {
        uint8_t* row = first + (int64_t)r * stride;
        float f[E];
#pragma unroll
        for (int e = 0; e < E; e++) f[e] = f8_decode(row[e], E5M2);
        f8_store<E, E5M2>(row, f, ratio);
      }
    }
    uint8_t* to = first + (int64_t)before * stride;
#pragma unroll
    for (int i = 0; i < R; i++) {
      // (past the end: the last row again, the same bytes)
      f8_store<E, E5M2>(to + (int64_t)min(i * warps + warp, n - 1) * stride, v[i], inv);
    }
  };
  if (a.e5m2) store(std::true_type{});
  else store(std::false_type{});
  if (threadIdx.x == 0) *scale = s;
}

__global__ void __launch_bounds__(256) kv8_write_kernel(Kv8WriteArgs a) {
  extern __shared__ float rows[];
  __shared__ float warp_max_[8];
  const int which = blockIdx.z & 1, b = blockIdx.z >> 1, head = blockIdx.y;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  int64_t start = a.start;
  if (a.positions) {
    const int p = a.positions[b];
    if (p < 0 || p > a.max_pos) return;  // an empty slot of the batch
    start = p;
  }
  const int64_t end = start + a.count;
  const int64_t blk = start / a.block + blockIdx.x;
  const int64_t lo = max(start, blk * a.block), hi = min(end, (blk + 1) * a.block);
  const int n = (int)(hi - lo), hd = a.hd;

  const void* src = which ? a.v : a.k;
  float amax = 0.f;
  for (int r = warp; r < n; r += 8) {
    float* row = rows + r * hd;
    const int64_t t = lo + r;
    const int64_t at = b * a.kv_bstride + (t - start) * a.kv_stride + (int64_t)head * hd;
    for (int d = lane; d < hd; d += 32) row[d] = ld_any(src, at + d, a.dtype_kv);
    __syncwarp();
    warp_row_norm(row, hd, which ? a.v_norm_w : a.k_norm_w, a.eps, lane);
    if (!which && a.cos_t)
      warp_row_rope(row, hd, a.cos_t + t * (hd / 2), a.sin_t + t * (hd / 2), lane);
    for (int d = lane; d < hd; d += 32) amax = f8_amax(amax, row[d]);
  }
  amax = warp_max(amax);
  if (lane == 0) warp_max_[warp] = amax;
  __syncthreads();
  for (int i = 0; i < 8; i++) amax = fmaxf(amax, warp_max_[i]);

  float* scale = (which ? a.v_scale : a.k_scale) + b * a.scale_bstride + blk * a.hkv + head;
  const int64_t stride = (int64_t)a.hkv * hd;
  uint8_t* cache = static_cast<uint8_t*>(which ? a.vcache : a.kcache) + b * a.cache_bstride +
                   (int64_t)head * hd;
  float s = f8_need_scale(amax, a.e5m2);
  const int before = (int)(lo - blk * a.block);  // rows of the block in front of the new ones
  if (before > 0) {
    const float old = *scale;
    __syncthreads();  // every thread has read the old scale before it is replaced
    s = fmaxf(s, old);
    if (s != old) {
      const float ratio = old / s;
      uint8_t* c = cache + blk * a.block * stride;
      for (int i = threadIdx.x; i < before * hd; i += 256) {
        uint8_t* p = c + (int64_t)(i / hd) * stride + i % hd;
        *p = f8_encode(f8_decode(*p, a.e5m2) * ratio, a.e5m2);
      }
    }
  }
  if (threadIdx.x == 0) *scale = s;
  const float inv = 1.0f / s;
  for (int i = threadIdx.x; i < n * hd; i += 256)
    cache[(lo + i / hd) * stride + i % hd] = f8_encode(rows[i] * inv, a.e5m2);
}

template <typename T, int E>
static void write_rows(const Kv8WriteArgs& a, int64_t per, cudaStream_t st) {
  const dim3 grid((unsigned)(per * a.hkv * 2), a.batch);
  // Rows of a warp: eight (of 256 values four) where there are enough CTAs to
  // fill the SMs, fewer in short pieces (93 rows of 4 heads of 256, normalised:
  // 9.1 us with eight, 4.8 with two); a decode step's row takes one of four
  // warps, the others are for rows that may be rounded again.
  constexpr int R = E == 8 ? 4 : 8;
  const int64_t ctas = per * a.hkv * 2 * a.batch;
  if (a.count == 1) kv8_write_rows_kernel<T, E, 1><<<grid, 128, 0, st>>>(a);
  else if (ctas >= 2 * sm_count()) kv8_write_rows_kernel<T, E, R><<<grid, 32 * a.block / R, 0, st>>>(a);
  else if (a.block <= 64) kv8_write_rows_kernel<T, E, 2><<<grid, 16 * a.block, 0, st>>>(a);
  else kv8_write_rows_kernel<T, E, 4><<<grid, 8 * a.block, 0, st>>>(a);
}

template <typename T>
static void write_rows_hd(const Kv8WriteArgs& a, int64_t per, cudaStream_t st) {
  if (a.hd == 64) write_rows<T, 2>(a, per, st);
  else if (a.hd == 128) write_rows<T, 4>(a, per, st);
  else write_rows<T, 8>(a, per, st);
}

cudaError_t launch_kv8_write(const Kv8WriteArgs& a0, cudaStream_t st) {
  Kv8WriteArgs a = a0;
  const int es = a.dtype_kv == kF32 ? 4 : 2;
  auto bits = [](const void* p) { return reinterpret_cast<uintptr_t>(p); };
  const bool aligned = ((bits(a.k) | bits(a.v) | (uintptr_t)(a.kv_stride * es) | (uintptr_t)(a.kv_bstride * es) |
                         bits(a.cos_t) | bits(a.sin_t) | bits(a.k_norm_w) | bits(a.v_norm_w)) & 15) == 0;
  const int64_t per = a.positions ? 1 : (a.start + a.count - 1) / a.block - a.start / a.block + 1;
  if (aligned && (a.hd == 64 || a.hd == 128 || a.hd == 256)) {
    if (per * a.hkv * 2 > INT32_MAX) return cudaErrorNotSupported;
    if (a.dtype_kv == kF32) write_rows_hd<float>(a, per, st);
    else if (a.dtype_kv == kF16) write_rows_hd<__half>(a, per, st);
    else write_rows_hd<__nv_bfloat16>(a, per, st);
    return cudaGetLastError();
  }
  const int rows = (int)(a.count < a.block ? a.count : a.block);
  const size_t smem = (size_t)rows * a.hd * sizeof(float);
  // (asked for at any size: the kernel's static shared memory counts too)
  static unsigned configured = 0;
  const cudaError_t e = allow_smem(kv8_write_kernel, 128 * 256 * 4, &configured);
  if (e != cudaSuccess) return e;
  kv8_write_kernel<<<dim3((unsigned)per, a.hkv, 2 * a.batch), 256, smem, st>>>(a);
  return cudaGetLastError();
}

// Decode attention for any even head_dim up to 256: one CTA per (sequence,
// query head), a warp per key row, an online softmax per warp.
constexpr int kSimtWarps = 8;
__global__ void __launch_bounds__(kSimtWarps * 32) kv8_decode_simt_kernel(Kv8DecodeArgs a) {
  __shared__ float q[256];
  __shared__ float acc_s[kSimtWarps][256];
  __shared__ float m_s[kSimtWarps], l_s[kSimtWarps];
  const int h = blockIdx.x, b = blockIdx.y, hd = a.hd;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int pos = a.positions ? a.positions[b] : a.max_pos;
  if (pos < 0 || pos > a.max_pos) return;
  const int kvh = h / (a.H / a.hkv);
  if (warp == 0) {
    const int64_t at = b * a.q_bstride + (int64_t)h * hd;
    for (int d = lane; d < hd; d += 32) q[d] = ld_any(a.q, at + d, a.dtype_q);
    __syncwarp();
    warp_row_norm(q, hd, a.q_norm_w, a.eps, lane);
    if (a.cos_t)
      warp_row_rope(q, hd, a.cos_t + (int64_t)pos * (hd / 2), a.sin_t + (int64_t)pos * (hd / 2),
                    lane);
  }
  __syncthreads();
  float qr[8], acc[8];
#pragma unroll
  for (int j = 0; j < 8; j++) {
    qr[j] = lane + 32 * j < hd ? q[lane + 32 * j] * a.scale_log2 : 0.f;
    acc[j] = 0.f;
  }
  float m = -INFINITY, l = 0.f;
  const uint8_t* kc = static_cast<const uint8_t*>(a.kcache) + b * a.cache_bstride;
  const uint8_t* vc = static_cast<const uint8_t*>(a.vcache) + b * a.cache_bstride;
  const float* ks = a.k_scale + b * a.scale_bstride + kvh;
  const float* vs = a.v_scale + b * a.scale_bstride + kvh;
  const int row_lo = a.window > 0 ? max(0, pos - a.window + 1) : 0;
  for (int t = row_lo + warp; t <= pos; t += kSimtWarps) {
    const int64_t at = ((int64_t)t * a.hkv + kvh) * hd;
    const int64_t sb = (int64_t)(t / a.block) * a.hkv;
    float dot = 0.f;
#pragma unroll
    for (int j = 0; j < 8; j++)
      if (lane + 32 * j < hd) dot = fmaf(qr[j], f8_decode(kc[at + lane + 32 * j], a.e5m2), dot);
    const float x = warp_sum(dot) * ks[sb];
    const float mn = fmaxf(m, x);
    const float corr = m == -INFINITY ? 0.f : exp2f(m - mn);
    const float p = exp2f(x - mn);
    l = l * corr + p;
    const float pv = p * vs[sb];
#pragma unroll
    for (int j = 0; j < 8; j++)
      if (lane + 32 * j < hd)
        acc[j] = fmaf(pv, f8_decode(vc[at + lane + 32 * j], a.e5m2), acc[j] * corr);
    m = mn;
  }
#pragma unroll
  for (int j = 0; j < 8; j++)
    if (lane + 32 * j < hd) acc_s[warp][lane + 32 * j] = acc[j];
  if (lane == 0) {
    m_s[warp] = m;
    l_s[warp] = l;
  }
  __syncthreads();
  float M = -INFINITY, L = 0.f, w[kSimtWarps];
  for (int i = 0; i < kSimtWarps; i++)
    if (l_s[i] != 0.f) M = fmaxf(M, m_s[i]);
  for (int i = 0; i < kSimtWarps; i++) {
    w[i] = l_s[i] != 0.f ? exp2f(m_s[i] - M) : 0.f;
    L += l_s[i] * w[i];
  }
  for (int d = threadIdx.x; d < hd; d += kSimtWarps * 32) {
    float o = 0.f;
    for (int i = 0; i < kSimtWarps; i++)
      if (l_s[i] != 0.f) o += acc_s[i][d] * w[i];
    st_any(a.o, b * a.o_bstride + (int64_t)h * hd + d, a.dtype_o, o / L);
  }
}

cudaError_t launch_kv8_decode(const Kv8DecodeArgs& a, cudaStream_t st) {
  kv8_decode_simt_kernel<<<dim3(a.H, a.batch), kSimtWarps * 32, 0, st>>>(a);
  return cudaGetLastError();
}

}  // namespace eb
