// eb_w4.cu -- projections with 4-bit weights and group scales (eb_linear_w4)
// and the host functions that lay the weights out.
//
//   y[r, o] = sum_g s[g, o] * sum_{i in g} (code[o, i] - z[g, o]) * x[r, i]
#include <math.h>
#include <string.h>

#include <algorithm>

#include <cooperative_groups.h>

#include "eb_common.cuh"
#include "eb_kernels.cuh"
#include "eb_rowops.cuh"
#include "eb_tc.cuh"

namespace cg = cooperative_groups;

namespace eb {

// linear_w4_kernel multiplies on the tensor cores in whole numbers: mma.sync
// m16n8k32, u8 codes by s8 activations, s32 sums. At a few rows of x the work is
// a stream of the weights, and what a warp does per code, not the matrix rate,
// has to keep under its share of the memory bandwidth (about 2.5 instruction
// slots per code and lane at 6.5 TB/s; one row takes 1.9). Eight codes in a word become two
// operand registers with a shift and two ANDs; f16 operands took eleven
// instructions (and twice the MMAs: both kinds issue at one per two clocks and
// SM here, with k16 and k32). A tcgen05 operand would have to pass through
// shared memory first, and its 128-row tiles would leave most SMs idle at
// decode sizes.
//
// - The columns are three s8 planes of x: each (row of x, block of 128 inputs)
//   is scaled by a power of two so that its largest value lies in [2^21, 2^22),
//   rounded to a whole number (off by 2^-22 of the largest value at most), and
//   split into bytes.
// - A group's sum over its codes is exact in s32, and zero point times the sum of
//   the same bytes is taken off it there, while nothing is rounded: both can be
//   far larger than what they leave. Sums below 2^22 turn to f32 by adding them
//   to the bits of 1.5 * 2^23. One or two column tiles: the planes' scales are
//   applied to each. Three: the planes are joined first, in groups of 32 all in
//   s32 (32 * 15 * 2^22 < 2^31), of more the two low ones in s32 (128 * 15 * 2^15
//   < 2^26) and the high one in f32. Then the group's scale, and the sum of the
//   row in f32.
// - The inputs of a k32 step may be any 32 as long as both operands agree, so
//   the packed layout gives thread c of a quad 8 consecutive codes (one
//   word) of each group of 32, even codes in one register, odd ones in the
//   other, and x is stored in that order.
// - The warps of a CTA: wr side by side over 32-row tiles, wk over pairs of
//   blocks of 128 inputs; a cluster splits the inputs further. CTAs stay and
//   walk over the tiles, so that x is staged once and the stream of weights
//   does not stop between tiles. Partial sums meet in shared memory, then in
//   the cluster's.
//
// Measured (calls in a row, weights from HBM; in brackets from L2 and out of a
// graph, and there with f16 operands): one row by 4096 x 28672 22.5 us (16.5,
// 26), eight rows by 14336 x 4096 26.6 us (23.5, 39), 37 rows by 4100 x 5003 in
// groups of 32 45 us (41, 52; joined in f32 49), one row by 1024 x 4096 6.6 us
// (4.6, 4.8), which is a launch, one trip to memory and the sums' two meetings.
// The large ones are bound by latency: 12 to 16 warps an SM (115 to 128
// registers a thread), each a chain of wait, unpack, products and join; an
// instruction is issued in 35 % (one row) to 49 % (37 rows) of the clocks in which
// an SM has work, and the grids leave a part of the SMs empty or half empty (224
// of 296 places, 128 and 125 of 148).
constexpr int kW4Ring = 2;   // pairs of blocks of a warp in its ring of shared memory
constexpr int kW4Pair = 4096;  // bytes of a tile's pair of blocks
constexpr int kW4Tile = 32;  // weight rows of a warp: two m16 tiles

// By columns / 8. One column tile: two CTAs of 8 warps on an SM. More: one CTA
// of 16, which stages x once for all.
constexpr int w4_warps(int nt) { return nt == 1 ? 8 : 16; }
constexpr int w4_ctas(int nt) { return nt == 1 ? 2 : 1; }
constexpr int w4_smem(int nt) { return (nt == 1 ? 112 : 226) * 1024; }
constexpr int w4_ring_bytes(int nt) { return w4_warps(nt) * kW4Ring * kW4Pair; }
// Partial sums of a CTA's warps, one m16 tile at a time.
constexpr int w4_red_bytes(int nt) { return w4_warps(nt) * 16 * (nt * 8 + 2) * 4; }

struct W4Plan {
  int wr, wk;      // warps of a CTA over row tiles and over pairs of input blocks
  int split;       // CTAs of a cluster over pairs
  int chunk;       // pairs (256 inputs) staged at a time
  int mt;          // x rows per CTA
  bool split_x;    // x's planes lie in the workspace
  int units;       // runs of wr tiles
  int nt, grid, smem;
};

constexpr int kW4Planes = 3;

__device__ __forceinline__ void mma_u8s8(int (&d)[4], const uint32_t (&a)[4], uint32_t b0,
                                         uint32_t b1) {
  asm("mma.sync.aligned.m16n8k32.row.col.s32.u8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
      "{%8,%9}, {%0,%1,%2,%3};"
      : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// Whole sums of a group that the join of three column tiles takes off, by
// groups in a block: of all planes together, or of the high one and of the others.
constexpr int w4_sums(int gb) { return gb == 4 ? 1 : 2; }

// Eight inputs of x row t into the planes' rows of shared memory (even ones,
// then odd ones). The 16 threads of a half warp hold a block of 128. With it
// the block's scales and the groups' whole sums: of each plane (three numbers
// each), or of planes together (JOINT: one scale, w4_sums sums `sum_next` apart).
template <int GROUP, bool JOINT>
__device__ __forceinline__ void w4_stage8(const W4Args& a, int64_t t, int64_t k0, uint8_t* dst,
                                          int row_bytes, float* scale, float* sums,
                                          int sum_stride, int sum_next) {
  float f[8];
  const int64_t at = t * a.x_stride + k0;
  const char* src = static_cast<const char*>(a.x) + at * (a.dtype_x == kF32 ? 4 : 2);
  if (k0 + 8 <= a.in_f && (reinterpret_cast<uintptr_t>(src) & 15) == 0) {
    load8_any(a.x, at, a.dtype_x, f);
  } else {
#pragma unroll
    for (int n = 0; n < 8; n++) f[n] = k0 + n < a.in_f ? ld_any(a.x, at + n, a.dtype_x) : 0.f;
  }
  float top = 0.f, odd = 0.f;  // odd: NaN if a value is not finite
#pragma unroll
  for (int n = 0; n < 8; n++) {
    top = fmaxf(top, fabsf(f[n]));
    odd = fmaf(f[n], 0.f, odd);
  }
  const uint32_t half = threadIdx.x & 16 ? 0xffff0000u : 0x0000ffffu;
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) {
    top = fmaxf(top, __shfl_xor_sync(half, top, o));
    odd += __shfl_xor_sync(half, odd, o);
  }
  const int e = min(max((int)(__float_as_uint(top) >> 23), 27), 254);  // at least 2^-100
  const float up = __uint_as_float((uint32_t)(127 + 21 + 127 - e) << 23);
  uint32_t w[kW4Planes][2] = {};
#pragma unroll
  for (int n = 0; n < 8; n++) {
    const int q = __float2int_rn(f[n] * up);
    const int lo = (int)(int8_t)q, q1 = (q - lo) >> 8, mid = (int)(int8_t)q1, hi = (q1 - mid) >> 8;
    const int sh = 8 * (n >> 1);
    w[0][n & 1] |= (uint32_t)(uint8_t)hi << sh;
    w[1][n & 1] |= (uint32_t)(uint8_t)mid << sh;
    w[2][n & 1] |= (uint32_t)(uint8_t)lo << sh;
  }
  const int lane = threadIdx.x & 15;
  int sum[kW4Planes];
#pragma unroll
  for (int p = 0; p < kW4Planes; p++) {
    *reinterpret_cast<uint2*>(dst + p * row_bytes) = make_uint2(w[p][0], w[p][1]);
    sum[p] = __dp4a((int)w[p][0], 0x01010101, __dp4a((int)w[p][1], 0x01010101, 0));
#pragma unroll
    for (int o = GROUP / 16; o > 0; o >>= 1) sum[p] += __shfl_xor_sync(half, sum[p], o);
  }
  // hi counts 2^(e - 127 - 21 + 16), and so on
  auto unit = [&](int p) { return __uint_as_float((uint32_t)(e - 5 - 8 * p) << 23) + odd; };
  float* at_group = sums + lane / (GROUP / 8) * sum_stride;
  if constexpr (JOINT) {
    if (lane % (GROUP / 8) == 0) {
      const int low = sum[1] * 256 + sum[2];
      at_group[0] = __int_as_float(GROUP == 32 ? sum[0] * 65536 + low : sum[0]);
      if (GROUP != 32) at_group[sum_next] = __int_as_float(low);
    }
    if (lane == 0) *scale = unit(2);
  } else {
#pragma unroll
    for (int p = 0; p < kW4Planes; p++) {
      if (lane % (GROUP / 8) == 0) at_group[p] = __int_as_float(sum[p]);
      if (lane == 0) scale[p] = unit(p);
    }
  }
}

// More than eight rows of x are split once, by w4_planes_kernel, instead of in
// every CTA. A (row, pair of blocks) in the workspace: the planes' 256 bytes
// each, the blocks' two scales, the 2 GB groups' sums, to a multiple of 16 bytes.
constexpr int w4_split_bytes(int gb) {
  return (kW4Planes * 256 + 2 * 4 * (1 + gb * w4_sums(gb)) + 15) / 16 * 16;
}

template <int GROUP>
__global__ void __launch_bounds__(256) w4_planes_kernel(W4Args a) {
  constexpr int GB = 128 / GROUP, BYTES = w4_split_bytes(GB);
  const int64_t pairs = (a.in_f + 255) / 256;
  const int64_t i = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);  // a warp per (row, pair)
  if (i >= a.m * pairs) return;
  const int lane = threadIdx.x & 31, blk = lane >> 4, e = lane & 15;
  uint8_t* out = static_cast<uint8_t*>(a.ws) + i * BYTES;
  float* scales = reinterpret_cast<float*>(out + kW4Planes * 256);
  w4_stage8<GROUP, true>(a, i / pairs, (i % pairs) * 256 + lane * 8,
                         out + blk * 128 + (e & 3) * 32 + (e >> 2) * 8, 256, scales + blk,
                         scales + 2 + blk * GB * w4_sums(GB), w4_sums(GB), 1);
}

__device__ __forceinline__ float w4_scale(uint32_t bits, bool bf16) {
  return bf16 ? __uint_as_float(bits << 16) : __half2float(__ushort_as_half((uint16_t)bits));
}

template <int NT, int GROUP>
__global__ void __launch_bounds__(w4_warps(NT) * 32, w4_ctas(NT)) linear_w4_kernel(W4Args a, W4Plan pl) {
  constexpr int GB = 128 / GROUP;  // groups in a block
  constexpr int LD = NT * 8 + 2, THREADS = w4_warps(NT) * 32;
  extern __shared__ __align__(16) uint8_t smem_raw[];
  float* red = reinterpret_cast<float*>(smem_raw + w4_ring_bytes(NT));  // [warps][16][LD]
  const int cta_rows = pl.wr * kW4Tile;
  float* part = red + w4_red_bytes(NT) / 4;  // [2][mt][cta_rows], with a cluster
  // Columns: one or two tiles hold the planes of each row of x side by side
  // (3 t + p). Three hold a plane each (8 p + t), so that a thread has all
  // planes of its two rows and joins them before it scales.
  constexpr bool JOINT = NT == 3;
  constexpr int XC = JOINT ? 8 : NT * 8;
  constexpr int SUMS = JOINT ? w4_sums(GB) : 1;
  // of a block's columns: scales [2 chunk][XC], a group's sums [2 chunk GB][SUMS][XC]
  float* xscale = part + (pl.split > 1 ? 2 * pl.mt * cta_rows : 0);
  float* xsum = xscale + 2 * pl.chunk * XC;
  uint8_t* zeros = reinterpret_cast<uint8_t*>(xsum + 2 * pl.chunk * GB * SUMS * XC);  // what columns past the last read
  uint8_t* xs = zeros + 256;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, c = lane & 3, n = lane >> 2;
  const int wk = warp % pl.wk, wr = warp / pl.wk;
  const int rank = blockIdx.x % pl.split;
  const int64_t m0 = (int64_t)blockIdx.y * pl.mt;
  const int mt = (int)min((int64_t)pl.mt, a.m - m0);
  constexpr int P = kW4Planes;
  auto column = [&](int t, int p) { return JOINT ? 8 * p + t : t * P + p; };
  auto has_column = [&](int t) { return JOINT ? n < mt : 8 * t + n < mt * P; };  // 8 t + n
  const int out_f = (int)a.out_f;
  const int blocks = (int)((a.in_f + 127) / 128), groups = (int)((a.in_f + GROUP - 1) / GROUP);
  const int pairs = (blocks + 1) / 2;
  const int p0 = (int)((int64_t)pairs * rank / pl.split);
  const int p1 = (int)((int64_t)pairs * (rank + 1) / pl.split);
  const int row_bytes = pl.chunk * 256 + 16;  // 16 past a multiple of 128: no bank is hit twice
  const uint16_t* scale = static_cast<const uint16_t*>(a.scale);
  const bool sbf = a.dtype_scale == kBF16;
  const int step = gridDim.x / pl.split;

  // The warp's pairs, tile after tile, pass through a ring of its own, each
  // thread reading back what it copied: no barrier, and two pairs of every
  // warp in flight without registers. Thread: rows n, n + 8, n + 16 and n + 24
  // of the tile (the last row again past the end), 16 bytes of each block. The
  // scales (low half) and zero points of a pair's groups come one pair ahead,
  // row `lane` of the tile in a thread.
  struct Meta {
    uint32_t v[2 * GB];
  };
  const uint32_t ring = smem_u32(smem_raw) + warp * kW4Ring * kW4Pair + lane * 16;
  const uint8_t* ring_p = smem_raw + warp * kW4Ring * kW4Pair + lane * 16;
  int fetch_unit = blockIdx.x / pl.split, fetch_p = p0 + wk;
  const uint8_t* from[4];
  auto aim = [&]() {
    const int row0 = (fetch_unit * pl.wr + wr) * kW4Tile;
#pragma unroll
    for (int j = 0; j < 4; j++)
      from[j] = static_cast<const uint8_t*>(a.q) + (int64_t)min(row0 + n + 8 * j, out_f - 1) * blocks * 64 +
                c * 16 + fetch_p * 128;
  };
  auto fetch = [&](int slot) {
    if (fetch_unit < pl.units && fetch_p < p1) {
#pragma unroll
      for (int j = 0; j < 4; j++) cp_async16(ring + slot * kW4Pair + j * 512, from[j]);
      if (2 * fetch_p + 1 < blocks)  // an odd last block has no partner: x is zero there
#pragma unroll
        for (int j = 0; j < 4; j++) cp_async16(ring + slot * kW4Pair + 2048 + j * 512, from[j] + 64);
#pragma unroll
      for (int j = 0; j < 4; j++) from[j] += pl.wk * 128;
      fetch_p += pl.wk;
      if (fetch_p >= p1) {
        fetch_p = p0 + wk;
        fetch_unit += step;
        aim();
      }
    }
    cp_async_commit();
  };
  int meta_unit = fetch_unit, meta_p = fetch_p;
  auto fetch_meta = [&](Meta& meta) {
    if (meta_unit < pl.units && meta_p < p1) {
      const int row = min((meta_unit * pl.wr + wr) * kW4Tile + lane, out_f - 1);
#pragma unroll
      for (int g = 0; g < 2 * GB; g++) {
        const int64_t at = (int64_t)min(meta_p * 2 * GB + g, groups - 1) * out_f + row;
        meta.v[g] = (uint32_t)__ldg(scale + at) | (a.zero ? (uint32_t)__ldg(a.zero + at) : 8u) << 16;
      }
      meta_p += pl.wk;
      if (meta_p >= p1) {
        meta_p = p0 + wk;
        meta_unit += step;
      }
    }
  };
  Meta ahead{};
  aim();
#pragma unroll
  for (int d = 0; d < kW4Ring; d++) fetch(d);
  fetch_meta(ahead);
  for (int i = threadIdx.x; i < 2 * pl.chunk * XC * (1 + GB * SUMS) + 64; i += THREADS)
    xscale[i] = 0.f;  // and xsum, and zeros
  constexpr int kMagic = 0x4b400000;  // 1.5 * 2^23: adding |v| < 2^22 gives the float 1.5 * 2^23 + v

  int slot = 0, buf = 0;
  for (int unit = blockIdx.x / pl.split; unit < pl.units; unit += step) {
    constexpr int AT = JOINT ? 1 : NT;
    float acc[2][AT][4];
#pragma unroll
    for (int rt = 0; rt < 2; rt++)
#pragma unroll
      for (int t = 0; t < AT; t++)
#pragma unroll
        for (int e = 0; e < 4; e++) acc[rt][t][e] = 0.f;

    for (int ch = p0; ch < p1; ch += pl.chunk) {
      const int end = min(ch + pl.chunk, p1);
      if (ch > p0 || unit == blockIdx.x / pl.split || pl.chunk < p1 - p0) {
        __syncthreads();  // what was staged before has been read
        const int eights = (end - ch) * 32;
        if (pl.split_x) {
          constexpr int BYTES = w4_split_bytes(GB), FLOATS = 2 + 2 * GB * SUMS;
          const uint8_t* src = static_cast<const uint8_t*>(a.ws) + (m0 * pairs + ch) * BYTES;
          const int n_pairs = end - ch, words = P * 16;
          for (int i = threadIdx.x; i < mt * n_pairs * words; i += THREADS) {
            const int word = i % words, q = i / words, t = q / n_pairs, pr = q % n_pairs;
            *reinterpret_cast<uint4*>(xs + column(t, word / 16) * row_bytes + pr * 256 + word % 16 * 16) =
                __ldg(reinterpret_cast<const uint4*>(src + ((int64_t)t * pairs + pr) * BYTES) + word);
          }
          for (int i = threadIdx.x; i < mt * n_pairs * FLOATS; i += THREADS) {
            const int j = i % FLOATS, q = i / FLOATS, t = q / n_pairs, pr = q % n_pairs;
            const float v = __ldg(reinterpret_cast<const float*>(src + ((int64_t)t * pairs + pr) * BYTES + P * 256) + j);
            if (j < 2) xscale[(pr * 2 + j) * XC + t] = v;
            else xsum[(pr * 2 * GB * SUMS + j - 2) * XC + t] = v;
          }
        } else {
          for (int i = threadIdx.x; i < eights * mt; i += THREADS) {
            const int t = i / eights, e = i % eights, at = JOINT ? t : t * P;
            w4_stage8<GROUP, JOINT>(a, m0 + t, (int64_t)ch * 256 + e * 8,
                                    xs + column(t, 0) * row_bytes + (e >> 4) * 128 + (e & 3) * 32 + ((e >> 2) & 3) * 8,
                                    (JOINT ? 8 : 1) * row_bytes, &xscale[(e >> 4) * XC + at],
                                    &xsum[(e >> 4) * GB * SUMS * XC + at], SUMS * XC, XC);
          }
        }
        __syncthreads();
      }
      for (int p = ch + wk; p < end; p += pl.wk) {
        cp_async_wait<kW4Ring - 1>();
        // With one column tile both blocks' words are in registers at once; with
        // more there is room for one block's.
        constexpr int KW = NT == 1 ? 2 : 1;
        uint4 w[KW][4];
        auto read = [&](int k) {
#pragma unroll
          for (int j = 0; j < 4; j++)
            w[k % KW][j] = *reinterpret_cast<const uint4*>(ring_p + slot * kW4Pair + k * 2048 + j * 512);
          if (k == 1) fetch(slot);  // into the place just read
        };
        const Meta meta = ahead;
        fetch_meta(ahead);
        const uint8_t* xb[NT];  // column 8 t + n, words 0 and 1
#pragma unroll
        for (int t = 0; t < NT; t++)
          xb[t] = (has_column(t) ? xs + (8 * t + n) * row_bytes + (p - ch) * 256 : zeros) + c * 32;
        const float* bs = xscale + (p - ch) * 2 * XC + 2 * c;
        const float* bz = xsum + (p - ch) * 2 * GB * SUMS * XC + 2 * c;
        // Two words of one block: 64 inputs of both m16 tiles.
        auto words = [&](int k, int i2, int (&sum)[2][NT][4]) {
          uint4 x[NT];
#pragma unroll
          for (int t = 0; t < NT; t++) x[t] = *reinterpret_cast<const uint4*>(xb[t] + k * 128 + i2 * 16);
#pragma unroll
          for (int h = 0; h < 2; h++) {
            const int i = 2 * i2 + h;
            const bool first = i * 32 % GROUP == 0, last = (i + 1) * 32 % GROUP == 0;
#pragma unroll
            for (int rt = 0; rt < 2; rt++) {
              const uint4 w0 = w[k % KW][2 * rt], w1 = w[k % KW][2 * rt + 1];
              const uint32_t u0 = i == 0 ? w0.x : i == 1 ? w0.y : i == 2 ? w0.z : w0.w;
              const uint32_t u1 = i == 0 ? w1.x : i == 1 ? w1.y : i == 2 ? w1.z : w1.w;
              const uint32_t f[4] = {u0 & 0x0f0f0f0fu, u1 & 0x0f0f0f0fu, (u0 >> 4) & 0x0f0f0f0fu,
                                     (u1 >> 4) & 0x0f0f0f0fu};
#pragma unroll
              for (int t = 0; t < NT; t++) {
                if (first)
#pragma unroll
                  for (int e = 0; e < 4; e++) sum[rt][t][e] = JOINT && (GROUP == 32 || t > 0) ? 0 : kMagic;
                mma_u8s8(sum[rt][t], f, h ? x[t].z : x[t].x, h ? x[t].w : x[t].y);
              }
            }
            if (last) {
              const int g = k * GB + i * 32 / GROUP;
#pragma unroll
              for (int rt = 0; rt < 2; rt++) {
                float s[2];
                int z[2];
#pragma unroll
                for (int r = 0; r < 2; r++) {
                  const uint32_t m = __shfl_sync(0xffffffffu, meta.v[g], n + 16 * rt + 8 * r);
                  s[r] = w4_scale(m & 0xffffu, sbf);
                  z[r] = (int)(m >> 16);
                }
                if constexpr (JOINT && GROUP == 32) {
                  const float2 b2 = *reinterpret_cast<const float2*>(bs + k * XC);
                  const int2 z2 = *reinterpret_cast<const int2*>(bz + g * XC);
#pragma unroll
                  for (int e = 0; e < 4; e++) {
                    const int whole = (sum[rt][0][e] * 256 + sum[rt][1][e]) * 256 + sum[rt][2][e] -
                                      z[e >> 1] * (e & 1 ? z2.y : z2.x);
                    acc[rt][0][e] = fmaf((float)whole, s[e >> 1] * (e & 1 ? b2.y : b2.x), acc[rt][0][e]);
                  }
                } else if constexpr (JOINT) {
                  const float2 b2 = *reinterpret_cast<const float2*>(bs + k * XC);
                  const int2 zh = *reinterpret_cast<const int2*>(bz + g * SUMS * XC);
                  const int2 zl = *reinterpret_cast<const int2*>(bz + (g * SUMS + 1) * XC);
#pragma unroll
                  for (int e = 0; e < 4; e++) {
                    const int high = sum[rt][0][e] - z[e >> 1] * (e & 1 ? zh.y : zh.x);
                    const int low = sum[rt][1][e] * 256 + sum[rt][2][e] - z[e >> 1] * (e & 1 ? zl.y : zl.x);
                    const float whole = fmaf(__int_as_float(high) - 12582912.f, 65536.f, (float)low);
                    acc[rt][0][e] = fmaf(whole, s[e >> 1] * (e & 1 ? b2.y : b2.x), acc[rt][0][e]);
                  }
                } else {
#pragma unroll
                  for (int t = 0; t < NT; t++) {
                    const float2 b2 = *reinterpret_cast<const float2*>(bs + k * XC + 8 * t);
                    const int2 z2 = *reinterpret_cast<const int2*>(bz + g * XC + 8 * t);
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                      const int v = sum[rt][t][e] - z[e >> 1] * (e & 1 ? z2.y : z2.x);
                      acc[rt][t][e] = fmaf(__int_as_float(v) - 12582912.f, s[e >> 1] * (e & 1 ? b2.y : b2.x),
                                           acc[rt][t][e]);
                    }
                  }
                }
              }
            }
          }
        };
        if constexpr (NT == 1) {
          // both blocks abreast: four chains of dependent products
          int sum[2][2][NT][4];
          read(0);
          read(1);
#pragma unroll
          for (int i2 = 0; i2 < 2; i2++)
#pragma unroll
            for (int k = 0; k < 2; k++) words(k, i2, sum[k]);
        } else {
          int sum[2][NT][4];
#pragma unroll
          for (int k = 0; k < 2; k++) {
            read(k);
#pragma unroll
            for (int i2 = 0; i2 < 2; i2++) words(k, i2, sum);
          }
        }
        slot ^= 1;
      }
    }

    // sums of the warps that share rows, one m16 tile after the other
    const int cta_row0 = unit * cta_rows;
#pragma unroll
    for (int rt = 0; rt < 2; rt++) {
      __syncthreads();  // the sums before have been read
#pragma unroll
      for (int t = 0; t < AT; t++)
#pragma unroll
        for (int h = 0; h < 2; h++)
          *reinterpret_cast<float2*>(&red[(warp * 16 + h * 8 + n) * LD + t * 8 + 2 * c]) =
              make_float2(acc[rt][t][2 * h], acc[rt][t][2 * h + 1]);
      __syncthreads();
      const int rows = pl.wr * 16;
      for (int i = threadIdx.x; i < rows * mt; i += THREADS) {
        const int r = i % rows, t = i / rows, w = r / 16, rr = r % 16;
        float v = 0.f;
        for (int k = 0; k < pl.wk; k++) {
          const float* s = red + ((w * pl.wk + k) * 16 + rr) * LD + (JOINT ? t : t * P);
          v += JOINT ? s[0] : (s[2] + s[1]) + s[0];
        }
        const int row = w * kW4Tile + rt * 16 + rr;
        if (pl.split > 1) part[(buf * pl.mt + t) * cta_rows + row] = v;
        else if (cta_row0 + row < out_f)
          st_any(a.y, (m0 + t) * a.y_stride + cta_row0 + row, a.dtype_y, v);
      }
    }
    if (pl.split > 1) {
      // and of the cluster. Two buffers: the one written next was read before
      // the barrier in between.
      cg::cluster_group cl = cg::this_cluster();
      cl.sync();
      for (int i = rank * THREADS + threadIdx.x; i < cta_rows * mt; i += pl.split * THREADS) {
        const int row = i % cta_rows, t = i / cta_rows;
        float v = 0.f;
        for (int s = 0; s < pl.split; s++) v += cl.map_shared_rank(part, s)[(buf * pl.mt + t) * cta_rows + row];
        if (cta_row0 + row < out_f)
          st_any(a.y, (m0 + t) * a.y_stride + cta_row0 + row, a.dtype_y, v);
      }
      buf ^= 1;
    }
  }
  cp_async_wait<0>();
  if (pl.split > 1) cg::this_cluster().sync();  // no CTA leaves while its sums are read
}

// Rows of x that a CTA multiplies at once, evened out over the passes.
constexpr int kW4Rows = 24 / kW4Planes;
static int w4_pass_rows(int64_t m) {
  const int64_t passes = (m + kW4Rows - 1) / kW4Rows;
  return (int)((m + passes - 1) / passes);
}
static int w4_column_tiles(int64_t m) {
  return m > kW4Rows ? 3 : (int)(m * kW4Planes + 7) / 8;
}

size_t linear_w4_workspace_bytes(int64_t m, int64_t in_f, int64_t) {
  if (m <= kW4Rows) return 0;
  return ((size_t)m * (size_t)((in_f + 255) / 256) * w4_split_bytes(4) + 255) / 256 * 256;  // any group
}

// The shape of a launch: of every (wk, split) whose staged x fits, the one
// with the least work on the busiest SM, counted in pairs of blocks of one warp
// (about 480 instructions; an eight of x staged by each thread is about a
// third of that, copied a twentieth, a tile's sums about a third, a cluster's
// about another), and at least
// what the longest row of pairs of one warp takes (a warp alone takes about as
// long for a pair as a full SM for 16). limit[split]: clusters of that size that
// are resident at once (an SM group holds whole clusters only: 148 SMs do not
// hold 21 clusters of 7). Measured against every other shape that fits (16 to 40
// each) at nine sizes of 1 to 64 rows, 1024 -> 4096 to 4096 -> 28672: within 5 % of
// the fastest (one row 4096 -> 28672 20.3 us, best 20.1, worst 78; eight rows
// 14336 -> 4096 26.1, best 26.1, worst 175; 37 rows 4100 -> 5003 41.5, best 41.4,
// worst 120).
static W4Plan plan_w4(int64_t m, int64_t in_f, int64_t out_f, int gb, const int* limit) {
  W4Plan p{};
  const int sms = sm_count();
  const int64_t passes = (m + kW4Rows - 1) / kW4Rows;
  p.mt = w4_pass_rows(m);
  p.split_x = m > kW4Rows;
  p.nt = w4_column_tiles(m);
  const int cols = p.nt == 3 ? 24 : p.mt * kW4Planes, xc = p.nt == 3 ? 8 : 8 * p.nt;
  const int floats = 1 + gb * (p.nt == 3 ? w4_sums(gb) : 1);  // of a block and column
  const int64_t tiles = (out_f + kW4Tile - 1) / kW4Tile, pairs = (in_f + 255) / 256;
  const int warps = w4_warps(p.nt);
  const int fixed = w4_ring_bytes(p.nt) + w4_red_bytes(p.nt);
  double best = 0;
  for (int wk = warps; wk >= 1; wk /= 2)
    for (int split = 1; split <= 8 && split <= pairs; split++) {
      const int wr = warps / wk;
      const int part = split > 1 ? 2 * p.mt * wr * kW4Tile * 4 : 0;
      const int64_t range = (pairs + split - 1) / split;
      const int64_t left = w4_smem(p.nt) - fixed - part - 16 * cols - 256;
      const int64_t fit = std::max<int64_t>(left, 0) / (256 * cols + 8 * xc * floats) / wk * wk;
      if (fit == 0) continue;  // chunks are whole turns of the wk warps
      const int64_t chunk = std::min(range, fit);
      const int64_t units = (tiles + wr - 1) / wr;
      const int64_t clusters = std::max<int64_t>(1, limit[split] / passes);
      const int64_t grid = std::min(units, clusters) * split;
      const int64_t turns = (units + clusters - 1) / clusters;
      // an SM's CTAs; at most one of them has the last turn if few have
      const int64_t per_sm = (grid * passes + sms - 1) / sms;
      const int64_t last = (units - (turns - 1) * clusters) * split * passes;
      const int64_t unit_sm = last <= sms ? per_sm * (turns - 1) + 1 : per_sm * turns;
      const double blocks_warp = (double)((range + wk - 1) / wk);
      const double stage = (p.split_x ? 0.06 : 0.3) * (double)((range * 32 * p.mt + warps * 32 - 1) / (warps * 32));
      const double sums = split > 1 ? 0.6 : 0.3;
      const double staged = chunk < range ? unit_sm * stage : per_sm * stage;
      const double busy = warps * (unit_sm * (blocks_warp + sums) + staged);
      const double alone = 16.0 * (turns * (blocks_warp + sums) + (chunk < range ? turns : 1) * stage);
      const double cost = std::max(busy, alone);
      if (best == 0 || cost < best) {
        best = cost;
        p.wk = wk;
        p.wr = wr;
        p.split = split;
        p.chunk = (int)chunk;
        p.units = (int)units;
        p.grid = (int)grid;
        p.smem = fixed + part + (int)chunk * 8 * xc * floats + 256 + cols * (int)(chunk * 256 + 16);
      }
    }
  return p;
}

// Resident clusters of every size, asked of the runtime once per kernel and
// device.
template <int NT, int GROUP>
static cudaError_t w4_limits(int (&limit)[9]) {
  static int cache[64][9] = {};
  auto kern = linear_w4_kernel<NT, GROUP>;
  int dev = 0;
  const cudaError_t have = cudaGetDevice(&dev);
  if (have != cudaSuccess) return have;
  int none[9] = {};
  int* known = dev < 64 ? cache[dev] : none;
  for (int split = 1; split <= 8; split++) {
    limit[split] = __atomic_load_n(&known[split], __ATOMIC_RELAXED);
    if (limit[split] > 0) continue;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(split);
    cfg.blockDim = dim3(w4_warps(NT) * 32);
    cfg.dynamicSmemBytes = w4_smem(NT);
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = split;
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    const cudaError_t e = cudaOccupancyMaxActiveClusters(&limit[split], kern, &cfg);
    if (e != cudaSuccess) return e;
    if (limit[split] < 1) limit[split] = 1;
    __atomic_store_n(&known[split], limit[split], __ATOMIC_RELAXED);
  }
  return cudaSuccess;
}

template <int NT, int GROUP>
static cudaError_t run_w4(const W4Args& a, cudaStream_t st) {
  auto kern = linear_w4_kernel<NT, GROUP>;
  static unsigned configured = 0;  // a bit per device
  cudaError_t e = allow_smem(kern, w4_smem(NT), &configured);
  int limit[9];
  if (e == cudaSuccess) e = w4_limits<NT, GROUP>(limit);
  if (e != cudaSuccess) return e;
  const W4Plan p = plan_w4(a.m, a.in_f, a.out_f, 128 / GROUP, limit);
  if (p.split_x) {
    const int64_t warps = a.m * ((a.in_f + 255) / 256);
    w4_planes_kernel<GROUP><<<(unsigned)((warps + 7) / 8), 256, 0, st>>>(a);
    e = cudaGetLastError();
    if (e != cudaSuccess) return e;
  }
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)p.grid, (unsigned)((a.m + p.mt - 1) / p.mt));
  cfg.blockDim = dim3(w4_warps(NT) * 32);
  cfg.dynamicSmemBytes = p.smem;
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = p.split;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = p.split > 1 ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, kern, a, p);
}

template <int GROUP>
static cudaError_t run_w4_nt(const W4Args& a, cudaStream_t st) {
  switch (w4_column_tiles(a.m)) {
    case 1: return run_w4<1, GROUP>(a, st);
    case 2: return run_w4<2, GROUP>(a, st);
    default: return run_w4<3, GROUP>(a, st);
  }
}

cudaError_t launch_linear_w4(const W4Args& a, cudaStream_t st) {
  switch (a.group) {
    case 32: return run_w4_nt<32>(a, st);
    case 64: return run_w4_nt<64>(a, st);
    default: return run_w4_nt<128>(a, st);
  }
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
