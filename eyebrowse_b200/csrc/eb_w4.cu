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

// linear_w4_kernel multiplies on the tensor cores with mma.sync (m16n8k16,
// f16, f32 sums): 16 weight rows by 16 inputs against 8 columns. At a few
// columns the work is a stream of the weights, and dequantisation in
// registers, not the matrix rate, is what a warp has to keep under its share
// of the memory bandwidth (about 2.5 instruction slots per code and lane at
// 6.5 TB/s); a tcgen05 operand would have to pass through shared memory
// first, and its 128-row tiles would leave most SMs idle at decode sizes.
//
// - Codes are exact in f16: 0x6400 | code is 1024 + code, 0x6400 | code << 4
//   is 1024 + 16 code, and one subtraction or FMA leaves code - zero.
// - The columns are f16 planes of x. Each (row of x, block of 128 inputs) is
//   scaled by the power of two that brings its largest value to [2^14, 2^15);
//   then a 16-bit value is one plane and an f32 value two, the second holding
//   what the first leaves (22 bits; what falls under f16's range is below
//   2^-39 of the block's largest). Products are exact; a group's sum is
//   scaled by its own and the block's scale in f32 and added to the row's.
// - The inputs of a k16 step may be any 16 as long as both operands agree, so
//   the packed layout gives thread c of a quad 8 consecutive codes (one
//   word) of each group of 32, and x is stored with its eights in the order
//   0 4 1 5 2 6 3 7 that the words' nibble pairs come out in.
// - The warps of a CTA: wr side by side over 32-row tiles, wk over the blocks
//   of 128 inputs; a cluster splits the inputs further. CTAs stay and walk
//   over the tiles, so that x is staged once and the stream of weights does
//   not stop between tiles. Partial sums meet in shared memory, then in the
//   cluster's.
constexpr int kW4Ring = 3;   // blocks of a warp in its ring of shared memory
constexpr int kW4Tile = 32;  // weight rows of a warp: two m16 tiles

// By columns / 8. One column tile: three CTAs of 8 warps on an SM (80
// registers a thread). More: one CTA of 16 (128), which stages x once for all.
constexpr int w4_warps(int nt) { return nt == 1 ? 8 : 16; }
constexpr int w4_ctas(int nt) { return nt == 1 ? 3 : 1; }
constexpr int w4_smem(int nt) { return (nt == 1 ? 74 : 226) * 1024; }
constexpr int w4_ring_bytes(int nt) { return w4_warps(nt) * kW4Ring * 2048; }
// Partial sums of a CTA's warps, one m16 tile at a time.
constexpr int w4_red_bytes(int nt) { return w4_warps(nt) * 16 * (nt * 8 + 2) * 4; }

struct W4Plan {
  int wr, wk;      // warps of a CTA over row tiles and over input blocks
  int split;       // CTAs of a cluster over input blocks
  int chunk;       // blocks of 128 inputs staged at a time
  int planes, mt;  // f16 planes per value, x rows per CTA
  int units;       // runs of wr tiles
  int nt, grid, smem;
};

__device__ __forceinline__ void mma_f16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0,
                                        uint32_t b1) {
  asm(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
      "{%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// The first product of a sum.
__device__ __forceinline__ void mma_f16_first(float (&d)[4], const uint32_t (&a)[4], uint32_t b0,
                                              uint32_t b1) {
  asm(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
      "{%8,%9}, {%10,%10,%10,%10};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.f));
}

__device__ __forceinline__ __half2 as_half2(uint32_t v) { return *reinterpret_cast<__half2*>(&v); }
__device__ __forceinline__ uint32_t as_u32(__half2 v) { return *reinterpret_cast<uint32_t*>(&v); }

// Codes 0 and 4, then 1 and 5, of a word, less the zero point, as f16 (exact).
// bias0 = -(1024 + zero), bias1 = -(64 + zero).
__device__ __forceinline__ uint32_t and_or(uint32_t a, uint32_t b, uint32_t c) {
  uint32_t d;
  asm("lop3.b32 %0, %1, %2, %3, 0xea;" : "=r"(d) : "r"(a), "r"(b), "r"(c));
  return d;
}
__device__ __forceinline__ void w4_pairs(uint32_t w, uint32_t magic, __half2 bias0, __half2 bias1, uint32_t& p0,
                                         uint32_t& p1) {
  p0 = as_u32(__hadd2(as_half2(and_or(w, 0x000f000fu, magic)), bias0));
  p1 = as_u32(__hfma2(as_half2(and_or(w, 0x00f000f0u, magic)), as_half2(0x2c002c00u), bias1));
}

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// Eight inputs of x row t into the planes' rows of shared memory. The 16
// threads of a half warp hold a block of 128.
__device__ __forceinline__ void w4_stage8(const W4Args& a, int planes, int64_t t, int64_t k0,
                                          uint8_t* dst, int row_bytes, float* block_scale) {
  float f[8];
  const int64_t at = t * a.x_stride + k0;
  const char* src = static_cast<const char*>(a.x) + at * (a.dtype_x == kF32 ? 4 : 2);
  if (k0 + 8 <= a.in_f && (reinterpret_cast<uintptr_t>(src) & 15) == 0) {
    load8_any(a.x, at, a.dtype_x, f);
  } else {
#pragma unroll
    for (int n = 0; n < 8; n++) f[n] = k0 + n < a.in_f ? ld_any(a.x, at + n, a.dtype_x) : 0.f;
  }
  float top = 0.f;  // of the finite values; the others go through as they are
#pragma unroll
  for (int n = 0; n < 8; n++) top = fabsf(f[n]) <= 3.402823466e38f ? fmaxf(top, fabsf(f[n])) : top;
  const uint32_t half = threadIdx.x & 16 ? 0xffff0000u : 0x0000ffffu;
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(half, top, o));
  const int e = max((int)(__float_as_uint(top) >> 23), 27);  // at least 2^-100
  const float up = __uint_as_float((uint32_t)(127 + 14 + 127 - e) << 23);
  if ((threadIdx.x & 15) == 0) {
    block_scale[0] = __uint_as_float((uint32_t)(e - 14) << 23);
    if (planes == 2) block_scale[1] = block_scale[0];
  }
  uint32_t h[4], l[4];
#pragma unroll
  for (int n = 0; n < 4; n++) {
    const float x0 = f[n] * up, x1 = f[n + 4] * up;
    const __half2 hi = __floats2half2_rn(x0, x1);
    const float2 hf = __half22float2(hi);
    h[n] = as_u32(hi);
    // an infinity or a NaN is all in the first plane
    l[n] = pack_half2(fabsf(hf.x) <= 65504.f ? x0 - hf.x : 0.f,
                      fabsf(hf.y) <= 65504.f ? x1 - hf.y : 0.f);
  }
  *reinterpret_cast<uint4*>(dst) = make_uint4(h[0], h[1], h[2], h[3]);
  if (planes == 2) *reinterpret_cast<uint4*>(dst + row_bytes) = make_uint4(l[0], l[1], l[2], l[3]);
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
  float* xscale = part + (pl.split > 1 ? 2 * pl.mt * cta_rows : 0);  // [chunk][8 NT]: of a block's columns
  uint8_t* zeros = reinterpret_cast<uint8_t*>(xscale + pl.chunk * NT * 8);  // what columns past the last read
  uint8_t* xs = zeros + 256;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, c = lane & 3, n = lane >> 2;
  const int wk = warp % pl.wk, wr = warp / pl.wk;
  const int rank = blockIdx.x % pl.split;
  const int64_t m0 = (int64_t)blockIdx.y * pl.mt;
  const int mt = (int)min((int64_t)pl.mt, a.m - m0);
  const int P = pl.planes, cols = mt * P;
  const int out_f = (int)a.out_f;
  const int blocks = (int)((a.in_f + 127) / 128), groups = (int)((a.in_f + GROUP - 1) / GROUP);
  const int kb0 = (int)((int64_t)blocks * rank / pl.split);
  const int kb1 = (int)((int64_t)blocks * (rank + 1) / pl.split);
  const int row_bytes = pl.chunk * 256 + 64;  // 64 past a multiple of 128: no bank is hit twice
  const uint16_t* scale = static_cast<const uint16_t*>(a.scale);
  const bool sbf = a.dtype_scale == kBF16;
  const int step = gridDim.x / pl.split;

  // The warp's blocks, tile after tile, pass through a ring of its own, each
  // thread reading back what it copied: no barrier, and several blocks of
  // every warp in flight without registers. Thread: rows n, n + 8, n + 16 and
  // n + 24 of the tile (the last row again past the end), 16 bytes of each.
  // The scales (low half) and zero points of a block's groups come with it,
  // row `lane` of the tile in a thread.
  struct Meta {
    uint32_t v[GB];
  };
  const uint32_t ring = smem_u32(smem_raw) + warp * kW4Ring * 2048 + lane * 16;
  int fetch_unit = blockIdx.x / pl.split, fetch_kb = kb0 + wk, fetch_slot = 0, fetch_row = 0;
  const uint8_t* from[4];
  auto aim = [&]() {
    const int row0 = (fetch_unit * pl.wr + wr) * kW4Tile;
    fetch_row = min(row0 + lane, out_f - 1);
#pragma unroll
    for (int j = 0; j < 4; j++)
      from[j] = static_cast<const uint8_t*>(a.q) + (int64_t)min(row0 + n + 8 * j, out_f - 1) * blocks * 64 + c * 16;
  };
  auto fetch = [&](Meta& meta) {
    if (fetch_unit < pl.units && fetch_kb < kb1) {
#pragma unroll
      for (int j = 0; j < 4; j++)
        cp_async16(ring + fetch_slot * 2048 + j * 512, from[j] + (uint32_t)(fetch_kb * 64));
#pragma unroll
      for (int g = 0; g < GB; g++) {
        const int64_t at = (int64_t)min(fetch_kb * GB + g, groups - 1) * out_f + fetch_row;
        meta.v[g] = (uint32_t)__ldg(scale + at) | (a.zero ? (uint32_t)__ldg(a.zero + at) : 8u) << 16;
      }
      fetch_kb += pl.wk;
      if (fetch_kb >= kb1) {
        fetch_kb = kb0 + wk;
        fetch_unit += step;
        aim();
      }
    }
    cp_async_commit();
    fetch_slot = fetch_slot + 1 == kW4Ring ? 0 : fetch_slot + 1;
  };
  for (int i = threadIdx.x; i < pl.chunk * NT * 8 + 64; i += THREADS) xscale[i] = 0.f;  // and zeros
  uint32_t magic = 0x64006400u;
  asm volatile("" : "+r"(magic));  // in a register: LOP3 takes one immediate
  static_assert(kW4Ring == 3, "two blocks ahead: meta0 and meta1");
  Meta meta0{}, meta1{};
  aim();
  fetch(meta0);
  fetch(meta1);

  int slot = 0, buf = 0;
  for (int unit = blockIdx.x / pl.split; unit < pl.units; unit += step) {
    float acc[2][NT][4];
#pragma unroll
    for (int rt = 0; rt < 2; rt++)
#pragma unroll
      for (int t = 0; t < NT; t++)
#pragma unroll
        for (int e = 0; e < 4; e++) acc[rt][t][e] = 0.f;

    for (int ch = kb0; ch < kb1; ch += pl.chunk) {
      const int end = min(ch + pl.chunk, kb1);
      if (ch > kb0 || unit == blockIdx.x / pl.split || pl.chunk < kb1 - kb0) {
        __syncthreads();  // what was staged before has been read
        const int eights = (end - ch) * 16;
        for (int i = threadIdx.x; i < eights * mt; i += THREADS) {
          const int t = i / eights, e = i % eights;
          w4_stage8(a, P, m0 + t, (int64_t)ch * 128 + e * 8, xs + t * P * row_bytes + e * 16,
                    row_bytes, &xscale[(e >> 4) * NT * 8 + t * P]);
        }
        __syncthreads();
      }
      for (int kb = ch + wk; kb < end; kb += pl.wk) {
        cp_async_wait<kW4Ring - 2>();
        uint4 w[4];
#pragma unroll
        for (int j = 0; j < 4; j++)
          w[j] = *reinterpret_cast<const uint4*>(smem_raw + (warp * kW4Ring + slot) * 2048 + j * 512 + lane * 16);
        slot = slot + 1 == kW4Ring ? 0 : slot + 1;
        const Meta meta = meta0;
        meta0 = meta1;
        fetch(meta1);
        const uint8_t* xb[NT];  // column 8 t + n, word 0
#pragma unroll
        for (int t = 0; t < NT; t++)
          xb[t] = (8 * t + n < cols ? xs + (8 * t + n) * row_bytes + (kb - ch) * 256 : zeros) + c * 16;
        // Chains of dependent products are kept short: a sum per m16 tile and,
        // at one column tile, per half of a word.
        constexpr int H = NT == 1 ? 2 : 1;
        float sum[2][NT][H][4];
        __half2 bias[2][2][2];
        float s[2][2];
#pragma unroll
        for (int i = 0; i < 4; i++) {
          const bool first = i * 32 % GROUP == 0, last = (i + 1) * 32 % GROUP == 0;
          if (first) {
#pragma unroll
            for (int rt = 0; rt < 2; rt++)
#pragma unroll
              for (int r = 0; r < 2; r++) {
                const uint32_t m = __shfl_sync(0xffffffffu, meta.v[i * 32 / GROUP], n + 16 * rt + 8 * r);
                s[rt][r] = w4_scale(m & 0xffffu, sbf);
                // -(1024 + z) and -(64 + z) in both halves: z is one, or 16, units of the last place
                bias[rt][r][0] = as_half2(((m >> 16) | 0xe400u) * 0x10001u);
                bias[rt][r][1] = as_half2((((m >> 12) & 0xf0u) | 0xd400u) * 0x10001u);
              }
          }
          uint4 x[NT];
#pragma unroll
          for (int t = 0; t < NT; t++) x[t] = *reinterpret_cast<const uint4*>(xb[t] + i * 64);
#pragma unroll
          for (int rt = 0; rt < 2; rt++) {
            const uint4 w0 = w[2 * rt], w1 = w[2 * rt + 1];
            const uint32_t u0 = i == 0 ? w0.x : i == 1 ? w0.y : i == 2 ? w0.z : w0.w;
            const uint32_t u1 = i == 0 ? w1.x : i == 1 ? w1.y : i == 2 ? w1.z : w1.w;
            uint32_t f0[4], f1[4];
            w4_pairs(u0, magic, bias[rt][0][0], bias[rt][0][1], f0[0], f0[2]);
            w4_pairs(u1, magic, bias[rt][1][0], bias[rt][1][1], f0[1], f0[3]);
            w4_pairs(u0 >> 8, magic, bias[rt][0][0], bias[rt][0][1], f1[0], f1[2]);
            w4_pairs(u1 >> 8, magic, bias[rt][1][0], bias[rt][1][1], f1[1], f1[3]);
#pragma unroll
            for (int t = 0; t < NT; t++) {
              if (first) mma_f16_first(sum[rt][t][0], f0, x[t].x, x[t].y);
              else mma_f16(sum[rt][t][0], f0, x[t].x, x[t].y);
            }
#pragma unroll
            for (int t = 0; t < NT; t++) {
              if (first && H == 2) mma_f16_first(sum[rt][t][H - 1], f1, x[t].z, x[t].w);
              else mma_f16(sum[rt][t][H - 1], f1, x[t].z, x[t].w);
            }
          }
          if (last) {
#pragma unroll
            for (int t = 0; t < NT; t++) {
              const float2 xb2 = *reinterpret_cast<const float2*>(xscale + (kb - ch) * NT * 8 + 8 * t + 2 * c);
#pragma unroll
              for (int rt = 0; rt < 2; rt++)
#pragma unroll
                for (int e = 0; e < 4; e++) {
                  const float v = H == 2 ? sum[rt][t][0][e] + sum[rt][t][H - 1][e] : sum[rt][t][0][e];
                  acc[rt][t][e] = fmaf(v * s[rt][e >> 1], e & 1 ? xb2.y : xb2.x, acc[rt][t][e]);
                }
            }
          }
        }
      }
    }

    // sums of the warps that share rows, one m16 tile after the other
    const int cta_row0 = unit * cta_rows;
#pragma unroll
    for (int rt = 0; rt < 2; rt++) {
      __syncthreads();  // the sums before have been read
#pragma unroll
      for (int t = 0; t < NT; t++)
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
          const float* s = red + ((w * pl.wk + k) * 16 + rr) * LD + t * P;
          v += P == 2 ? s[1] + s[0] : s[0];
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

size_t linear_w4_workspace_bytes(int64_t, int64_t, int64_t) { return 0; }

// The shape of a launch: of every (wk, split) whose staged x fits, the one
// with the least work on the busiest SM, counted in blocks of 128 inputs of
// one warp (an eight of x staged by each thread is about a quarter, a tile's
// sums about one, a cluster's about another), and at least what the longest
// row of blocks of one warp takes (a warp alone takes about as long for a
// block as a full SM for 24).
static W4Plan plan_w4(int64_t m, int64_t in_f, int64_t out_f, int planes) {
  W4Plan p{};
  p.planes = planes;
  const int64_t most = 24 / planes, passes = (m + most - 1) / most;
  p.mt = (int)((m + passes - 1) / passes);
  const int cols = p.mt * planes;
  p.nt = (cols + 7) / 8;
  const int64_t tiles = (out_f + kW4Tile - 1) / kW4Tile, blocks = (in_f + 127) / 128;
  const int64_t slots = (int64_t)w4_ctas(p.nt) * sm_count();
  const int warps = w4_warps(p.nt);
  const int fixed = w4_ring_bytes(p.nt) + w4_red_bytes(p.nt);
  double best = 0;
  for (int wk = warps; wk >= 1; wk /= 2)
    for (int split = 1; split <= 8 && split <= blocks; split++) {
      const int wr = warps / wk;
      const int part = split > 1 ? 2 * p.mt * wr * kW4Tile * 4 : 0;
      const int64_t range = (blocks + split - 1) / split;
      const int64_t left = w4_smem(p.nt) - fixed - part - 64 * cols - 256;
      const int64_t fit = std::max<int64_t>(left, 0) / (256 * cols + 32 * p.nt) / wk * wk;
      if (fit == 0) continue;  // chunks are whole turns of the wk warps
      const int64_t chunk = std::min(range, fit);
      const int64_t units = (tiles + wr - 1) / wr;
      const int64_t clusters = std::max<int64_t>(1, slots / passes / split);
      const int64_t grid = std::min(units, clusters) * split;
      const int64_t turns = (units + clusters - 1) / clusters;
      // an SM's CTAs; at most one of them has the last turn if few have
      const int64_t per_sm = (grid * passes + sm_count() - 1) / sm_count();
      const int64_t last = (units - (turns - 1) * clusters) * split * passes;
      const int64_t unit_sm = last <= sm_count() ? per_sm * (turns - 1) + 1 : per_sm * turns;
      const double blocks_warp = (double)((range + wk - 1) / wk);
      const double stage = 0.25 * (double)((range * 16 * p.mt + warps * 32 - 1) / (warps * 32));
      const double sums = split > 1 ? 2 : 1;
      const double staged = chunk < range ? unit_sm * stage : per_sm * stage;
      const double busy = warps * (unit_sm * (blocks_warp + sums) + staged);
      const double alone = 24.0 * (turns * (blocks_warp + sums) + (chunk < range ? turns : 1) * stage);
      const double cost = std::max(busy, alone);
      if (best == 0 || cost < best) {
        best = cost;
        p.wk = wk;
        p.wr = wr;
        p.split = split;
        p.chunk = (int)chunk;
        p.units = (int)units;
        p.grid = (int)grid;
        p.smem = fixed + part + (int)chunk * 32 * p.nt + 256 + cols * (int)(chunk * 256 + 64);
      }
    }
  return p;
}

template <int NT, int GROUP>
static cudaError_t run_w4(const W4Args& a, const W4Plan& p, cudaStream_t st) {
  auto kern = linear_w4_kernel<NT, GROUP>;
  static unsigned configured = 0;  // a bit per device
  const cudaError_t e = allow_smem(kern, w4_smem(NT), &configured);
  if (e != cudaSuccess) return e;
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
static cudaError_t run_w4_nt(const W4Args& a, const W4Plan& p, cudaStream_t st) {
  switch (p.nt) {
    case 1: return run_w4<1, GROUP>(a, p, st);
    case 2: return run_w4<2, GROUP>(a, p, st);
    default: return run_w4<3, GROUP>(a, p, st);
  }
}

cudaError_t launch_linear_w4(const W4Args& a, cudaStream_t st) {
  const W4Plan p = plan_w4(a.m, a.in_f, a.out_f, a.dtype_x == kF32 ? 2 : 1);
  switch (a.group) {
    case 32: return run_w4_nt<32>(a, p, st);
    case 64: return run_w4_nt<64>(a, p, st);
    default: return run_w4_nt<128>(a, p, st);
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
