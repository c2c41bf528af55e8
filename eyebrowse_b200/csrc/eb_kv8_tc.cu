// eb_kv8_tc.cu -- decode attention over the 8-bit cache on tcgen05 tensor cores
// (head_dim 64, 128 and 256).
//
// The cache's bytes go from HBM through TMA into shared memory and from there
// into the tensor core as they are: no thread touches them. For a KV head and
// its G query heads, over tiles of 128 rows t:
//
//   S^T [t, (h, j)] = K [t, d] * Q^T     A = the K tile (K-major)
//   O^T [d, (h, j)] += V^T [d, t] * P^T  A = the V tile (MN-major)
//
// with kind::f8f6f4, whose operands may be E4M3 and E5M2 in any pairing. The
// other operand has to be 8 bits wide too, so a value x of Q or P becomes
// planes j = 0, 1, ..: the nearest E4M3 number, then 16 times what is left,
// and so on, four bits each, which the readers add up again with weights
// 16^-j. Four planes (16 bits) serve 16-bit outputs, five (20 bits) f32. The
// G * planes columns are few, so the tensor work stays far below the time the
// bytes take (N = 48: two MMAs of 24 clocks per 4 KB).
//
// At head_dim 64 a CTA takes two neighbouring KV heads, whose bytes of a row lie
// side by side: their tile looks like one of head_dim 128. S is made for each
// from its own half of the bytes; O for the heads of both, of which each keeps
// its own half of the lanes.
//
// Scales: a row's K scale multiplies its scores, its V scale its weight, both
// in the softmax thread that owns the row (one TMEM lane each). Weights are
// kept relative to a running maximum of score + log2(V scale) per head, so
// that what P holds stays in E4M3's range; it is raised (and O rescaled) only
// when a tile passes it by more than 2^3.5.
//
// One CTA = (KV head or pair [, 8 heads of it], sequence, chunk of rows), 192
// threads: warps 0-3 softmax and output, warp 4 TMA producer, warp 5 TMEM owner
// and MMA issuer (S of tile j + 1 runs during the softmax of tile j). Chunks
// start on multiples of 128 rows, so a block of rows never spans two; the CTA of
// the last one appends the step's new row first (two warps each for K and V),
// where one CTA has all heads of the KV head. The last CTA of a (sequence, head
// group) merges the chunks' partial (m, l, O) in chunk order (atomic ticket, no
// spin-wait).
//
// Measured: 64 sequences of 512 to 16384 rows, 8 KV heads of 128 with four query
// heads each, 196 to 207 us, of which HBM needs 165: it is bound by the softmax
// threads, four exponentials and four splits of a weight into planes for each
// 256 bytes a row has. One sequence of 2048 rows 12 us: the
// launch, the append, one trip to HBM, four barriers a tile and the merge. At
// head_dim 256 the ring (192 KB) leaves one CTA an SM: 24 sequences with a window
// of 1024, 4 KV heads, 28.5 us, 192 CTAs in 148 places. head_dim 64: 64
// sequences of 8192 rows, 8 KV heads, 124 us (the bytes need 82).
#include "eb_kv8.cuh"
#include "eb_rowops.cuh"
#include "eb_tc.cuh"

namespace eb {

constexpr int kKvTile = 128;
constexpr int kKvChunks = 256;         // of a context, at most (the host's plan keeps to it)
constexpr float kPScale = 32.f;        // P's plane 0 holds 32 * weight, at most 32 * 2^3.5 < 448
constexpr float kKvRescale = 3.5f;
constexpr float kMinLogScale = -64.f;  // of a V scale of zero

template <int HD, int GP, int P>
struct Kv8Cfg {
  static constexpr bool PAIR = HD == 64;  // two KV heads, GP / 2 query heads of each
  static constexpr int HALVES = PAIR ? 2 : 1, GH = GP / HALVES;
  static constexpr int HB = PAIR ? 1 : HD / 128;
  static constexpr int NH = (GH * P + 15) / 16 * 16, N = HALVES * NH;  // columns of a KV head, of a tile
  // column of plane p of head h
  static constexpr __host__ __device__ int col(int h, int p) { return h / GH * NH + h % GH * P + p; }
  static constexpr int ROWS = N * 128;  // bytes of a [N][128] operand block
  static constexpr int TILE = kKvTile * 128;
  static constexpr int K_BYTES = HB * TILE;
  static constexpr int Q_OFF = 0, P_OFF = HB * ROWS, KV_OFF = P_OFF + 2 * ROWS;
  // two CTAs on an SM at head_dim 128, one at 256
  static constexpr int NST = HB == 2 ? 3 : (KV_OFF + 6 * K_BYTES <= 110 * 1024 ? 3 : 2);
  static constexpr int BAR_OFF = KV_OFF + NST * 2 * K_BYTES;
  static constexpr int MISC_OFF = BAR_OFF + 256;  // warp maxima [2][4][8], sums [4][8], flags
  static constexpr int SMEM = MISC_OFF + 512 + 1024;
  static constexpr int O_COL = 0, S_COL = HB * N;
  static constexpr int TMEM_COLS = constexpr_pow2ceil(HB * N + 2 * N);
  static_assert(NST * 2 * K_BYTES >= GP * (kKvChunks + 1) * 4, "the merge's weights");
  static_assert(SMEM <= 232448 && TMEM_COLS <= 512 / (HB == 1 ? 2 : 1), "on-chip budgets");
};

__device__ __forceinline__ void umma_f8(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc,
                                        uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
      "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}
// kind::f8f6f4, f32 sums: A E4M3 (0) or E5M2 (1), K- or MN-major, B E4M3 K-major, M = 128.
__device__ __forceinline__ uint32_t idesc_f8(int N, bool a_e5m2, bool a_mn) {
  return (1u << 4) | ((a_e5m2 ? 1u : 0u) << 7) | ((a_mn ? 1u : 0u) << 15) |
         ((uint32_t)(N >> 3) << 17) | (8u << 24);
}
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
        "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]),
        "=r"(r[14]), "=r"(r[15])
      : "r"(taddr));
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
      "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
      "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}

// Byte of (row n, byte k) in a [N][128] operand block with 128-byte swizzle.
__device__ __forceinline__ uint32_t sw128_byte(uint32_t n, uint32_t k) {
  return (n << 7) | (((k >> 4) ^ (n & 7u)) << 4) | (k & 15u);
}

// x's planes: E4M3 codes c[0], c[1], .. with x ~ sum_j 16^-j value(c[j]).
template <int P>
__device__ __forceinline__ void f8_planes(float x, uint8_t (&c)[P]) {
#pragma unroll
  for (int j = 0; j < P; j++) {
    c[j] = f8_encode(x, false);
    x = (x - f8_decode(c[j], false)) * 16.f;
  }
}

// The same of two values: codes of x0 in the low, of x1 in the high byte.
template <int P>
__device__ __forceinline__ void f8_planes2(float x0, float x1, uint16_t (&c)[P]) {
#pragma unroll
  for (int j = 0; j < P; j++) {
    c[j] = __nv_cvt_float2_to_fp8x2(make_float2(x0, x1), __NV_SATFINITE, __NV_E4M3);
    if (j + 1 < P) {
      const float2 v = __half22float2(__half2(__nv_cvt_fp8x2_to_halfraw2(c[j], __NV_E4M3)));
      x0 = (x0 - v.x) * 16.f;
      x1 = (x1 - v.y) * 16.f;
    }
  }
}

template <int HD, int GP, int P>
__global__ void __launch_bounds__(192)
    kv8_decode_tc_kernel(const __grid_constant__ CUtensorMap tmK,
                         const __grid_constant__ CUtensorMap tmV, Kv8DecodeArgs a) {
  using C = Kv8Cfg<HD, GP, P>;
  constexpr int E = HD / 32, N = C::N, NST = C::NST, GH = C::GH, HALVES = C::HALVES;
  const int grp = blockIdx.x, b = blockIdx.y, ck = blockIdx.z;
  const int kvh = grp / a.gsubs * HALVES, sub = grp % a.gsubs;
  const int heads = a.H / a.hkv;
  const int G = min(GH, heads - sub * GH);           // heads of each KV head
  const int halves = min(HALVES, a.hkv - kvh);       // an odd last KV head has no neighbour
  auto has = [&](int h) { return h % GH < G && h / GH < halves; };
  auto head = [&](int h) { return (kvh + h / GH) * heads + sub * GH + h % GH; };
  const int pos = a.positions ? a.positions[b] : a.max_pos;
  if (pos < 0 || pos > a.max_pos) return;  // an empty slot of the batch
  const int row_lo = a.window > 0 ? max(0, pos - a.window + 1) : 0;
  const int first = row_lo & ~(kKvTile - 1);
  const int n_chunks = (pos - first) / a.chunk + 1;
  if (ck >= n_chunks) return;
  const int row_begin = first + ck * a.chunk;
  const int row_end = min(row_begin + a.chunk, pos + 1);
  const int n_tiles = (row_end - row_begin + kKvTile - 1) / kKvTile;
  const bool append = a.k_new && ck == n_chunks - 1;  // this chunk holds the new row and its block

  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~uintptr_t(1023));
  const uint32_t s0 = smem_u32(smem);
  const uint32_t sQ = s0 + C::Q_OFF, sP = s0 + C::P_OFF, sKV = s0 + C::KV_OFF;
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + C::BAR_OFF);
  float* wmax = reinterpret_cast<float*>(smem + C::MISC_OFF);  // [2][4][8]
  float* wsum = wmax + 64;                                     // [4][8]
  volatile int* abort_flag = reinterpret_cast<volatile int*>(wsum + 32);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(wsum + 33);
  auto bar = [&](int i) { return smem_u32(&bars[i]); };
  constexpr int kQ = 0, kFinal = 1, kSFull0 = 2, kPFull0 = 4, kODone0 = 6, kKFull0 = 8;
  constexpr int kKEmpty0 = kKFull0 + NST, kVFull0 = kKEmpty0 + NST, kVEmpty0 = kVFull0 + NST;
  constexpr int kAppended = kVEmpty0 + NST, kNumBars = kAppended + 1;
  static_assert(kNumBars * 8 <= 256, "barrier area");

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    mbar_init(bar(kQ), 128);
    mbar_init(bar(kFinal), 1);
    for (int i = kSFull0; i < kNumBars; i++)
      mbar_init(bar(i), i == kPFull0 || i == kPFull0 + 1 || i == kAppended ? 128 : 1);
    *abort_flag = 0;
    fence_mbar_init();
    fence_async_smem();
  }
  if (warp == 4 && lane == 0) {
    tma_prefetch_map(&tmK);
    tma_prefetch_map(&tmV);
  }
  if (warp == 5) {
    tmem_alloc(smem_u32(tmem_slot), C::TMEM_COLS);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  if (warp == 4) {
    // ------------------------------------------------------------ TMA producer
    if (lane == 0) {
      int issued = 0;
      // only the chunk that is appended to waits for it
      bool ok = !append || mbar_wait(bar(kAppended), 0, abort_flag, a.err, kErrTimeoutTma);
      for (int j = 0; ok && j < n_tiles; j++) {
        const int st = j % NST, row = row_begin + j * kKvTile;
        for (int which = 0; which < 2; which++) {
          const int full = (which ? kVFull0 : kKFull0) + st, empty = (which ? kVEmpty0 : kKEmpty0) + st;
          if (j >= NST &&
              !mbar_wait(bar(empty), (j / NST - 1) & 1, abort_flag, a.err, kErrTimeoutTma)) {
            ok = false;
            break;
          }
          const uint32_t dst = sKV + (st * 2 + which) * C::K_BYTES;
          mbar_arrive_expect_tx(bar(full), C::K_BYTES);
#pragma unroll
          for (int hb = 0; hb < C::HB; hb++)
            tma_load_4d(dst + hb * C::TILE, which ? &tmV : &tmK, bar(full),
                        C::PAIR ? kvh * HD : hb * 128, C::PAIR ? 0 : kvh, row, b);
          issued++;
        }
      }
      // every load that was issued has landed before the CTA may leave
      for (int i = 0; i < 2 * NST; i++) {
        const int st = i >> 1, which = i & 1;
        const int n = (issued - (which ? 0 : -1)) / 2;  // loads of this kind: K first
        const int uses = n > st ? (n - 1 - st) / NST + 1 : 0;
        if (uses)
          mbar_drain(bar((which ? kVFull0 : kKFull0) + st), (uses - 1) & 1, a.err, kErrTimeoutTma);
      }
    }
    __syncwarp();
  } else if (warp == 5) {
    // ------------------------------------------------------------ MMA issuer
    if (lane == 0) {
      const uint32_t id_qk = idesc_f8(C::NH, a.e5m2, false), id_pv = idesc_f8(N, a.e5m2, true);
      auto issue_qk = [&](int buf, int st) {
#pragma unroll
        for (int u = 0; u < HALVES; u++)  // (a pair's second KV head: bytes 64.. of the rows)
#pragma unroll
          for (int k = 0; k < HD / 32; k++) {
            const int at = u * 2 + k;
            umma_f8(tmem + C::S_COL + buf * N + u * C::NH,
                    sdesc_sw128(sKV + st * 2 * C::K_BYTES + (at >> 2) * C::TILE + (at & 3) * 32, 16, 1024),
                    sdesc_sw128(sQ + (at >> 2) * C::ROWS + u * C::NH * 128 + (at & 3) * 32, 16, 1024),
                    id_qk, k > 0);
          }
      };
      auto issue_pv = [&](int buf, int st, bool first_tile) {
#pragma unroll
        for (int hb = 0; hb < C::HB; hb++)
#pragma unroll
          for (int k = 0; k < kKvTile / 32; k++)
            umma_f8(tmem + C::O_COL + hb * N,
                    sdesc_sw128(sKV + (st * 2 + 1) * C::K_BYTES + hb * C::TILE + k * 32 * 128, C::TILE, 1024),
                    sdesc_sw128(sP + buf * C::ROWS + k * 32, 16, 1024), id_pv,
                    (!first_tile || k > 0) ? 1u : 0u);
      };
      bool ok = mbar_wait(bar(kQ), 0, abort_flag, a.err, kErrTimeoutMma) &&
                mbar_wait(bar(kKFull0), 0, abort_flag, a.err, kErrTimeoutMma);
      if (ok) {
        tc_fence_after();
        issue_qk(0, 0);
        umma_commit(bar(kSFull0));
        umma_commit(bar(kKEmpty0));
      }
      for (int j = 0; ok && j < n_tiles; j++) {
        const int st = j % NST, nj = j + 1, nst = nj % NST;
        if (nj < n_tiles) {
          if (!mbar_wait(bar(kKFull0 + nst), (nj / NST) & 1, abort_flag, a.err, kErrTimeoutMma)) break;
          tc_fence_after();
          issue_qk(nj & 1, nst);
          umma_commit(bar(kSFull0 + (nj & 1)));
          umma_commit(bar(kKEmpty0 + nst));
        }
        if (!mbar_wait(bar(kPFull0 + (j & 1)), (j >> 1) & 1, abort_flag, a.err, kErrTimeoutMma) ||
            !mbar_wait(bar(kVFull0 + st), (j / NST) & 1, abort_flag, a.err, kErrTimeoutMma))
          break;
        tc_fence_after();
        issue_pv(j & 1, st, j == 0);
        umma_commit(bar(kODone0 + (j & 1)));
        umma_commit(bar(kVEmpty0 + st));
      }
      umma_commit(bar(kFinal));
      mbar_drain(bar(kFinal), 0, a.err, kErrTimeoutMma);
    }
    __syncwarp();
  } else {
    // ------------------------------------------------------------ softmax (warps 0-3)
    const int tid = threadIdx.x;
    if (append) {  // warps 0 and 1 the K row, 2 and 3 the V row
      for (int u = 0; u < halves; u++)
        kv8_append<E>(a, warp >> 1, b, kvh + u, pos, warp & 1, lane, 2 + (warp >> 1));
      // generic-proxy writes -> visible to the TMA loads that follow
      asm volatile("fence.proxy.async.global;" ::: "memory");
      mbar_arrive(bar(kAppended));
    }
    // Q's planes: a warp per head, a head's largest value brought to [128, 256)
    float* qscale = wsum;  // [8] until the sums need the place
    for (int g = warp; g < GP; g += 4) {
      if (!has(g)) continue;
      float v[E];
      const int64_t at = (int64_t)b * a.q_bstride + (int64_t)head(g) * HD + lane * E;
      if (((reinterpret_cast<uintptr_t>(a.q) | (uintptr_t)(a.q_bstride * (a.dtype_q == kF32 ? 4 : 2))) & 15) == 0) {
        ld_row<E>(a.q, at, a.dtype_q, v);
      } else {
#pragma unroll
        for (int e = 0; e < E; e++) v[e] = ld_any(a.q, at + e, a.dtype_q);
      }
      warp_kv_row<E>(v, a.q_norm_w, a.eps, a.cos_t ? a.cos_t + (int64_t)pos * (HD / 2) : nullptr,
                     a.sin_t ? a.sin_t + (int64_t)pos * (HD / 2) : nullptr, lane);
      float top = 0.f;
#pragma unroll
      for (int e = 0; e < E; e++) top = f8_amax(top, v[e]);
      top = warp_max(top);
      const int ex = min(max((int)(__float_as_uint(top) >> 23), 27), 227);
      const float up = __uint_as_float((uint32_t)(254 + 7 - ex) << 23);
      if (lane == 0) qscale[g] = __uint_as_float((uint32_t)(ex - 7) << 23);
      uint8_t c[E][P];
#pragma unroll
      for (int e = 0; e < E; e++)
        f8_planes<P>(fabsf(v[e]) <= 3.402823466e38f ? v[e] * up : __uint_as_float(0x7fc00000u), c[e]);
      const int d = g / GH * 64 + lane * E;
#pragma unroll
      for (int j = 0; j < P; j++) {
        uint8_t* dst = smem + C::Q_OFF + (d >> 7) * C::ROWS + sw128_byte(C::col(g, j), d & 127);
        if constexpr (E == 2) {
          *reinterpret_cast<uint16_t*>(dst) = (uint16_t)(c[0][j] | c[1][j] << 8);
        } else {
#pragma unroll
          for (int e = 0; e < E; e += 4)
            *reinterpret_cast<uint32_t*>(dst + e) = (uint32_t)c[e][j] | (uint32_t)c[e + 1][j] << 8 |
                                                    (uint32_t)c[e + 2][j] << 16 | (uint32_t)c[e + 3][j] << 24;
        }
      }
    }
    fence_async_smem();
    mbar_arrive(bar(kQ));
    named_bar_and(1, 128, true);
    float qs[GP];
#pragma unroll
    for (int h = 0; h < GP; h++) qs[h] = has(h) ? qscale[h] * a.scale_log2 : 0.f;

    const float* ks = a.k_scale + b * a.scale_bstride + kvh;
    const float* vs = a.v_scale + b * a.scale_bstride + kvh;
    const int shift = 31 - __clz(a.block);
    auto scales = [&](int j, float (&k)[HALVES], float (&v)[HALVES]) {  // of this thread's row of tile j
      const int row = row_begin + j * kKvTile + tid;
      const bool in = row >= row_lo && row < row_end;
#pragma unroll
      for (int u = 0; u < HALVES; u++) {  // (through L2: the append wrote one of them)
        k[u] = in && u < halves ? __ldcg(ks + (int64_t)(row >> shift) * a.hkv + u) : 0.f;
        v[u] = in && u < halves ? __ldcg(vs + (int64_t)(row >> shift) * a.hkv + u) : 0.f;
      }
    };
    float m[GP], l[GP];
#pragma unroll
    for (int h = 0; h < GP; h++) {
      m[h] = -INFINITY;
      l[h] = 0.f;
    }
    float ksc[HALVES], vsc[HALVES], ksn[HALVES] = {}, vsn[HALVES] = {};
    scales(0, ksc, vsc);
    const uint32_t lanes = (uint32_t)(warp * 32) << 16;
    bool ok = true;
    for (int j = 0; j < n_tiles; j++) {
      const int buf = j & 1, st = j % NST;
      if (j + 1 < n_tiles) scales(j + 1, ksn, vsn);
      ok = ok && mbar_wait(bar(kSFull0 + buf), (j >> 1) & 1, abort_flag, a.err, kErrTimeoutSoftmax);
      __syncwarp();
      tc_fence_after();
      uint32_t raw[N];
#pragma unroll
      for (int i = 0; i < N; i += 16) tmem_ld16(tmem + lanes + C::S_COL + buf * N + i, raw + i);
      tmem_ld_wait();
      const int row = row_begin + j * kKvTile + tid;
      const bool in = row >= row_lo && row < row_end;
      float lv[HALVES], vp[HALVES];
#pragma unroll
      for (int u = 0; u < HALVES; u++) {
        lv[u] = vsc[u] > 0x1p-64f ? __log2f(vsc[u]) : kMinLogScale;
        vp[u] = in ? vsc[u] * kPScale : 0.f;
      }
      float s[GP];
#pragma unroll
      for (int h = 0; h < GP; h++) {
        float x = __uint_as_float(raw[C::col(h, P - 1)]);
#pragma unroll
        for (int p = P - 2; p >= 0; p--) x = fmaf(x, 0.0625f, __uint_as_float(raw[C::col(h, p)]));
        s[h] = in ? x * (qs[h] * ksc[h / GH]) : -INFINITY;
      }
      // Does a row pass the reference of its head by too much? One barrier tells
      // all four warps; only then are the tile's maxima exchanged.
      bool over = false;
#pragma unroll
      for (int h = 0; h < GP; h++) over = over || (has(h) && s[h] + lv[h / GH] > m[h] + kKvRescale);
      bool raise = !named_bar_and(1, 128, ok && !over);
      float mn[GP];
      if (raise) {
#pragma unroll
        for (int h = 0; h < GP; h++) {
          const float top = warp_max(s[h] + lv[h / GH]);
          if (lane == 0 && has(h)) wmax[(buf * 4 + warp) * 8 + h] = top;
        }
        ok = named_bar_and(1, 128, ok);
        if (!ok) break;
#pragma unroll
        for (int h = 0; h < GP; h++) {
          const float* w = wmax + buf * 32 + h;
          mn[h] = has(h) ? fmaxf(fmaxf(w[0], w[8]), fmaxf(w[16], w[24])) : 0.f;
        }
      }
      if (raise) {  // the same in all four warps
        float corr[GP];
#pragma unroll
        for (int h = 0; h < GP; h++) {
          corr[h] = 1.f;
          if (!has(h)) continue;
          const float up = fmaxf(m[h], mn[h]);
          corr[h] = m[h] == up ? 1.f : ex2(m[h] - up);
          m[h] = up;
          l[h] *= corr[h];
        }
        if (j > 0) {
          ok = mbar_wait(bar(kODone0 + ((j - 1) & 1)), ((j - 1) >> 1) & 1, abort_flag, a.err,
                         kErrTimeoutSoftmax);
          __syncwarp();
          tc_fence_after();
#pragma unroll
          for (int hb = 0; hb < C::HB; hb++) {
            uint32_t o[N];
#pragma unroll
            for (int i = 0; i < N; i += 16) tmem_ld16(tmem + lanes + C::O_COL + hb * N + i, o + i);
            tmem_ld_wait();
#pragma unroll
            for (int h = 0; h < GP; h++)
#pragma unroll
              for (int p = 0; p < P; p++)
                o[C::col(h, p)] = __float_as_uint(__uint_as_float(o[C::col(h, p)]) * corr[h]);
#pragma unroll
            for (int i = 0; i < N; i += 16) tmem_st16(tmem + lanes + C::O_COL + hb * N + i, o + i);
          }
          tmem_st_wait();
        }
      }
      // P's buffer is free once the PV before the last one is done
      if (j >= 2)
        ok = ok && mbar_wait(bar(kODone0 + buf), ((j >> 1) - 1) & 1, abort_flag, a.err, kErrTimeoutSoftmax);
      uint8_t* pt = smem + C::P_OFF + buf * C::ROWS;
#pragma unroll
      for (int h = 0; h < GP; h += 2) {
        if (!has(h)) continue;
        // (a head past the last has a score of garbage: its columns are not read)
        const float w0 = in ? ex2(s[h] - m[h]) : 0.f;
        l[h] += w0;
        if constexpr (GP == 1) {
          uint8_t c[P];
          f8_planes<P>(in ? w0 * vp[0] : 0.f, c);
#pragma unroll
          for (int p = 0; p < P; p++) pt[sw128_byte(p, tid)] = c[p];
        } else {
          const float w1 = in ? ex2(s[h + 1] - m[h + 1]) : 0.f;
          l[h + 1] += w1;
          uint16_t c[P];
          f8_planes2<P>(in ? w0 * vp[h / GH] : 0.f, in ? w1 * vp[(h + 1) / GH] : 0.f, c);
#pragma unroll
          for (int p = 0; p < P; p++) {
            pt[sw128_byte(C::col(h, p), tid)] = (uint8_t)c[p];
            pt[sw128_byte(C::col(h + 1, p), tid)] = (uint8_t)(c[p] >> 8);
          }
        }
      }
      if (row_begin + j * kKvTile < row_lo || row_begin + (j + 1) * kKvTile > row_end) {
        // Rows outside [row_lo, row_end) hold whatever the cache holds, NaN
        // codes too: zero them in the V tile, 0 * NaN would reach O.
        ok = ok && mbar_wait(bar(kVFull0 + st), (j / NST) & 1, abort_flag, a.err, kErrTimeoutSoftmax);
        if (ok && !in) {
          uint8_t* vt = smem + C::KV_OFF + (st * 2 + 1) * C::K_BYTES + tid * 128;
#pragma unroll
          for (int hb = 0; hb < C::HB; hb++)
#pragma unroll
            for (int i = 0; i < 8; i++)
              *reinterpret_cast<uint4*>(vt + hb * C::TILE + i * 16) = make_uint4(0, 0, 0, 0);
        }
      }
      fence_async_smem();
      tc_fence_before();
      mbar_arrive(bar(kPFull0 + buf));
#pragma unroll
      for (int u = 0; u < HALVES; u++) {
        ksc[u] = ksn[u];
        vsc[u] = vsn[u];
      }
    }

    // ---- partial or final output: thread = one d (and d + 128) of every head
    ok = ok && mbar_wait(bar(kFinal), 0, abort_flag, a.err, kErrTimeoutEpilogue);
#pragma unroll
    for (int h = 0; h < GP; h++) {
      l[h] = warp_sum(l[h]);
      if (lane == 0 && has(h)) wsum[warp * 8 + h] = l[h];
    }
    ok = named_bar_and(1, 128, ok);
    if (ok) {
      tc_fence_after();
      const bool split = n_chunks > 1;
#pragma unroll
      for (int h = 0; h < GP; h++)
        if (has(h)) l[h] = (wsum[h] + wsum[8 + h]) + (wsum[16 + h] + wsum[24 + h]);
#pragma unroll
      for (int hb = 0; hb < C::HB; hb++) {
        uint32_t raw[N];
#pragma unroll
        for (int i = 0; i < N; i += 16) tmem_ld16(tmem + lanes + C::O_COL + hb * N + i, raw + i);
        tmem_ld_wait();
        const int d = C::PAIR ? tid & 63 : hb * 128 + tid;
#pragma unroll
        for (int h = 0; h < GP; h++) {
          if (!has(h) || (C::PAIR && tid >> 6 != h / GH)) continue;
          float x = __uint_as_float(raw[C::col(h, P - 1)]);
#pragma unroll
          for (int p = P - 2; p >= 0; p--) x = fmaf(x, 0.0625f, __uint_as_float(raw[C::col(h, p)]));
          x *= 1.f / kPScale;
          if (split) a.ws_acc[(((int64_t)b * a.H + head(h)) * a.cmax + ck) * HD + d] = x;
          else st_any(a.o, b * a.o_bstride + (int64_t)head(h) * HD + d, a.dtype_o, x / l[h]);
        }
      }
      if (split) {
        if (tid == 0)
#pragma unroll
          for (int h = 0; h < GP; h++)
            if (has(h)) {
              float* ml = a.ws_ml + (((int64_t)b * a.H + head(h)) * a.cmax + ck) * 2;
              ml[0] = m[h];
              ml[1] = l[h];
            }
        __threadfence();
        named_bar_and(1, 128, true);
        unsigned* cnt = a.ws_cnt + (int64_t)b * gridDim.x + grp;
        bool mine = false;
        if (tid == 0) mine = atomicAdd(cnt, 1u) == (unsigned)(n_chunks - 1);
        mine = !named_bar_and(1, 128, !(tid == 0 && mine));
        if (mine) {
          // The last CTA merges the chunks, in their order: weights by a warp per
          // head, a chunk per lane, into the ring (nothing uses it any more);
          // then a thread sums its d over them, eight loads in flight.
          __threadfence();
          float* weight = reinterpret_cast<float*>(smem + C::KV_OFF);  // [GP][kKvChunks], then sums [GP]
          for (int h = warp; h < GP; h += 4) {
            if (!has(h)) continue;
            const float2* ml = reinterpret_cast<const float2*>(a.ws_ml) + ((int64_t)b * a.H + head(h)) * a.cmax;
            float2 v[kKvChunks / 32];
            float M = -INFINITY, L = 0.f;
#pragma unroll
            for (int i = 0; i < kKvChunks / 32; i++) {
              v[i] = i * 32 + lane < n_chunks ? __ldcg(ml + i * 32 + lane) : make_float2(-INFINITY, 0.f);
              M = fmaxf(M, v[i].x);
            }
            M = warp_max(M);
#pragma unroll
            for (int i = 0; i < kKvChunks / 32; i++) {
              if (i * 32 + lane >= n_chunks) continue;
              const float w = ex2(v[i].x - M);
              weight[h * kKvChunks + i * 32 + lane] = w;
              L = fmaf(v[i].y, w, L);
            }
            L = warp_sum(L);
            if (lane == 0) weight[GP * kKvChunks + h] = L;
          }
          named_bar_and(1, 128, true);
          const int half = C::PAIR ? tid >> 6 : 0, d = C::PAIR ? tid & 63 : tid;
          for (int g = 0; g < G && half < halves; g++) {
            const int h = half * GH + g;
            const float* acc = a.ws_acc + ((int64_t)b * a.H + head(h)) * a.cmax * HD + d;
            const float* w = weight + h * kKvChunks;
            float x[C::HB] = {};
#pragma unroll 8
            for (int c = 0; c < n_chunks; c++)
#pragma unroll
              for (int hb = 0; hb < C::HB; hb++)
                x[hb] = fmaf(__ldcg(acc + (int64_t)c * HD + hb * 128), w[c], x[hb]);
#pragma unroll
            for (int hb = 0; hb < C::HB; hb++)
              st_any(a.o, b * a.o_bstride + (int64_t)head(h) * HD + hb * 128 + d, a.dtype_o,
                     x[hb] / weight[GP * kKvChunks + h]);
          }
          if (tid == 0) *cnt = 0u;
        }
      }
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 5) {
    tc_fence_after();
    tmem_dealloc(tmem, C::TMEM_COLS);
  }
}

// 4-D map over B caches [max_seq][Hkv][hd] of bytes, box {128, 1, 128, 1}; at
// head_dim 64 a row's KV heads are one run of bytes, 128 of them a pair (an odd
// last one's other half is filled with zeros).
static bool make_kv8_map(CUtensorMap* m, const void* base, const Kv8DecodeArgs& a) {
  auto fn = encode_fn();
  if (!fn) return false;
  const bool pair = a.hd == 64;
  cuuint64_t dims[4] = {(cuuint64_t)(pair ? a.hd * a.hkv : a.hd), (cuuint64_t)(pair ? 1 : a.hkv),
                        (cuuint64_t)a.max_seq, (cuuint64_t)a.batch};
  cuuint64_t strides[3] = {dims[0], (cuuint64_t)a.hkv * a.hd,
                           a.batch > 1 ? (cuuint64_t)a.cache_bstride
                                       : (cuuint64_t)a.max_seq * a.hkv * a.hd};
  cuuint32_t box[4] = {128, 1, kKvTile, 1};
  cuuint32_t estr[4] = {1, 1, 1, 1};
  return fn(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 4, const_cast<void*>(base), dims, strides, box, estr,
            CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
            CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int HD, int GP, int P>
static cudaError_t run_kv8_tc(const Kv8DecodeArgs& a, cudaStream_t st) {
  using C = Kv8Cfg<HD, GP, P>;
  auto kern = kv8_decode_tc_kernel<HD, GP, P>;
  static unsigned configured = 0;
  const cudaError_t e = allow_smem(kern, C::SMEM, &configured);
  if (e != cudaSuccess) return e;
  CUtensorMap mk, mv;
  if (!make_kv8_map(&mk, a.kcache, a) || !make_kv8_map(&mv, a.vcache, a)) return cudaErrorInvalidValue;
  kern<<<dim3((a.hkv + C::HALVES - 1) / C::HALVES * a.gsubs, a.batch, a.cmax), 192, C::SMEM, st>>>(mk, mv, a);
  return cudaGetLastError();
}

template <int HD, int P>
static cudaError_t run_kv8_group(const Kv8DecodeArgs& a, cudaStream_t st) {
  const int heads = a.H / a.hkv * (HD == 64 ? 2 : 1);
  if (heads > 4) return run_kv8_tc<HD, 8, P>(a, st);
  if (heads > 2) return run_kv8_tc<HD, 4, P>(a, st);
  if constexpr (HD != 64)
    if (heads == 1) return run_kv8_tc<HD, 1, P>(a, st);
  return run_kv8_tc<HD, 2, P>(a, st);
}

bool kv8_tc_supported(int hd) { return hd == 64 || hd == 128 || hd == 256; }

cudaError_t launch_kv8_decode_tc(const Kv8DecodeArgs& a, cudaStream_t st) {
  const bool wide = a.dtype_o == kF32;
  if (a.hd == 64) return wide ? run_kv8_group<64, 5>(a, st) : run_kv8_group<64, 4>(a, st);
  if (a.hd == 128) return wide ? run_kv8_group<128, 5>(a, st) : run_kv8_group<128, 4>(a, st);
  return wide ? run_kv8_group<256, 5>(a, st) : run_kv8_group<256, 4>(a, st);
}

}  // namespace eb
