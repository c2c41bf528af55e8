// eb_sample.cu -- the next token's id from a row of logits: temperature, top-k,
// top-p, min-p and a given uniform number.
//
// Tokens are ordered by (logit descending, index ascending): every filter
// keeps a prefix of that order. A composite key, the logit's ordered bits
// above the complemented index, turns the order into one of distinct 64-bit
// integers, so a prefix is {key >= cut}; the token is then found by a running
// sum in index order over the kept ones. Nothing is sorted but a list of at
// most kCap tokens around the cut:
//
//   pass 1  the largest logit M (with no filter: the sums too, and pass 4)
//   pass 2  a histogram of (M - logit) / T in 1/32 octaves of weight, counts
//           only. Where it shows that top_k's cut, or all that top_p's can
//           need, lies within kCap tokens, the window is those bins from the
//           top; else the bins around the estimated cut.
//   pass 3  the window's tokens into the list; above it, and in all for top_p,
//           the weights' exact sums. The list is sorted and the cut found
//           among exact sums. A cut outside the window, or a bin of more than
//           kCap tokens at the cut, is left to a bisection over the keys with
//           a pass per bit: exact for any input, and slow.
//   pass 4  sums of the kept weights, a run of the row per warp; the run in
//           which u's share falls is then walked by its CTA. With all kept
//           tokens in the list, the list sorted by index takes its place.
//
// Weights are f64 (2^t by a 32-entry table and a Taylor polynomial of degree
// 4: 2 * 10^-12 relative): in f32 the running sum over a vocabulary would be
// off by more than many a token's share. Sums meet in a fixed order, so
// results do not depend on timing (the list's order of arrival is undone by
// the sort).
//
// A row is shared by a cluster of 1 to 16 CTAs; passes after the first read it
// from L1 or L2. What bounds it: for one row the chain of five cluster barriers
// (of ten where the quick bound fails) with rank 0 alone at work in between; for
// many rows latency, at 24 warps an SM of 80 registers (and some spills): 256 open
// rows take 98 us, of which the f64 pipe needs 22 (12 operations a token), with
// 512 CTAs in 444 places. A bisection is far slower: rows of 151936 take 0.23 to
// 0.53 ms alone, 64 of them 0.8 to 1.9 ms.
#include <cooperative_groups.h>

#include <algorithm>

#include "eb_common.cuh"
#include "eb_kernels.cuh"
#include "eb_rowops.cuh"

namespace cg = cooperative_groups;

namespace eb {

constexpr int kSampleWarps = 8, kSampleThreads = kSampleWarps * 32;
constexpr int kMaxCluster = 16;
constexpr int kCap = 2048;   // tokens the list holds
constexpr int kAround = 1024; // tokens taken around an estimated cut
constexpr int kCount = 256;   // tokens sorted by counting
constexpr int kOctaves = 60, kPerOctave = 32, kBins = kOctaves * kPerOctave;
typedef unsigned long long u64;

struct SampleShared {
  u64 list[kCap];  // in rank 0: the window's tokens
  union {
    u64 mine[kCap];  // pass 3: this CTA's, on their way there
    struct {         // pass 2: sums of the tokens' places in their bin, in 1/256
      unsigned place[kBins], place_total[kBins];
    };
  };
  double tab[32];
  double seg[kMaxCluster * kSampleWarps];  // sums of the row's runs
  float seg_ref[kMaxCluster * kSampleWarps];
  double part[2][kMaxCluster];  // CTAs' sums, by turn
  double warp_d[kSampleWarps];
  u64 warp_best[kSampleWarps];
  u64 best[kMaxCluster];
  u64 cut;
  unsigned hist[kBins];   // this CTA's counts
  unsigned total[kBins];  // in rank 0: the row's
  int offset[kBins];      // in rank 0: tokens in front of a bin
  unsigned warp_u[kSampleWarps];
  unsigned count, n_mine;  // tokens in list (in rank 0) and in mine
  int mode, lo, hi, k_cut;
  unsigned above, in, base;
  int found, last;
};

enum SampleMode { kAll, kList, kWide, kBisect, kAgain, kShift };

// Floats as unsigned integers of the same order, and back.
__device__ __forceinline__ uint32_t ordered_bits(float x) {
  const uint32_t b = __float_as_uint(x);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float from_ordered(uint32_t o) {
  return __uint_as_float(o & 0x80000000u ? o & 0x7fffffffu : ~o);
}
__device__ __forceinline__ u64 token_key(float l, int i) {
  return (u64)ordered_bits(l) << 32 | (0xffffffffu - (uint32_t)i);
}

__device__ __forceinline__ void count_up(unsigned* p, unsigned by) {
  asm volatile("red.shared::cta.add.u32 [%0], %1;" ::"r"(smem_u32(p)), "r"(by) : "memory");
}

// A logit as the definition takes it: NaN is -infinity, -0 is 0.
__device__ __forceinline__ float clean(float x) { return fmaxf(x, -INFINITY) + 0.f; }

// Taylor coefficients of 2^r and the rounding constant, as operands of the
// f64 instructions (an immediate would take two moves).
__constant__ double kEx2[5] = {0.69314718055994530942, 0.24022650695910071233,
                               0.05550410866482157995, 0.00961812910762847716, 0x1.8p47};

// 2^t for -61 < t <= 0 (1 exactly for 0); elsewhere and for NaN see `on`.
__device__ __forceinline__ double ex2_raw(double t, const double* tab) {
  const double z = t + kEx2[4];  // multiples of 1/32 in its lowest bits
  const int n = __double2loint(z);
  const double r = t - (z - kEx2[4]);  // |r| <= 1/64
  const double q = fma(fma(fma(kEx2[3], r, kEx2[2]), r, kEx2[1]), r, kEx2[0]);
  const double v = tab[n & 31];
  const double p = fma(v * r, q, v);
  return __hiloint2double((int)((unsigned)__double2hiint(p) + ((unsigned)(n >> 5) << 20)),
                          __double2loint(p));
}
__device__ __forceinline__ double ex2_f64(double t, const double* tab) {
  return t > -61.0 ? ex2_raw(t, tab) : 0.0;
}

// f(values, first index) for the row's tokens [a, b), a warp's run: first the
// ends, single tokens padded with -infinity, then 16-byte words. U words of a
// lane are loaded at once: four where the row comes from memory; one (and the
// next on its way) in later passes, which find it in L1 or L2 and are so short
// that fetching U copies of a long body would take longer than running them.
template <int U, typename T, typename F>
__device__ __forceinline__ void each_word(const T* row, int a, int b, F f) {
  constexpr int VEC = 16 / (int)sizeof(T);
  const int lane = threadIdx.x & 31;
  const int mis = (int)((reinterpret_cast<uintptr_t>(row + a) / sizeof(T)) % VEC);
  const int head = min(b - a, (VEC - mis) % VEC);
  const int words = (b - a - head) / VEC, tail = b - a - head - words * VEC;
  const int a1 = a + head;
  const uint4* src = reinterpret_cast<const uint4*>(row + a1);
  float x[VEC];
  {  // head and tail together are fewer than 32
    const int at = lane < head ? a + lane : b - tail + lane - head;
#pragma unroll
    for (int k = 0; k < VEC; k++) x[k] = -INFINITY;
    if (lane < head + tail) {
      x[0] = clean(Elem<T>::to_f32(row[at]));
      f(x, at);
    }
  }
  auto word = [&](const uint4& w, int v) {
    const T* e = reinterpret_cast<const T*>(&w);
#pragma unroll
    for (int k = 0; k < VEC; k++) x[k] = clean(Elem<T>::to_f32(e[k]));
    f(x, a1 + v * VEC);
  };
  int v = lane;
  if constexpr (U > 1) {
#pragma unroll 1
    for (; v + 32 * (U - 1) < words; v += 32 * U) {
      uint4 w[U];
#pragma unroll
      for (int u = 0; u < U; u++) w[u] = src[v + 32 * u];
#pragma unroll
      for (int u = 0; u < U; u++) word(w[u], v + 32 * u);
    }
  }
  uint4 next = make_uint4(0, 0, 0, 0);
  if (v < words) next = src[v];
#pragma unroll 1
  for (; v < words; v += 32) {
    const uint4 w = next;
    if (v + 32 < words) next = src[v + 32];
    word(w, v);
  }
}
// f(value, index), the padding too: -infinity has no weight, no bin and no
// place among the largest. Words without a value of at least `from` are passed
// over (NaN: none is).
template <typename T, typename F>
__device__ __forceinline__ void each_token(const T* row, int a, int b, float from, F f) {
  constexpr int VEC = 16 / (int)sizeof(T);
  each_word<1, T>(row, a, b, [&](const float (&l)[VEC], int i) {
    float m = l[0];
#pragma unroll
    for (int k = 1; k < VEC; k++) m = fmaxf(m, l[k]);
    if (m < from) return;
#pragma unroll
    for (int k = 0; k < VEC; k++) f(l[k], i + k);
  });
}

__device__ __forceinline__ double warp_sum_d(double x) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
  return x;
}

// Exclusive running sum over the CTA's threads, and the total.
template <typename V>
__device__ __forceinline__ V block_scan(V v, V* part, V& all) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  V run = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const V t = __shfl_up_sync(0xffffffffu, run, o);
    if (lane >= o) run += t;
  }
  __syncthreads();
  if (lane == 31) part[warp] = run;
  __syncthreads();
  V before = 0;
  all = 0;
  for (int w = 0; w < kSampleWarps; w++) {
    if (w == warp) before = all;
    all += part[w];
  }
  return before + run - v;
}

// Up to kCount distinct keys, descending, each placed by counting the larger ones.
__device__ __forceinline__ void sort_few(u64* k, int m) {
  __syncthreads();
  u64 mine = 0;
  int at = 0;
  if (threadIdx.x < m) {
    mine = k[threadIdx.x];
#pragma unroll 8
    for (int i = 0; i < m; i++) at += k[i] > mine;
  }
  __syncthreads();
  if (threadIdx.x < m) k[at] = mine;
  __syncthreads();
}

template <typename T>
__global__ void __launch_bounds__(kSampleThreads, 3) sample_kernel(SampleArgs a) {
  extern __shared__ __align__(16) uint8_t smem_raw[];
  SampleShared& s = *reinterpret_cast<SampleShared*>(smem_raw);
  cg::cluster_group cl = cg::this_cluster();
  const int C = a.cluster, rank = blockIdx.x % C;
  const int64_t r = blockIdx.x / C;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int n = (int)a.vocab, runs = C * kSampleWarps;
  const T* row = static_cast<const T*>(a.logits) + r * a.row_stride;
  auto run_start = [&](int g) { return (int)((int64_t)n * g / runs); };
  const int g = rank * kSampleWarps + warp, i0 = run_start(g), i1 = run_start(g + 1);
  auto sync = [&]() {
    if (C > 1) cl.sync();
    else __syncthreads();
  };
  auto at_rank = [&](auto* p, int to) { return C > 1 ? cl.map_shared_rank(p, to) : p; };

  const float temp = a.temperature ? a.temperature[r] : 1.f;
  const bool greedy = !(temp > 0.f);
  const int top_k = a.top_k ? a.top_k[r] : 0;
  const float top_p = a.top_p ? a.top_p[r] : 1.f;
  // past 1 nothing would be kept: as 1, the largest logit and its equals are
  const double min_p = a.min_p && a.min_p[r] > 0.f ? (double)fminf(a.min_p[r], 1.f) : 0.0;
  const bool k_on = !greedy && top_k > 0 && top_k < n, p_on = !greedy && top_p < 1.f;
  // One variable decides which passes a row takes. (With the conditions
  // spelled out at each branch nvcc 12.9 dropped the one before pass 2.)
  enum Kind { kGreedy, kCut, kFloor, kOpen };
  const int kind = greedy ? kGreedy : (k_on || p_on) ? kCut : min_p > 0.0 ? kFloor : kOpen;
  const bool summed = kind == kOpen || (kind == kCut && !k_on);  // pass 1 sums the weights too
  float u = a.u[r];
  u = u > 0.f ? fminf(u, 0x1.fffffep-1f) : 0.f;
  const double c = 1.4426950408889634 / (double)temp;  // octaves per unit of logit

  if (tid < 32) s.tab[tid] = exp2((double)tid / 32);
  for (int i = tid; i < kBins; i += kSampleThreads) s.hist[i] = s.total[i] = s.place[i] = s.place_total[i] = 0;
  if (tid == 0) {
    s.count = s.n_mine = 0;
    s.found = n;
    s.last = -1;
  }
  __syncthreads();

  // ---- pass 1: the largest logit and where it comes first; or the weights'
  // sum with it, against each thread's own largest so far
  float top = -INFINITY;
  int top_i = n;
  float largest;  // this thread's
  double sum = 0;
  constexpr int VEC = 16 / (int)sizeof(T);
  if (summed) {
    double far = 0;         // the thread's largest
    double part[4] = {0, 0, 0, 0};  // four chains of additions
    each_word<4, T>(row, i0, i1, [&](const float (&l)[VEC], int) {
      float m = l[0];
#pragma unroll
      for (int k = 1; k < VEC; k++) m = fmaxf(m, l[k]);
      if (m > top) {
        const double f = top == -INFINITY ? 0.0 : ex2_f64(((double)top - (double)m) * c, s.tab);
#pragma unroll
        for (int k = 0; k < 4; k++) part[k] *= f;
        top = m;
        far = (double)m;
      }
      if (top == INFINITY) {
#pragma unroll
        for (int k = 0; k < VEC; k++) part[0] += l[k] == INFINITY ? 1.0 : 0.0;
      } else if (top > -INFINITY) {
        // -infinity leaves t -infinity or NaN: not counted
#pragma unroll
        for (int k = 0; k < VEC; k++) {
          const double t = ((double)l[k] - far) * c;  // 0 for the largest itself
          const double w = ex2_raw(t, s.tab);
          if (t > -61.0) part[k & 3] += w;
        }
      }
    });
    sum = (part[0] + part[1]) + (part[2] + part[3]);
  } else {
    each_word<4, T>(row, i0, i1, [&](const float (&l)[VEC], int i) {
#pragma unroll
      for (int k = 0; k < VEC; k++)
        if (l[k] > top || (l[k] == top && i + k < top_i)) {  // the ends come first
          top = l[k];
          top_i = i + k;
        }
    });
  }
  {
    u64 best = token_key(top, top_i);
    const float mine = top;
    largest = top;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const u64 t = __shfl_xor_sync(0xffffffffu, best, o);
      best = t > best ? t : best;
    }
    top = from_ordered((uint32_t)(best >> 32));
    if (summed) {
      // the run's sum against its largest
      const double f = mine == top ? 1.0 : mine == -INFINITY ? 0.0 : ex2_f64(((double)mine - (double)top) * c, s.tab);
      sum = warp_sum_d(top == -INFINITY ? 0.0 : sum * f);
      if (lane < C) {
        *at_rank(&s.seg[g], lane) = sum;
        *at_rank(&s.seg_ref[g], lane) = top;
      }
    }
    if (lane == 0) s.warp_best[warp] = best;
    __syncthreads();
    for (int w = 0; w < kSampleWarps; w++) best = s.warp_best[w] > best ? s.warp_best[w] : best;
    if (tid < C) *at_rank(&s.best[rank], tid) = best;
    sync();
    for (int q = 0; q < C; q++) best = s.best[q] > best ? s.best[q] : best;
    top = from_ordered((uint32_t)(best >> 32));
    top_i = (int)(0xffffffffu - (uint32_t)best);
  }
  // From here on a CTA may leave where no other will read its memory again.
  if (top == -INFINITY || kind == kGreedy) {
    if (rank == 0 && tid == 0) a.ids[r] = top == -INFINITY ? -1 : top_i;
    return;
  }
  const double top_d = (double)top;
  auto weight = [&](float l) {  // -infinity leaves t -infinity or NaN: none
    const double t = ((double)l - top_d) * c;
    const double w = ex2_raw(t, s.tab);
    return l == top ? 1.0 : t >= -60.0 ? w : 0.0;
  };

  // 1/32 octaves of weight below the largest, not smaller for a smaller logit;
  // a token past the last bin has no weight. (fminf takes the NaN of -infinity
  // at an infinite temperature there.)
  const float cb = (float)(c * kPerOctave);
  auto bins_below = [&](float l) {
    const float d = l == top ? 0.f : (top - l) * cb;
    return fminf(d, (float)kBins);
  };
  auto bin_of = [&](float l) { return (int)bins_below(l); };

  // The runs' sums of pass 1, against the row's largest; their sum.
  double whole = 0;
  if (summed) {
    if (tid < runs) s.seg[tid] *= weight(s.seg_ref[tid]);
    __syncthreads();
    constexpr int PER = kMaxCluster * kSampleWarps / 32;
#pragma unroll
    for (int j = 0; j < PER; j++)
      if (lane * PER + j < runs) whole += s.seg[lane * PER + j];
    whole = warp_sum_d(whole);
  }

  u64 cut = 0;
  double above = 0;             // this thread's tokens above the window
  int win_lo = 0, win_hi = -1;  // and the window: pass 4 reads it alone
  float from = -INFINITY;       // no value below matters
  if (kind == kCut) {
    // ---- pass 2: counts by bin; for top_p alone the places in the bins too.
    // Tokens that weigh less than (1 - top_p) / n of the whole are less than
    // 1 - top_p of it together: top_p drops them all, and they are not counted.
    const bool sums = p_on && !k_on;
    auto value_at = [&](float bins) {  // not above any value in that many bins
      return top - bins / cb - fabsf(top) * 1e-6f;
    };
    if (sums) {
      const double least = (1.0 - (double)fmaxf(top_p, 0.f)) * whole / n;
      from = value_at((float)kPerOctave * (1.f - __log2f((float)least)) + 1.f);
    }
    // With top_k, first only each thread's largest: the bin that holds top_k of
    // those bounds the cut from below, and little more than top_k tokens are
    // in it or above. Where too few threads or too many tokens are: every one.
    bool quick = k_on && top_k <= kCount * 3 / 4 && top_k <= C * kSampleThreads / 4;
    int mode;
    for (;;) {
      if (quick) {
        const int b = bin_of(largest);
        if (b < kBins) count_up(&s.hist[b], 1);
      } else if (sums) {
        each_token(row, i0, i1, from, [&](float l, int) {
          const float d = bins_below(l);
          const int b = (int)d;
          if (b < kBins) {
            count_up(&s.hist[b], 1);
            count_up(&s.place[b], (unsigned)((d - (float)b) * 256.f));
          }
        });
      } else {
        each_token(row, i0, i1, from, [&](float l, int) {
          const int b = bin_of(l);
          if (b < kBins) count_up(&s.hist[b], 1);
        });
      }
      __syncthreads();
      if (C > 1) {
        unsigned* to = cl.map_shared_rank(s.total, 0);
        unsigned* to_place = cl.map_shared_rank(s.place_total, 0);
        for (int i = tid; i < kBins; i += kSampleThreads)
          if (s.hist[i]) {
            atomicAdd(to + i, s.hist[i]);
            if (sums) atomicAdd(to_place + i, s.place[i]);
          }
      }
      sync();
      const unsigned* total = C > 1 ? s.total : s.hist;
      const unsigned* places = C > 1 ? s.place_total : s.place;
      if (rank == 0) {
        // some bins to a thread: counts and estimated masses, from the top. A
        // bin's mass is taken as its count at the mean place of its tokens (plus
        // what an even spread adds: (ln 2 / 32)^2 / 24).
        constexpr int PER = (kBins + kSampleThreads - 1) / kSampleThreads;
        unsigned cnt[PER], mine = 0, before, all;
        double mass = 0, est[PER];
#pragma unroll
        for (int j = 0; j < PER; j++) {
          const int b = tid * PER + j;
          cnt[j] = b < kBins ? total[b] : 0;
          mine += cnt[j];
          est[j] = 0;
          if (sums && cnt[j]) {
            const float mean = ((float)places[b] + 0.5f * cnt[j]) / (256.f * cnt[j]);
            est[j] = cnt[j] * ex2_f64(-((double)b + (double)mean) / kPerOctave, s.tab) * (cnt[j] > 8 ? 1.0000195 : 1.0);
          }
          mass += est[j];
        }
        before = block_scan(mine, s.warp_u, all);
        double all_mass;
        const double m_before = block_scan(mass, s.warp_d, all_mass);
        const bool k_cut = quick || (k_on && (unsigned)top_k < all);  // else fewer tokens have weight
        const double want = sums ? (double)fmaxf(top_p, 0x1p-100f) * whole : 0.0;
        if (tid == 0) {
          s.lo = 0;
          s.hi = kBins - 1;  // where no bin is the cut's
        }
        __syncthreads();
        unsigned run = before;
        double m_run = m_before;
#pragma unroll
        for (int j = 0; j < PER; j++) {  // the cut's bin
          const bool here = k_cut ? run < (unsigned)top_k && run + cnt[j] >= (unsigned)top_k
                                  : m_run < want && m_run + est[j] >= want;
          if (here && cnt[j]) atomicMin(&s.hi, tid * PER + j);
          run += cnt[j];
          m_run += est[j];
        }
        __syncthreads();
        const int cut_bin = s.hi;
        run = before;
#pragma unroll
        for (int j = 0; j < PER; j++) {
          if (tid * PER + j < kBins) s.offset[tid * PER + j] = (int)run;
          if (tid * PER + j == cut_bin) {
            s.above = run;
            s.in = cnt[j];
          }
          run += cnt[j];
        }
        __syncthreads();
        const unsigned above = s.above, in = s.in;
        int mode = kList;
        if (quick) mode = all >= (unsigned)top_k ? kList : kAgain;
        else if (!k_cut && !p_on) mode = kAll;
        else if (in > kCap || (k_on && p_on && (k_cut ? above + in > kCap : all > kAround))) mode = kBisect;
        else if (above + in > (k_cut ? kCap : kAround)) mode = kWide;
        __syncthreads();
        if (mode == kWide && tid == 0) s.lo = cut_bin;
        __syncthreads();
        // top_p's cut was estimated: take as many bins around as the list holds,
        // below it first (half of the room left, in the wide case), then above
        if (!k_cut && (mode == kList || mode == kWide)) {
          const unsigned room = mode == kList ? kAround : above + in + (in < kAround ? (kAround - in) / 2 : 0);
          run = before;
#pragma unroll
          for (int j = 0; j < PER; j++) {
            run += cnt[j];
            const int b = tid * PER + j;
            if (b > cut_bin && b < kBins && run <= room) atomicMax(&s.hi, b);
          }
          __syncthreads();
          if (mode == kWide) {
            const int hi = s.hi;
            run = before;
#pragma unroll
            for (int j = 0; j < PER; j++) {
              run += cnt[j];
              if (tid * PER + j == hi) s.in = run;  // tokens down to hi
            }
            __syncthreads();
            const unsigned down = s.in;
            run = before;
#pragma unroll
            for (int j = 0; j < PER; j++) {
              const int b = tid * PER + j;
              if (b < cut_bin && down - run <= kAround) atomicMin(&s.lo, b);
              run += cnt[j];
            }
            __syncthreads();
          }
        }
        const int lo = s.lo, hi = s.hi;
        if (tid < C) {
          *at_rank(&s.mode, tid) = mode;
          *at_rank(&s.lo, tid) = lo;
          *at_rank(&s.hi, tid) = hi;
          *at_rank(&s.k_cut, tid) = k_cut ? 1 : 0;
        }
      }
      sync();
      mode = s.mode;
      int lo = s.lo, hi = s.hi;
      const bool k_cut = s.k_cut != 0;
      const float from_all = from;

      for (int turn = 0; mode == kList || mode == kWide; turn++) {
        // ---- pass 3: the window into rank 0's list, the sum (for top_k: the
        // count) of what is above it
        unsigned n_above = 0;
        from = fmaxf(from_all, value_at((float)hi + 2.f));
        above = 0;
        const bool count = k_cut && lo > 0;
        auto gather = [&](float l, int i, int b) {
          if (b >= lo && b <= hi) {
            const unsigned at = atomicAdd(&s.n_mine, 1u);
            if (at < kCap) s.mine[at] = token_key(l, i);  // the window holds no more
          }
        };
        if (lo == 0) {
          each_token(row, i0, i1, from, [&](float l, int i) { gather(l, i, bin_of(l)); });
        } else {
          each_token(row, i0, i1, from, [&](float l, int i) {
            const int b = bin_of(l);
            gather(l, i, b);
            if (b < lo) {
              above += weight(l);
              n_above++;
            }
          });
          double all_a;
          block_scan(count ? (double)n_above : above, s.warp_d, all_a);
          if (tid == 0) *at_rank(&s.part[0][rank], 0) = all_a;
        }
        __syncthreads();
        {
          const unsigned have = s.n_mine;
          if (tid == 0) s.base = atomicAdd(at_rank(&s.count, 0), have);
          __syncthreads();
          u64* list = at_rank(s.list, 0);
          const unsigned base = s.base;
          for (unsigned i = tid; i < have && i < kCap; i += kSampleThreads)
            if (base + i < kCap) list[base + i] = s.mine[i];
        }
        sync();
        if (rank == 0 && s.count > (quick ? kCount : kCap)) {  // a quick bound that was too low
          if (tid < C) *at_rank(&s.mode, tid) = quick ? kAgain : kBisect;
        } else if (rank == 0) {
          const int m = (int)s.count;
          // sorted: a short list by counting, a long one by bin (whose places
          // pass 2 counted) and then within each bin
          if (m <= kCount) {
            sort_few(s.list, m);
          } else {
            const int start = s.offset[lo];
            __syncthreads();
            for (int i = tid; i < m; i += kSampleThreads) {
              const u64 key = s.list[i];
              const int b = bin_of(from_ordered((uint32_t)(key >> 32)));
              const int at = atomicAdd(&s.offset[b], 1) - start;
              if (at >= 0 && at < m) s.mine[at] = key;  // (always: the counts are these tokens')
            }
            __syncthreads();
            for (int i = tid; i < m; i += kSampleThreads) {
              const u64 key = s.mine[i];
              const int b = bin_of(from_ordered((uint32_t)(key >> 32)));
              const int end = min(s.offset[b] - start, m), begin = max(end - (int)total[b], 0);
              int at = begin;
              for (int j = begin; j < end; j++) at += s.mine[j] > key;
              if (at < m) s.list[at] = key;
            }
            __syncthreads();
            for (int b = lo + tid; b <= hi; b += kSampleThreads) s.offset[b] -= (int)total[b];
          }
          double over = 0;  // of what is above the window
          if (lo > 0)
            for (int q = 0; q < C; q++) over += s.part[0][q];
          // running sums of the sorted list's weights, four to a thread
          constexpr int PER = kCap / kSampleThreads;
          double w[PER], mine = 0, all, b4[PER];
          const int left = k_cut ? top_k - (count ? (int)over : 0) : m;  // places in the list
#pragma unroll
          for (int j = 0; j < PER; j++) {
            const int i = tid * PER + j;
            w[j] = i < m && i < left ? weight(from_ordered((uint32_t)(s.list[i] >> 32))) : 0.0;
            b4[j] = mine;
            mine += w[j];
          }
          const double start = block_scan(mine, s.warp_d, all) + (sums ? over : 0.0);
          if (!sums) whole = all;  // of the top_k tokens, or of all that have weight
          const double want = (double)top_p * whole;
          unsigned keep = 0, kept;
#pragma unroll
          for (int j = 0; j < PER; j++) {
            const int i = tid * PER + j;
            const bool first = i == 0 && lo == 0;
            if (i < m && i < left && (first || !p_on || count || start + b4[j] < want) &&
                (first || w[j] >= min_p))
              keep++;
          }
          block_scan(keep, s.warp_u, kept);
          // top_p's cut is not in the window: above it, or below. The next window
          // is as many of the bins there as the list holds.
          const bool up = sums && lo > 0 && over >= want;
          const bool down = sums && !up && (int)kept == m && hi + 1 < kBins && over + all < want;
          if (up || down) {
            mode = kShift;
            __syncthreads();
            if (tid == 0) {
              s.lo = up ? lo : hi + 1;
              s.hi = up ? lo - 1 : hi;
            }
            __syncthreads();
            const int edge = up ? lo : hi + 1, tokens = s.offset[edge];
            for (int b = tid; b < kBins; b += kSampleThreads) {
              if (up && b < lo && tokens - s.offset[b] <= kCap) atomicMin(&s.lo, b);
              if (down && b > hi && s.offset[b] + (int)total[b] - tokens <= kCap) atomicMax(&s.hi, b);
            }
            __syncthreads();
            if (s.lo > s.hi || turn >= 8) mode = kBisect;  // a bin of more than the list holds
          } else if ((int)kept > kCount && mode == kList) {
            mode = kWide;  // pass 4 finds the token
          }
          if (mode == kList) {
            // all kept tokens are here: in index order, the running sum again
            u64 k2[PER];
            __syncthreads();
#pragma unroll
            for (int j = 0; j < PER; j++) k2[j] = tid * PER + j < (int)kept ? s.list[tid * PER + j] : 0;
            __syncthreads();
#pragma unroll
            for (int j = 0; j < PER; j++)  // complemented index first: descending is index ascending
              if (tid * PER + j < (int)kept) s.list[tid * PER + j] = k2[j] << 32 | k2[j] >> 32;
            sort_few(s.list, (int)kept);
            mine = 0;
#pragma unroll
            for (int j = 0; j < PER; j++) {
              const int i = tid * PER + j;
              w[j] = i < (int)kept ? weight(from_ordered((uint32_t)s.list[i])) : 0.0;
              mine += w[j];
            }
            double run = block_scan(mine, s.warp_d, all);
            const double target = (double)u * all;
            // the first place at which the sum passes the target
#pragma unroll
            for (int j = 0; j < PER; j++) {
              const int i = tid * PER + j;
              run += w[j];
              if (w[j] > 0) {
                if (run > target) atomicMin(&s.found, i);
                atomicMax(&s.last, i);
              }
            }
            __syncthreads();
            if (tid == 0) {
              const int i = s.found < n ? s.found : s.last;
              a.ids[r] = (int)(0xffffffffu - (uint32_t)(s.list[i] >> 32));
            }
          } else if (mode == kWide) {
            // the last kept key; none in the window: what is above its first
            if (tid == 0) s.cut = kept > 0 ? s.list[kept - 1] : m > 0 ? s.list[0] + 1 : ~0ull;
            __syncthreads();
          }
          if (tid < C) {
            *at_rank(&s.mode, tid) = mode;
            *at_rank(&s.cut, tid) = s.cut;
            const int to_lo = s.lo, to_hi = s.hi;
            *at_rank(&s.lo, tid) = to_lo;
            *at_rank(&s.hi, tid) = to_hi;
          }
        }
        if (mode == kList) {
          // rank 0 alone knows whether the list sufficed
          sync();
          if (s.mode == kList) return;
        } else {
          sync();
        }
        mode = s.mode;
        cut = s.cut;
        if (mode == kShift) {
          lo = s.lo;
          hi = s.hi;
          mode = kWide;
          if (tid == 0) s.count = s.n_mine = 0;
          sync();
          continue;
        }
        if (mode == kWide && min_p == 0.0) {
          win_lo = lo;
          win_hi = hi;
        }
        break;
      }
      if (mode != kAgain) break;
      quick = false;
      from = -INFINITY;
      for (int i = tid; i < kBins; i += kSampleThreads) s.hist[i] = s.total[i] = 0;
      if (tid == 0) s.count = s.n_mine = 0;
      sync();
    }
    if (mode == kBisect) {
      // ---- a pass per bit of the key: counts, then exact sums
      int turn = 0;
      auto reduce = [&](double v) {
        double all;
        block_scan(v, s.warp_d, all);
        if (tid < C) *at_rank(&s.part[turn & 1][rank], tid) = all;
        sync();
        all = 0;
        for (int q = 0; q < C; q++) all += s.part[turn & 1][q];
        turn++;
        return all;
      };
      cut = 0;
      if (k_on)
        for (int bit = 63; bit >= 0; bit--) {
          const u64 at = cut | 1ull << bit;
          int v = 0;
          each_token(row, i0, i1, -INFINITY, [&](float l, int i) { v += token_key(l, i) >= at; });
          if (reduce(v) >= top_k) cut = at;
        }
      if (p_on) {
        const u64 low = cut;
        auto mass = [&](u64 at) {
          double v = 0;
          each_token(row, i0, i1, -INFINITY, [&](float l, int i) {
            if (token_key(l, i) >= at) v += weight(l);
          });
          return reduce(v);
        };
        const double want = (double)top_p * mass(low);
        cut = 0;
        for (int bit = 63; bit >= 0; bit--) {
          const u64 at = cut | 1ull << bit;
          const double v = mass(at);
          if (v >= want && v > 0) cut = at;
        }
        cut = cut > low ? cut : low;
      }
    }
  }

  // ---- pass 4: sums of the kept weights by run; open rows have them
  auto kept_weight = [&](float l, int i) {
    if (token_key(l, i) < cut) return 0.0;
    const double w = weight(l);
    return w >= min_p || l == top ? w : 0.0;
  };
  if (kind != kOpen) {
    if (win_hi >= 0) {
      sum = above;
      each_token(row, i0, i1, from, [&](float l, int i) {
        const int b = bin_of(l);
        if (b >= win_lo && b <= win_hi) sum += kept_weight(l, i);
      });
    } else {
      sum = 0;
      each_token(row, i0, i1, -INFINITY, [&](float l, int i) { sum += kept_weight(l, i); });
    }
    sum = warp_sum_d(sum);
    if (lane < C) *at_rank(&s.seg[g], lane) = sum;
    sync();
  }
  // The run in which the running sum passes the target (every warp finds the
  // same): four runs to a lane.
  double before = 0, target;
  int run;
  {
    constexpr int PER = kMaxCluster * kSampleWarps / 32;
    double v[PER], mine = 0;
#pragma unroll
    for (int j = 0; j < PER; j++) {
      v[j] = lane * PER + j < runs ? s.seg[lane * PER + j] : 0.0;
      mine += v[j];
    }
    double at = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const double t = __shfl_up_sync(0xffffffffu, at, o);
      if (lane >= o) at += t;
    }
    target = (double)u * __shfl_sync(0xffffffffu, at, 31);
    at -= mine;
    int first = runs, last = -1;  // this lane's first run past the target, its last with weight
    double b_first = 0, b_last = 0;
#pragma unroll
    for (int j = 0; j < PER; j++) {
      if (v[j] > 0) {
        if (at + v[j] > target && first == runs) {
          first = lane * PER + j;
          b_first = at;
        }
        last = lane * PER + j;
        b_last = at;
      }
      at += v[j];
    }
    run = __reduce_min_sync(0xffffffffu, first);
    if (run < runs) {
      before = __shfl_sync(0xffffffffu, b_first, run / PER);
    } else {  // u so near 1 that rounding passes the end: the last with weight
      run = __reduce_max_sync(0xffffffffu, last);
      before = __shfl_sync(0xffffffffu, b_last, max(run, 0) / PER);
    }
  }
  if (run < 0 || run / kSampleWarps != rank) return;  // (the largest has weight: some run has)

  // ---- the run, in pieces of consecutive tokens to a thread
  const int a0 = run_start(run), a1 = run_start(run + 1);
  const int per = (a1 - a0 + kSampleThreads - 1) / kSampleThreads;
  const int b0 = min(a1, a0 + tid * per), b1 = min(a1, b0 + per);
  sum = 0;
  for (int i = b0; i < b1; i++) sum += kept_weight(clean(Elem<T>::to_f32(row[i])), i);
  double all;
  double at = before + block_scan(sum, s.warp_d, all);
  for (int i = b0; i < b1 && sum > 0; i++) {
    const double w = kept_weight(clean(Elem<T>::to_f32(row[i])), i);
    at += w;
    if (w > 0) {
      if (at > target) {
        atomicMin(&s.found, i);
        break;
      }
      atomicMax(&s.last, i);
    }
  }
  __syncthreads();
  if (tid == 0) a.ids[r] = s.found < n ? s.found : s.last;
}

size_t sample_workspace_bytes(int64_t, int64_t) { return 0; }

template <typename T>
static cudaError_t run_sample(SampleArgs a, cudaStream_t st) {
  auto kern = sample_kernel<T>;
  static unsigned configured = 0;
  cudaError_t e = allow_smem(kern, (int)sizeof(SampleShared), &configured);
  if (e != cudaSuccess) return e;
  // CTAs per row: up to six for every SM (three are resident), with 4096 tokens
  // each at least. Rows whose filters take longer then have more SMs: 64 rows
  // of mixed settings take 90 us with 8 CTAs each, 117 with 4 (rows of top-k 50
  // alone 44, and 26 with 4).
  a.cluster = 1;
  while (a.cluster < kMaxCluster && a.rows * a.cluster * 2 <= 6 * sm_count() &&
         a.vocab >= 4096ll * 2 * a.cluster)
    a.cluster *= 2;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)(a.rows * a.cluster));
  cfg.blockDim = dim3(kSampleThreads);
  cfg.dynamicSmemBytes = sizeof(SampleShared);
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = a.cluster;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = a.cluster > 1 ? 1 : 0;
  if (a.cluster > 8) {  // more than the portable size
    e = cudaFuncSetAttribute(kern, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    if (e != cudaSuccess) return e;
  }
  return cudaLaunchKernelEx(&cfg, kern, a);
}

cudaError_t launch_sample(const SampleArgs& a, cudaStream_t st) {
  switch (a.dtype) {
    case kF32: return run_sample<float>(a, st);
    case kF16: return run_sample<__half>(a, st);
    default: return run_sample<__nv_bfloat16>(a, st);
  }
}

}  // namespace eb
