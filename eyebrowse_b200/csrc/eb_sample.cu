// eb_sample.cu -- the next token's id from a row of logits: temperature, top-k,
// top-p, min-p and a given uniform number.
//
// Tokens are ordered by (logit descending, index ascending): every filter
// keeps a prefix of that order. A composite key, the logit's ordered bits
// above the complemented index, turns the order into one of distinct 64-bit
// integers, so a prefix is {key >= cut}.
#include "eb_common.cuh"
#include "eb_kernels.cuh"
#include "eb_rowops.cuh"

namespace eb {

constexpr int kSampleThreads = 1024;

// Floats as unsigned integers of the same order.
__device__ __forceinline__ uint32_t ordered_bits(float x) {
  const uint32_t b = __float_as_uint(x);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}

template <typename T>
__device__ __forceinline__ T block_sum(T v, T* part) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  __syncthreads();
  if (lane == 0) part[warp] = v;
  __syncthreads();
  v = part[lane];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

__global__ void __launch_bounds__(kSampleThreads) sample_kernel(SampleArgs a) {
  __shared__ double part_d[32];
  __shared__ int part_i[32];
  __shared__ float part_f[32];
  __shared__ int found;
  const int64_t r = blockIdx.x;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int n = (int)a.vocab;
  auto logit = [&](int i) {
    const float l = ld_any(a.logits, r * a.row_stride + i, a.dtype);
    return l != l ? -INFINITY : l;
  };
  float top = -INFINITY;
  for (int i = tid; i < n; i += kSampleThreads) top = fmaxf(top, logit(i));
  top = warp_max(top);
  if (lane == 0) part_f[warp] = top;
  if (tid == 0) found = n;
  __syncthreads();
  top = warp_max(part_f[lane]);
  if (top == -INFINITY) {
    if (tid == 0) a.ids[r] = -1;
    return;
  }
  const float temp = a.temperature ? a.temperature[r] : 1.f;
  if (!(temp > 0.f)) {
    for (int i = tid; i < n; i += kSampleThreads)
      if (logit(i) == top) atomicMin(&found, i);
    __syncthreads();
    if (tid == 0) a.ids[r] = found;
    return;
  }
  auto weight = [&](float l) {
    if (l == top) return 1.0;
    if (l == -INFINITY) return 0.0;
    const double w = exp(((double)l - (double)top) / (double)temp);
    return w < 0x1p-60 ? 0.0 : w;
  };
  auto key = [&](float l, int i) {
    return (unsigned long long)ordered_bits(l) << 32 | (0xffffffffu - (uint32_t)i);
  };
  unsigned long long cut = 0;
  auto mass = [&](unsigned long long at) {
    double s = 0;
    for (int i = tid; i < n; i += kSampleThreads) {
      const float l = logit(i);
      if (key(l, i) >= at) s += weight(l);
    }
    return block_sum(s, part_d);
  };
  const int k = a.top_k ? a.top_k[r] : 0;
  if (k > 0 && k < n) {
    for (int bit = 63; bit >= 0; bit--) {
      const unsigned long long at = cut | 1ull << bit;
      int c = 0;
      for (int i = tid; i < n; i += kSampleThreads) c += key(logit(i), i) >= at;
      if (block_sum(c, part_i) >= k) cut = at;
    }
  }
  const float p = a.top_p ? a.top_p[r] : 1.f;
  if (p < 1.f) {
    const double want = (double)p * mass(cut);
    const unsigned long long low = cut;
    cut = 0;
    for (int bit = 63; bit >= 0; bit--) {
      const unsigned long long at = cut | 1ull << bit;
      const double s = mass(at);
      if (s >= want && s > 0) cut = at;
    }
    cut = cut > low ? cut : low;
  }
  const double least = a.min_p && a.min_p[r] > 0.f ? (double)a.min_p[r] : 0.0;
  auto kept = [&](int i) {
    const float l = logit(i);
    if (key(l, i) < cut) return 0.0;
    const double w = weight(l);
    return w >= least || l == top ? w : 0.0;
  };
  // the running sum in the vocabulary's order: a run of tokens per thread
  const int per = (n + kSampleThreads - 1) / kSampleThreads;
  const int i0 = min(n, tid * per), i1 = min(n, i0 + per);
  double s = 0;
  for (int i = i0; i < i1; i++) s += kept(i);
  double run = s;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const double t = __shfl_up_sync(0xffffffffu, run, o);
    if (lane >= o) run += t;
  }
  if (lane == 31) part_d[warp] = run;
  __syncthreads();
  double before = 0, total = 0;
  for (int w = 0; w < 32; w++) {
    if (w < warp) before += part_d[w];
    total += part_d[w];
  }
  before += run - s;
  float u = a.u[r];
  u = u > 0.f ? fminf(u, 0x1.fffffep-1f) : 0.f;
  const double target = (double)u * total;
  if (s > 0 && before + s > target) {
    double c = before;
    for (int i = i0; i < i1; i++) {
      const double w = kept(i);
      c += w;
      if (w > 0 && c > target) {
        atomicMin(&found, i);
        break;
      }
    }
  }
  __syncthreads();
  if (tid == 0) a.ids[r] = found;
}

cudaError_t launch_sample(const SampleArgs& a, cudaStream_t st) {
  sample_kernel<<<(unsigned)a.rows, kSampleThreads, 0, st>>>(a);
  return cudaGetLastError();
}

size_t sample_workspace_bytes(int64_t, int64_t) { return 0; }

}  // namespace eb
