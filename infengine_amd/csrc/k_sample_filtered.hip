// Sampling with temperature, top-k, top-p and min-p by row, from given uniforms (no reference
// counterpart: the reference samples greedily).
//
// The tokens in the order (logit descending, id ascending), with the weights
// w = exp((l - max l) / T):
//   n_k  = top_k (off: all);   Z = the mass of the first n_k
//   n_p  = the shortest prefix of those with mass >= top_p Z (off: n_k)
//   n_m  = the tokens with w >= min_p (off: all)
//   kept = the first max(1, min(n_p, n_m)); the token: the first id, in id order, whose kept
//          cumulative mass exceeds u x the kept mass.
// Weights are computed in fp64 and added in 64-bit fixed point (2^-42 units): sums are exact and
// free of order, so that a draw next to a border of the distribution falls as it does in 64 bits.
#include "ie_kernels.h"

namespace ie {

namespace {

constexpr int kThreads = 1024, kWaves = kThreads / 64;
constexpr double kUnit = 4398046511104.0;  // 2^42: sums over kSampleMaxVocab = 2^21 tokens fit 63 bits
typedef unsigned long long u64;

// Order-preserving key of a logit; NaN counts as -inf, -0 as +0.
__device__ __forceinline__ uint32_t logit_key(float v) {
  if (v != v) v = -INFINITY;
  if (v == 0.f) v = 0.f;
  const uint32_t u = __float_as_uint(v);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
constexpr uint32_t kKeyNegInf = 0x007FFFFFu;  // logit_key(-inf)

__device__ __forceinline__ double weight(float l, float mx, double t) {
  if (l == mx) return 1.0;              // (infinite maxima too)
  if (!(l > -INFINITY)) return 0.0;     // -inf, NaN
  return exp(((double)l - (double)mx) / t);
}
__device__ __forceinline__ u64 fixed(double w) { return (u64)(w * kUnit + 0.5); }

template <typename T>
__device__ __forceinline__ T wave_scan_inc(T v) {
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const T w = __shfl_up(v, o, 64);
    if (lane >= o) v += w;
  }
  return v;
}

// Inclusive scan over the workgroup; `red` is a scratch of kWaves values.
__device__ __forceinline__ u64 block_scan(u64 v, u64* red, u64* total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  u64 inc = wave_scan_inc(v);
  __syncthreads();
  if (lane == 63) red[wave] = inc;
  __syncthreads();
  u64 all = 0;
  for (int w = 0; w < kWaves; ++w) {
    if (w < wave) inc += red[w];
    all += red[w];
  }
  *total = all;
  return inc;
}

// A cut of the order: tokens with key > key, and those with key == key and id < id, are kept.
struct Cut {
  uint32_t key;
  int id;
};

// One workgroup a row, several passes over its logits.
__global__ __launch_bounds__(kThreads) void sample_row_kernel(SampleParams p) {
  __shared__ u64 hist[256];
  __shared__ u64 red[kWaves];
  __shared__ uint32_t s_max;
  __shared__ int s_bin, s_id;
  __shared__ u64 s_above;
  const int row = blockIdx.x, tid = threadIdx.x, lane = tid & 63;
  const float* L = p.logits + (size_t)row * p.vocab;
  const int n = p.vocab;

  // the largest logit
  if (tid == 0) s_max = 0, s_id = 0x7FFFFFFF;
  __syncthreads();
  uint32_t best = 0;
  for (int i = tid; i < n; i += kThreads) best = max(best, logit_key(L[i]));
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) best = max(best, (uint32_t)__shfl_xor((int)best, o, 64));
  if (lane == 0) atomicMax(&s_max, best);
  __syncthreads();
  const uint32_t kmax = s_max;
  if (kmax <= kKeyNegInf) {  // nothing to choose from
    if (tid == 0) p.out[row] = -1;
    return;
  }
  const float mx = __uint_as_float(kmax & 0x80000000u ? kmax ^ 0x80000000u : ~kmax);
  const float tf = p.temperature ? p.temperature[row] : 1.0f;
  const float min_p = p.min_p ? p.min_p[row] : 0.0f;
  if (!(tf > 0.f) || min_p > 1.0f) {  // greedy: the first of the largest
    int id = 0x7FFFFFFF;
    for (int i = tid; i < n; i += kThreads)
      if (logit_key(L[i]) == kmax) id = min(id, i);
    atomicMin(&s_id, id);
    __syncthreads();
    if (tid == 0) p.out[row] = s_id;
    return;
  }
  const double t = tf;
  const int top_k = p.top_k ? p.top_k[row] : 0;
  const float top_p = p.top_p ? p.top_p[row] : 1.0f;
  // min-p is a cut of its own, by weight
  const auto passes = [&](double w) { return !(min_p > 0.f) || w >= (double)min_p; };

  Cut cut{0, 0x7FFFFFFF};
  const auto kept = [&](uint32_t k, int i) { return k > cut.key || (k == cut.key && i < cut.id); };
  // The cut where the sum of f over the order (within the present cut) reaches target >= 1: by a
  // radix select of the key, then, among equal keys (equal f), the id of the last one needed.
  const auto select = [&](auto f, u64 target) {
    uint32_t prefix = 0, mask = 0;
    for (int shift = 24; shift >= 0; shift -= 8) {
      if (tid < 256) hist[tid] = 0;
      __syncthreads();
      for (int i = tid; i < n; i += kThreads) {
        const float l = L[i];
        const uint32_t k = logit_key(l);
        if ((k & mask) == prefix && kept(k, i)) {
          const u64 q = f(l);
          if (q) atomicAdd(&hist[k >> shift & 255u], q);
        }
      }
      __syncthreads();
      if (tid < 64) {  // lane l: digits 255 - 4 l .. 252 - 4 l
        u64 h[4], own = 0;
#pragma unroll
        for (int j = 0; j < 4; ++j) own += h[j] = hist[255 - 4 * lane - j];
        const u64 inc = wave_scan_inc(own);
        const u64 hit = __ballot(inc >= target);
        if (lane == (hit ? __ffsll((long long)hit) - 1 : 63)) {
          u64 above = inc - own;
          int j = 0;
          while (j < 3 && above + h[j] < target) above += h[j++];
          s_bin = 255 - 4 * lane - j;
          s_above = above;
        }
      }
      __syncthreads();
      prefix |= (uint32_t)s_bin << shift;
      mask |= 255u << shift;
      target -= s_above;
      __syncthreads();
    }
    // among the tokens with that key, in id order
    u64 base = 0;
    if (tid == 0) s_id = n - 1;
    for (int i0 = 0; i0 < n; i0 += kThreads) {
      const int i = i0 + tid;
      u64 q = 0;
      if (i < n && logit_key(L[i]) == prefix && kept(prefix, i)) q = f(L[i]);
      u64 all;
      const u64 inc = base + block_scan(q, red, &all);
      if (q && inc >= target && inc - q < target) s_id = i;
      base += all;
      if (base >= target) break;
    }
    __syncthreads();
    const Cut c{prefix, s_id + 1};
    __syncthreads();
    return c;
  };

  if (top_k > 0 && top_k < n) cut = select([](float) { return (u64)1; }, (u64)top_k);
  const auto mass = [&](float l) { return fixed(weight(l, mx, t)); };
  const auto sum_kept = [&](bool with_min_p) {
    u64 z = 0, all;
    for (int i = tid; i < n; i += kThreads) {
      const float l = L[i];
      if (!kept(logit_key(l), i)) continue;
      const double w = weight(l, mx, t);
      if (!with_min_p || passes(w)) z += fixed(w);
    }
    block_scan(z, red, &all);
    return all;
  };
  if (top_p < 1.0f) {
    const u64 z = sum_kept(false);
    const double want = ceil((double)z * (top_p > 0.f ? (double)top_p : 0.0));
    cut = select(mass, want < 1.0 ? 1 : want > (double)z ? z : (u64)want);
  }
  const u64 z = sum_kept(true);
  const float u = p.uniform[row];
  const u64 at = min((u64)((double)z * (u > 0.f ? (double)u : 0.0)), z - 1);
  // the first id whose kept cumulative mass exceeds it
  u64 base = 0;
  for (int i0 = 0; i0 < n; i0 += kThreads) {
    const int i = i0 + tid;
    u64 q = 0;
    if (i < n && kept(logit_key(L[i]), i)) {
      const double w = weight(L[i], mx, t);
      if (passes(w)) q = fixed(w);
    }
    u64 all;
    const u64 inc = base + block_scan(q, red, &all);
    if (q && inc > at && inc - q <= at) p.out[row] = i;  // exactly one token
    base += all;
    if (base > at) break;
  }
}

}  // namespace

size_t sample_filtered_workspace_bytes(int rows, int vocab) { return 16; }

int launch_sample_filtered(const SampleParams& p, void* workspace, hipStream_t st) {
  hipLaunchKernelGGL(sample_row_kernel, dim3(p.rows), dim3(kThreads), 0, st, p);
  IE_CHECK_LAUNCH();
  return IE_OK;
}

}  // namespace ie
