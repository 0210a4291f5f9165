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
// Greedy rows (T not > 0, min_p > 1) are top_k = 1.  Weights are computed in fp64 and added in 64-bit
// fixed point within a chunk of the row (exact, free of order), the chunks' sums in fp64 in
// order: a draw next to a border of the distribution falls as it does in 64 bits.  Tokens below
// 2^-46 of the largest (some: 2^-43) round to no unit and weigh nothing.
//
// A row is cut into 8 or 16 chunks, a workgroup each, over three launches:
//   hist    the chunk's max, and its tokens binned by B(l) = floor(8 l / T), which is the same scale
//           in every chunk: counts and masses of the bins from the chunk max's down (relative to the chunk
//           max: nothing of another chunk is needed).  Only what the row's settings need; with top_k only
//           the bins that can hold the chunk's first top_k
//   gather  every workgroup adds up the chunks' histograms and finds the bins that hold the cuts (the
//           same in all of them), then the mass of its tokens in the bins above (kept for certain) and
//           the list of those in the cuts' bins, in id order
//   finish  a workgroup per row: the cuts by a radix select over the listed tokens, the chunks' kept
//           masses, the chunk that holds the draw, its token by a scan in id order
// The bins are 1/8 of a nat wide: of 128256 N(0, 2) logits at T = 1 at most 3200 are listed.  The list
// has room for every token (flatter rows list more and take longer).
//
// What it takes, us by kernel for a row of 128256: top-k 50 hist 5.4, gather 7.8, finish 5.6; top-p 0.9 6.3,
// 10.9, 17.4; min-p 3.1, 5.2, 9.2; no filter 5.4, 3.3, 9.1; for 64 rows 12.9, 12.2, 5.3; 18.0, 19.2, 20.0;
// 5.8, 13.4, 11.3; 14.0, 4.0, 9.7.  One row is bound by the waits of three launches for each other's results
// (a launch that only reads the row's state takes 3-4); 64 rows by the weights' fp64 steps and the histogram's
// LDS additions in the first two launches, and in the last, which one CU a row runs, by the barriers of the
// selects and the weights of the draw's chunk (top-p 0.9, of 45500 cycles: 3300 the row's state, 1800 its lists,
// 16900 the select (4800 the smallest and largest key, 4000 a digit, two of them, 4000 the id), 3700 the chunks' kept
// masses, 1150 the draw's chunk, 16500 the weights of its 16032 logits, 2200 the last 64).
#include "ie_kernels.h"

namespace ie {

namespace {

typedef unsigned long long u64;

constexpr int kThreads = 1024, kWaves = kThreads / 64;
constexpr int kChunks = 16, kBins = 256;    // (at most 16 chunks)
constexpr int kRound = 8;                   // logits a thread and round
constexpr int kGroup = 4;                   // weights a thread computes together
constexpr int kSmall = 64;                  // tokens listed whole, one a lane of the finish
constexpr double kUnit = 4398046511104.0;   // 2^42: masses of listed tokens (2^21 of them: 2^63)
constexpr double kChunkUnit = 35184372088832.0;  // 2^45: of a chunk's tokens (2^18 of them: 2^63)
static_assert(kSampleMaxVocab <= 1 << 21 && kSampleMaxVocab / (kChunks / 2) <= 1 << 18, "sums in 64 bits");

// A row's state in the workspace; the listed tokens follow it, chunk by chunk.
struct Row {
  float pmax[kChunks];
  int n_listed[kChunks];
  u64 total[kChunks];         // rows without top_k: the chunk's mass, relative to its max
  double kept[kChunks];       // mass of the chunk's tokens in bins above the cuts'
  int p_lo, p_hi, k_bin;
  int small;                  // -1, or: every token that can be kept is listed (bins up to this one)
  u64 k_above;                // tokens in the bins above k_bin
  double mass_k, mass_p;      // masses of the bins above k_bin, above p_lo
  unsigned int count[kChunks][kBins];
  u64 mass[kChunks][kBins];
};
struct Listed {
  float l;
  int id;
};

// Chunks a row: 16 while all the chunks' 1024-thread workgroups run at once, two a CU, 8 past that.  Mixed
// settings, us in 8 and in 16 chunks: 16 rows 48.2 and 41.7, 32 rows 49.7 and 48.8, 48 rows 58.4 and 59.5, 64
// rows 61.1 and 68.7.
__host__ __device__ __forceinline__ int row_chunks(int rows) { return rows <= 32 ? kChunks : kChunks / 2; }
__host__ __device__ __forceinline__ int chunk_len(int vocab, int chunks) { return (vocab + chunks - 1) / chunks; }
__host__ __device__ __forceinline__ size_t row_bytes(int vocab) {
  return ((sizeof(Row) + 255) & ~(size_t)255) +
         ((((size_t)vocab + kChunks) * sizeof(Listed) + 255) & ~(size_t)255);
}
__device__ __forceinline__ Row& row_state(void* ws, int row, int vocab) {
  return *reinterpret_cast<Row*>(static_cast<char*>(ws) + row * row_bytes(vocab));
}
__device__ __forceinline__ Listed* row_list(Row& R, int chunk, int len) {
  return reinterpret_cast<Listed*>(reinterpret_cast<char*>(&R) + ((sizeof(Row) + 255) & ~(size_t)255)) +
         (size_t)chunk * len;
}

// A row's settings.
struct Setting {
  double inv_t;
  int top_k;       // 0: off
  float top_p;     // used when p
  float min_p;
  int m_bins;      // no token of a bin past it reaches min_p (used when m)
  int p_bins;      // no bin past it holds top_p's cut (used when p without top_k)
  bool p, m;
};
__device__ __forceinline__ Setting setting(const SampleParams& p, int row) {
  const float t = p.temperature ? p.temperature[row] : 1.0f;
  const int k = p.top_k ? p.top_k[row] : 0;
  const float tp = p.top_p ? p.top_p[row] : 1.0f, mp = p.min_p ? p.min_p[row] : 0.0f;
  const bool greedy = !(t > 0.f) || mp > 1.0f;
  Setting s;
  s.inv_t = 1.0 / (greedy ? 1.0 : (double)t);
  s.top_k = greedy ? 1 : k > 0 && k < p.vocab ? k : 0;
  s.p = !greedy && tp < 1.0f;
  s.top_p = tp > 0.f ? tp : 0.f;
  s.m = !greedy && mp > 0.f;
  s.min_p = mp;
  s.m_bins = s.m ? (int)fminf(-8.0f * __logf(mp), (float)kBins) + 2 : 0;
  // the tokens past d nats below the largest weigh at most vocab exp(-d), which is less than the share
  // left out, (1 - top_p) of at least 1, from here on
  s.p_bins = s.p ? (int)fminf(8.0f * (__logf((float)p.vocab) - __logf(1.0f - s.top_p)), (float)kBins - 3) + 2 : 0;
  return s;
}

// 2^(j / 64), for the weights: held in LDS by each workgroup that computes many.
constexpr double two_to(double x) {  // 0 <= x < 1, by the exponential series
  const double r = x * 0.6931471805599453;
  double y = 1.0;
  for (int k = 24; k > 0; --k) y = 1.0 + y * r / k;
  return y;
}
struct Powers {
  double v[64];
};
constexpr Powers make_powers() {
  Powers t{};
  for (int j = 0; j < 64; ++j) t.v[j] = two_to(j / 64.0);
  return t;
}
__device__ const Powers kPowers = make_powers();

// Weights exp((l - mx) / T) of a row, nothing for tokens past 33 nats below mx (they round to no
// unit), -inf and NaN.  (l - mx) / T = (64 e + j + f) ln 2 / 64 with |f| <= 1/2: 2^e 2^(j/64) times the
// exponential series of f ln 2 / 64 to the fifth power (what is left out is below 4e-17 of it).  Two
// additions of 1.5 x 2^52 round to whole numbers.
struct Weigher {
  const double* powers;  // the table in LDS
  double mx, scale;      // 64 / (T ln 2)
  float fmx;
  __device__ Weigher(const double* t, float m, double inv_t)
      : powers(t), mx(m), scale(inv_t * 92.33248261893583), fmx(m) {}
  __device__ __forceinline__ double operator()(float l) const {
    constexpr double c1 = 0.010830424696249145, c2 = c1 * c1 / 2, c3 = c2 * c1 / 3, c4 = c3 * c1 / 4,
                     c5 = c4 * c1 / 5, whole = 6755399441055744.0;
    const double z = ((double)l - mx) * scale;
    const double t = z + whole, f = z - (t - whole);
    double y = fma(f, c5, c4);
    y = fma(y, f, c3);
    y = fma(y, f, c2);
    y = fma(y, f, c1);
    y = fma(y, f, 1.0);
    const int n = (int)__double_as_longlong(t);
    const u64 w = (u64)__double_as_longlong(y * powers[n & 63]) + ((u64)(uint32_t)(n >> 6) << 52);
    return l == fmx ? 1.0 : z > -33.0 * 92.33248261893583 ? __longlong_as_double((long long)w) : 0.0;
  }
  // The same for N tokens whose weights are only counted in whole units: without a branch, so that their steps
  // overlap (one token at a time took 276 cycles a wave's 64).  What weighs nothing here weighs less than
  // half a unit there.
  template <int N>
  __device__ __forceinline__ void many(const float (&l)[N], double (&w)[N]) const {
    constexpr double c1 = 0.010830424696249145, c2 = c1 * c1 / 2, c3 = c2 * c1 / 3, c4 = c3 * c1 / 4,
                     c5 = c4 * c1 / 5, whole = 6755399441055744.0;
    if (fmx == INFINITY) {
#pragma unroll
      for (int u = 0; u < N; ++u) w[u] = l[u] == fmx ? 1.0 : 0.0;
      return;
    }
#pragma unroll
    for (int u = 0; u < N; ++u) {
      const double z = fmax(((double)l[u] - mx) * scale, -3100.0);  // (33.6 nats, and for NaN)
      const double t = z + whole, f = z - (t - whole);
      const int n = (int)__double_as_longlong(t);
      double y = fma(f, c5, c4);
      y = fma(y, f, c3);
      y = fma(y, f, c2);
      y = fma(y, f, c1);
      y = fma(y, f, 1.0) * powers[n & 63];
      w[u] = __hiloint2double(__double2hiint(y) + ((n & ~63) << 14), __double2loint(y));
    }
  }
};
// w in whole units (2^42 or 2^45) for 0 <= w <= 1.
__device__ __forceinline__ u64 in_units(double w, double unit) {
  return (u64)__double_as_longlong(fma(w, unit, 4503599627370496.0)) & 0xFFFFFFFFFFFFFull;
}

// The token's bin below that of `mx`, kBins for those that weigh nothing (further below, -inf, NaN).
// Non-decreasing in falling l, and the same steps whatever mx: B(l) = floor(l x scale) of the exact product,
// held as the floor of its fp32 rounding plus, where that is a whole number, the floor of what the rounding
// left out (8 l / T passes 24 bits for small T: with the rounded product alone neighbouring logits come to
// lie many bins off); differences below kBins are exact at any size of l.  scale = 8 / T, held finite: below
// that T bins are wider than 1/8 nat, and tokens past kBins only weigh less.
struct Binner {
  float mx, scale, top, top_rest;
  __device__ Binner(float m, double inv_t) : mx(m), scale((float)fmin(8.0 * inv_t, 3.4e38)) { parts(m, top, top_rest); }
  __device__ __forceinline__ void parts(float l, float& whole, float& rest) const {
    const float x = l * scale;
    whole = floorf(x);
    rest = whole == x ? floorf(fmaf(l, scale, -x)) : 0.f;
  }
  __device__ __forceinline__ int operator()(float l) const {
    float whole, rest;
    parts(l, whole, rest);
    const float d = (top - whole) + (top_rest - rest);
    return l == mx ? 0 : l > -INFINITY && d < (float)kBins ? max((int)d, 0) : kBins;
  }
  // No product below it is of a bin up to `needed` (NaN: every one may be).
  __device__ __forceinline__ float least(int needed) const {
    const float b = (top - (float)needed) + top_rest;
    return b - fabsf(b) * 0x1p-22f;  // (its own roundings)
  }
};

// Lane moves within the VALU (the LDS-crossbar shuffles cost over ten times as much): CTRL a DPP control,
// lanes without a source and rows outside ROWS get 0.
template <int CTRL, int ROWS, typename T>
__device__ __forceinline__ T dpp_move(T v) {
  if constexpr (sizeof(T) == 4) {
    return __builtin_bit_cast(
        T, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CTRL, ROWS, 0xF, false));
  } else {
    const u64 x = __builtin_bit_cast(u64, v);
    const uint32_t lo = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)x, CTRL, ROWS, 0xF, false);
    const uint32_t hi = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)(x >> 32), CTRL, ROWS, 0xF, false);
    return __builtin_bit_cast(T, (u64)hi << 32 | lo);
  }
}
// Inclusive scan of each row of 16 lanes (row_shr 1, 2, 4, 8), and of the wave (row_bcast 15, 31).
template <typename T>
__device__ __forceinline__ T row_scan_inc(T v) {
  v += dpp_move<0x111, 0xF>(v);
  v += dpp_move<0x112, 0xF>(v);
  v += dpp_move<0x114, 0xF>(v);
  v += dpp_move<0x118, 0xF>(v);
  return v;
}
template <typename T>
__device__ __forceinline__ T wave_scan_inc(T v) {
  v = row_scan_inc(v);
  v += dpp_move<0x142, 0xA>(v);
  v += dpp_move<0x143, 0xC>(v);
  return v;
}
// The value of one lane (the same lane for the whole wave).
template <typename T>
__device__ __forceinline__ T lane_value(T v, int lane) {
  if constexpr (sizeof(T) == 4) {
    return __builtin_bit_cast(T, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), lane));
  } else {
    const u64 x = __builtin_bit_cast(u64, v);
    const uint32_t lo = __builtin_amdgcn_readlane((int)(uint32_t)x, lane);
    const uint32_t hi = __builtin_amdgcn_readlane((int)(uint32_t)(x >> 32), lane);
    return __builtin_bit_cast(T, (u64)hi << 32 | lo);
  }
}

// Smallest of the wave, on every lane.
__device__ __forceinline__ uint32_t wave_min_u32(uint32_t v) {
  const auto step = [](uint32_t a, uint32_t b) { return a < b ? a : b; };
  v = step(v, __builtin_amdgcn_update_dpp(~0, (int)v, kDppQuadXor1, 0xF, 0xF, false));
  v = step(v, __builtin_amdgcn_update_dpp(~0, (int)v, kDppQuadXor2, 0xF, 0xF, false));
  v = step(v, __builtin_amdgcn_update_dpp(~0, (int)v, kDppRowHalfMirror, 0xF, 0xF, false));
  v = step(v, __builtin_amdgcn_update_dpp(~0, (int)v, kDppRowMirror, 0xF, 0xF, false));
  return step(step(lane_value(v, 0), lane_value(v, 16)), step(lane_value(v, 32), lane_value(v, 48)));
}

// Inclusive scan over the workgroup and its total; `red` is a scratch of kWaves values.
template <typename T>
__device__ __forceinline__ T block_scan(T v, T* red, T* total) {
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const T inc = wave_scan_inc(v);
  __syncthreads();
  if (lane == 63) red[wave] = inc;
  __syncthreads();
  static_assert(kWaves == 16, "a wave a lane of a row");
  const T own = red[lane & 15], upto = row_scan_inc(own);
  *total = lane_value(upto, 15);
  return inc + lane_value(upto - own, wave);
}

template <typename T>
__device__ __forceinline__ T block_sum(T v, T* red) {
  T all;
  block_scan(v, red, &all);
  return all;
}

// Thread t's kRound logits of a round of the ids [i, end): a wave has 64 kRound ids in a row, 64 a load
// (past the end: NaN, which weighs nothing).
__device__ __forceinline__ int round_id(int i, int u) {
  return i + (int)(threadIdx.x >> 6) * (64 * kRound) + u * 64 + (int)(threadIdx.x & 63);
}
__device__ __forceinline__ void load_round(const float* L, int i, int end, float (&v)[kRound]) {
#pragma unroll
  for (int u = 0; u < kRound; ++u) v[u] = L[min(round_id(i, u), end - 1)];
#pragma unroll
  for (int u = 0; u < kRound; ++u)
    if (round_id(i, u) >= end) v[u] = NAN;
}

// First of the wave's 256 bins (4 a lane: inc, own the inclusive scan and the lane's own sum of h) whose
// cumulative value reaches the target, and what lies above it; kBins: none.
template <typename T>
__device__ __forceinline__ int first_bin(T inc, T own, const T (&h)[4], T target, T* above) {
  const u64 hit = __ballot(inc >= target);
  const int at = hit ? __ffsll((long long)hit) - 1 : 63;
  T a = inc - own;
  int j = 0;
  while (j < 3 && a + h[j] < target) a += h[j++];
  const int bin = hit ? 4 * (int)(threadIdx.x & 63) + j : kBins;
  *above = lane_value(a, at);
  return lane_value(bin, at);
}

// (64 VGPRs: two workgroups a CU)
__global__ __launch_bounds__(kThreads, 8) void sample_hist_kernel(SampleParams p, void* ws) {
  // four histograms, by lane: lanes of a wave that meet in a bin wait for each other
  constexpr int kCopies = 4;
  __shared__ unsigned int count[kCopies * kBins];
  __shared__ u64 mass[kCopies * kBins];
  __shared__ double powers[64];
  __shared__ float redf[kWaves];
  __shared__ u64 red[kWaves];
  __shared__ int s_bin;
  const int c = blockIdx.x, row = blockIdx.y, tid = threadIdx.x, lane = tid & 63;
  Row& R = row_state(ws, row, p.vocab);
  const float* L = p.logits + (size_t)row * p.vocab;
  const int cl = chunk_len(p.vocab, p.chunks), beg = min(p.vocab, c * cl), end = min(p.vocab, beg + cl);
  const Setting s = setting(p, row);
  static_assert(kCopies * kBins == kThreads, "a bin a thread");
  count[tid] = 0;
  mass[tid] = 0;
  if (tid < 64) powers[tid] = kPowers.v[tid];
  float v[kRound], own_max = -INFINITY;
  for (int i = beg; i < end; i += kRound * kThreads) {
    load_round(L, i, end, v);
#pragma unroll
    for (int u = 0; u < kRound; ++u) own_max = fmaxf(own_max, v[u]);  // (of a NaN and a number, the number)
  }
  float mx = wave_max(own_max);
  if (lane == 0) redf[tid >> 6] = mx;
  __syncthreads();
  mx = wave_max(redf[lane & (kWaves - 1)]);
  if (tid == 0) R.pmax[c] = mx;
  const Weigher weight(powers, mx, s.inv_t);
  if (!s.top_k && !s.p && s.m) return;
  u64 sum = 0;
  if (mx > -INFINITY) {
    const Binner bin(mx, s.inv_t);
    const int copy = (lane & (kCopies - 1)) * kBins;
    int last = s.p ? s.p_bins : -1;  // bins counted
    if (s.top_k) {
      // as many threads' largest tokens as top_k lie in the bins up to `last`: the chunk's first top_k do
      // too, and the bins behind need no count (they keep those threads' part of it)
      const int b = bin(own_max);
      if (b < kBins) atomicAdd(&count[copy + b], 1u);
      __syncthreads();
      if (tid < 64) {
        unsigned int h[4], own = 0, above;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          h[j] = 0;
#pragma unroll
          for (int k = 0; k < kCopies; ++k) h[j] += count[k * kBins + 4 * lane + j];
          own += h[j];
        }
        const int at = first_bin(wave_scan_inc(own), own, h, (unsigned int)s.top_k, &above);
        if (lane == 0) s_bin = min(at, kBins - 1);
      }
      __syncthreads();
      last = s_bin;
    }
    bool counted = false;  // the thread's largest token, once
    // the last round first: it is still held
    const int rounds = (end - beg + kRound * kThreads - 1) / (kRound * kThreads);
    for (int k = rounds - 1; k >= 0; --k) {
      if (k < rounds - 1) load_round(L, beg + k * kRound * kThreads, end, v);
      if (s.top_k) {
#pragma unroll
        for (int u = 0; u < kRound; ++u) {
          const int b = bin(v[u]);
          if (b > last) continue;
          const bool again = !counted && v[u] == own_max;
          counted |= again;
          if (!again) atomicAdd(&count[copy + b], 1u);
          if (s.p) atomicAdd(&mass[copy + b], in_units(weight(v[u]), kChunkUnit));
        }
      } else {
#pragma unroll
        for (int u0 = 0; u0 < kRound; u0 += kGroup) {
          float l[kGroup];
          double w[kGroup];
#pragma unroll
          for (int u = 0; u < kGroup; ++u) l[u] = v[u0 + u];
          weight.many(l, w);
#pragma unroll
          for (int u = 0; u < kGroup; ++u) {
            const u64 q = in_units(w[u], kChunkUnit);
            sum += q;
            if (s.p) {
              const int b = bin(l[u]);
              if (b <= last) atomicAdd(&mass[copy + b], q);
            }
          }
        }
      }
    }
  }
  if (!s.top_k) {
    sum = block_sum(sum, red);
    if (tid == 0) R.total[c] = sum;
    if (!s.p) return;
  }
  __syncthreads();
  if (tid < kBins) {
    if (s.top_k)
      R.count[c][tid] = (count[tid] + count[tid + kBins]) + (count[tid + 2 * kBins] + count[tid + 3 * kBins]);
  } else if (tid < 2 * kBins && s.p) {
    const int b = tid - kBins;
    R.mass[c][b] = (mass[b] + mass[b + kBins]) + (mass[b + 2 * kBins] + mass[b + 3 * kBins]);
  }
}

__device__ __forceinline__ float row_max(const Row& R, int chunks) {
  const int lane = threadIdx.x & 63;
  return wave_max(lane < chunks ? R.pmax[lane] : -INFINITY);
}

// The bins that hold the cuts: tokens of bins < lo are kept, those of k_bin and of p_lo .. p_hi are
// undecided, the others dropped.  (-1 .. -2: no such cut)
struct CutBins {
  int lo, p_lo, p_hi, k_bin;
};

__global__ __launch_bounds__(kThreads, 8) void sample_gather_kernel(SampleParams p, void* ws) {
  __shared__ u64 red[kWaves];
  __shared__ double redd[kWaves];
  __shared__ u64 part_c[4][kBins];
  __shared__ double part_m[4][kBins];
  __shared__ double powers[64];
  __shared__ CutBins s_cut;
  __shared__ bool s_small;
  __shared__ int s_cnt[kWaves];
  const int c = blockIdx.x, row = blockIdx.y, tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  Row& R = row_state(ws, row, p.vocab);
  const float* L = p.logits + (size_t)row * p.vocab;
  const int cl = chunk_len(p.vocab, p.chunks), beg = min(p.vocab, c * cl), end = min(p.vocab, beg + cl);
  const Setting s = setting(p, row);
  if (tid < 64) powers[tid] = kPowers.v[tid];
  const float mx = row_max(R, p.chunks);
  if (!(mx > -INFINITY)) return;  // nothing to choose from
  const Binner bin(mx, s.inv_t);
  const Weigher weight(powers, mx, s.inv_t);
  __syncthreads();
  const bool cuts = s.top_k || s.p;
  CutBins cut{kBins, -1, -2, -1};
  // the row's histogram: thread (bin, quarter of the chunks), then the quarters in order
  const int b = tid & (kBins - 1), q = tid / kBins;
  bool small = false;
  if (s.top_k) {
    u64 count = 0;
    for (int j = 0; j < p.chunks / 4; ++j) {
      const int ch = q * (p.chunks / 4) + j;
      const int from = b - bin(R.pmax[ch]);  // (bin(-inf) = kBins: none)
      if (from >= 0) count += R.count[ch][from];
    }
    part_c[q][b] = count;
    __syncthreads();
    if (wave == 0) {  // lane l: bins 4 l .. 4 l + 3
      u64 n[4], nsum = 0, above;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int b4 = 4 * lane + j;
        nsum += n[j] = (part_c[0][b4] + part_c[1][b4]) + (part_c[2][b4] + part_c[3][b4]);
      }
      const u64 ninc = wave_scan_inc(nsum);
      const int k_bin = first_bin(ninc, nsum, n, (u64)s.top_k, &above);
      u64 upto = ninc - nsum;  // tokens up to and with that bin, in its lane
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (4 * lane + j <= k_bin) upto += n[j];
      upto = lane_value(upto, min(k_bin >> 2, 63));
      if (lane == 0) {
        // (kBins: the first top_k reach past every token that weighs anything)
        s_cut.k_bin = k_bin < kBins ? k_bin : -1;
        s_small = upto <= kSmall;
        if (c == 0) R.k_above = above, R.small = upto <= kSmall ? (int)min(k_bin, kBins - 1) : -1;
      }
    }
    __syncthreads();
    cut.k_bin = s_cut.k_bin;
    small = s_small;
    // a row whose first tokens are few has them all listed: nothing else of it is needed
    if (small) cut = CutBins{0, 0, cut.k_bin < 0 ? kBins - 1 : cut.k_bin, cut.k_bin};
    else if (cut.k_bin >= 0) cut.lo = cut.k_bin;
  } else if (c == 0 && tid == 0) {
    R.small = -1;
  }
  if (s.p && !small) {
    double mass = 0.0;
    for (int j = 0; j < p.chunks / 4; ++j) {
      const int ch = q * (p.chunks / 4) + j;
      const float cm = R.pmax[ch];
      const int from = b - bin(cm);
      if (from >= 0) mass += (double)R.mass[ch][from] * weight(cm);
    }
    part_m[q][b] = mass;
    __syncthreads();
    if (wave == 0) {
      double m[4], msum = 0.0;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int b4 = 4 * lane + j;
        msum += m[j] = ((part_m[0][b4] + part_m[1][b4]) + (part_m[2][b4] + part_m[3][b4])) * (1.0 / kChunkUnit);
      }
      const double minc = wave_scan_inc(msum);
      double mass_k = lane_value(minc, 63);
      if (!s.top_k) {  // (bins past those that can hold the cut are not summed)
        const float cm = lane < p.chunks ? R.pmax[lane] : -INFINITY;
        const double own = cm > -INFINITY ? (double)R.total[lane] * weight(cm) * (1.0 / kChunkUnit) : 0.0;
        mass_k = fmax(mass_k, lane_value(wave_scan_inc(own), 63));
      }
      double mass_k_incl = mass_k, mass_p = 0.0, none;
      if (cut.k_bin >= 0) {
        // masses up to that bin, without it and with it
        double below = minc - msum, own = 0.0;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          if (4 * lane + j < cut.k_bin) below += m[j];
          if (4 * lane + j == cut.k_bin) own = m[j];
        }
        mass_k = lane_value(below, cut.k_bin >> 2);
        mass_k_incl = mass_k + lane_value(own, cut.k_bin >> 2);
      }
      // Z lies between the masses without and with k_bin (which part of it is kept is not known yet)
      const double tiny = 1.0 / kUnit, last = lane_value(minc, 63);
      const int p_lo = first_bin(minc, msum, m, fmin(fmax(mass_k * s.top_p * (1.0 - 1e-12), tiny), last), &mass_p);
      const int p_hi = first_bin(minc, msum, m, fmin(fmax(mass_k_incl * s.top_p * (1.0 + 1e-12), tiny), last), &none);
      if (lane == 0) {
        s_cut.p_hi = min(p_hi, cut.k_bin >= 0 ? cut.k_bin : kBins - 1);
        s_cut.p_lo = min(p_lo, s_cut.p_hi);
        if (c == 0) R.mass_k = mass_k, R.mass_p = mass_p;
      }
    }
    __syncthreads();
    cut.lo = cut.p_lo = s_cut.p_lo;
    cut.p_hi = s_cut.p_hi;
  }
  if (c == 0 && tid == 0) R.p_lo = cut.p_lo, R.p_hi = cut.p_hi, R.k_bin = cut.k_bin;
  // The chunk's certain mass: from the histogram (or the total) where there is one and no min-p, else
  // token by token
  const bool summed = !s.m && !small && (s.p || !cuts);
  double low = 0.0;
  if (summed) {
    const float cm = R.pmax[c];
    // (a chunk whose largest token rounds to no unit has none that a draw could find)
    const double top = cm > -INFINITY ? weight(cm) : 0.0;
    const double scale = in_units(top, kChunkUnit) ? top * (1.0 / kChunkUnit) : 0.0;
    if (scale > 0.0) {
      if (!cuts) {
        low = (double)R.total[c] * scale;
      } else {
        const int from = tid - bin(cm);
        if (tid < cut.lo && from >= 0) low = (double)R.mass[c][from] * scale;  // (lo <= kBins)
        low = block_sum(low, redd);
      }
    } else if (cuts) {
      block_sum(low, redd);
    }
    if (!cuts) {
      if (tid == 0) R.kept[c] = low, R.n_listed[c] = 0;
      return;
    }
  }
  Listed* list = row_list(R, c, cl);
  const int sum_bins = summed ? 0 : s.m ? min(cut.lo, s.m_bins) : cut.lo;  // bins summed token by token
  // no bin past `needed` matters
  const int needed = max(max(sum_bins - 1, cut.k_bin), cut.p_hi);
  const float least = bin.least(needed);
  u64 sum = 0;
  int listed = 0;
  // (beg and end are the workgroup's: every thread runs every round and its barriers)
  for (int i = beg; i < end; i += kRound * kThreads) {
    float v[kRound];
    load_round(L, i, end, v);
    unsigned int hits = 0;
    int before = 0, place[kRound];
#pragma unroll
    for (int u = 0; u < kRound; ++u) {
      place[u] = 0;
      // (most rows need few tokens: one product and comparison for the others)
      if (!__ballot(!(v[u] * bin.scale < least))) continue;
      const int b = bin(v[u]);
      if (b < sum_bins && b < kBins) {
        const double w = weight(v[u]);
        if (!s.m || w >= (double)s.min_p) sum += in_units(w, kChunkUnit);
      }
      const bool hit = b >= cut.lo && b < kBins && (b == cut.k_bin || (b >= cut.p_lo && b <= cut.p_hi));
      const u64 vote = __ballot(hit);
      place[u] = before + __popcll(vote & ((1ull << lane) - 1));
      before += __popcll(vote);
      hits |= (unsigned int)hit << u;
    }
    if (!cuts) continue;
    // places in id order: wave after wave
    if (lane == 0) s_cnt[wave] = before;
    __syncthreads();
    const int own = s_cnt[lane & (kWaves - 1)], upto = row_scan_inc(own);
    const int at = listed + lane_value(upto - own, wave);
    listed += lane_value(upto, kWaves - 1);
    __syncthreads();
#pragma unroll
    for (int u = 0; u < kRound; ++u)
      if (hits >> u & 1) list[at + place[u]] = Listed{v[u], round_id(i, u)};
  }
  if (!summed) low = (double)block_sum(sum, red) * (1.0 / kChunkUnit);
  if (tid == 0) {
    R.kept[c] = low;
    R.n_listed[c] = listed;
  }
}

// A cut of the order: tokens with l > l, and those with l == l and id < id, are kept.
struct Cut {
  float l;
  int id;
  __device__ __forceinline__ bool keeps(float x, int i) const { return x > l || (x == l && i < id); }
};

// Order-preserving key of a logit (no NaN here), -0 as +0.
__device__ __forceinline__ uint32_t logit_key(float v) {
  if (v == 0.f) v = 0.f;
  const uint32_t u = __float_as_uint(v);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float key_logit(uint32_t k) {
  return __uint_as_float(k & 0x80000000u ? k ^ 0x80000000u : ~k);
}

constexpr int kDigits = 2048;
constexpr int kHeld = 4;          // listed tokens a thread holds
constexpr int kScan = 16;         // logits a thread and round of the last scan

// Memory accesses of a wave's lanes keep their order across it.
__device__ __forceinline__ void wave_fence() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// A row whose tokens are all listed, at most one a lane: one wave, no barrier.
__device__ __forceinline__ int finish_small(const SampleParams& p, const Setting& s, Row& R, int own_n, double uniform,
                                            int cl, const Weigher& weight, u64* by_rank) {
  const int lane = threadIdx.x & 63;
  const int upto = wave_scan_inc(own_n);
  const int n = lane_value(upto, 63);
  int c = 0, before = 0;
  for (int k = 0; k < p.chunks - 1; ++k) {
    const int end = lane_value(upto, k);
    if (lane >= end) c = k + 1, before = end;
  }
  Listed t{-INFINITY, -1};
  if (lane < n) t = row_list(R, c, cl)[lane - before];
  // places in the order (the list is in id order)
  int rank = 0;
  for (int j = 0; j < n; ++j) {
    const float l = lane_value(t.l, j);
    rank += l > t.l || (l == t.l && j < lane);
  }
  const double w = weight(t.l);
  const bool in_k = lane < n && (!s.top_k || rank < s.top_k);
  u64 q = in_k ? in_units(w, kUnit) : 0;
  bool keep = in_k && (!s.m || w >= (double)s.min_p);
  if (s.p) {
    // the masses in the order: those before a token short of the share of them all
    // (one wave: the hardware does its LDS accesses in order; the fences hold the compiler to it)
    by_rank[lane] = 0;
    wave_fence();
    if (lane < n) by_rank[rank] = q;
    wave_fence();
    const u64 sorted = by_rank[lane], inc = wave_scan_inc(sorted), z = lane_value(inc, 63);
    wave_fence();
    by_rank[lane] = inc - sorted;
    wave_fence();
    const double share = ceil((double)z * (double)s.top_p);
    const u64 want = share < 1.0 ? 1 : share > (double)z ? z : (u64)share;
    keep = keep && by_rank[min(rank, 63)] < want;
  }
  keep = keep || (lane < n && rank == 0);
  if (!keep) q = 0;
  const u64 inc = wave_scan_inc(q), z = lane_value(inc, 63);
  const double x = (double)z * fmax(uniform, 0.0);  // (a NaN too: 0)
  const u64 at = x < (double)z ? min((u64)x, z - 1) : z - 1;
  return lane_value(t.id, __ffsll((long long)__ballot(inc > at)) - 1);
}

__global__ __launch_bounds__(kThreads) void sample_finish_kernel(SampleParams p, void* ws) {
  __shared__ u64 hist[kDigits];
  __shared__ u64 red[kWaves];
  __shared__ u64 listed_of[kChunks];
  __shared__ double powers[64];
  __shared__ int offset[kChunks + 1];
  __shared__ uint32_t s_min, s_max;
  __shared__ int s_digit, s_id;
  __shared__ u64 s_above, s_at;
  const int row = blockIdx.x, tid = threadIdx.x, lane = tid & 63;
  Row& R = row_state(ws, row, p.vocab);
  const float* L = p.logits + (size_t)row * p.vocab;
  // (what the row's state holds in one go: a load after the other is a wait each)
  const int own_listed = lane < p.chunks ? R.n_listed[lane] : 0;
  const double own_kept = lane < p.chunks ? R.kept[lane] : 0.0;
  const double u_row = p.uniform[row];
  const int small = R.small, p_lo = R.p_lo, p_hi = R.p_hi, k_bin = R.k_bin;
  const Setting s = setting(p, row);
  const float mx = row_max(R, p.chunks);
  if (!(mx > -INFINITY)) {
    if (tid == 0) p.out[row] = -1;
    return;
  }
  if (tid < 64) powers[tid] = kPowers.v[tid];
  const Binner bin(mx, s.inv_t);
  const Weigher weight(powers, mx, s.inv_t);
  const int cl = chunk_len(p.vocab, p.chunks);
  if (small >= 0) {
    if (tid >= 64) return;
    const int token = finish_small(p, s, R, own_listed, u_row, cl, weight, hist);
    if (tid == 0) p.out[row] = token;
    return;
  }
  if (tid < 64) {
    const int inc = wave_scan_inc(own_listed);
    if (tid < kChunks) {
      offset[tid + 1] = inc;
      listed_of[tid] = 0;
    }
    if (tid == 0) offset[0] = 0;
  }
  __syncthreads();
  const int n = offset[kChunks];
  const auto chunk_of = [&](int j) {
    int c = 0;
#pragma unroll
    for (int k = 1; k < kChunks; ++k) c += j >= offset[k];
    return c;
  };
  // The listed tokens in rounds of kHeld a thread, in id order slab by slab; most rows have one round, whose
  // tokens stay in registers.  (past the end: bin kBins)
  Listed held[kHeld];
  const auto load_held = [&](int j0) {
#pragma unroll
    for (int u = 0; u < kHeld; ++u) {
      const int j = j0 + u * kThreads + tid, c = chunk_of(j);
      held[u] = j < n ? row_list(R, c, cl)[j - offset[c]] : Listed{-INFINITY, -1};
    }
  };
  const bool one_round = n <= kHeld * kThreads;
  if (one_round) load_held(0);

  // The cut where the sum of f over the listed tokens (0: not among them; some are), in the order, reaches
  // target >= 1 (never: all of them stay): a radix select of the key from the first bits in which they differ, then,
  // among equal keys (equal f), the id of the last one needed.
  const auto select = [&](auto f, u64 target) {
    if (tid == 0) s_min = 0xFFFFFFFFu, s_max = 0;
    __syncthreads();
    uint32_t key[kHeld], kmin = 0xFFFFFFFFu, kmax = 0;
    u64 q[kHeld];
    const auto weigh = [&]() {
#pragma unroll
      for (int u = 0; u < kHeld; ++u) key[u] = logit_key(held[u].l), q[u] = f(held[u]);
    };
    for (int j0 = 0; j0 < n; j0 += kHeld * kThreads) {
      if (!one_round) load_held(j0);
      weigh();
#pragma unroll
      for (int u = 0; u < kHeld; ++u)
        if (q[u]) kmin = min(kmin, key[u]), kmax = max(kmax, key[u]);
    }
    // (a wave's first: 1024 additions to one place wait for each other, 16000 cycles)
    kmin = wave_min_u32(kmin), kmax = ~wave_min_u32(~kmax);
    if (lane == 0 && kmin <= kmax) atomicMin(&s_min, kmin), atomicMax(&s_max, kmax);
    __syncthreads();
    uint32_t base = s_min, span = s_max - s_min;  // keys base .. base + span are left
    while (span) {
      const int shift = max(0, 32 - __clz(span) - 11);
      hist[tid] = 0, hist[tid + kThreads] = 0;
      __syncthreads();
      for (int j0 = 0; j0 < n; j0 += kHeld * kThreads) {
        if (!one_round) load_held(j0), weigh();
#pragma unroll
        for (int u = 0; u < kHeld; ++u) {
          if (j0 + u * kThreads >= n) break;  // (the workgroup's)
          bool left = q[u] && key[u] - base <= span;
          // logits that were 16-bit numbers have few values: equal ones are added together while a wave has
          // several (64 additions to one place wait for each other)
          for (u64 todo = __ballot(left); todo; todo = __ballot(left)) {
            const int first = __ffsll((long long)todo) - 1;
            const uint32_t k = lane_value(key[u], first);
            const u64 same = __ballot(left && key[u] == k);
            if (__popcll(same) < 4) {
              if (left) atomicAdd(&hist[(key[u] - base) >> shift], q[u]);
              break;
            }
            if (lane == first) atomicAdd(&hist[(k - base) >> shift], q[u] * (u64)__popcll(same));
            left = left && key[u] != k;
          }
        }
      }
      __syncthreads();
      // digits from the largest: thread t has kDigits - 1 - 2 t and the one below
      static_assert(kDigits == 2 * kThreads, "two digits a thread");
      const u64 h0 = hist[kDigits - 1 - 2 * tid], h1 = hist[kDigits - 2 - 2 * tid];
      u64 all;
      const u64 inc = block_scan(h0 + h1, red, &all);
      if (target > all) target = all;
      if (inc >= target && inc - (h0 + h1) < target) {  // exactly one thread
        const bool first = inc - h1 >= target;
        s_digit = kDigits - (first ? 1 : 2) - 2 * tid;
        s_above = inc - h1 - (first ? h0 : 0);
      }
      __syncthreads();
      base += (uint32_t)s_digit << shift;
      target -= s_above;
      span = min((1u << shift) - 1, span - ((uint32_t)s_digit << shift));
      __syncthreads();
    }
    // the tokens with that key, in id order
    if (tid == 0) s_id = 0x7FFFFFFE;
    u64 before = 0;
    for (int j0 = 0; j0 < n && before < target; j0 += kHeld * kThreads) {
      if (!one_round) load_held(j0), weigh();
#pragma unroll
      for (int u = 0; u < kHeld; ++u) {
        if (j0 + u * kThreads >= n) break;  // (the workgroup's)
        const u64 own = key[u] == base ? q[u] : 0;
        u64 all;
        const u64 inc = before + block_scan(own, red, &all);
        if (own && inc >= target && inc - own < target) s_id = held[u].id;
        before += all;
      }
    }
    __syncthreads();
    const Cut c{key_logit(base), s_id + 1};
    __syncthreads();
    return c;
  };
  const auto mass = [&](float l) { return in_units(weight(l), kUnit); };

  Cut k_cut{-INFINITY, 0x7FFFFFFF}, cut = k_cut;
  if (k_bin >= 0) {
    k_cut = select([&](const Listed& t) { return (u64)(bin(t.l) == k_bin); }, (u64)s.top_k - R.k_above);
    cut = k_cut;
  }
  if (s.p) {
    double z = R.mass_k;  // of the bins above k_bin (of all: no such cut)
    if (k_bin >= 0) {
      u64 in_bin = 0;
      for (int j0 = 0; j0 < n; j0 += kHeld * kThreads) {
        if (!one_round) load_held(j0);
#pragma unroll
        for (int u = 0; u < kHeld; ++u)
          if (bin(held[u].l) == k_bin && k_cut.keeps(held[u].l, held[u].id)) in_bin += mass(held[u].l);
      }
      z += (double)block_sum(in_bin, red) * (1.0 / kUnit);
    }
    const double want = ceil((z * (double)s.top_p - R.mass_p) * kUnit);
    // (a token that rounds to no unit counts one here: a bin of such tokens holds its cut as any other)
    cut = select([&](const Listed& t) -> u64 {
                   const int b = bin(t.l);
                   return b >= p_lo && b <= p_hi && k_cut.keeps(t.l, t.id) ? max(mass(t.l), (u64)1) : 0;
                 },
                 want > 1.0 ? (u64)want : (u64)1);
  }
  // (what is kept lies at or above the cut, the bins above it with it; a cut keeps all that weighs
  // something where there is none)
  const auto kept_mass = [&](float l, int id, double unit) -> u64 {
    if (!cut.keeps(l, id)) return 0;
    const double w = weight(l);
    return !s.m || w >= (double)s.min_p ? in_units(w, unit) : 0;
  };
  // the chunks' kept masses
  for (int j0 = 0; j0 < n; j0 += kHeld * kThreads) {
    if (!one_round) load_held(j0);
#pragma unroll
    for (int u = 0; u < kHeld; ++u) {
      if (j0 + u * kThreads >= n) break;  // (the workgroup's)
      const u64 q = held[u].id >= 0 ? kept_mass(held[u].l, held[u].id, kUnit) : 0;
      if (!__ballot(q != 0)) continue;
      // (the list goes chunk by chunk, so a wave has one or two; 64 additions to one place wait for each other)
      const int own = chunk_of(min(j0 + u * kThreads + tid, n - 1)), to = lane_value(own, 63);
      for (int c = lane_value(own, 0); c <= to; ++c) {
        const u64 all = lane_value(wave_scan_inc(own == c ? q : 0), 63);
        if (lane == 0) atomicAdd(&listed_of[c], all);
      }
    }
  }
  __syncthreads();
  if (tid < 64) {
    const double own =
        tid < p.chunks ? own_kept + (double)listed_of[tid] * (1.0 / kUnit) : 0.0;
    // added one after the other: sums that never fall, which a scan's, rounded in another order a lane,
    // may do
    double z = 0.0, before = 0.0;
    for (int k = 0; k < p.chunks; ++k) {
      if (tid == k) before = z;
      z += lane_value(own, k);
    }
    const double u = u_row, x = z * fmax(u, 0.0);  // (a NaN too: 0)
    // (u >= 1, or a product rounded up: the last chunk that keeps anything)
    const u64 some = __ballot(own > 0.0), more = __ballot(before + own > x) & some;
    const int c = more ? __ffsll((long long)more) - 1 : some ? 63 - __clzll((long long)some) : 0;
    // (a chunk's sum reaches 2^63; u >= 1: past all of its tokens, wherever the sums were rounded)
    const u64 draw = u >= 1.0 ? ~0ull : (u64)fmin(fmax(x - before, 0.0) * kChunkUnit, 1.8e19);
    if (tid == c) s_digit = c, s_at = draw, s_id = -1;
  }
  __syncthreads();
  // the chunk's first id whose kept cumulative mass exceeds the draw (its last kept id where the sums'
  // roundings, or a uniform past 1, leave none): first the 1024 ids that hold it, a wave's of the
  // round, then the 64 of those, a wave each
  const u64 at = s_at;
  const int beg = s_digit * cl, end = min(p.vocab, beg + cl);
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  // from a value a wave: what lies before this wave's, and whether it holds `at`; adds all to `before`
  const auto place = [&](u64 own, u64& before) {
    __syncthreads();
    if (lane == 0) red[wave] = own;
    __syncthreads();
    const u64 mine = red[lane & (kWaves - 1)], inc = row_scan_inc(mine);
    const u64 upto = before + lane_value(inc - mine, wave);
    before += lane_value(inc, kWaves - 1);
    return upto;
  };
  const bool dense = !s.m && cut.l == -INFINITY;  // (nothing is dropped)
  u64 before = 0;
  int last = -1;
  if (tid == 0) s_min = 0xFFFFFFFFu;
  for (int i = beg; i < end && before <= at; i += kScan * kThreads) {
    const int id0 = i + wave * (64 * kScan) + lane;  // 64 a load
    float v[kScan];
    u64 own = 0;
#pragma unroll
    for (int u = 0; u < kScan; ++u) v[u] = L[min(id0 + u * 64, end - 1)];
    if (dense) {
#pragma unroll
      for (int u0 = 0; u0 < kScan; u0 += kGroup) {
        float l[kGroup];
        double w[kGroup];
#pragma unroll
        for (int u = 0; u < kGroup; ++u) l[u] = v[u0 + u];
        weight.many(l, w);
#pragma unroll
        for (int u = 0; u < kGroup; ++u) {
          const int id = id0 + (u0 + u) * 64;
          const u64 q = id < end ? in_units(w[u], kChunkUnit) : 0;
          own += q;
          if (q) last = id;
        }
      }
    } else {
#pragma unroll
      for (int u = 0; u < kScan; ++u) {
        const int id = id0 + u * 64;
        if (!__ballot(v[u] >= cut.l)) continue;
        const u64 q = id < end ? kept_mass(v[u], id, kChunkUnit) : 0;
        own += q;
        if (q) last = id;
      }
    }
    own = lane_value(wave_scan_inc(own), 63);
    const u64 upto = place(own, before);
    if (lane == 0 && upto <= at && at < upto + own) s_min = (uint32_t)(id0), s_above = upto;
  }
  __syncthreads();
  if (before > at) {  // (uniform)
    static_assert(kScan == kWaves, "64 ids a wave");
    const int id = (int)s_min + wave * 64 + lane;
    const float v = L[min(id, end - 1)];
    const u64 q = id < end ? kept_mass(v, id, kChunkUnit) : 0, inc = wave_scan_inc(q);
    u64 from = s_above;
    const u64 upto = place(lane_value(inc, 63), from);
    if (upto + inc - q <= at && at < upto + inc) p.out[row] = id;  // one token
  }
  if (before <= at) {  // (uniform)
    if (last >= 0) atomicMax(&s_id, last);
    __syncthreads();
    if (tid == 0) p.out[row] = s_id;
  }
}

}  // namespace

size_t sample_filtered_workspace_bytes(int rows, int vocab) { return rows * row_bytes(vocab); }

int launch_sample_filtered(SampleParams p, void* ws, hipStream_t st) {
  p.chunks = row_chunks(p.rows);
  const dim3 chunks(p.chunks, p.rows);
  hipLaunchKernelGGL(sample_hist_kernel, chunks, dim3(kThreads), 0, st, p, ws);
  hipLaunchKernelGGL(sample_gather_kernel, chunks, dim3(kThreads), 0, st, p, ws);
  hipLaunchKernelGGL(sample_finish_kernel, dim3(p.rows), dim3(kThreads), 0, st, p, ws);
  IE_CHECK_LAUNCH();
  return IE_OK;
}

}  // namespace ie
