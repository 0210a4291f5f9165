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
// fixed point: sums are exact and free of order, and a draw next to a border of the distribution
// falls as it does in 64 bits.  Kept masses are in 2^-42 units, so that the tokens below exp(-30)
// of the largest weigh nothing.
//
// A row is cut into kChunks chunks, a workgroup each, over three launches:
//   hist    the chunk's max, and its tokens binned by B(l) = floor(8 l / T), which is the same scale
//           in every chunk: counts and masses of the bins from the chunk max's down (relative to the chunk
//           max: nothing of another chunk is needed).  Only what the row's settings need.
//   gather  every workgroup adds up the chunks' histograms and finds the bins that hold the cuts (the
//           same in all of them), then sums the mass of its tokens in the bins above (kept for
//           certain) and lists those in the cuts' bins, in id order
//   finish  a workgroup per row: the cuts by a radix select over the listed tokens, the chunks' kept
//           masses, the chunk that holds the draw, its token by a scan in id order
// The bins are 1/8 of a nat wide: of 128256 N(0, 2) logits at T = 1 at most 3200 are listed.  The list
// has room for every token (flatter rows list more and take longer).
#include "ie_kernels.h"

namespace ie {

namespace {

typedef unsigned long long u64;

constexpr int kThreads = 1024, kWaves = kThreads / 64;
constexpr int kChunks = 16, kBins = 256;
constexpr int kRound = 8;                   // logits a thread and round
constexpr double kUnit = 4398046511104.0;   // 2^42: sums over kSampleMaxVocab = 2^21 tokens fit 63 bits
constexpr double kBinUnit = 70368744177664.0;  // 2^46: a chunk's sums (2^17 tokens) fit 63 bits
static_assert(kSampleMaxVocab / kChunks <= 1 << 17, "a bin's mass in 64 bits");

// A row's state in the workspace; the listed tokens follow it, chunk by chunk.
struct Row {
  float pmax[kChunks];
  int n_listed[kChunks];
  u64 kept[kChunks];          // mass of the chunk's tokens in bins above the cuts'
  int cut_bins[4];            // lo, p_lo, p_hi, k_bin
  u64 k_above;                // tokens in the bins above k_bin
  double mass_k, mass_p;      // masses of the bins above k_bin, above p_lo
  unsigned int count[kChunks][kBins];
  u64 mass[kChunks][kBins];
};
struct Listed {
  float l;
  int id;
};

__host__ __device__ __forceinline__ int chunk_len(int vocab) { return (vocab + kChunks - 1) / kChunks; }
__host__ __device__ __forceinline__ size_t row_bytes(int vocab) {
  return ((sizeof(Row) + 255) & ~(size_t)255) +
         (((size_t)chunk_len(vocab) * kChunks * sizeof(Listed) + 255) & ~(size_t)255);
}
__device__ __forceinline__ Row& row_state(void* ws, int row, int vocab) {
  return *reinterpret_cast<Row*>(static_cast<char*>(ws) + row * row_bytes(vocab));
}
__device__ __forceinline__ Listed* row_list(Row& R, int chunk, int vocab) {
  return reinterpret_cast<Listed*>(reinterpret_cast<char*>(&R) + ((sizeof(Row) + 255) & ~(size_t)255)) +
         (size_t)chunk * chunk_len(vocab);
}

// A row's settings.
struct Setting {
  double inv_t;
  int top_k;       // 0: off
  float top_p;     // used when p
  float min_p;
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
  return s;
}

// e^x for x <= 0, in 64 bits: 2^n e^r with |r| <= ln 2 / 2 and the exponential series to r^11 / 11!
// (what is left out is below 7e-15 of it).
__device__ __forceinline__ double exp_neg(double x) {
  const double n = rint(x * 1.4426950408889634);
  const double r = fma(n, -0.6931471805599453, x);
  double y = 1.0 / 39916800.0;
  y = fma(y, r, 1.0 / 3628800.0);
  y = fma(y, r, 1.0 / 362880.0);
  y = fma(y, r, 1.0 / 40320.0);
  y = fma(y, r, 1.0 / 5040.0);
  y = fma(y, r, 1.0 / 720.0);
  y = fma(y, r, 1.0 / 120.0);
  y = fma(y, r, 1.0 / 24.0);
  y = fma(y, r, 1.0 / 6.0);
  y = fma(y, r, 0.5);
  y = fma(y, r, 1.0);
  y = fma(y, r, 1.0);
  return ldexp(y, (int)n);
}

// Weight of a token: nothing past 33 nats below the max (it rounds to no unit), -inf, NaN.
__device__ __forceinline__ double weight(float l, float mx, double inv_t) {
  if (l == mx) return 1.0;  // (infinite maxima too)
  const double x = ((double)l - (double)mx) * inv_t;
  return x > -33.0 ? exp_neg(x) : 0.0;
}
__device__ __forceinline__ u64 fixed(double w) { return (u64)(w * kUnit + 0.5); }

// The token's bin below that of `mx`, kBins for those that weigh nothing (further below, -inf, NaN).
// Non-decreasing in falling l, and the same steps whatever mx: B(l) = floor(l x scale) in fp32, whose
// rounding is monotone, and whose differences below kBins are exact at any size of l.  scale = 8 / T,
// held finite: below that T bins are wider than 1/8 nat, and tokens past kBins only weigh less.
struct Binner {
  float mx, scale, top;
  __device__ Binner(float m, double inv_t)
      : mx(m), scale((float)fmin(8.0 * inv_t, 3.4e38)), top(floorf(m * scale)) {}
  __device__ __forceinline__ int operator()(float l) const {
    const float d = top - floorf(l * scale);
    return l == mx ? 0 : l > -INFINITY && d < (float)kBins ? max((int)d, 0) : kBins;
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

__device__ __forceinline__ u64 block_sum(u64 v, u64* red) {
  u64 all;
  block_scan(v, red, &all);
  return all;
}

// kRound logits of [i, end) a thread, kThreads apart (past the end: NaN, which weighs nothing).
__device__ __forceinline__ void load_round(const float* L, int i, int end, float (&v)[kRound]) {
#pragma unroll
  for (int u = 0; u < kRound; ++u) v[u] = L[min(i + u * kThreads, end - 1)];
#pragma unroll
  for (int u = 0; u < kRound; ++u)
    if (i + u * kThreads >= end) v[u] = NAN;
}

__global__ __launch_bounds__(kThreads) void sample_hist_kernel(SampleParams p, void* ws) {
  // four histograms, by lane: lanes of a wave that meet in a bin wait for each other
  constexpr int kCopies = 4;
  __shared__ unsigned int count[kCopies * kBins];
  __shared__ u64 mass[kCopies * kBins];
  __shared__ float red[kWaves];
  const int c = blockIdx.x, row = blockIdx.y, tid = threadIdx.x, lane = tid & 63;
  Row& R = row_state(ws, row, p.vocab);
  const float* L = p.logits + (size_t)row * p.vocab;
  const int cl = chunk_len(p.vocab), beg = min(p.vocab, c * cl), end = min(p.vocab, beg + cl);
  const Setting s = setting(p, row);
  static_assert(kCopies * kBins == kThreads, "a bin a thread");
  count[tid] = 0;
  mass[tid] = 0;
  float v[kRound], mx = -INFINITY;
  for (int i = beg; i < end; i += kRound * kThreads) {
    load_round(L, i + tid, end, v);
#pragma unroll
    for (int u = 0; u < kRound; ++u) mx = fmaxf(mx, v[u]);  // (of a NaN and a number, the number)
  }
  mx = wave_max(mx);
  if (lane == 0) red[tid >> 6] = mx;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kWaves; ++w) mx = fmaxf(mx, red[w]);
  if (tid == 0) R.pmax[c] = mx;
  if (!s.top_k && !s.p) return;
  if (mx > -INFINITY) {
    const Binner bin(mx, s.inv_t);
    const int copy = (lane & (kCopies - 1)) * kBins;
    for (int i = beg; i < end; i += kRound * kThreads) {
      if (end - beg > kRound * kThreads) load_round(L, i + tid, end, v);
#pragma unroll
      for (int u = 0; u < kRound; ++u) {
        const int b = bin(v[u]);
        if (b == kBins) continue;
        if (s.top_k) atomicAdd(&count[copy + b], 1u);
        if (s.p) atomicAdd(&mass[copy + b], (u64)(weight(v[u], mx, s.inv_t) * kBinUnit + 0.5));
      }
    }
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

__device__ __forceinline__ float row_max(const Row& R) {
  float mx = -INFINITY;
#pragma unroll
  for (int c = 0; c < kChunks; ++c) mx = fmaxf(mx, R.pmax[c]);
  return mx;
}

// The bins that hold the cuts: tokens of bins < lo are kept, those of k_bin and of p_lo .. p_hi are
// undecided, the others dropped.  (-1 .. -2: no such cut)
struct CutBins {
  int lo, p_lo, p_hi, k_bin;
};

__global__ __launch_bounds__(kThreads) void sample_gather_kernel(SampleParams p, void* ws) {
  __shared__ u64 red[kWaves];
  __shared__ u64 part_c[4][kBins];
  __shared__ double part_m[4][kBins];
  __shared__ CutBins s_cut;
  __shared__ int s_cnt[kRound * kWaves];
  const int c = blockIdx.x, row = blockIdx.y, tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  Row& R = row_state(ws, row, p.vocab);
  const float* L = p.logits + (size_t)row * p.vocab;
  const int cl = chunk_len(p.vocab), beg = min(p.vocab, c * cl), end = min(p.vocab, beg + cl);
  const Setting s = setting(p, row);
  float v[kRound];
  if (beg < end) load_round(L, beg + tid, end, v);
  const float mx = row_max(R);
  if (!(mx > -INFINITY)) return;  // nothing to choose from
  const Binner bin(mx, s.inv_t);
  CutBins cut{kBins, -1, -2, -1};
  if (s.top_k || s.p) {
    // the row's histogram: thread (bin, quarter of the chunks), then the quarters in order
    const int b = tid & (kBins - 1), q = tid / kBins;
    u64 count = 0;
    double mass = 0.0;
#pragma unroll
    for (int j = 0; j < kChunks / 4; ++j) {
      const int ch = q * (kChunks / 4) + j;
      const float cm = R.pmax[ch];
      const int from = b - bin(cm);  // (bin(-inf) = kBins: none)
      if (from < 0) continue;
      if (s.top_k) count += R.count[ch][from];
      if (s.p) mass += (double)R.mass[ch][from] * weight(cm, mx, s.inv_t);
    }
    part_c[q][b] = count;
    part_m[q][b] = mass;
    __syncthreads();
    if (wave == 0) {  // lane l: bins 4 l .. 4 l + 3
      u64 n[4], nsum = 0;
      double m[4], msum = 0.0;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int b4 = 4 * lane + j;
        nsum += n[j] = (part_c[0][b4] + part_c[1][b4]) + (part_c[2][b4] + part_c[3][b4]);
        msum += m[j] = ((part_m[0][b4] + part_m[1][b4]) + (part_m[2][b4] + part_m[3][b4])) * (1.0 / kBinUnit);
      }
      const u64 ninc = wave_scan_inc(nsum);
      const double minc = wave_scan_inc(msum);
      // first bin whose cumulative value reaches the target (kBins: none), and what lies above it
      const auto first_bin = [&](auto inc, auto own, const auto (&h)[4], auto target, auto* above) {
        const u64 hit = __ballot(inc >= target);
        const int at = hit ? __ffsll((long long)hit) - 1 : 63;
        auto a = inc - own;
        int j = 0;
        while (j < 3 && a + h[j] < target) a += h[j++];
        const int bin4 = hit ? 4 * lane + j : kBins;
        *above = lane_value(a, at);
        return lane_value(bin4, at);
      };
      u64 k_above = 0;
      double mass_k = lane_value(minc, 63), mass_k_incl = mass_k, mass_p = 0.0, none;
      if (s.top_k) {
        cut.k_bin = first_bin(ninc, nsum, n, (u64)s.top_k, &k_above);
        if (cut.k_bin == kBins) {
          cut.k_bin = -1;  // the first top_k reach past every token that weighs anything
        } else {
          // masses up to that bin, without it and with it
          double below = minc - msum, own = 0.0;
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            if (4 * lane + j < cut.k_bin) below += m[j];
            if (4 * lane + j == cut.k_bin) own = m[j];
          }
          mass_k = lane_value(below, cut.k_bin >> 2);
          mass_k_incl = mass_k + lane_value(own, cut.k_bin >> 2);
          cut.lo = cut.k_bin;
        }
      }
      if (s.p) {
        // Z lies between the masses without and with k_bin (which part of it is kept is not known yet)
        const double tiny = 1.0 / kUnit, last = mass_k_incl;
        cut.p_lo = first_bin(minc, msum, m, fmin(fmax(mass_k * s.top_p * (1.0 - 1e-12), tiny), last), &mass_p);
        cut.p_hi = first_bin(minc, msum, m, fmin(fmax(mass_k_incl * s.top_p * (1.0 + 1e-12), tiny), last), &none);
        const int most = cut.k_bin >= 0 ? cut.k_bin : kBins - 1;
        cut.p_hi = min(cut.p_hi, most);
        cut.p_lo = min(cut.p_lo, cut.p_hi);
        cut.lo = cut.p_lo;
      }
      if (lane == 0) {
        s_cut = cut;
        if (c == 0) {
          R.cut_bins[0] = cut.lo, R.cut_bins[1] = cut.p_lo;
          R.cut_bins[2] = cut.p_hi, R.cut_bins[3] = cut.k_bin;
          R.k_above = k_above;
          R.mass_k = mass_k;
          R.mass_p = mass_p;
        }
      }
    }
    __syncthreads();
    cut = s_cut;
  } else if (c == 0 && tid == 0) {
    R.cut_bins[0] = cut.lo, R.cut_bins[1] = cut.p_lo;
    R.cut_bins[2] = cut.p_hi, R.cut_bins[3] = cut.k_bin;
  }
  Listed* list = row_list(R, c, p.vocab);
  u64 low = 0;
  int listed = 0;
  // (beg and end are the workgroup's: every thread runs every round and its barriers)
  for (int i = beg; i < end; i += kRound * kThreads) {
    if (i > beg) load_round(L, i + tid, end, v);
    unsigned int hits = 0;
#pragma unroll
    for (int u = 0; u < kRound; ++u) {
      const int b = bin(v[u]);
      if (b < cut.lo && b < kBins) {
        const double w = weight(v[u], mx, s.inv_t);
        if (!s.m || w >= (double)s.min_p) low += fixed(w);
      } else if (b < kBins && (b == cut.k_bin || (b >= cut.p_lo && b <= cut.p_hi))) {
        hits |= 1u << u;
      }
      const u64 vote = __ballot(hits >> u & 1);
      if (lane == 0) s_cnt[u * kWaves + wave] = __popcll(vote);
    }
    __syncthreads();
    // places in id order: the slabs of kThreads ids one after the other, wave by wave
    static_assert(kRound * kWaves == 128, "two counts a lane");
    const int a = s_cnt[2 * lane], b2 = s_cnt[2 * lane + 1];
    const int inc = wave_scan_inc(a + b2);
    __syncthreads();
#pragma unroll
    for (int u = 0; u < kRound; ++u) {
      const int slot = u * kWaves + wave;
      const int upto = lane_value(inc, slot >> 1) - lane_value(slot & 1 ? b2 : a + b2, slot >> 1);
      const u64 vote = __ballot(hits >> u & 1);
      if (hits >> u & 1)
        list[listed + upto + __popcll(vote & ((1ull << lane) - 1))] = Listed{v[u], i + tid + u * kThreads};
    }
    listed += lane_value(inc, 63);
  }
  low = block_sum(low, red);
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
constexpr int kInLds = 4096;  // listed tokens kept in LDS

__global__ __launch_bounds__(kThreads) void sample_finish_kernel(SampleParams p, void* ws) {
  __shared__ u64 hist[kDigits];
  __shared__ Listed held[kInLds];
  __shared__ u64 red[kWaves];
  __shared__ u64 kept_of[kChunks];
  __shared__ int offset[kChunks + 1];
  __shared__ uint32_t s_min, s_max;
  __shared__ int s_digit, s_id;
  __shared__ u64 s_above, s_at;
  const int row = blockIdx.x, tid = threadIdx.x, lane = tid & 63;
  Row& R = row_state(ws, row, p.vocab);
  const float* L = p.logits + (size_t)row * p.vocab;
  const Setting s = setting(p, row);
  const float mx = row_max(R);
  if (!(mx > -INFINITY)) {
    if (tid == 0) p.out[row] = -1;
    return;
  }
  const Binner bin(mx, s.inv_t);
  const int p_lo = R.cut_bins[1], p_hi = R.cut_bins[2], k_bin = R.cut_bins[3];
  if (tid < 64) {
    const int n = tid < kChunks ? R.n_listed[tid] : 0;
    const int inc = wave_scan_inc(n);
    if (tid < kChunks) {
      offset[tid + 1] = inc;
      kept_of[tid] = R.kept[tid];
    }
    if (tid == 0) offset[0] = 0;
  }
  __syncthreads();
  const int n = offset[kChunks];
  const bool in_lds = n <= kInLds;
  // listed token j, in id order
  const auto fetch = [&](int j) {
    int c = 0;
#pragma unroll
    for (int k = 1; k < kChunks; ++k) c += j >= offset[k];
    return row_list(R, c, p.vocab)[j - offset[c]];
  };
  if (in_lds)
    for (int j = tid; j < n; j += kThreads) held[j] = fetch(j);
  __syncthreads();
  const auto token = [&](int j) { return in_lds ? held[j] : fetch(j); };

  // The cut where the sum of f over the listed tokens that `in` takes, in the order, reaches target >= 1
  // (never: all of them stay): a radix select of the key from the first bits in which they differ, then,
  // among equal keys (equal f), the id of the last one needed.
  const auto select = [&](auto in, auto f, u64 target) {
    if (tid == 0) s_min = 0xFFFFFFFFu, s_max = 0;
    __syncthreads();
    uint32_t kmin = 0xFFFFFFFFu, kmax = 0;
    for (int j = tid; j < n; j += kThreads) {
      const Listed t = token(j);
      if (!in(t)) continue;
      const uint32_t k = logit_key(t.l);
      kmin = min(kmin, k), kmax = max(kmax, k);
    }
    if (kmin <= kmax) atomicMin(&s_min, kmin), atomicMax(&s_max, kmax);
    __syncthreads();
    uint32_t base = s_min, span = s_max - s_min;  // keys base .. base + span are left
    while (span) {
      const int shift = max(0, 32 - __clz(span) - 11);
      for (int d = tid; d < kDigits; d += kThreads) hist[d] = 0;
      __syncthreads();
      for (int j = tid; j < n; j += kThreads) {
        const Listed t = token(j);
        const uint32_t k = logit_key(t.l) - base;
        if (in(t) && k <= span) atomicAdd(&hist[k >> shift], f(t));
      }
      __syncthreads();
      // digits from the largest: thread t has kDigits - 1 - 2 t and the one below
      const u64 h0 = hist[kDigits - 1 - 2 * tid], h1 = hist[kDigits - 2 - 2 * tid];
      u64 all;
      const u64 inc = block_scan(h0 + h1, red, &all);
      if (all == 0) return Cut{-INFINITY, 0x7FFFFFFF};  // (they weigh nothing)
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
    for (int j0 = 0; j0 < n && before < target; j0 += kThreads) {
      const int j = j0 + tid;
      u64 q = 0;
      int id = 0;
      if (j < n) {
        const Listed t = token(j);
        id = t.id;
        if (in(t) && logit_key(t.l) == base) q = f(t);
      }
      u64 all;
      const u64 inc = before + block_scan(q, red, &all);
      if (q && inc >= target && inc - q < target) s_id = id;
      before += all;
    }
    __syncthreads();
    const Cut c{key_logit(base), s_id + 1};
    __syncthreads();
    return c;
  };
  const auto mass = [&](float l) { return fixed(weight(l, mx, s.inv_t)); };

  Cut k_cut{-INFINITY, 0x7FFFFFFF}, cut = k_cut;
  if (k_bin >= 0) {
    k_cut = select([&](Listed t) { return bin(t.l) == k_bin; }, [](Listed) { return (u64)1; },
                   (u64)s.top_k - R.k_above);
    cut = k_cut;
  }
  if (s.p) {
    double z = R.mass_k;  // of the bins above k_bin (of all: no such cut)
    if (k_bin >= 0) {
      u64 in_bin = 0;
      for (int j = tid; j < n; j += kThreads) {
        const Listed t = token(j);
        if (bin(t.l) == k_bin && k_cut.keeps(t.l, t.id)) in_bin += mass(t.l);
      }
      z += (double)block_sum(in_bin, red) * (1.0 / kUnit);
    }
    const double want = ceil((z * (double)s.top_p - R.mass_p) * kUnit);
    cut = select([&](Listed t) {
                   const int b = bin(t.l);
                   return b >= p_lo && b <= p_hi && k_cut.keeps(t.l, t.id);
                 },
                 [&](Listed t) { return mass(t.l); }, want > 1.0 ? (u64)want : (u64)1);
  }
  // (what is kept lies at or above the cut, the bins above it with it; a cut keeps all that weighs
  // something where there is none)
  const auto kept_mass = [&](float l, int id) -> u64 {
    if (!cut.keeps(l, id)) return 0;
    const double w = weight(l, mx, s.inv_t);
    return !s.m || w >= (double)s.min_p ? fixed(w) : 0;
  };
  // the chunks' kept masses
  for (int j = tid; j < n; j += kThreads) {
    const Listed t = token(j);
    const u64 q = kept_mass(t.l, t.id);
    if (!q) continue;
    int c = 0;
#pragma unroll
    for (int k = 1; k < kChunks; ++k) c += j >= offset[k];
    atomicAdd(&kept_of[c], q);
  }
  __syncthreads();
  if (tid < 64) {
    const u64 own = tid < kChunks ? kept_of[tid] : 0, inc = wave_scan_inc(own);
    const u64 z = lane_value(inc, 63);
    const float u = p.uniform[row];
    const double x = (double)z * (u > 0.f ? (double)u : 0.0);
    const u64 at = x < (double)z ? min((u64)x, z - 1) : z - 1;
    const int c = __ffsll((long long)__ballot(inc > at)) - 1;
    if (lane == c) s_digit = c, s_at = at - (inc - own);
  }
  __syncthreads();
  // the chunk's first id whose kept cumulative mass exceeds the draw
  const u64 at = s_at;
  const int cl = chunk_len(p.vocab), beg = s_digit * cl, end = min(p.vocab, beg + cl);
  u64 before = 0;
  for (int i = beg; i < end && before <= at; i += kRound * kThreads) {
    // kRound ids in a row a thread: one scan a round
    float v[kRound];
    u64 q[kRound], own = 0;
#pragma unroll
    for (int u = 0; u < kRound; ++u) v[u] = L[min(i + tid * kRound + u, end - 1)];
#pragma unroll
    for (int u = 0; u < kRound; ++u) {
      const int id = i + tid * kRound + u;
      own += q[u] = id < end ? kept_mass(v[u], id) : 0;
    }
    u64 all;
    u64 upto = before + block_scan(own, red, &all) - own;
#pragma unroll
    for (int u = 0; u < kRound; ++u) {
      if (upto <= at && at < upto + q[u]) p.out[row] = i + tid * kRound + u;  // exactly one token
      upto += q[u];
    }
    before += all;
  }
}

}  // namespace

size_t sample_filtered_workspace_bytes(int rows, int vocab) { return rows * row_bytes(vocab); }

int launch_sample_filtered(const SampleParams& p, void* ws, hipStream_t st) {
  const dim3 chunks(kChunks, p.rows);
  hipLaunchKernelGGL(sample_hist_kernel, chunks, dim3(kThreads), 0, st, p, ws);
  hipLaunchKernelGGL(sample_gather_kernel, chunks, dim3(kThreads), 0, st, p, ws);
  hipLaunchKernelGGL(sample_finish_kernel, dim3(p.rows), dim3(kThreads), 0, st, p, ws);
  IE_CHECK_LAUNCH();
  return IE_OK;
}

}  // namespace ie
