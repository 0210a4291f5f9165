// Attention of ragged chunks of new tokens over a paged K/V cache of bf16 or 8-bit pages, where groups of
// sequences may share the pages of their first positions (no reference counterparts: the reference
// attends one sequence over one bf16 plane).
//
// The row at position p sees the keys j <= p with j > p - window or j < n_sinks whose page is there:
//   o = sum_j softmax_j(q . k_j / sqrt(128)) v_j,  zeros where it sees none.
// An 8-bit row is read as its codes times its scale 2^e, which bf16 holds exactly, so that both kinds of pages
// run the same products (k_attn_window.hip: S^T = K . Q^T, online softmax, O^T = V^T . P^T in bf16 with fp32
// sums, weights rounded to bf16).
//
// Softmax over a union of key sets is joined from (o, m, l) of each.  So the keys that a group of sequences
// shares are attended once, by the rows of all of them (a prefix segment: rows of different sequences
// are columns of one block, each with its own position), and each sequence's other keys by its rows (an own
// segment).  Sequences that fill the columns of a block by themselves gain nothing from that and attend all
// their keys in their own segment.
//
// A workgroup of 4 waves takes one kv head of a segment in one of two forms.
// Narrow (up to 16 columns, a column being a (row, q head of the kv head's group)): the key tiles go round
// the waves, each of which holds all the columns: nothing is shared until the waves' (o, m, l) are
// joined at the end.  K comes from memory in the layout of the product's operand (the order of the 128 dims
// within the sum is free, and Q's fragments are taken in the same order), V through registers into a tile of the
// wave's own in LDS, from which it is read transposed.  No barrier, a tile of loads in flight a wave.
// Wide: 16 or 32 columns a wave, the tiles staged in LDS for all four, double-buffered, as k_attn_window.hip
// does it; 8-bit tiles pass through registers, where they become bf16.
#include <algorithm>
#include <atomic>
#include <random>

#include "ie_attn_tiles.h"

namespace ie {

namespace {

constexpr int NW = 4;
constexpr int kNarrowCols = 16;
constexpr int kOutStride = kHeadDim + 4;  // of a column's sums in LDS, floats (no bank conflicts)

// A workgroup's work: rows r0 .. r0 + nr - 1 of a segment of n rows, one kv head, the tiles i0 .. i1 - 1
// of the segment's run: na blocks from a0 on (sinks), then those from b0 on.
struct Work {
  int g, n, nqb, splits, split, r0, nr, part0, i0, i1;
  int a0, na, b0;
  int p0, row0;     // own: position and batch row of the block's first row
  int first, end;   // prefix: its sequences
  int nkeys;        // keys of the segment: positions below
  int seq;          // own: the sequence, whose table is read (prefix: the first's)
  bool prefix;
  bool whole;       // its rows have no other partials
  const int* table;
  __device__ __forceinline__ int tile(int i) const { return i < na ? a0 + i : b0 + i - na; }
};

// The blocks lo .. hi - 1 that a row from position p0 on may see, at most up to position p1's block.
struct Run {
  int a0, na, b0, count;
};
__host__ __device__ __forceinline__ Run run_of(int p0, int p1, int lo, int hi, int window, int n_sinks) {
  const int oldest = p0 - window + 1;
  const int first = oldest > 0 ? oldest / BKEY : 0;
  const int st = (n_sinks + BKEY - 1) / BKEY, top = p1 / BKEY + 1;
  Run r;
  r.a0 = lo;
  const int sinks_end = st < first ? st : first;
  const int a_end = sinks_end < hi ? sinks_end : hi;
  r.na = a_end > lo ? a_end - lo : 0;
  r.b0 = first > lo ? first : lo;
  const int b_end = top < hi ? top : hi;
  r.count = r.na + (b_end > r.b0 ? b_end - r.b0 : 0);
  return r;
}

// Rows of a block of a segment of n rows.
__host__ __device__ __forceinline__ int block_rows(int n, int gs, int qi) {
  return (n << gs) <= kNarrowCols ? n : (64 * qi) >> gs;
}

// Workgroup -> (segment, split, row block, kv head): kv heads go round the XCDs, whose L2 then holds the head's
// keys for the blocks that share them; prefixes come first, then the sequences, of each the last blocks (the
// longest runs) first.  (the segments' arguments in one go, a lane each)
__device__ __forceinline__ Work work_of(const AttnSharedParams& p, int qi) {
  const int lane = threadIdx.x & 63, gs = p.group_shift;
  Work w;
  w.g = blockIdx.x % kKVHeads;
  int item = blockIdx.x / kKVHeads;
  w.prefix = item < p.prefix_items;
  int lo, hi, pmax;
  if (w.prefix) {
    const int l32 = lane & 31;
    const int item_end = p.p_item_end[l32];
    const int k = __popcll(__ballot(lane < p.n_prefixes && item_end <= item));
    w.first = p.p_first[k], w.end = p.p_end[k];
    w.splits = p.p_splits[k], w.part0 = p.p_part0[k];
    w.row0 = w.first ? p.member_end[max(w.first - 1, 0)] : 0;  // (members before the prefix's)
    w.n = p.member_end[w.end - 1] - w.row0;
    item -= k ? p.p_item_end[max(k - 1, 0)] : 0;
    w.p0 = p.p_start[k];
    lo = 0, hi = p.p_blocks[k];
    w.nkeys = hi * BKEY;
    w.seq = w.first;
    pmax = w.nkeys - 1;
  } else {
    item -= p.prefix_items;
    const int item_end = p.item_end[lane];
    const int b = __popcll(__ballot(lane < p.n_seqs && item_end <= item));
    w.seq = b, w.first = b, w.end = b + 1;
    w.splits = p.splits[b], w.part0 = p.part0[b];
    w.row0 = b ? p.row_end[max(b - 1, 0)] : 0;
    w.n = p.row_end[b] - w.row0;
    item -= b ? p.item_end[max(b - 1, 0)] : 0;
    w.p0 = p.start[b];
    lo = p.lo[b], hi = kMaxLongCtx / BKEY;
    w.nkeys = w.p0 + w.n;
    pmax = 0;
  }
  const int rb = block_rows(w.n, gs, qi);
  w.nqb = (w.n + rb - 1) / rb;
  w.r0 = (w.nqb - 1 - item % w.nqb) * rb;
  w.split = item / w.nqb;
  w.nr = min(rb, w.n - w.r0);
  if (!w.prefix) {
    w.p0 += w.r0;
    w.row0 += w.r0;
    pmax = w.p0 + w.nr - 1;
  }
  const Run r = run_of(w.p0, pmax, lo, hi, p.window, p.n_sinks);
  w.a0 = r.a0, w.na = r.na, w.b0 = r.b0;
  const int tps = (r.count + w.splits - 1) / w.splits;
  w.i0 = min(r.count, w.split * tps);
  w.i1 = min(r.count, w.i0 + tps);
  w.whole = !w.prefix && w.splits == 1 && p.prefix[w.seq] < 0;
  w.table = p.block_tables + (size_t)w.seq * p.table_stride;
  return w;
}

// ---------------------------------------------------------------- columns
// The (batch row, position) of row r of the block.
struct RowPos {
  int row, pos;
};
__device__ __forceinline__ RowPos row_of(const AttnSharedParams& p, const Work& w, int r) {
  RowPos x{w.row0 + r, w.p0 + r};
  if (w.prefix) {
    // members' rows one after the other, row `at` of them
    const int at = w.row0 + w.r0 + r;
    int before = w.row0;
    for (int b = w.first; b < w.end; ++b) {
      const int upto = p.member_end[b];
      if (at >= before && at < upto) {
        x.row = (b ? p.row_end[max(b - 1, 0)] : 0) + at - before;
        x.pos = p.start[b] + at - before;
      }
      before = upto;
    }
  }
  return x;
}

template <int QI>
struct Columns : ColumnState<QI> {
  using ColumnState<QI>::q, ColumnState<QI>::pos, ColumnState<QI>::o, ColumnState<QI>::m, ColumnState<QI>::l;
  int least, most;  // of the wave's positions

  // Columns past the rows repeat the last row.  PERM: Q's dims in the order in which the narrow form
  // takes 8-bit keys.
  template <bool PERM>
  __device__ __forceinline__ void load(const AttnSharedParams& p, const Work& w, int col0) {
    const int fr = threadIdx.x & 15, G = threadIdx.x >> 4 & 3, gs = p.group_shift;
    int lo = INT32_MAX, hi = 0;
#pragma unroll
    for (int qi = 0; qi < QI; ++qi) {
      const int col = col0 + 16 * qi + fr;
      const RowPos x = row_of(p, w, min(col >> gs, w.nr - 1));
      pos[qi] = x.pos;
      const size_t at = ((size_t)x.row << gs << 3) + ((size_t)w.g << gs) + (col & ((1 << gs) - 1));
      const u32x4_t* row = reinterpret_cast<const u32x4_t*>(p.q + at * kHeadDim);
#pragma unroll
      for (int ks = 0; ks < 4; ++ks)
        q[qi][ks] = __builtin_bit_cast(bf16x8_t, row[PERM ? 8 * (ks >> 1) + 2 * G + (ks & 1) : 4 * ks + G]);
      lo = min(lo, x.pos), hi = max(hi, x.pos);
    }
#pragma unroll
    for (int s = 1; s < 16; s <<= 1) {
      lo = min(lo, __shfl_xor(lo, s, 64));
      hi = max(hi, __shfl_xor(hi, s, 64));
    }
    least = __builtin_amdgcn_readfirstlane(lo);
    most = __builtin_amdgcn_readfirstlane(hi);
    this->clear();
    // The compiler does not see what the kernels' own waits cover: without one here it would guard the
    // fragments inside their loops, where that is a wait for the tile in flight.
    __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0)
  }
};

// Device-scope stores and loads: what one workgroup hands to another within a launch.
__device__ __forceinline__ void agent_store2(float* p, float a, float b) {
  const uint64_t v = (uint64_t)__float_as_uint(b) << 32 | __float_as_uint(a);
  __hip_atomic_store(reinterpret_cast<uint64_t*>(p), v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ float2 agent_load2(const float* p) {
  const uint64_t v = __hip_atomic_load(reinterpret_cast<const uint64_t*>(p), __ATOMIC_RELAXED,
                                       __HIP_MEMORY_SCOPE_AGENT);
  return make_float2(__uint_as_float((uint32_t)v), __uint_as_float((uint32_t)(v >> 32)));
}

// ---------------------------------------------------------------- pages
// A head's K and V planes in a page, `rows` of their 64 rows there; a page outside the pool has none: what
// is read of them is zero.
struct Planes {
  __amdgpu_buffer_rsrc_t k, v, scales;
  int rows;
};
template <bool F8>
__device__ __forceinline__ Planes planes_of(const AttnSharedParams& p, int g, int page, int rows) {
  constexpr int kRow = F8 ? kHeadDim : kRowBytes;
  constexpr size_t kHead = F8 ? kPage8Head : kPageHead * 2;
  const bool ok = page >= 0 && page < p.n_pages;
  const uint8_t* at = p.pages + (size_t)(ok ? page : 0) * (F8 ? kPage8Bytes : kPageElems * 2);
  Planes x;
  x.rows = __builtin_amdgcn_readfirstlane(ok ? max(min(BKEY, rows), 0) : 0);
  x.k = __builtin_amdgcn_make_buffer_rsrc((void*)(at + g * kHead), 0, x.rows * kRow, kBufferFlags);
  x.v = __builtin_amdgcn_make_buffer_rsrc((void*)(at + (kKVHeads + g) * kHead), 0, x.rows * kRow, kBufferFlags);
  // (K's bytes of all heads, then V's)
  if constexpr (F8)
    x.scales = __builtin_amdgcn_make_buffer_rsrc((void*)(at + kPage8Codes), 0, ok ? 2 * kKVHeads * kPagePos : 0,
                                                 kBufferFlags);
  return x;
}

// The scale of byte k of w; 0 for a row that is not there (its codes read as zero, its scale may be anything).
__device__ __forceinline__ float scale_at_byte(uint32_t w, int k, bool there) {
  return scale_of(there ? w >> (8 * k) & 0xFF : 0);
}

// 16 codes as two chunks of 8 bf16.
__device__ __forceinline__ void chunks_of(u32x4_t (&c)[2], const u32x4_t& w, float scale) {
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const u32x2v_t a = dequantise4(w[2 * i], scale), b = dequantise4(w[2 * i + 1], scale);
    c[i] = u32x4_t{a[0], a[1], b[0], b[1]};
  }
}

// ---------------------------------------------------------------- narrow form
// A wave's K tile as operands: lane (fr, G) holds of the rows fr + 16 kb (kb 0 .. 3) the dims
// 32 ks + 8 G .. +8 (bf16), or the 16 codes from 64 j + 16 G on, j 0 and 1: two operands.
template <bool F8, int AUX>
struct NarrowK {
  static constexpr int kLoads = F8 ? 2 : 4;
  u32x4_t w[4][kLoads];
  uint32_t scales;
  int rows;
  __device__ __forceinline__ void issue(const Planes& x, int g) {
    const int fr = threadIdx.x & 15, G = threadIdx.x >> 4 & 3;
    rows = x.rows;
    const int off = fr * (F8 ? kHeadDim : kRowBytes) + 16 * G;
    if constexpr (F8)
      scales = __builtin_amdgcn_raw_buffer_load_b32(x.scales, 4 * fr, g * kPagePos, AUX);
#pragma unroll
    for (int kb = 0; kb < 4; ++kb)
#pragma unroll
      for (int j = 0; j < kLoads; ++j)
        w[kb][j] = __builtin_amdgcn_raw_buffer_load_b128(
            x.k, off + kb * 16 * (F8 ? kHeadDim : kRowBytes) + 64 * j, 0, AUX);
  }
  __device__ __forceinline__ void scores(f32x4_t (&s)[1][4], const ColumnState<1>& c) const {
    const int fr = threadIdx.x & 15;
#pragma unroll
    for (int kb = 0; kb < 4; ++kb) {
      s[0][kb] = f32x4_t{0.f, 0.f, 0.f, 0.f};
      if constexpr (F8) {
        const float scale = scale_at_byte(scales, kb, 16 * kb + fr < rows);
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          u32x4_t a[2];
          chunks_of(a, w[kb][j], scale);
#pragma unroll
          for (int h = 0; h < 2; ++h)
            s[0][kb] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, a[h]), c.q[0][2 * j + h],
                                                               s[0][kb], 0, 0, 0);
        }
      } else {
#pragma unroll
        for (int ks = 0; ks < 4; ++ks)
          s[0][kb] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, w[kb][ks]), c.q[0][ks],
                                                             s[0][kb], 0, 0, 0);
      }
    }
  }
};

// A wave's V tile on its way to LDS.  16 lanes a row of bf16, 8 a row of codes; of those, lane group
// e takes the rows 16 u + 2 e + v (their scales are 8 bytes in a row).
template <bool F8, int AUX>
struct NarrowV {
  static constexpr int kLoads = F8 ? 8 : 16;
  u32x4_t w[kLoads];
  u32x2_t scales;
  int rows;
  static __device__ __forceinline__ int row(int i) {
    const int lane = threadIdx.x & 63;
    return F8 ? 16 * (i >> 1) + 2 * (lane >> 3) + (i & 1) : 4 * i + (lane >> 4);
  }
  __device__ __forceinline__ void issue(const Planes& x, int g) {
    const int lane = threadIdx.x & 63;
    rows = x.rows;
    if constexpr (F8)
      scales = __builtin_bit_cast(u32x2_t, __builtin_amdgcn_raw_buffer_load_b64(x.scales, 8 * (lane >> 3),
                                                                               (kKVHeads + g) * kPagePos, AUX));
    const int off = F8 ? row(0) * kHeadDim + 16 * (lane & 7) : row(0) * kRowBytes + 16 * (lane & 15);
#pragma unroll
    for (int i = 0; i < kLoads; ++i)
      w[i] = __builtin_amdgcn_raw_buffer_load_b128(
          x.v, off + (F8 ? (16 * (i >> 1) + (i & 1)) * kHeadDim : 4 * i * kRowBytes), 0, AUX);
  }
  __device__ __forceinline__ void stage(u32x4_t* tile) const {
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      const int r = row(i);
      if constexpr (F8) {
        u32x4_t c[2];
        chunks_of(c, w[i], scale_at_byte(scales[i & 1], i >> 1, r < rows));
        tile[kv_slot(r, 2 * (lane & 7))] = c[0];
        tile[kv_slot(r, 2 * (lane & 7) + 1)] = c[1];
      } else {
        tile[kv_slot(r, lane & 15)] = w[i];
      }
    }
  }
};

// The softmax sums of some splits or waves joined: for each, its (m, l) and four values of its o.
struct Joined {
  f32x4_t o = {0.f, 0.f, 0.f, 0.f};
  float M = -INFINITY, L = 0.f;
  // N more, those from `count` on and those without keys (l = 0) passed over
  template <int N>
  __device__ __forceinline__ void add(const f32x4_t (&po)[N], const float2 (&ml)[N], int count) {
    float mn = M;
#pragma unroll
    for (int u = 0; u < N; ++u)
      if (u < count) mn = fmaxf(mn, ml[u].x);
    const float a = L == 0.f ? 0.f : __builtin_amdgcn_exp2f((M - mn) * kScoreScale);
    L *= a;
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] *= a;
#pragma unroll
    for (int u = 0; u < N; ++u) {
      if (u >= count || ml[u].y == 0.f) continue;
      const float w = __builtin_amdgcn_exp2f((ml[u].x - mn) * kScoreScale);
      L = fmaf(ml[u].y, w, L);
#pragma unroll
      for (int e = 0; e < 4; ++e) o[e] = fmaf(po[u][e], w, o[e]);
    }
    M = mn;
  }
  __device__ __forceinline__ void write(uint16_t* out) const {
    const float inv = L == 0.f ? 0.f : 1.0f / L;
    const u32x2_t w = {pack_bf2(o[0] * inv, o[1] * inv), pack_bf2(o[2] * inv, o[3] * inv)};
    *reinterpret_cast<u32x2_t*>(out) = w;
  }
};

template <bool F8, int AUX>
__device__ __forceinline__ void narrow_tiles(const AttnSharedParams& p, const Work& w, ColumnState<1>& c, int least,
                                             int most, int wave, u32x4_t* tile) {
  NarrowK<F8, AUX> k;
  NarrowV<F8, AUX> v;
  const Frags f;
  int i = w.i0 + wave;
  int page = i < w.i1 ? w.table[w.tile(i)] : -1;
  {
    const Planes x = planes_of<F8>(p, w.g, page, w.nkeys - w.tile(i) * BKEY);
    k.issue(x, w.g);
    v.issue(x, w.g);
  }
#pragma unroll 1
  for (; i < w.i1; i += NW) {
    const bool there = page >= 0 && page < p.n_pages;
    const int key0 = w.tile(i) * BKEY;
    const Sight see = there ? sight(key0, least, most, p.window, p.n_sinks) : kNone;
    page = i + NW < w.i1 ? w.table[w.tile(i + NW)] : -1;
    // (past the last tile nothing is read)
    const Planes x = planes_of<F8>(p, w.g, page, w.nkeys - w.tile(i + NW) * BKEY);
    f32x4_t s[1][4];
    bf16x8_t pb[1][2];
    k.scores(s, c);
    k.issue(x, w.g);
    if (see == kAll)
      weights<false>(pb, c, s, key0, p.window, p.n_sinks);
    else if (see == kSome)
      weights<true>(pb, c, s, key0, p.window, p.n_sinks);
    if (see != kNone) v.stage(tile);
    v.issue(x, w.g);
    // (the wave's own tile: the hardware does its LDS accesses in order; the compiler is held to it)
    asm volatile("" ::: "memory");
    if (see == kAll)
      values<false>(c, pb, f, tile, key0, p.window, p.n_sinks);
    else if (see == kSome)
      values<true>(c, pb, f, tile, key0, p.window, p.n_sinks);
    asm volatile("" ::: "memory");
  }
}

template <bool F8>
__device__ __forceinline__ void narrow(const AttnSharedParams& p, const Work& w, u32x4_t (*lds)[TC]) {
  __shared__ int s_last;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int tid = threadIdx.x, gs = p.group_shift, heads = kKVHeads << gs;
  Columns<1> c;
  c.template load<F8>(p, w, 0);
  if (p.nt)
    narrow_tiles<F8, 2>(p, w, c, c.least, c.most, wave, lds[wave]);
  else
    narrow_tiles<F8, 0>(p, w, c, c.least, c.most, wave, lds[wave]);
  // the waves' sums side by side: [column][128], then (m, l)
  {
    const int fr = tid & 15, G = tid >> 4 & 3;
    float* mine = reinterpret_cast<float*>(lds[wave]);
#pragma unroll
    for (int db = 0; db < 8; ++db) *reinterpret_cast<f32x4_t*>(mine + fr * kOutStride + 16 * db + 4 * G) = c.o[0][db];
    if (G == 0) *reinterpret_cast<float2*>(mine + kNarrowCols * kOutStride + 2 * fr) = make_float2(c.m[0], c.l[0][0]);
  }
  __syncthreads();
  const int ncols = w.nr << gs;
  const bool join = p.join && !w.whole;
  for (int i = tid; i < ncols * 32; i += 64 * NW) {
    const int col = i >> 5, d = 4 * (i & 31);
    f32x4_t po[NW];
    float2 ml[NW];
#pragma unroll
    for (int u = 0; u < NW; ++u) {
      const float* from = reinterpret_cast<const float*>(lds[u]);
      po[u] = *reinterpret_cast<const f32x4_t*>(from + col * kOutStride + d);
      ml[u] = *reinterpret_cast<const float2*>(from + kNarrowCols * kOutStride + 2 * col);
    }
    Joined j;
    j.add(po, ml, NW);
    const int h = (w.g << gs) + (col & ((1 << gs) - 1)), r = col >> gs;
    if (w.whole) {
      j.write(p.out + ((size_t)(w.row0 + r) * heads + h) * kHeadDim + d);
      continue;
    }
    const size_t slot = ((size_t)w.part0 + (size_t)w.split * w.n + w.r0 + r) * heads + h;
    if (join) {
      agent_store2(p.part + slot * kHeadDim + d, j.o[0], j.o[1]);
      agent_store2(p.part + slot * kHeadDim + d + 2, j.o[2], j.o[3]);
      if (d == 0) agent_store2(p.part_ml + 2 * slot, j.M, j.L);
    } else {
      *reinterpret_cast<f32x4_t*>(p.part + slot * kHeadDim + d) = j.o;
      if (d == 0) *reinterpret_cast<float2*>(p.part_ml + 2 * slot) = make_float2(j.M, j.L);
    }
  }
  if (!join) return;
  // The last split of the (sequence, kv head) to arrive joins them, in the splits' order.  The word that
  // counts them is the caller's memory, which may hold anything: a count is one with this call's tag,
  // whatever else is there counts as none.  The last leaves 0.
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // the partials are there, before the arrival counts
  __syncthreads();
  if (tid == 0) {
    unsigned long long* word = p.arrived + (size_t)w.seq * kKVHeads + w.g;
    unsigned long long cur = __hip_atomic_load(word, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT), next;
    do {
      next = cur >> 16 == p.tag ? cur + 1 : p.tag << 16 | 1;
    } while (!__hip_atomic_compare_exchange_strong(word, &cur, next, __ATOMIC_RELAXED, __ATOMIC_RELAXED,
                                                   __HIP_MEMORY_SCOPE_AGENT));
    const bool last = (int)(next & 0xFFFF) == w.splits;
    if (last) __hip_atomic_store(word, 0ull, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    s_last = last;
  }
  __syncthreads();
  if (!s_last) return;
  for (int i = tid; i < ncols * 32; i += 64 * NW) {
    const int col = i >> 5, d = 4 * (i & 31);
    const int h = (w.g << gs) + (col & ((1 << gs) - 1)), r = col >> gs;
    const size_t slot0 = ((size_t)w.part0 + w.r0 + r) * heads + h, step = (size_t)w.n * heads;
    Joined j;
    for (int s0 = 0; s0 < w.splits; s0 += 8) {
      f32x4_t po[8];
      float2 ml[8];
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        const size_t slot = slot0 + min(s0 + u, w.splits - 1) * step;
        ml[u] = agent_load2(p.part_ml + 2 * slot);
        const float2 a = agent_load2(p.part + slot * kHeadDim + d), b = agent_load2(p.part + slot * kHeadDim + d + 2);
        po[u] = f32x4_t{a.x, a.y, b.x, b.y};
      }
      j.add(po, ml, w.splits - s0);
    }
    j.write(p.out + ((size_t)(w.row0 + r) * heads + h) * kHeadDim + d);
  }
}

// ---------------------------------------------------------------- wide form
// A thread's part of an 8-bit tile: chunk t % 8 (16 codes) of rows t / 8 and t / 8 + 32, of K and V.
struct Raw8 {
  u32x4_t k[2], v[2];
  uint32_t ks, vs;
  int rows;
  template <int AUX>
  __device__ __forceinline__ void issue(const Planes& x, int g) {
    const int t = threadIdx.x;
    rows = x.rows;
    // the scales of rows t / 8 % 16 + 16 i
    ks = __builtin_amdgcn_raw_buffer_load_b32(x.scales, 4 * (t >> 3 & 15), g * kPagePos, AUX);
    vs = __builtin_amdgcn_raw_buffer_load_b32(x.scales, 4 * (t >> 3 & 15), (kKVHeads + g) * kPagePos, AUX);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      k[i] = __builtin_amdgcn_raw_buffer_load_b128(x.k, 16 * t, 4096 * i, AUX);
      v[i] = __builtin_amdgcn_raw_buffer_load_b128(x.v, 16 * t, 4096 * i, AUX);
    }
  }
  __device__ __forceinline__ void stage(u32x4_t* kt, u32x4_t* vt) const {
    const int t = threadIdx.x, c = 2 * (t & 7);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int r = (t >> 3) + 32 * i, byte = (t >> 7) + 2 * i;
      u32x4_t x[2];
      chunks_of(x, k[i], scale_at_byte(ks, byte, r < rows));
      kt[kv_slot(r, c)] = x[0];
      kt[kv_slot(r, c + 1)] = x[1];
      chunks_of(x, v[i], scale_at_byte(vs, byte, r < rows));
      vt[kv_slot(r, c)] = x[0];
      vt[kv_slot(r, c + 1)] = x[1];
    }
  }
};

template <bool F8, int QI>
__device__ __forceinline__ void wide(const AttnSharedParams& p, const Work& w, u32x4_t (*lds)[TC]) {
  constexpr int CW = 16 * QI;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const bool idle = (wave * CW) >> p.group_shift >= w.nr;  // (no rows)
  const bool nt = p.nt && w.nqb == 1;
  const TileLoad<NW> ld(wave);
  Raw8 raw;
  auto issue = [&](u32x4_t* ks, u32x4_t* vs, int i, int page) {
    const Planes x = planes_of<F8>(p, w.g, page, w.nkeys - w.tile(i) * BKEY);
    if constexpr (F8) {
      if (nt) raw.issue<2>(x, w.g);
      else raw.issue<0>(x, w.g);
    } else if (nt) {
      issue_tile<NW, 2>(ks, x.k, ld);
      issue_tile<NW, 2>(vs, x.v, ld);
    } else {
      issue_tile<NW, 0>(ks, x.k, ld);
      issue_tile<NW, 0>(vs, x.v, ld);
    }
  };
  // page of the tile in flight, and of the one after it (loaded a step ahead)
  int page = -1, next = -1;
  if (w.i0 < w.i1) {
    const int here = w.table[w.tile(w.i0)];
    next = w.table[w.tile(min(w.i0 + 1, w.i1 - 1))];
    page = __builtin_amdgcn_readfirstlane(here);
    issue(lds[0], lds[1], w.i0, page);
  }
  Columns<QI> c;
  c.template load<false>(p, w, wave * CW);
  const Frags f;

  auto step = [&](int i, u32x4_t* kc, u32x4_t* vc, u32x4_t* kn, u32x4_t* vn) {
    // 8 bits: tile i becomes bf16 in the buffers of tile i - 2, which every wave left before the last
    // barrier.  Then tile i has landed and every wave is done with tile i - 1.
    if constexpr (F8) {
      raw.stage(kc, vc);
      asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
    } else {
      asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
    }
    const bool there = page >= 0 && page < p.n_pages;
    // tile i + 1 is issued unconditionally: past the last tile it has no bytes
    page = i + 1 < w.i1 ? __builtin_amdgcn_readfirstlane(next) : -1;
    issue(kn, vn, i + 1, page);
    next = w.table[w.tile(min(i + 2, w.i1 - 1))];
    const int key0 = w.tile(i) * BKEY;
    const Sight see = there && !idle ? sight(key0, c.least, c.most, p.window, p.n_sinks) : kNone;
    if (see == kNone) return;  // (wave-uniform)
    f32x4_t s[QI][4];
    bf16x8_t pb[QI][2];
    scores(s, c, f, kc);
    __builtin_amdgcn_sched_barrier(0);
    if (see == kAll) {
      weights<false>(pb, c, s, key0, p.window, p.n_sinks);
      values<false>(c, pb, f, vc, key0, p.window, p.n_sinks);
    } else {
      weights<true>(pb, c, s, key0, p.window, p.n_sinks);
      __builtin_amdgcn_sched_barrier(0);  // (no fragments held over the softmax: registers)
      values<true>(c, pb, f, vc, key0, p.window, p.n_sinks);
    }
  };
  for (int i = w.i0; i < w.i1; i += 2) {
    step(i, lds[0], lds[1], lds[2], lds[3]);
    if (i + 1 < w.i1) step(i + 1, lds[2], lds[3], lds[0], lds[1]);
  }

  const int fr = threadIdx.x & 15, G = threadIdx.x >> 4 & 3, gs = p.group_shift;
  const int heads = kKVHeads << gs;
#pragma unroll
  for (int qi = 0; qi < QI; ++qi) {
    const int col = wave * CW + 16 * qi + fr, r = col >> gs;
    if (r >= w.nr) continue;
    const int h = (w.g << gs) + (col & ((1 << gs) - 1));
    if (!w.whole) {
      const size_t slot = ((size_t)w.part0 + (size_t)w.split * w.n + w.r0 + r) * heads + h;
      float* dst = p.part + slot * kHeadDim + 4 * G;
#pragma unroll
      for (int db = 0; db < 8; ++db) *reinterpret_cast<f32x4_t*>(dst + 16 * db) = c.o[qi][db];
      if (G == 0) *reinterpret_cast<float2*>(p.part_ml + 2 * slot) = make_float2(c.m[qi], c.l[qi][0]);
    } else {
      const float inv = c.l[qi][0] == 0.f ? 0.f : 1.0f / c.l[qi][0];
      uint16_t* dst = p.out + ((size_t)(w.row0 + r) * heads + h) * kHeadDim;
#pragma unroll
      for (int db = 0; db < 8; ++db) {
        const u32x2_t v = {pack_bf2(c.o[qi][db][0] * inv, c.o[qi][db][1] * inv),
                           pack_bf2(c.o[qi][db][2] * inv, c.o[qi][db][3] * inv)};
        *reinterpret_cast<u32x2_t*>(dst + db * 16 + 4 * G) = v;
      }
    }
  }
}

template <bool F8, int QI>
__global__ __launch_bounds__(64 * NW, 2) void attn_shared_kernel(AttnSharedParams p) {
  __shared__ u32x4_t lds[4][TC];
  const Work w = work_of(p, QI);
  if ((w.n << p.group_shift) <= kNarrowCols)
    narrow<F8>(p, w, lds);
  else
    wide<F8, QI>(p, w, lds);
}

// Joins the partials of each (row, q head) that has more than one: 32 lanes each, 4 dims a lane, the
// prefix's splits first, then the row's own.
__global__ __launch_bounds__(256) void attn_shared_merge_kernel(AttnSharedParams p) {
  const int lane = threadIdx.x & 63;
  const int row_end = p.row_end[lane];
  const int heads = kKVHeads << p.group_shift;
  const int row = blockIdx.x * 8 / heads;  // (8 heads a workgroup: heads is a multiple of 8)
  const int b = __popcll(__ballot(lane < p.n_seqs && row_end <= row));
  const int k = p.prefix[b], splits = p.splits[b];
  if (k < 0 && splits < 2) return;
  const int row0 = b ? p.row_end[max(b - 1, 0)] : 0, n = p.row_end[b] - row0;
  const int h = blockIdx.x * 8 % heads + (threadIdx.x >> 5), d = (threadIdx.x & 31) * 4;
  const float2* ml = reinterpret_cast<const float2*>(p.part_ml);
  Joined j;
  const auto add = [&](size_t slot0, size_t step, int count) {
    for (int s0 = 0; s0 < count; s0 += 8) {
      float2 v[8];
      f32x4_t po[8];
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        const size_t slot = slot0 + min(s0 + u, count - 1) * step;
        v[u] = ml[slot];
        po[u] = *reinterpret_cast<const f32x4_t*>(p.part + slot * kHeadDim + d);
      }
      j.add(po, v, count - s0);
    }
  };
  if (k >= 0) {
    const int first = p.p_first[k], before = first ? p.member_end[max(first - 1, 0)] : 0;
    const int all = p.member_end[p.p_end[k] - 1] - before;
    const int at = (b ? p.member_end[max(b - 1, 0)] : 0) - before + row - row0;
    add(((size_t)p.p_part0[k] + at) * heads + h, (size_t)all * heads, p.p_splits[k]);
  }
  add(((size_t)p.part0[b] + row - row0) * heads + h, (size_t)n * heads, splits);
  j.write(p.out + ((size_t)row * heads + h) * kHeadDim + d);
}

// Sequences of up to this many columns share a prefix; others fill a block of the wide form by themselves.
constexpr int kMemberCols = 64;
constexpr int kMaxSplits = 64;

// Rows of at most `rows` that share a prefix.
int members_of(int rows, int heads) { return std::min(rows, kMaxSeqs * std::max(1, kMemberCols / (heads / kKVHeads))); }
// Partial rows (a row and split) that a workspace for `rows` rows holds: 64 splits of up to 64 rows, and a
// prefix's and an own partial of each row that shares.  It never falls with the rows.
long long part_rows(int rows, int heads) { return (long long)std::min(rows, 64) * kMaxSplits + 2ll * members_of(rows, heads); }

constexpr size_t kArrivedBytes = (size_t)kMaxSeqs * kKVHeads * sizeof(unsigned long long);

// A call's tag of the arrival counts, 48 bits.
unsigned long long next_tag() {
  static std::atomic<unsigned long long> n{[] {
    std::random_device r;
    return (unsigned long long)r() << 32 | r();
  }()};
  const unsigned long long t = n.fetch_add(1, std::memory_order_relaxed) & ((1ull << 48) - 1);
  return t ? t : next_tag();
}

// A segment as the plan sees it.
struct Segment {
  int n, tiles;  // rows; tiles of its longest row block
  bool narrow;
};

// Columns a wave of the wide form; tiles a split of either form.
struct Plan {
  int qi, wide, narrow;
  int splits(const Segment& x) const {
    const int t = x.narrow ? narrow : wide;
    return std::clamp((x.tiles + t - 1) / t, 1, kMaxSplits);
  }
  int blocks(const Segment& x, int gs) const {
    const int rb = block_rows(x.n, gs, qi);
    return (x.n + rb - 1) / rb;
  }
};

Plan plan_of(const Segment* own, int n_own, const Segment* pre, int n_pre, const int* prefix, int gs, long long room) {
  long long narrow = 0, wide = 0;
  int longest = 1;
  const auto count = [&](const Segment& x) {
    if (!x.n) return;
    if (x.narrow) narrow += x.tiles;
    else wide += (long long)x.tiles * ((x.n << gs) + 63) / 64;
    longest = std::max(longest, x.tiles);
  };
  for (int b = 0; b < n_own; ++b) count(own[b]);
  for (int k = 0; k < n_pre; ++k) count(pre[k]);
  Plan plan{1, 1, 4};
  plan.narrow = (int)std::max(4ll, (narrow * kKVHeads + 511) / 512);
  plan.wide = (int)std::max(1ll, (wide * kKVHeads + 511) / 512);
  // (at one split a segment the partials fit)
  for (;;) {
    long long part = 0;
    for (int b = 0; b < n_own; ++b) {
      const int k = plan.splits(own[b]);
      if (k > 1 || prefix[b] >= 0) part += (long long)own[b].n * k;
    }
    for (int k = 0; k < n_pre; ++k) part += (long long)pre[k].n * plan.splits(pre[k]);
    if (part <= room) return plan;
    plan.wide *= 2, plan.narrow *= 2;
  }
}

}  // namespace

size_t attn_shared_workspace_bytes(int rows, int heads) {
  return kArrivedBytes + (size_t)part_rows(rows, heads) * heads * (kHeadDim + 2) * sizeof(float);
}

int launch_attn_shared(AttnSharedParams p, const SeqBatch& s, const SharedGroups& g, bool fp8, void* workspace,
                       hipStream_t st) {
  const int gs = p.group_shift, heads = kKVHeads << gs;
  p.n_seqs = s.n;
  int rows = 0, members = 0;
  long long keys = 0;
  for (int b = 0; b < s.n; ++b) p.prefix[b] = -1, p.lo[b] = 0;
  // the prefixes: groups of two sequences at least that have few rows each
  for (int i = 0, b0 = 0; i < g.n; b0 += g.seqs[i++]) {
    const int b1 = b0 + g.seqs[i], blocks = g.shared[i] / BKEY;
    int many = 0, least = kMaxLongCtx;
    for (int b = b0; b < b1; ++b)
      if (s.n_new[b] && (s.n_new[b] << gs) <= kMemberCols) ++many, least = std::min(least, s.start[b]);
    if (!blocks || many < 2) continue;
    const int k = p.n_prefixes++;
    p.p_first[k] = b0, p.p_end[k] = b1, p.p_blocks[k] = blocks, p.p_start[k] = least;
    for (int b = b0; b < b1; ++b)
      if (s.n_new[b] && (s.n_new[b] << gs) <= kMemberCols) p.prefix[b] = k, p.lo[b] = blocks;
  }
  Segment own[kMaxSeqs], pre[kMaxPrefixes];
  for (int b = 0; b < s.n; ++b) {
    const int n = s.n_new[b];
    p.start[b] = s.start[b];
    p.row_end[b] = rows += n;
    p.member_end[b] = members += p.prefix[b] >= 0 ? n : 0;
    keys += std::min(s.start[b] + n - p.lo[b] * BKEY, p.window + p.n_sinks + n);
  }
  if (!rows) return IE_OK;
  for (int k = 0; k < p.n_prefixes; ++k) {
    const int n = p.member_end[p.p_end[k] - 1] - (p.p_first[k] ? p.member_end[p.p_first[k] - 1] : 0);
    keys += p.p_blocks[k] * BKEY;
    pre[k] = {n, run_of(p.p_start[k], p.p_blocks[k] * BKEY - 1, 0, p.p_blocks[k], p.window, p.n_sinks).count,
              (n << gs) <= kNarrowCols};
  }
  for (int b = 0; b < s.n; ++b) {
    const int n = s.n_new[b], rb = n ? block_rows(n, gs, 2) : 1, last = n ? (n - 1) / rb * rb : 0;
    own[b] = {n, 0, (n << gs) <= kNarrowCols};
    if (!n) continue;
    const auto tiles = [&](int r0) {
      return run_of(s.start[b] + r0, s.start[b] + std::min(r0 + rb, n) - 1, p.lo[b], kMaxLongCtx / BKEY, p.window,
                    p.n_sinks).count;
    };
    own[b].tiles = std::max(tiles(0), last ? tiles(last) : 0);
  }
  const Plan plan = plan_of(own, s.n, pre, p.n_prefixes, p.prefix, gs, part_rows(rows, heads));
  // splits, items and partial rows, segment by segment
  int items = 0, part = 0;
  bool split_wide = false, split_any = false;
  const auto place = [&](const Segment& x, bool alone, int& item_end, int& splits, int& part0) {
    splits = plan.splits(x);
    if (x.n) items += splits * plan.blocks(x, gs);
    item_end = items;
    part0 = part;
    if (!x.n || (alone && splits == 1)) return;
    part += x.n * splits;
    split_any = true;
    split_wide |= !x.narrow;
  };
  for (int k = 0; k < p.n_prefixes; ++k) place(pre[k], false, p.p_item_end[k], p.p_splits[k], p.p_part0[k]);
  p.prefix_items = items;
  items = 0;
  for (int b = 0; b < s.n; ++b) place(own[b], p.prefix[b] < 0, p.item_end[b], p.splits[b], p.part0[b]);
  items += p.prefix_items;
  p.join = split_any && !split_wide && !p.n_prefixes;
  // a batch whose keys of all layers exceed the 256 MB cache finds none of them there: such keys, where one
  // workgroup reads them, pass it by
  p.nt = keys > 2048;
  p.arrived = static_cast<unsigned long long*>(workspace);
  p.tag = p.join ? next_tag() : 0;
  p.part = reinterpret_cast<float*>(static_cast<char*>(workspace) + kArrivedBytes);
  p.part_ml = p.part + (size_t)part * heads * kHeadDim;
  const dim3 grid(items * kKVHeads), block(64 * NW);
  if (fp8 && plan.qi == 1)
    hipLaunchKernelGGL((attn_shared_kernel<true, 1>), grid, block, 0, st, p);
  else if (fp8)
    hipLaunchKernelGGL((attn_shared_kernel<true, 2>), grid, block, 0, st, p);
  else if (plan.qi == 1)
    hipLaunchKernelGGL((attn_shared_kernel<false, 1>), grid, block, 0, st, p);
  else
    hipLaunchKernelGGL((attn_shared_kernel<false, 2>), grid, block, 0, st, p);
  IE_CHECK_LAUNCH();
  if (split_any && !p.join) {
    hipLaunchKernelGGL(attn_shared_merge_kernel, dim3(rows << gs), dim3(256), 0, st, p);
    IE_CHECK_LAUNCH();
  }
  return IE_OK;
}

}  // namespace ie
