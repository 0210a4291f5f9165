// Attention of ragged chunks of new tokens over a paged K/V cache of bf16 or 8-bit pages, where groups of
// sequences may share the pages of their first positions (no reference counterparts: the reference
// attends one sequence over one bf16 plane).
//
// The row at position p sees the keys j <= p with j > p - window or j < n_sinks whose page is there:
//   o = sum_j softmax_j(q . k_j / sqrt(128)) v_j,  zeros where it sees none.
// An 8-bit row stands for its codes times its scale 2^e, exact in bf16 (past its largest, an infinity); keys and values
// become that on their way to the products, which are k_attn_window.hip's: S^T = K . Q^T, online softmax, O^T = V^T . P^T in bf16 with fp32 sums, weights
// rounded to bf16 (2^-8 of a weight, the sum is of the rounded ones).  The matrix unit would take the codes as they lie,
// with the scales in an operand of their own and the queries in two e4m3 parts, in as many cycles (8192 rows over 4096 keys
// 572 us, not 615); but it sums 8-bit products eight at a time to 13 bits below the largest of the eight (measured, with
// and without scales: a product of less than 2^-13 of its neighbour adds nothing), so that a channel in which keys and
// queries are large takes the others' bits: with products of up to 53 in the scores, outputs were 5 times further
// off than the bf16 roundings allow.
//
// Softmax over a union of key sets is joined from (o, m, l) of each.  So the keys that a group of sequences
// shares are attended once, by the rows of all of them (a prefix segment: rows of different sequences
// are columns of one block, each with its own position), and each sequence's other keys by its rows (an own
// segment).  Sequences that fill the columns of a block by themselves (kMemberCols) gain nothing from that and attend
// all their keys in their own segment.
//
// A workgroup takes one kv head of a block of a segment, in one of two forms.
// Narrow (4 or 8 waves, up to 16 columns, a column being a (row, q head of the kv head's group)): the key tiles go round
// the waves, each of which holds all the columns: nothing is shared until the waves' (o, m, l) are
// joined at the end.  K comes from memory in the layout of the product's operand (the order of the 128 dims
// within the sum is free, and Q's fragments are taken in the same order), V through registers into a tile of the
// wave's own in LDS, from which it is read transposed.  No barrier, a tile of loads in flight a wave (256 registers: in
// 128, half a tile at a time, 16 tokens over 4096 keys take 92 us, not 30).  Bound by latency for few keys (one token
// over 600 keys 8.6 us, of which the launch is 3; over 60000 33), by HBM past that (16 tokens over 4096
// keys each 29.9, 4.5 TB/s; 6.5 but for the 9 of a run of one tile).  Splits are joined by the last to arrive.
// Wide (4 or 8 waves of 16 columns): the tiles are staged in LDS for all waves, bf16 ones directly and
// double-buffered, 8-bit ones through registers.  Bound by the vector units (busy 54% of the cycles), LDS (48%) and
// the matrix units (41%), partly one after the other: 8192 rows over 4096 keys 611-622 us, 0.90-0.92 PFLOP/s.
// A batch with wide and few narrow items runs both in one launch; short narrow items that would fill the chip by themselves
// take a wave each there (64 sequences behind 1024 8-bit positions 19.5 -> 17.3 us, behind 16384 54 -> 51).  Rows with a prefix, or cut wide items, are
// joined by a launch of their own (4.0 us for 16 tokens, 5.5 for 64; joining the prefix's partials in the narrow
// kernel, behind a count, took longer than that launch).  Few prefix tiles a workgroup are bound by latency: 16 tokens
// behind 4992 bf16 positions take 19.1 us, of the first launch's 11 us 1 the arguments, 1.6 the first loads' addresses
// and the queries, 1.5 the first tile, 1.8 a tile, 1 the end.
#include <algorithm>
#include <atomic>
#include <chrono>
#include <cmath>

#include "ie_attn_tiles.h"

namespace ie {

namespace {

constexpr int NN = 4;  // waves of the narrow form's workgroups (8 where the plan says so)
constexpr int kNarrowCols = 16;

// A workgroup's work: rows r0 .. r0 + nr - 1 of a segment of n rows, one kv head, the tiles i0 .. i1 - 1
// of the segment's run: na blocks from a0 on (sinks), then those from b0 on.
struct Work {
  int g, n, nqb, splits, split, r0, nr, part0, i0, i1;
  int a0, na, b0;
  int p0, row0;     // own: position and batch row of the block's first row
  int first, end;   // prefix: its sequences
  int nkeys;        // keys of the segment: positions below
  int seq;          // own: the sequence; prefix: the one furthest back, whose table is read
  bool prefix;
  bool whole;       // its rows have no other partials
  bool with_prefix; // they have a prefix's
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

// Sequences of up to so many columns share a prefix; others fill blocks of the wide form by themselves.
constexpr int kMemberCols = 64;
// A sequence's own keys go to the narrow form: up to 16 columns, one block; and those of members, in blocks of 16.  (A member's
// long own keys are then read by each of its blocks: 4 x 16 rows of 32 heads over 20000 own keys of 8 bits take 77 us
// behind 64 shared positions, 52 without the group.)  A prefix never does.
__host__ __device__ __forceinline__ bool is_narrow(int n, int gs, bool member) {
  return n <= (member ? kMemberCols : kNarrowCols) >> gs;
}
// Rows of a block of the wide form.
__host__ __device__ __forceinline__ int block_rows(int gs, int waves) { return (16 * waves) >> gs; }

// Workgroup and item -> (segment, split, row block, kv head): kv heads go round the XCDs, whose L2 then holds the head's
// keys for the blocks that share them; prefixes come first, then the sequences, of each the last blocks (the
// longest runs) first.  (the segments' arguments in one go, a lane each)
template <bool NARROW>
__device__ __forceinline__ Work work_of(const AttnSharedParams& p, int waves, int item) {
  const int lane = threadIdx.x & 63, gs = p.group_shift;
  Work w;
  w.g = blockIdx.x % kKVHeads;
  w.prefix = !NARROW && item < p.prefix_items;
  int lo, hi, pmax;
  const int member_end = p.member_end[lane];
  if (w.prefix) {
    const int l = lane & 31;
    const int item_end = p.p_item_end[l], firsts = p.p_first[l], ends = p.p_end[l], splits = p.p_splits[l],
              part0 = p.p_part0[l], seqs = p.p_seq[l], blocks = p.p_blocks[l], starts = p.start[lane];
    const int k = __popcll(__ballot(lane < p.n_prefixes && item_end <= item));
    w.first = __builtin_amdgcn_readlane(firsts, k), w.end = __builtin_amdgcn_readlane(ends, k);
    w.splits = __builtin_amdgcn_readlane(splits, k), w.part0 = __builtin_amdgcn_readlane(part0, k);
    // (members before the prefix's)
    w.row0 = w.first ? __builtin_amdgcn_readlane(member_end, max(w.first - 1, 0)) : 0;
    w.n = __builtin_amdgcn_readlane(member_end, w.end - 1) - w.row0;
    item -= k ? __builtin_amdgcn_readlane(item_end, max(k - 1, 0)) : 0;
    w.seq = __builtin_amdgcn_readlane(seqs, k);
    w.p0 = __builtin_amdgcn_readlane(starts, w.seq);
    lo = 0, hi = __builtin_amdgcn_readlane(blocks, k);
    w.nkeys = hi * BKEY;
    w.whole = w.with_prefix = false;
    pmax = w.nkeys - 1;
  } else {
    item -= NARROW ? 0 : p.prefix_items;
    const int item_end = NARROW ? p.narrow_end[lane] : p.wide_end[lane], row_end = p.row_end[lane],
              starts = p.start[lane], splits = p.splits[lane], part0 = p.part0[lane], los = p.lo[lane],
              prefixes = p.prefix[lane];
    const int b = __popcll(__ballot(lane < p.n_seqs && item_end <= item)), before = max(b - 1, 0);
    w.seq = b, w.first = b, w.end = b + 1;
    w.splits = __builtin_amdgcn_readlane(splits, b), w.part0 = __builtin_amdgcn_readlane(part0, b);
    w.row0 = b ? __builtin_amdgcn_readlane(row_end, before) : 0;
    w.n = __builtin_amdgcn_readlane(row_end, b) - w.row0;
    item -= b ? __builtin_amdgcn_readlane(item_end, before) : 0;
    w.p0 = __builtin_amdgcn_readlane(starts, b);
    lo = __builtin_amdgcn_readlane(los, b), hi = kMaxLongCtx / BKEY;
    w.nkeys = w.p0 + w.n;
    w.with_prefix = __builtin_amdgcn_readlane(prefixes, b) >= 0;
    w.whole = w.splits == 1 && !w.with_prefix;
    pmax = 0;
  }
  const int rb = NARROW ? kNarrowCols >> gs : block_rows(gs, waves);
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
  w.table = p.block_tables + (size_t)w.seq * p.table_stride;
  return w;
}

// ---------------------------------------------------------------- columns
// The (batch row, position) of row r of the block.
struct RowPos {
  int row, pos;
};
__device__ __forceinline__ RowPos row_of(const AttnSharedParams& p, const Work& w, int r) {
  if (!w.prefix) return RowPos{w.row0 + r, w.p0 + r};
  // members' rows one after the other, row `at` of them all: the first sequence b with member_end > at
  const int lane = threadIdx.x & 63;
  const int member_end = lane < p.n_seqs ? p.member_end[lane] : INT32_MAX, row_end = p.row_end[lane],
            start = p.start[lane];
  const int at = w.row0 + w.r0 + r;
  int b = 0;
#pragma unroll
  for (int s = 32; s; s >>= 1) b += __shfl(member_end, b + s - 1, 64) <= at ? s : 0;
  const int m = __shfl(member_end, max(b - 1, 0), 64), e = __shfl(row_end, max(b - 1, 0), 64);
  const int before = b ? m : 0, rows = b ? e : 0;
  return RowPos{rows + at - before, __shfl(start, b, 64) + at - before};
}

// CODES: of the keys' operands made of 16 codes a lane (NarrowK): the dims 64 j + 16 G .. +16, j 0 and 1, of a row, in
// two operands each (which dims an operand holds is free, as long as keys and queries agree).
template <bool CODES>
struct Columns : ColumnState<1> {
  int least, most;  // of the wave's positions

  // Columns past the rows repeat the last row.
  __device__ __forceinline__ void load(const AttnSharedParams& p, const Work& w, int col0) {
    const int fr = threadIdx.x & 15, G = threadIdx.x >> 4 & 3, gs = p.group_shift;
    const int col = col0 + fr;
    const RowPos x = row_of(p, w, min(col >> gs, w.nr - 1));
    pos[0] = x.pos;
    const size_t at = ((size_t)x.row << gs << 3) + ((size_t)w.g << gs) + (col & ((1 << gs) - 1));
    const bf16x8_t* row = reinterpret_cast<const bf16x8_t*>(p.q + at * kHeadDim);
#pragma unroll
    for (int ks = 0; ks < 4; ++ks) q[0][ks] = row[CODES ? 8 * (ks >> 1) + 2 * G + (ks & 1) : 4 * ks + G];
    clear();
  }
  __device__ __forceinline__ void set() {
    int lo = pos[0], hi = pos[0];
#pragma unroll
    for (int s = 1; s < 16; s <<= 1) {
      lo = min(lo, __shfl_xor(lo, s, 64));
      hi = max(hi, __shfl_xor(hi, s, 64));
    }
    least = __builtin_amdgcn_readfirstlane(lo);
    most = __builtin_amdgcn_readfirstlane(hi);
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

// Codes and a scale that bf16 does not hold as numbers: bit 7 of a byte is set for a NaN code; scales past 2^119, whose
// codes may go past the largest bf16, count as such too.
__device__ __forceinline__ uint32_t nonfinite8(const u32x4_t& w, float scale) {
  uint32_t n = scale >= 0x1p120f ? 0x80u : 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) n |= (w[i] & 0x7F7F7F7Fu) + 0x01010101u;
  return n & 0x80808080u;
}

// 16 codes as two chunks of 8 bf16.
__device__ __forceinline__ void chunks_of(u32x4_t (&c)[2], const u32x4_t& w, float scale) {
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const u32x2v_t a = dequantise4(w[2 * i], scale), b = dequantise4(w[2 * i + 1], scale);
    c[i] = u32x4_t{a[0], a[1], b[0], b[1]};
  }
}

// A wave's columns from col0 on: what they come to, or a partial of it.
__device__ __forceinline__ void put(const AttnSharedParams& p, const Work& w, const ColumnState<1>& c, int col0) {
  const int fr = threadIdx.x & 15, G = threadIdx.x >> 4 & 3, gs = p.group_shift;
  const int heads = kKVHeads << gs;
  const int col = col0 + fr, r = col >> gs;
  if (r >= w.nr) return;
  const int h = (w.g << gs) + (col & ((1 << gs) - 1));
  if (!w.whole) {
    const size_t slot = ((size_t)w.part0 + (size_t)w.split * w.n + w.r0 + r) * heads + h;
    float* dst = p.part + slot * kHeadDim + 4 * G;
#pragma unroll
    for (int db = 0; db < 8; ++db) *reinterpret_cast<f32x4_t*>(dst + 16 * db) = c.o[0][db];
    if (G == 0) *reinterpret_cast<float2*>(p.part_ml + 2 * slot) = make_float2(c.m[0], c.l[0][0]);
  } else {
    const float inv = c.l[0][0] == 0.f ? 0.f : 1.0f / c.l[0][0];
    uint16_t* dst = p.out + ((size_t)(w.row0 + r) * heads + h) * kHeadDim;
#pragma unroll
    for (int db = 0; db < 8; ++db) {
      const u32x2_t v = {pack_bf2(c.o[0][db][0] * inv, c.o[0][db][1] * inv),
                         pack_bf2(c.o[0][db][2] * inv, c.o[0][db][3] * inv)};
      *reinterpret_cast<u32x2_t*>(dst + db * 16 + 4 * G) = v;
    }
  }
}

// ---------------------------------------------------------------- narrow form
// A wave's K tile as operands: lane (fr, G) holds of the rows fr + 16 kb (kb 0 .. 3) the dims 32 ks + 8 G .. +8 (bf16),
// or the codes 64 j + 16 G .. +16, j 0 and 1, two operands each.
template <bool F8, int AUX>
struct NarrowK {
  static constexpr int kLoads = F8 ? 2 : 4;
  u32x4_t w[4][kLoads];
  uint32_t scales;  // (of a row that is not there anything: no row sees it)
  __device__ __forceinline__ void issue(const Planes& x, int g) {
    const int fr = threadIdx.x & 15, G = threadIdx.x >> 4 & 3;
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
  __device__ __forceinline__ void scores(f32x4_t (&s)[1][4], const Columns<F8>& c) const {
#pragma unroll
    for (int kb = 0; kb < 4; ++kb) {
      u32x4_t a[4];
      if constexpr (F8) {
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          u32x4_t two[2];
          chunks_of(two, w[kb][j], scale_of(scales >> (8 * kb) & 0xFF));
          a[2 * j] = two[0], a[2 * j + 1] = two[1];
        }
      } else {
#pragma unroll
        for (int ks = 0; ks < 4; ++ks) a[ks] = w[kb][ks];
      }
      s[0][kb] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int ks = 0; ks < 4; ++ks)
        s[0][kb] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, a[ks]), c.q[0][ks], s[0][kb],
                                                           0, 0, 0);
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
  // CHECK: whether the tile has an infinity or a NaN (8 bits: or may have).  Masked tiles need it: those without run the
  // product of the others (a third of the instructions; 32 tokens over windows of 512 14.5 -> 12.2 us).
  template <bool CHECK>
  __device__ __forceinline__ bool stage(u32x4_t* tile) const {
    const int lane = threadIdx.x & 63;
    uint32_t bad = 0;
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      const int r = row(i);
      if constexpr (F8) {
        u32x4_t c[2];
        const float scale = scale_at_byte(scales[i & 1], i >> 1, r < rows);
        if constexpr (CHECK) bad |= nonfinite8(w[i], scale);
        chunks_of(c, w[i], scale);
        tile[kv_slot(r, 2 * (lane & 7))] = c[0];
        tile[kv_slot(r, 2 * (lane & 7) + 1)] = c[1];
      } else {
        if constexpr (CHECK)
#pragma unroll
          for (int e = 0; e < 4; ++e) bad |= nonfinite2(w[i][e]);
        tile[kv_slot(r, lane & 15)] = w[i];
      }
    }
    return CHECK && __ballot(bad != 0) != 0;
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
__device__ __forceinline__ void narrow_tiles(const AttnSharedParams& p, const Work& w, Columns<F8>& c, int from,
                                             int stride, u32x4_t* tile) {
  NarrowK<F8, AUX> k;
  NarrowV<F8, AUX> v;
  const Frags f;
  // The wave's tiles' pages, 64 at a time, a lane each: a load of each by itself would be waited for together with
  // the tile in flight.
  const int lane = threadIdx.x & 63;
  int pages = -1;
  const auto look_up = [&](int first) {
    const int i = first + stride * lane;
    pages = i < w.i1 ? w.table[w.tile(i)] : -1;
  };
  int i = w.i0 + from, n = 0;
  look_up(i);
  c.load(p, w, 0);
  int page = __builtin_amdgcn_readlane(pages, 0);
  {
    const Planes x = planes_of<F8>(p, w.g, page, w.nkeys - w.tile(i) * BKEY);
    k.issue(x, w.g);
    v.issue(x, w.g);
  }
  c.set();
#pragma unroll 1
  for (; i < w.i1; i += stride) {
    const bool there = page >= 0 && page < p.n_pages;
    const int key0 = w.tile(i) * BKEY;
    const Sight see = there ? sight(key0, c.least, c.most, p.window, p.n_sinks) : kNone;
    if ((++n & 63) == 0) look_up(i + stride);
    page = __builtin_amdgcn_readlane(pages, n & 63);
    // (past the last tile nothing is read)
    const Planes x = planes_of<F8>(p, w.g, page, w.nkeys - w.tile(i + stride) * BKEY);
    f32x4_t s[1][4];
    bf16x8_t pb[1][2];
    k.scores(s, c);
    k.issue(x, w.g);
    if (see == kAll)
      weights_grown<false>(pb, c, s, key0, p.window, p.n_sinks);
    else if (see == kSome)
      weights_grown<true>(pb, c, s, key0, p.window, p.n_sinks);
    bool bad = false;
    if (see == kAll)
      v.template stage<false>(tile);
    else if (see == kSome)
      bad = v.template stage<true>(tile);
    v.issue(x, w.g);
    // (the wave's own tile: the hardware does its LDS accesses in order; the compiler is held to it)
    asm volatile("" ::: "memory");
    if (bad)
      values<true>(c, pb, f, tile, key0, p.window, p.n_sinks);
    else if (see != kNone)
      values<false>(c, pb, f, tile, key0, p.window, p.n_sinks);
    asm volatile("" ::: "memory");
  }
}

// Adds the partials from..end - 1 of a row and head to j, four values of o and (m, l) of each: slot_of(i) is the i-th's
// slot.  AGENT: of workgroups of this launch.
template <bool AGENT, typename Slot>
__device__ __forceinline__ void add_splits(Joined& j, const AttnSharedParams& p, int from, int end, int d,
                                           const Slot& slot_of) {
  for (int s0 = from; s0 < end; s0 += 8) {
    f32x4_t po[8];
    float2 ml[8];
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      const size_t slot = slot_of(min(s0 + u, end - 1));
      const float *o = p.part + slot * kHeadDim + d, *m = p.part_ml + 2 * slot;
      if constexpr (AGENT) {
        ml[u] = agent_load2(m);
        const float2 a = agent_load2(o), b = agent_load2(o + 2);
        po[u] = f32x4_t{a.x, a.y, b.x, b.y};
      } else {
        ml[u] = *reinterpret_cast<const float2*>(m);
        po[u] = *reinterpret_cast<const f32x4_t*>(o);
      }
    }
    j.add(po, ml, end - s0);
  }
}

template <bool F8, int NW>
__device__ __forceinline__ void narrow(const AttnSharedParams& p, const Work& w, u32x4_t (*lds)[TC]) {
  __shared__ int s_last;
  __shared__ float2 ml_of[NW][kNarrowCols];  // (m, l) of the waves' columns, then of parts of the splits
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int tid = threadIdx.x, gs = p.group_shift, heads = kKVHeads << gs;
  const int ncols = w.nr << gs;
  Columns<F8> c;
  if (p.nt && w.nqb == 1)
    narrow_tiles<F8, 2>(p, w, c, wave, NW, lds[wave]);
  else
    narrow_tiles<F8, 0>(p, w, c, wave, NW, lds[wave]);
  // the waves' sums side by side: [column][128], and (m, l); the 16-byte pieces of a column in an order of its own (16
  // columns' meet no bank twice)
  {
    const int fr = tid & 15, G = tid >> 4 & 3;
    f32x4_t* mine = reinterpret_cast<f32x4_t*>(lds[wave]) + fr * 32;
#pragma unroll
    for (int db = 0; db < 8; ++db) mine[(4 * db + G) ^ fr] = c.o[0][db];
    if (G == 0) ml_of[wave][fr] = make_float2(c.m[0], c.l[0][0]);
  }
  __syncthreads();
  for (int i = tid; i < ncols * 32; i += 64 * NW) {
    const int col = i >> 5, d = 4 * (i & 31);
    f32x4_t po[NW];
    float2 ml[NW];
#pragma unroll
    for (int u = 0; u < NW; ++u) {
      po[u] = reinterpret_cast<const f32x4_t*>(lds[u])[col * 32 + ((i & 31) ^ col)];
      ml[u] = ml_of[u][col];
    }
    const int h = (w.g << gs) + (col & ((1 << gs) - 1)), r = col >> gs;
    Joined j;
    j.add(po, ml, NW);
    if (w.whole) {
      j.write(p.out + ((size_t)(w.row0 + r) * heads + h) * kHeadDim + d);
      continue;
    }
    const size_t slot = ((size_t)w.part0 + (size_t)w.split * w.n + w.r0 + r) * heads + h;
    if (w.with_prefix) {  // (joined by a launch of its own)
      *reinterpret_cast<f32x4_t*>(p.part + slot * kHeadDim + d) = j.o;
      if (d == 0) *reinterpret_cast<float2*>(p.part_ml + 2 * slot) = make_float2(j.M, j.L);
      continue;
    }
    agent_store2(p.part + slot * kHeadDim + d, j.o[0], j.o[1]);
    agent_store2(p.part + slot * kHeadDim + d + 2, j.o[2], j.o[3]);
    if (d == 0) agent_store2(p.part_ml + 2 * slot, j.M, j.L);
  }
  if (w.whole || w.with_prefix) return;
  // The last split of the sequence (one block: up to 16 columns) and kv head to arrive joins them, in the splits'
  // order.  The word that counts them is the caller's memory, which may hold anything: a count is one with this
  // call's tag, whatever else is there counts as none.  The last leaves 0.
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // the partials are there, before the arrival counts
  __syncthreads();
  if (tid == 0) {
    unsigned long long* word = p.arrived + w.seq * kKVHeads + w.g;
    unsigned long long cur = __hip_atomic_load(word, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT), next = 0;
    // (without this call's tag: the first to put it there counts one; with it, it stays until the last)
    while (cur >> 16 != p.tag && !next)
      if (__hip_atomic_compare_exchange_strong(word, &cur, p.tag << 16 | 1, __ATOMIC_RELAXED, __ATOMIC_RELAXED,
                                               __HIP_MEMORY_SCOPE_AGENT))
        next = p.tag << 16 | 1;
    if (!next) next = __hip_atomic_fetch_add(word, 1ull, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) + 1;
    const bool last = (int)(next & 0xFFFF) == w.splits;
    if (last) __hip_atomic_store(word, 0ull, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    s_last = last;
  }
  __syncthreads();
  if (!s_last) return;
  // few columns: several threads a (column, four values), a part of the splits each, joined through LDS
  const int pairs = ncols * 32, parts = max(1, 64 * NW / pairs), each = (w.splits + parts - 1) / parts;
  f32x4_t* part_o = reinterpret_cast<f32x4_t*>(lds[0]);
  for (int i = tid; i < parts * pairs; i += 64 * NW) {
    const int part = i / pairs, col = (i - part * pairs) >> 5, d = 4 * (i & 31);
    const int h = (w.g << gs) + (col & ((1 << gs) - 1)), r = col >> gs;
    const size_t step = (size_t)w.n * heads, slot0 = ((size_t)w.part0 + w.r0 + r) * heads + h;
    Joined j;
    add_splits<true>(j, p, part * each, min(part * each + each, w.splits), d,
                     [&](int s) { return slot0 + s * step; });
    if (parts == 1) {
      j.write(p.out + ((size_t)(w.row0 + r) * heads + h) * kHeadDim + d);
    } else {
      part_o[i] = j.o;
      if (d == 0) ml_of[0][part * ncols + col] = make_float2(j.M, j.L);
    }
  }
  if (parts == 1) return;
  __syncthreads();
  for (int i = tid; i < pairs; i += 64 * NW) {
    const int col = i >> 5, d = 4 * (i & 31);
    const int h = (w.g << gs) + (col & ((1 << gs) - 1)), r = col >> gs;
    Joined j;
    for (int k = 0; k < parts; ++k) {
      const f32x4_t o[1] = {part_o[k * pairs + i]};
      const float2 ml[1] = {ml_of[0][k * ncols + col]};
      j.add(o, ml, 1);
    }
    j.write(p.out + ((size_t)(w.row0 + r) * heads + h) * kHeadDim + d);
  }
}

// An item of a wave's own: no waves to join.
template <bool F8>
__device__ __forceinline__ void narrow_alone(const AttnSharedParams& p, const Work& w, u32x4_t* tile) {
  Columns<F8> c;
  if (p.nt && w.nqb == 1)
    narrow_tiles<F8, 2>(p, w, c, 0, 1, tile);
  else
    narrow_tiles<F8, 0>(p, w, c, 0, 1, tile);
  put(p, w, c, 0);
}

// ---------------------------------------------------------------- wide form
// A thread's part of an 8-bit tile: chunk at() of row row() (and of the row 32 on, with 4 waves) of K and V, which become
// bf16 on the way to LDS.  Rows and chunks go over the lanes so that eight lanes' stores are half a row and half of
// the row 4 on, whose swizzle differs: they meet no bank twice.
template <int NW>
struct Wide8 {
  static constexpr int kEach = 8 / NW;
  u32x4_t k[kEach], v[kEach];
  uint32_t ks, vs;  // the scales of rows row() % 16 + 16 i
  int rows;
  static __device__ __forceinline__ int row() {
    const int t = threadIdx.x;
    return (t >> 6) * 8 + (t >> 2 & 1) * 4 + (t >> 3 & 3);
  }
  static __device__ __forceinline__ int at() { return (threadIdx.x >> 5 & 1) * 4 + (threadIdx.x & 3); }
  template <int AUX>
  __device__ __forceinline__ void issue(const Planes& x, int g) {
    rows = x.rows;
    ks = __builtin_amdgcn_raw_buffer_load_b32(x.scales, 4 * (row() & 15), g * kPagePos, AUX);
    vs = __builtin_amdgcn_raw_buffer_load_b32(x.scales, 4 * (row() & 15), (kKVHeads + g) * kPagePos, AUX);
#pragma unroll
    for (int i = 0; i < kEach; ++i) {  // (the row 32 on has the same swizzle)
      k[i] = __builtin_amdgcn_raw_buffer_load_b128(x.k, row() * kHeadDim + at() * 16, 32 * i * kHeadDim, AUX);
      v[i] = __builtin_amdgcn_raw_buffer_load_b128(x.v, row() * kHeadDim + at() * 16, 32 * i * kHeadDim, AUX);
    }
  }
  __device__ __forceinline__ void stage(u32x4_t* kt, u32x4_t* vt, int wave) const {
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      const int r = row() + 32 * i, byte = (wave >> 1) + 2 * i;  // (8 rows a wave)
      const int first = kv_slot(r, 2 * at()), second = kv_slot(r, 2 * at() + 1);
      u32x4_t x[2];
      chunks_of(x, k[i], scale_at_byte(ks, byte, r < rows));
      kt[first] = x[0], kt[second] = x[1];
      chunks_of(x, v[i], scale_at_byte(vs, byte, r < rows));
      vt[first] = x[0], vt[second] = x[1];
    }
  }
};

template <bool F8, int NW>
__device__ __forceinline__ void wide(const AttnSharedParams& p, const Work& w, u32x4_t* kt, u32x4_t* vt) {
  constexpr int kAhead = 2;
  constexpr int kBuffer = F8 ? 0 : 1;  // (of two, or one)
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const bool idle = (wave * 16) >> p.group_shift >= w.nr;  // (no rows)
  const bool nt = p.nt && w.nqb == 1;
  const TileLoad<NW> ld(wave);
  Wide8<NW> raw;
  const auto planes = [&](int i, int page) { return planes_of<F8>(p, w.g, page, w.nkeys - w.tile(i) * BKEY); };
  // (past the last tile there are no bytes)
  const auto page_of = [&](int i) { return w.table[w.tile(min(i, w.i1 - 1))]; };
  const auto checked = [&](int i, int page) { return i < w.i1 ? __builtin_amdgcn_readfirstlane(page) : -1; };
  // 8 bits: to registers; bf16: to LDS.
  const auto issue = [&](int i, int page) {
    const Planes x = planes(i, page);
    u32x4_t *ks = kt + (i & kBuffer) * TC, *vs = vt + (i & kBuffer) * TC;
    if constexpr (F8) {
      if (nt) raw.template issue<2>(x, w.g);
      else raw.template issue<0>(x, w.g);
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
    const int here = page_of(w.i0);
    next = page_of(w.i0 + 1);
    page = checked(w.i0, here);
    issue(w.i0, page);
  }
  Columns<false> c;
  c.load(p, w, wave * 16);
  c.set();
  // The compiler does not see what the kernel's own waits cover: without one here it would guard the
  // fragments inside the loops, where that is a wait for the tile in flight.
  __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0)
  const Frags f;

  // Tile i is there, for all waves; tile i + 1 is on its way.  bf16: it has landed in LDS, and every wave is done with tile
  // i - 1, whose buffer tile i + 1 takes.  8 bits: it becomes bf16 in the one buffer, once every wave has left that; with
  // two buffers, and no barrier before, a CU holds two workgroups of four waves, not three (6 x 333 rows 88 -> 68
  // us, 8192 rows 626 -> 615).
  auto arrive = [&](int i) {
    if constexpr (F8) {
      asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
      raw.stage(kt, vt, wave);
    }
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
    page = checked(i + 1, next);
    issue(i + 1, page);
    next = page_of(i + 2);
  };
  auto tile_scores = [&](f32x4_t (&s)[1][4], int i) {
    scores(s, c, f, kt + (i & kBuffer) * TC);
    __builtin_amdgcn_sched_barrier(0);
  };
  const auto see = [&](int i) {
    return page >= 0 && page < p.n_pages ? sight(w.tile(i) * BKEY, c.least, c.most, p.window, p.n_sinks) : kNone;
  };
  // Tiles that all rows see in full, one after the other, in a loop of their own: with the other kinds in
  // one body the compiler moves the sums between two sets of registers in each step.
  if (idle)
    for (int i = w.i0; i < w.i1; ++i) arrive(i);
  for (int i = idle ? w.i1 : w.i0; i < w.i1;) {
#pragma unroll 1
    for (; i < w.i1 && see(i) == kAll; ++i) {
      arrive(i);
      f32x4_t s[1][4];
      bf16x8_t pb[1][2];
      tile_scores(s, i);
      weights_grown<false>(pb, c, s, 0, p.window, p.n_sinks);
      values<false, kAhead>(c, pb, f, vt + (i & kBuffer) * TC, 0, p.window, p.n_sinks);
    }
    if (i == w.i1) break;
    const bool some = see(i) == kSome;
    arrive(i);
    if (some) {
      const int key0 = w.tile(i) * BKEY;
      f32x4_t s[1][4];
      bf16x8_t pb[1][2];
      tile_scores(s, i);
      weights_grown<true>(pb, c, s, key0, p.window, p.n_sinks);
      __builtin_amdgcn_sched_barrier(0);  // (no fragments held over the softmax: registers)
      values<true>(c, pb, f, vt + (i & kBuffer) * TC, key0, p.window, p.n_sinks);
    }
    ++i;
  }

  put(p, w, c, wave * 16);
}

template <bool F8, int NW>
__global__ __launch_bounds__(64 * NW, 2) void attn_shared_narrow_kernel(AttnSharedParams p) {
  __shared__ u32x4_t lds[NW][TC];
  narrow<F8, NW>(p, work_of<true>(p, 1, blockIdx.x / kKVHeads), lds);
}

// Both forms; the narrow items a workgroup each, or a wave each where they are short and many.
template <bool F8, bool ALONE>
__global__ __launch_bounds__(64 * NN, 2) void attn_shared_both_kernel(AttnSharedParams p) {
  __shared__ u32x4_t lds[NN][TC];
  const int item = blockIdx.x / kKVHeads - p.wide_items;
  if (item < 0) {
    wide<F8, NN>(p, work_of<false>(p, NN, blockIdx.x / kKVHeads), lds[0], lds[2]);
  } else if constexpr (ALONE) {
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), mine = item * NN + wave;
    if (mine < p.narrow_items) narrow_alone<F8>(p, work_of<true>(p, 1, mine), lds[wave]);
  } else {
    narrow<F8, NN>(p, work_of<true>(p, 1, item), lds);
  }
}

template <bool F8, int NW>
__global__ __launch_bounds__(64 * NW, NW == 8 ? 4 : F8 ? 3 : 2) void attn_shared_wide_kernel(AttnSharedParams p) {
  constexpr int kTiles = F8 ? 1 : 2;
  __shared__ u32x4_t kt[kTiles * TC], vt[kTiles * TC];
  wide<F8, NW>(p, work_of<false>(p, NW, blockIdx.x / kKVHeads), kt, vt);
}

// Joins the partials of each (row, q head) that has more than one, but for those that the narrow form has joined: 32
// lanes each, 4 dims a lane, the prefix's splits first, then the row's own; PARTS threads share a lane's splits.
template <int PARTS>
__global__ __launch_bounds__(256) void attn_shared_merge_kernel(AttnSharedParams p) {
  constexpr int kEach = 8 / PARTS;  // (row, head) pairs a workgroup
  const int lane = threadIdx.x & 63;
  const int row_end = p.row_end[lane], member_end = p.member_end[lane], lane_splits = p.splits[lane],
            part0 = p.part0[lane], prefix = p.prefix[lane];
  const int heads = kKVHeads << p.group_shift;
  const int row = p.merge_row0 + blockIdx.x * kEach / heads;  // (heads is a multiple of 8)
  const int b = __popcll(__ballot(lane < p.n_seqs && row_end <= row)), before = max(b - 1, 0);
  const int k = __builtin_amdgcn_readlane(prefix, b), splits = __builtin_amdgcn_readlane(lane_splits, b);
  const int row0 = b ? __builtin_amdgcn_readlane(row_end, before) : 0;
  const int n = __builtin_amdgcn_readlane(row_end, b) - row0;
  if (k < 0 && (splits < 2 || is_narrow(n, p.group_shift, false))) return;  // (the whole workgroup)
  const int part = threadIdx.x / (32 * kEach), pair = (threadIdx.x >> 5) % kEach;
  const int h = blockIdx.x * kEach % heads + pair, d = (threadIdx.x & 31) * 4;
  size_t pre = 0, pre_step = 0;
  int n_pre = 0;
  if (k >= 0) {
    const int first = p.p_first[k], end = p.p_end[k], p_part0 = p.p_part0[k];
    n_pre = p.p_splits[k];
    const int base = first ? __builtin_amdgcn_readlane(member_end, max(first - 1, 0)) : 0;
    const int all = __builtin_amdgcn_readlane(member_end, end - 1) - base;
    const int at = (b ? __builtin_amdgcn_readlane(member_end, before) : 0) - base + row - row0;
    pre = ((size_t)p_part0 + at) * heads + h, pre_step = (size_t)all * heads;
  }
  const size_t own = ((size_t)__builtin_amdgcn_readlane(part0, b) + row - row0) * heads + h, own_step = (size_t)n * heads;
  // this part's share of the two lists, one behind the other
  const int count = n_pre + splits, each = (count + PARTS - 1) / PARTS;
  Joined j;
  add_splits<false>(j, p, part * each, min(part * each + each, count), d,
                    [&](int s) { return s < n_pre ? pre + s * pre_step : own + (s - n_pre) * own_step; });
  if constexpr (PARTS > 1) {
    __shared__ f32x4_t part_o[PARTS][kEach][32];
    __shared__ float2 part_ml[PARTS][kEach];
    part_o[part][pair][threadIdx.x & 31] = j.o;
    if (d == 0) part_ml[part][pair] = make_float2(j.M, j.L);
    __syncthreads();
    if (part) return;
    f32x4_t o[PARTS];
    float2 ml[PARTS];
#pragma unroll
    for (int u = 0; u < PARTS; ++u) o[u] = part_o[u][pair][threadIdx.x & 31], ml[u] = part_ml[u][pair];
    j = Joined();
    j.add(o, ml, PARTS);
  }
  j.write(p.out + ((size_t)row * heads + h) * kHeadDim + d);
}

constexpr int kMaxSplits = 64;

// Rows of at most `rows` that share a prefix.
int members_of(int rows, int heads) { return std::min(rows, kMaxSeqs * std::max(1, kMemberCols / (heads / kKVHeads))); }
// Partial rows (a row and split) that a workspace for `rows` rows holds: 64 splits of up to 64 rows, and a
// prefix's and an own partial of each row that shares.  It never falls with the rows.
long long part_rows(int rows, int heads) {
  return (long long)std::min(rows, 64) * kMaxSplits + 2ll * members_of(rows, heads);
}

constexpr size_t kArrivedBytes = (size_t)kMaxSeqs * kKVHeads * sizeof(unsigned long long);

// A call's tag of the arrival counts, 48 bits.
unsigned long long next_tag() {
  // (from a place of its own in each process)
  static std::atomic<unsigned long long> n{
      splitmix64((unsigned long long)std::chrono::steady_clock::now().time_since_epoch().count() ^
                 splitmix64(reinterpret_cast<uintptr_t>(&n)))};
  const unsigned long long t = n.fetch_add(1, std::memory_order_relaxed) & ((1ull << 48) - 1);
  return t ? t : next_tag();
}

// A segment as the plan sees it.
struct Segment {
  int n, tiles;  // rows; tiles of its longest row block
  double mean;   // and of a row block in the mean
  bool narrow, parts;  // its form; it leaves partials even where it is not cut
};

int blocks_of(const Segment& x, int gs, int columns) { return (x.n + (columns >> gs) - 1) / (columns >> gs); }

// The join takes a lane's splits by four threads where that fills a launch.
bool few_pairs(int rows, int gs) { return rows < 512 >> gs; }

// What is launched: `both` forms in one kernel (the wide one with 4 waves, the narrow items a wave each if `alone`), or each
// in its own; the tiles a split of either form.
struct Plan {
  bool both, alone;
  int waves, wide, narrow;
  int nwaves = NN;  // of the narrow kernel
  int splits(const Segment& x) const {
    // (16 tiles, four a wave, take as long as the join of two halves does)
    if (x.narrow && !x.parts && x.tiles <= 16) return 1;
    const int t = x.narrow ? narrow : wide;
    return std::clamp((x.tiles + t - 1) / t, 1, kMaxSplits);
  }
};

// A form's time for a tile where 1, 2 or 3 workgroups share a CU (0: they do not fit), us.  Measured over 196 tiles
// of 30 rows, 66 of 8192 rows and 67-126 of four sequences of 742-2500 rows (32 heads); 8 bits: by these and 25 more
// batches, all counts of splits of each form.
struct Rate {
  int waves;
  double c[3];
};
constexpr Rate kRates[2][3] = {{{8, {1.92, 2.33, 0}}, {4, {1.75, 1.75, 0}}, {4, {1.75, 1.9, 0}}},    // bf16; the last:
                               {{8, {1.83, 2.1, 0}}, {4, {1.18, 1.5, 2.0}}, {4, {1.15, 1.6, 0}}}};  // both forms

// The time of `items` workgroups of `us` (at one a CU) each, by the rates' growth with their number; even: 1 where they are
// all as long as the longest, 0 where half as long in the mean.
double turns(const Rate& r, double items, double us, double even) {
  const int most = r.c[2] > 0 ? 3 : 2;
  const double round = 256 * most, each = us / r.c[0];
  const auto part = [&](double n) { return each * r.c[n > 512 ? 2 : n > 256 ? 1 : 0]; };
  if (items <= round) return part(items);
  // (the longest come first, so that more than a round ends evenly)
  const double mixed = each * r.c[most - 1] * items / round + 0.25 * us;
  if (items > 2 * round) return mixed;
  // equal ones: the second round takes what its workgroups take by themselves (2048 rows over 2048 8-bit keys each 89 us, 2100
  // and 3000 rows 134 with 8 waves, 128 and 150 with 4)
  return mixed + even * (each * r.c[most - 1] + part(items - round) - mixed);
}

// The launches with the least modelled time.  A workgroup starts and ends in 4 us and takes its tiles (1.5 more for the
// masked ones of a run), a narrow one 1.25 for four, and all narrow ones what HBM takes for their keys; a launch more is
// 3, the join 4.5 and 0.2 a split (0.06 by four threads), its partials written and read at 5 TB/s.  8 bits: within 6% of the
// best of 14 split counts and all forms over 29 batches of 1-8192 rows, with prefixes and without (1 x 200 rows over
// 16000 keys 371 us uncut, 89 in 8; 2500 rows 79 uncut, 111 in two; 2 x 1000 over 4096 keys 165 and 177), within 12% over
// six of 64 sequences behind a prefix.  bf16: within 12% over 13 batches, and over five of 64 sequences behind a prefix; a sixth, 64
// rows behind 1024 positions with 200 of their own, takes 24 us, not 19.
Plan plan_of(const Segment* x, int n, int rows, bool prefixes, bool fp8, int gs, long long room) {
  long long narrow = 0, narrow_runs = 0;
  int wide_longest = 0, narrow_longest = 0, narrow_items = 0;
  bool any_narrow = false;
  const Segment* wide[kMaxPrefixes + kMaxSeqs];
  int n_wide = 0;
  for (int i = 0; i < n; ++i) {
    if (!x[i].n) continue;
    if (x[i].narrow) {
      narrow += (long long)x[i].tiles * blocks_of(x[i], gs, kNarrowCols);
      narrow_runs += x[i].tiles;
      narrow_longest = std::max(narrow_longest, x[i].tiles);
      any_narrow = true;
    } else {
      wide_longest = std::max(wide_longest, x[i].tiles);
      wide[n_wide++] = x + i;
    }
  }
  Plan best{false, false, 8, 1, 4, NN};
  // narrow: a workgroup a CU, in whole rounds of its waves, two at least
  best.narrow = NN * (int)std::max<long long>(2, (narrow * kKVHeads + 256 * NN - 1) / (256 * NN));
  // (halves of unequal runs are no better than a run)
  if (2 * narrow_longest <= 3 * best.narrow) best.narrow = std::max(narrow_longest, 1);
  double narrow_us = 0;
  if (any_narrow) {
    for (int i = 0; i < n; ++i)
      if (x[i].n && x[i].narrow) narrow_items += best.splits(x[i]) * blocks_of(x[i], gs, kNarrowCols) * kKVHeads;
    // A run of few tiles, where a workgroup has a CU for itself: by eight waves in two steps, not three (8 bits: 5 tiles 7.6 ->
    // 7.2 us, 10 tiles 9.1 -> 8.7; of 16 tiles on, and with twice the bytes, a CU's loads take the time: 2-5% slower, and
    // with more workgroups than CUs 18-49%).
    if (fp8 && narrow_longest > NN && narrow_longest <= 3 * NN && narrow_items <= 256) best.nwaves = 8;
    narrow_us = 1.25 * ((std::min(best.narrow, narrow_longest) + NN - 1) / NN);
  }
  // what the narrow segments' keys take at 5.5 TB/s
  const double narrow_hbm = 4 + narrow_runs * (double)(kKVHeads * BKEY) * (fp8 ? 2 * kHeadDim + 2 : 4 * kHeadDim) / 5.5e6;
  double least = 1e30;
  for (int form = 0; form < 4 && wide_longest; ++form) {
    const bool both = form >= 2, alone = form == 3;
    // (a wave each: uncut items that would fill the chip with workgroups)
    if (both && (!any_narrow || (alone && (narrow_longest > best.narrow || narrow_items < 512)))) continue;
    const Rate& r = kRates[fp8][std::min(form, 2)];
    const double small = alone ? (double)narrow_items / NN : narrow_items;  // workgroups
    const double small_us = 4 + (alone ? 1.25 * narrow_longest : narrow_us);
    int tried = 0;
    for (const int k : {1, 2, 3, 4, 6, 8, 10, 12, 16, 20, 26, 32, 48, kMaxSplits}) {
      Plan plan = best;
      plan.both = both, plan.alone = alone, plan.waves = r.waves, plan.wide = (wide_longest + k - 1) / k;
      if (k > wide_longest || plan.wide == tried) continue;
      tried = plan.wide;
      double items = 0, tiles = 0, parts = 0;
      int most = 1;  // splits
      for (int i = 0; i < n_wide; ++i) {
        const Segment& y = *wide[i];
        const int s = plan.splits(y), b = blocks_of(y, gs, 16 * r.waves);
        items += (double)s * b * kKVHeads;
        tiles += y.mean * b * kKVHeads;
        if (s > 1 || y.parts) parts += (double)y.n * s;
        most = std::max(most, s);
      }
      const double each = 4 + (tiles / items + 1.5) * r.c[0];
      const double even = std::clamp(2 * tiles / (items * plan.wide) - 1, 0.0, 1.0);
      double cost = std::max(both ? turns(r, items + small, (items * each + small * small_us) / (items + small), even)
                                  : turns(r, items, each, even),
                             4 + (plan.wide + 1.5) * r.c[0]);
      if (!both && any_narrow) cost += 3 + std::max(turns(kRates[fp8][2], narrow_items, 4 + narrow_us, 0), narrow_hbm);
      if (both) cost = std::max(cost, narrow_hbm);
      if (parts || prefixes)
        cost += 4.5 + (few_pairs(rows, gs) ? 0.06 : 0.2) * most + parts * (kKVHeads << gs) * (kHeadDim + 2) * 4 * 2 / 5e6;
      if (cost < least) least = cost, best = plan;
    }
  }
  // (at one split a segment the partials fit)
  for (;;) {
    long long part = 0;
    for (int i = 0; i < n; ++i) {
      const int k = best.splits(x[i]);
      if (k > 1 || x[i].parts) part += (long long)x[i].n * k;
    }
    if (part <= room) return best;
    best.wide *= 2, best.narrow *= 2;
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
    const auto member = [&](int b) { return s.n_new[b] && s.n_new[b] <= kMemberCols >> gs; };
    int many = 0, back = b0, first = b0;
    for (int b = b0; b < b1; ++b) {
      if (!member(b)) continue;
      if (!many++) first = back = b;
      if (s.start[b] < s.start[back]) back = b;
    }
    if (!blocks || many < 2) continue;
    const int k = p.n_prefixes++;
    // The table row of the member furthest back is read: behind a window the others' may have lost pages that it
    // still sees, while what it has lost none of them sees.  (One without new rows may be over, its pages gone.)
    p.p_first[k] = first, p.p_end[k] = b1, p.p_blocks[k] = blocks, p.p_seq[k] = back;
    for (int b = b0; b < b1; ++b)
      if (member(b)) p.prefix[b] = k, p.lo[b] = blocks;
  }
  Segment all[kMaxPrefixes + kMaxSeqs];  // the prefixes, then the sequences
  for (int b = 0; b < s.n; ++b) {
    const int n = s.n_new[b];
    p.start[b] = s.start[b];
    p.row_end[b] = rows += n;
    p.member_end[b] = members += p.prefix[b] >= 0 ? n : 0;
    keys += std::min(s.start[b] + n - p.lo[b] * BKEY, p.window + p.n_sinks + n);
  }
  if (!rows) return IE_OK;
  Segment* const pre = all;
  Segment* const own = all + p.n_prefixes;
  for (int k = 0; k < p.n_prefixes; ++k) {
    const int n = p.member_end[p.p_end[k] - 1] - (p.p_first[k] ? p.member_end[p.p_first[k] - 1] : 0);
    keys += p.p_blocks[k] * BKEY;
    const int tiles = run_of(s.start[p.p_seq[k]], p.p_blocks[k] * BKEY - 1, 0, p.p_blocks[k], p.window, p.n_sinks).count;
    pre[k] = {n, tiles, (double)tiles, false, true};
  }
  for (int b = 0; b < s.n; ++b) {
    const int n = s.n_new[b], rb = block_rows(gs, 8), last = n ? (n - 1) / rb : 0;
    own[b] = {n, 0, 0, is_narrow(n, gs, p.prefix[b] >= 0), p.prefix[b] >= 0};
    if (!n) continue;
    const auto tiles = [&](int block) {
      const int r0 = block * rb;
      return run_of(s.start[b] + r0, s.start[b] + std::min(r0 + rb, n) - 1, p.lo[b], kMaxLongCtx / BKEY, p.window,
                    p.n_sinks).count;
    };
    for (int i = 0; i < 8; ++i) {
      const int x = tiles((int)((long long)last * i / 7));
      own[b].tiles = std::max(own[b].tiles, x);
      own[b].mean += x / 8.0;
    }
  }
  const Plan plan = plan_of(all, p.n_prefixes + s.n, rows, p.n_prefixes > 0, fp8, gs, part_rows(rows, heads));
  // splits, items and partial rows, segment by segment
  int wide = 0, narrow = 0, part = 0;
  bool merge = false, tagged = false;
  for (int k = 0; k < p.n_prefixes; ++k) {
    p.p_splits[k] = plan.splits(pre[k]);
    p.p_part0[k] = part;
    part += pre[k].n * p.p_splits[k];
    wide += p.p_splits[k] * blocks_of(pre[k], gs, 16 * plan.waves);
    p.p_item_end[k] = wide;
  }
  p.prefix_items = wide;
  for (int b = 0; b < s.n; ++b) {
    const Segment& x = own[b];
    const int splits = p.splits[b] = plan.splits(x);
    p.part0[b] = part;
    if (x.n && x.narrow) {
      narrow += splits * blocks_of(x, gs, kNarrowCols);
      part += splits > 1 || x.parts ? x.n * splits : 0;
      tagged |= splits > 1;
      merge |= x.parts;
    } else if (x.n) {
      wide += splits * blocks_of(x, gs, 16 * plan.waves);
      part += splits > 1 ? x.n * splits : 0;
      merge |= splits > 1;
    }
    p.narrow_end[b] = narrow;
    p.wide_end[b] = wide - p.prefix_items;
  }
  // a batch whose keys of all layers are about the 256 MB cache and more (2048 are 268 MB in bf16, 135 in 8 bits) finds
  // few of them there: such keys, where one workgroup reads them, pass it by
  p.nt = keys > 2048;
  p.arrived = static_cast<unsigned long long*>(workspace);
  p.tag = tagged ? next_tag() : 0;
  p.part = reinterpret_cast<float*>(static_cast<char*>(workspace) + kArrivedBytes);
  p.part_ml = p.part + (size_t)part * heads * kHeadDim;
  p.wide_items = plan.both ? wide : 0;
  p.narrow_items = narrow;
  if (plan.both) {
    const dim3 grid((wide + (plan.alone ? (narrow + NN - 1) / NN : narrow)) * kKVHeads), block(64 * NN);
    if (fp8 && plan.alone)
      hipLaunchKernelGGL((attn_shared_both_kernel<true, true>), grid, block, 0, st, p);
    else if (fp8)
      hipLaunchKernelGGL((attn_shared_both_kernel<true, false>), grid, block, 0, st, p);
    else if (plan.alone)
      hipLaunchKernelGGL((attn_shared_both_kernel<false, true>), grid, block, 0, st, p);
    else
      hipLaunchKernelGGL((attn_shared_both_kernel<false, false>), grid, block, 0, st, p);
    IE_CHECK_LAUNCH();
    wide = narrow = 0;
  }
  if (wide) {
    const dim3 grid(wide * kKVHeads), block(64 * plan.waves);
    if (fp8 && plan.waves == 8)
      hipLaunchKernelGGL((attn_shared_wide_kernel<true, 8>), grid, block, 0, st, p);
    else if (fp8)
      hipLaunchKernelGGL((attn_shared_wide_kernel<true, 4>), grid, block, 0, st, p);
    else if (plan.waves == 8)
      hipLaunchKernelGGL((attn_shared_wide_kernel<false, 8>), grid, block, 0, st, p);
    else
      hipLaunchKernelGGL((attn_shared_wide_kernel<false, 4>), grid, block, 0, st, p);
    IE_CHECK_LAUNCH();
  }
  if (narrow) {
    const dim3 grid(narrow * kKVHeads), block(64 * plan.nwaves);
    if (fp8 && plan.nwaves == 8)
      hipLaunchKernelGGL((attn_shared_narrow_kernel<true, 8>), grid, block, 0, st, p);
    else if (fp8)
      hipLaunchKernelGGL((attn_shared_narrow_kernel<true, 4>), grid, block, 0, st, p);
    else
      hipLaunchKernelGGL((attn_shared_narrow_kernel<false, 4>), grid, block, 0, st, p);
    IE_CHECK_LAUNCH();
  }
  if (merge) {
    // (few rows: their partials a few at a time; a grid holds 2^32 threads)
    constexpr int kRows = 1 << 20;
    if (few_pairs(rows, gs)) {
      hipLaunchKernelGGL((attn_shared_merge_kernel<4>), dim3(rows << gs << 2), dim3(256), 0, st, p);
      IE_CHECK_LAUNCH();
    } else {
      for (; p.merge_row0 < rows; p.merge_row0 += kRows) {
        const int n = std::min(rows - p.merge_row0, kRows);
        hipLaunchKernelGGL((attn_shared_merge_kernel<1>), dim3(n << gs), dim3(256), 0, st, p);
        IE_CHECK_LAUNCH();
      }
    }
  }
  return IE_OK;
}

}  // namespace ie
