// Attention of ragged chunks of new tokens over the paged K/V cache, with a sliding window and
// sinks (no reference counterpart: the reference attends one sequence, all keys, one plane).
//
// Sequence b's new rows sit at positions start .. start + n_new - 1; the row at position p sees the
// keys j <= p with j > p - window or j < n_sinks whose page is there:
//   o = sum_j softmax_j(q . k_j / sqrt(128)) v_j,  zeros where it sees none.
//
// A workgroup of 4 waves takes one kv head and a block of query columns, 16 or 32 a wave, a column
// being a (row, q head of the kv head's group): consecutive columns are the group's heads, then the
// next row, so that a single token of a 4-head group fills 4 of a wave's 16 columns and a chunk fills
// all of them, whatever the group.  It walks the 64-key tiles that the block's rows see (a tile is a page:
// the sink tiles, then the window's), each staged once in LDS for all its waves.  Per tile and wave, with
// v_mfma_f32_16x16x32_bf16:
//   S^T[key][col] = K . Q^T       (A = K rows from LDS, B = Q fragments in registers)
//   online softmax per column     (running max and sum in fp32)
//   O^T[d][col] += V^T . P^T      (P^T straight from the S^T accumulators, rounded to bf16: at most
//                                  half a step, 2^-8, a weight, and the sum l is of the rounded weights)
// K and V go global -> LDS by direct loads, row-major with swizzled 16-byte chunks, double-buffered;
// V^T fragments are transposed LDS reads (ds_read_b64_tr_b16).  Rows past the sequence's end read
// as zero (buffer bounds).
//
// Few columns over many keys: the tiles are cut into splits, a workgroup each, whose (o, m, l) go to
// the caller's workspace in fp32 and are combined by a second kernel.
//
// Measured (32 q heads): one token over 600 keys 9.6-10.1 us (6.0 and 4.0 for the merge: two launches' starts, one
// tile of work); one token of 16 sequences over 4096 keys 47.5, of which 43 read their 268 MB at 6.2 TB/s; 8192 rows
// over 4096 keys each 598, 611 and 647 on three cards, 0.86-0.93 PF: the MFMAs are busy 45% of the cycles and the
// vector units 60% (exponents, maxima, rescales, packing), and the fragment reads of a CU's 8 waves take about 0.9
// of a tile step's 2.24 (128 KiB at 382 B/ns and 128 at 238), which two waves a SIMD overlap in part; 6 sequences
// of up to 333 rows over 1500 keys 72: 328 workgroups, so that 72 CUs hold two and set the time (cut in three over the
// keys the merge's 20 MB of partials a split take what that gains: 75).
#include <algorithm>

#include "ie_kernels.h"

namespace ie {

namespace {

typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef short short4_t __attribute__((ext_vector_type(4)));
typedef float f32x4_t __attribute__((ext_vector_type(4)));
typedef unsigned int u32x2_t __attribute__((ext_vector_type(2)));
typedef __attribute__((address_space(3))) void lds_void;
typedef __attribute__((address_space(3))) short4_t lds_short4;

constexpr int BKEY = kPagePos;        // keys per tile: a page
constexpr int TC = BKEY * 16;         // 16-byte chunks per K (or V) tile
constexpr int kRowBytes = kHeadDim * 2;
constexpr int kBufferFlags = 0x00020000;  // buffer descriptor word 3 (raw 32-bit access)
constexpr float kScoreScale = 0.08838834764831845f * 1.4426950408889634f;  // 1/sqrt(128) * log2(e)

// Chunk c of key row r at slot c ^ swz(r), swz the bijection b3 b2 b1 b0 -> (b2^b3) b1 b0 b2 of the
// row's low bits: no bank conflicts for the K fragment reads (16 rows of a chunk column) nor
// for the transposed V reads (rows 4G..4G+3, or 8j..8j+7, of a chunk pair).
__device__ __forceinline__ int kv_swz(int r) {
  return ((((r >> 2) ^ (r >> 3)) & 1) << 3) | ((r & 3) << 1) | ((r >> 2) & 1);
}
__device__ __forceinline__ int kv_slot(int r, int c) { return r * 16 + (c ^ kv_swz(r)); }

// The tiles that the rows at positions p0 .. p1 see: tile i is block i of the first `sinks`, then
// first, first + 1, ...; `count` in all.  Host and device agree on it.
struct TileRun {
  int sinks, first, count;
};
__host__ __device__ __forceinline__ TileRun tile_run(int p0, int p1, int window, int n_sinks) {
  const int oldest = p0 - window + 1;
  TileRun r;
  r.first = oldest > 0 ? oldest / BKEY : 0;
  const int st = (n_sinks + BKEY - 1) / BKEY;
  r.sinks = st < r.first ? st : r.first;
  r.count = r.sinks + p1 / BKEY - r.first + 1;
  return r;
}

// Both halves of a dword as bf16: true where one of them is an infinity or a NaN.
__device__ __forceinline__ uint32_t nonfinite2(uint32_t w) {
  return ((w & 0x7F807F80u) + 0x00800080u) & 0x80008000u;
}

// A workgroup's work: the rows r0 .. r0 + nr - 1 (positions p0 ..) of sequence b's new rows, one kv
// head, the tiles i0 .. i1 - 1 of the run that they see.
struct Work {
  int g, b, row0, n_new, nqb, splits, split, r0, nr, p0, nkeys, i0, i1;
  TileRun run;
  const int* table;
  __device__ __forceinline__ int tile(int i) const { return i < run.sinks ? i : run.first + i - run.sinks; }
};

// Workgroup -> (sequence, split, row block, kv head): kv heads go round the XCDs, whose L2 then holds the
// head's keys for the blocks that share them; a sequence's last blocks (the longest runs) come first.
// (the sequences' arguments in one go, a lane each: one after the other they are a wait each)
__device__ __forceinline__ Work work_of(const AttnWindowParams& p, int columns) {
  const int lane = threadIdx.x & 63;
  const int item_end = p.item_end[lane], row_end = p.row_end[lane], start = p.start[lane],
            splits = p.splits[lane];
  Work w;
  w.g = blockIdx.x % kKVHeads;
  const int item = blockIdx.x / kKVHeads;
  w.b = __popcll(__ballot(lane < p.n_seqs && item_end <= item));
  const int before = max(w.b - 1, 0);
  w.row0 = w.b ? __builtin_amdgcn_readlane(row_end, before) : 0;
  w.n_new = __builtin_amdgcn_readlane(row_end, w.b) - w.row0;
  w.splits = __builtin_amdgcn_readlane(splits, w.b);
  const int first = __builtin_amdgcn_readlane(start, w.b);
  const int local = item - (w.b ? __builtin_amdgcn_readlane(item_end, before) : 0);
  const int rb = columns >> p.group_shift;
  w.nqb = (w.n_new + rb - 1) / rb;
  w.r0 = (w.nqb - 1 - local % w.nqb) * rb;
  w.split = local / w.nqb;
  w.nr = min(rb, w.n_new - w.r0);
  w.p0 = first + w.r0;
  w.nkeys = first + w.n_new;
  w.run = tile_run(w.p0, w.p0 + w.nr - 1, p.window, p.n_sinks);
  const int tps = (w.run.count + w.splits - 1) / w.splits;
  w.i0 = min(w.run.count, w.split * tps);
  w.i1 = min(w.run.count, w.i0 + tps);
  w.table = p.block_tables + (size_t)w.b * p.table_stride;
  return w;
}

// A wave's query columns: lane fr of each group of 16 holds column col0 + 16 qi + fr.
template <int QI>
struct Columns {
  bf16x8_t q[QI][4];  // Q^T fragments: Q[column][32 ks + 8 G .. +8]
  int pos[QI];        // the columns' positions
  f32x4_t o[QI][8];   // unnormalised: [db][r] = O[column][16 db + 4 G + r]
  float m[QI];        // running max of the raw scores (the scale is applied inside the exponent)
  f32x4_t l[QI];      // [0]: the running sum (the ones-MFMA's other rows are not rescaled)

  // columns past the rows repeat the last row
  __device__ __forceinline__ void load(const AttnWindowParams& p, const Work& w, int col0) {
    const int fr = threadIdx.x & 15, G = threadIdx.x >> 4 & 3, gs = p.group_shift;
#pragma unroll
    for (int qi = 0; qi < QI; ++qi) {
      const int col = col0 + 16 * qi + fr, r = min(col >> gs, w.nr - 1);
      pos[qi] = w.p0 + r;
      const size_t at = ((size_t)(w.row0 + w.r0 + r) << gs << 3) + ((size_t)w.g << gs) + (col & ((1 << gs) - 1));
      const u32x4_t* row = reinterpret_cast<const u32x4_t*>(p.q + at * kHeadDim);
#pragma unroll
      for (int ks = 0; ks < 4; ++ks) q[qi][ks] = __builtin_bit_cast(bf16x8_t, row[4 * ks + G]);
      m[qi] = -INFINITY, l[qi] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int db = 0; db < 8; ++db) o[qi][db] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    }
    // The compiler does not see what the kernels' own waits cover: without one here it would guard the
    // fragments inside their loops, where that is a wait for the tile in flight.
    __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0)
  }

  __device__ __forceinline__ void store(const AttnWindowParams& p, const Work& w, int col0) const {
    const int fr = threadIdx.x & 15, G = threadIdx.x >> 4 & 3, gs = p.group_shift;
    const int heads = kKVHeads << gs;
#pragma unroll
    for (int qi = 0; qi < QI; ++qi) {
      const int col = col0 + 16 * qi + fr, r = col >> gs;
      if (r >= w.nr) continue;
      const int h = (w.g << gs) + (col & ((1 << gs) - 1));
      if (w.splits > 1) {
        // this split's partial, [slot][head][128] and [slot][head](m, l), slots split by split of the
        // sequence's rows
        const size_t slot = ((size_t)p.part0[w.b] + (size_t)w.split * w.n_new + w.r0 + r) * heads + h;
        float* dst = p.part + slot * kHeadDim + 4 * G;
#pragma unroll
        for (int db = 0; db < 8; ++db) *reinterpret_cast<f32x4_t*>(dst + 16 * db) = o[qi][db];
        if (G == 0) *reinterpret_cast<float2*>(p.part_ml + 2 * slot) = make_float2(m[qi], l[qi][0]);
      } else {
        const float inv = l[qi][0] == 0.f ? 0.f : 1.0f / l[qi][0];
        uint16_t* dst = p.out + ((size_t)(w.row0 + w.r0 + r) * heads + h) * kHeadDim;
#pragma unroll
        for (int db = 0; db < 8; ++db) {
          const u32x2_t v = {pack_bf2(o[qi][db][0] * inv, o[qi][db][1] * inv),
                             pack_bf2(o[qi][db][2] * inv, o[qi][db][3] * inv)};
          *reinterpret_cast<u32x2_t*>(dst + db * 16 + 4 * G) = v;
        }
      }
    }
  }
};

// Byte offsets of a lane's fragment reads in a tile of 64 rows: K fragment ks of key row fr (+ 4096 per
// 16 keys); the transposed V read of dims 16 db + 4 (fr % 4) .. of keys 4 G + fr / 4 (+ 8192 per 32
// keys, + 4096 for keys + 16).  ks and db are XORs of the swizzled chunk.
struct Frags {
  uint32_t k0, v0;
  __device__ __forceinline__ Frags() {
    const int fr = threadIdx.x & 15, G = threadIdx.x >> 4 & 3;
    k0 = (uint32_t)kv_slot(fr, G) * 16;
    v0 = (uint32_t)kv_slot(4 * G + (fr >> 2), (fr & 3) >> 1) * 16 + (fr & 1) * 8;
  }
  __device__ __forceinline__ uint32_t k(int ks) const { return k0 ^ (uint32_t)(ks * 64); }
  __device__ __forceinline__ uint32_t v(int db) const { return v0 ^ (uint32_t)(db * 32); }
};

// s[qi][kb][r] = raw score of the column and key 16 kb + 4 G + r of the tile.
template <int QI>
__device__ __forceinline__ void scores(f32x4_t (&s)[QI][4], const Columns<QI>& c, const Frags& f,
                                       const u32x4_t* ktile) {
  const char* kb8 = reinterpret_cast<const char*>(ktile);
#pragma unroll
  for (int kb = 0; kb < 4; ++kb) {
#pragma unroll
    for (int qi = 0; qi < QI; ++qi) s[qi][kb] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int ks = 0; ks < 4; ++ks) {
      const bf16x8_t a = *reinterpret_cast<const bf16x8_t*>(kb8 + f.k(ks) + kb * 4096);
#pragma unroll
      for (int qi = 0; qi < QI; ++qi)
        s[qi][kb] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, c.q[qi][ks], s[qi][kb], 0, 0, 0);
    }
  }
}

// The scores to weights (bf16, as P^T operands), the outputs and sums so far rescaled.  MASK applies the
// window, the sinks and the diagonal.  A column may have seen no key so far: its max stays -inf and its
// weights are 0 (the exponent's offset is then taken from a finite stand-in).
template <bool MASK, int QI>
__device__ __forceinline__ void weights(bf16x8_t (&pb)[QI][2], Columns<QI>& c, f32x4_t (&s)[QI][4],
                                        int key0, int window, int n_sinks) {
  int first = 4 * (threadIdx.x >> 4 & 3);  // the lane's first key in each 16
  if constexpr (MASK) asm volatile("" : "+v"(first));  // (opaque: nothing made of it is kept over the tiles)
#pragma unroll
  for (int qi = 0; qi < QI; ++qi) {
    float mt = -INFINITY;
#pragma unroll
    for (int kb = 0; kb < 4; ++kb)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        if constexpr (MASK) {
          const int key = key0 + first + 16 * kb + r;
          const bool seen = (key <= c.pos[qi]) & ((key > c.pos[qi] - window) | (key < n_sinks));
          s[qi][kb][r] = seen ? s[qi][kb][r] : -INFINITY;
        }
        mt = fmaxf(mt, s[qi][kb][r]);
      }
    mt = xor32_max(xor16_max(mt));
    const float mn = fmaxf(c.m[qi], mt);
    const float nb = -fmaxf(mn, -3.0e38f) * kScoreScale;
    const float alpha = __builtin_amdgcn_exp2f(fmaf(c.m[qi], kScoreScale, nb));  // m = -inf: 0
    c.m[qi] = mn;
#pragma unroll
    for (int kb = 0; kb < 4; ++kb)
#pragma unroll
      for (int r = 0; r < 4; ++r)
        s[qi][kb][r] = __builtin_amdgcn_exp2f(fmaf(s[qi][kb][r], kScoreScale, nb));
#pragma unroll
    for (int db = 0; db < 8; ++db) c.o[qi][db] *= alpha;
    c.l[qi][0] *= alpha;
#pragma unroll
    for (int ks2 = 0; ks2 < 2; ++ks2) {
      const u32x4_t w = {pack_bf2(s[qi][2 * ks2][0], s[qi][2 * ks2][1]),
                         pack_bf2(s[qi][2 * ks2][2], s[qi][2 * ks2][3]),
                         pack_bf2(s[qi][2 * ks2 + 1][0], s[qi][2 * ks2 + 1][1]),
                         pack_bf2(s[qi][2 * ks2 + 1][2], s[qi][2 * ks2 + 1][3])};
      pb[qi][ks2] = __builtin_bit_cast(bf16x8_t, w);
    }
  }
}

// o += V^T . P^T and the sums.  MASK: 0 x (an infinity or NaN) of a key that a column does not see must
// stay 0: such values are kept out of the product and added to the columns that see them.
template <bool MASK, int QI>
__device__ __forceinline__ void values(Columns<QI>& c, const bf16x8_t (&pb)[QI][2], const Frags& f,
                                       const u32x4_t* vtile, int key0, int window, int n_sinks) {
  const u32x4_t ones_w = {0x3F803F80u, 0x3F803F80u, 0x3F803F80u, 0x3F803F80u};
  const bf16x8_t ones = __builtin_bit_cast(bf16x8_t, ones_w);
  const char* vb8 = reinterpret_cast<const char*>(vtile);
#pragma unroll
  for (int qi = 0; qi < QI; ++qi)
#pragma unroll
    for (int ks2 = 0; ks2 < 2; ++ks2)
      c.l[qi] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(ones, pb[qi][ks2], c.l[qi], 0, 0, 0);
  uint32_t bad = 0;
#pragma unroll
  for (int db = 0; db < 8; ++db) {
    if constexpr (MASK) __builtin_amdgcn_sched_barrier(0);  // (fewer fragments at once: registers)
#pragma unroll
    for (int ks2 = 0; ks2 < 2; ++ks2) {
      const char* va = vb8 + f.v(db) + ks2 * 8192;
      const short4_t lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_short4*)va);
      const short4_t hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_short4*)(va + 4096));
      const short4_t both[2] = {lo, hi};
      u32x4_t w = __builtin_bit_cast(u32x4_t, both);
      if constexpr (MASK) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const uint32_t n = nonfinite2(w[e]);
          bad |= n;
          w[e] &= ~((n >> 15) * 0xFFFFu);
        }
      }
      const bf16x8_t a = __builtin_bit_cast(bf16x8_t, w);
#pragma unroll
      for (int qi = 0; qi < QI; ++qi)
        c.o[qi][db] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, pb[qi][ks2], c.o[qi][db], 0, 0, 0);
    }
  }
  if constexpr (MASK) {
    if (__builtin_expect(__ballot(bad != 0) != 0, 0)) {
      int G = threadIdx.x >> 4 & 3;
      asm volatile("" : "+v"(G));
#pragma unroll
      for (int qi = 0; qi < QI; ++qi) {
#pragma unroll 1
        for (int key = 0; key < BKEY; ++key) {
          const int k = key0 + key;
          const bool seen = k <= c.pos[qi] && (k > c.pos[qi] - window || k < n_sinks);
#pragma unroll
          for (int db = 0; db < 8; ++db) {
            // V[key][16 db + 4 G ..+3]
            const u32x2_t v = *reinterpret_cast<const u32x2_t*>(
                vb8 + kv_slot(key, 2 * db + (G >> 1)) * 16 + (G & 1) * 8);
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const uint32_t n = seen ? nonfinite2(v[e]) : 0;
              if (n & 0x8000u) c.o[qi][db][2 * e] += bf_lo(v[e]);
              if (n >> 16) c.o[qi][db][2 * e + 1] += bf_hi(v[e]);
            }
          }
        }
      }
    }
  }
}

// The part of one tile (K or V) that a wave of NW loads: rows 4 (wave + NW j) + lane / 16, a lane filling slot
// lane % 16 of its row from chunk (lane % 16) ^ swz(row).
template <int NW>
struct TileLoad {
  uint32_t voff[16 / NW];
  int wave;
  __device__ __forceinline__ TileLoad(int w) : wave(w) {
#pragma unroll
    for (int j = 0; j < 16 / NW; ++j) {
      const int r = 4 * (wave + NW * j) + ((int)threadIdx.x >> 4 & 3);
      voff[j] = (uint32_t)(r * kRowBytes + (((threadIdx.x & 15) ^ kv_swz(r)) * 16));
    }
  }
};
template <int NW, int AUX>
__device__ __forceinline__ void issue_tile(u32x4_t* stage, __amdgpu_buffer_rsrc_t rs, const TileLoad<NW>& ld) {
#pragma unroll
  for (int j = 0; j < 16 / NW; ++j)
    __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (lds_void*)(stage + (ld.wave + NW * j) * 64), 16, ld.voff[j], 0, 0, AUX);
}
// The 64 rows of the head's plane in a page (a tile's K or V), `rows` of them there; a page outside the
// pool has none (zeros).
__device__ __forceinline__ __amdgpu_buffer_rsrc_t page_rows(const AttnWindowParams& p, const uint16_t* plane,
                                                            int g, int page, int rows) {
  const bool ok = page >= 0 && page < p.n_pages;
  const size_t base = (size_t)(ok ? page : 0) * kPageElems + (size_t)g * kPageHead;
  const int bytes = __builtin_amdgcn_readfirstlane(ok ? min(BKEY, rows) * kRowBytes : 0);
  return __builtin_amdgcn_make_buffer_rsrc((void*)(plane + base), 0, bytes, kBufferFlags);
}

// How the rows at positions wp0 .. wp1 see the tile from key0 on.
enum Sight { kNone, kSome, kAll };
__device__ __forceinline__ Sight sight(int key0, int wp0, int wp1, int window, int n_sinks) {
  const int last = key0 + BKEY - 1;
  if (wp1 < wp0 || key0 > wp1 || (last <= wp0 - window && key0 >= n_sinks)) return kNone;
  return last <= wp0 && (key0 > wp1 - window || last < n_sinks) ? kAll : kSome;
}

// 4 waves of 16 QI columns, the tiles double-buffered (64 KiB: two workgroups a CU).
template <int QI>
__device__ __forceinline__ void attend(const AttnWindowParams& p) {
  constexpr int NW = 4, CW = 16 * QI;
  __shared__ u32x4_t k0[TC], v0[TC], k1[TC], v1[TC];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const Work w = work_of(p, CW * NW);
  const int wr0 = (wave * CW) >> p.group_shift;
  const int wp0 = w.p0 + wr0, wp1 = w.p0 + min(w.nr, wr0 + (CW >> p.group_shift)) - 1;
  const bool nt = p.nt && w.nqb == 1;
  const TileLoad<NW> ld(wave);
  auto issue = [&](u32x4_t* ks, u32x4_t* vs, int i, int page) {
    const int rows = w.nkeys - w.tile(i) * BKEY;
    const auto krs = page_rows(p, p.k, w.g, page, rows), vrs = page_rows(p, p.v, w.g, page, rows);
    if (nt) {
      issue_tile<NW, 2>(ks, krs, ld);
      issue_tile<NW, 2>(vs, vrs, ld);
    } else {
      issue_tile<NW, 0>(ks, krs, ld);
      issue_tile<NW, 0>(vs, vrs, ld);
    }
  };
  // page of the tile in flight, and of the one after it (loaded a step ahead)
  int page = -1, next = -1;
  if (w.i0 < w.i1) {
    const int here = w.table[w.tile(w.i0)];
    next = w.table[w.tile(min(w.i0 + 1, w.i1 - 1))];
    page = __builtin_amdgcn_readfirstlane(here);
    issue(k0, v0, w.i0, page);
  }
  Columns<QI> c;
  c.load(p, w, wave * CW);
  const Frags f;

  auto step = [&](int i, const u32x4_t* kc, const u32x4_t* vc, u32x4_t* kn, u32x4_t* vn) {
    // tile i has landed (the only loads in flight) and every wave is done with tile i - 1
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
    const bool there = page >= 0 && page < p.n_pages;
    // tile i + 1 is issued unconditionally: past the last tile it has no bytes
    page = i + 1 < w.i1 ? __builtin_amdgcn_readfirstlane(next) : -1;
    issue(kn, vn, i + 1, page);
    next = w.table[w.tile(min(i + 2, w.i1 - 1))];
    const int key0 = w.tile(i) * BKEY;
    const Sight see = there ? sight(key0, wp0, wp1, p.window, p.n_sinks) : kNone;
    if (see == kNone) return;  // (wave-uniform)
    f32x4_t s[QI][4];
    bf16x8_t pb[QI][2];
    scores(s, c, f, kc);
    __builtin_amdgcn_sched_barrier(0);  // (8192 rows over 4096 keys: 611 us without, 598 with)
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
    step(i, k0, v0, k1, v1);
    if (i + 1 < w.i1) step(i + 1, k1, v1, k0, v0);
  }
  c.store(p, w, wave * CW);
}

__global__ __launch_bounds__(256, 2) void attn_window_16_kernel(AttnWindowParams p) { attend<1>(p); }
__global__ __launch_bounds__(256, 2) void attn_window_32_kernel(AttnWindowParams p) { attend<2>(p); }

// Combines the splits of each (row, q head) of the sequences that have them: 32 lanes each, 4
// dims a lane, in split order.  A split without keys for the row (l = 0) is passed over.
__global__ __launch_bounds__(256) void attn_window_merge_kernel(AttnWindowParams p) {
  const int lane = threadIdx.x & 63;
  const int row_end = p.row_end[lane], lane_splits = p.splits[lane], part0 = p.part0[lane];
  const int heads = kKVHeads << p.group_shift;
  const int row = blockIdx.x * 8 / heads;  // (8 heads a workgroup: heads is a multiple of 8)
  const int b = __popcll(__ballot(lane < p.n_seqs && row_end <= row));
  const int splits = __builtin_amdgcn_readlane(lane_splits, b);
  if (splits < 2) return;
  const int row0 = b ? __builtin_amdgcn_readlane(row_end, max(b - 1, 0)) : 0;
  const int n_new = __builtin_amdgcn_readlane(row_end, b) - row0;
  const int h = blockIdx.x * 8 % heads + (threadIdx.x >> 5), d = (threadIdx.x & 31) * 4;
  const size_t slot0 = ((size_t)__builtin_amdgcn_readlane(part0, b) + row - row0) * heads + h;
  const size_t step = (size_t)n_new * heads;
  const float2* ml = reinterpret_cast<const float2*>(p.part_ml);
  float M = -INFINITY, L = 0.f;
  f32x4_t o = {0.f, 0.f, 0.f, 0.f};
  for (int s0 = 0; s0 < splits; s0 += 8) {
    float2 v[8];
    f32x4_t po[8];
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      const size_t slot = slot0 + min(s0 + u, splits - 1) * step;
      v[u] = ml[slot];
      po[u] = *reinterpret_cast<const f32x4_t*>(p.part + slot * kHeadDim + d);
    }
    float mn = M;
#pragma unroll
    for (int u = 0; u < 8; ++u) mn = fmaxf(mn, v[u].x);
    const float a = L == 0.f ? 0.f : __builtin_amdgcn_exp2f((M - mn) * kScoreScale);
    L *= a;
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] *= a;
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      if (s0 + u >= splits || v[u].y == 0.f) continue;
      const float w = __builtin_amdgcn_exp2f((v[u].x - mn) * kScoreScale);
      L = fmaf(v[u].y, w, L);
#pragma unroll
      for (int e = 0; e < 4; ++e) o[e] = fmaf(po[u][e], w, o[e]);
    }
    M = mn;
  }
  const float inv = L == 0.f ? 0.f : 1.0f / L;
  const u32x2_t w = {pack_bf2(o[0] * inv, o[1] * inv), pack_bf2(o[2] * inv, o[3] * inv)};
  *reinterpret_cast<u32x2_t*>(p.out + ((size_t)row * heads + h) * kHeadDim + d) = w;
}

}  // namespace

// Partial rows (a row and split) that a workspace for `rows` rows holds: every row's in 64 splits, up to
// kAttnWindowPartRows.  It never falls with the rows: a workspace serves all smaller batches.
static int attn_window_part_rows(int rows) {
  return std::min(rows, kAttnWindowPartRows / kAttnWindowMaxSplits) * kAttnWindowMaxSplits;
}

size_t attn_window_workspace_bytes(int rows, int heads) {
  return (size_t)attn_window_part_rows(rows) * heads * (kHeadDim + 2) * sizeof(float);
}

namespace {

// A form (columns a wave) and its tiles a split.
struct Plan {
  int qi, tps;
  double cost;
};

// The form and split with the least modelled time, us: a workgroup's step over a tile takes c1 where it
// has a CU for itself and c2 where two share one (measured at 64 rows over 65 tiles and at 8192 rows over 66:
// 1.12 and 1.39 for 16 columns a wave, 1.63 and 2.24 for 32), and 512 run at once; a launch 3.5, the merge
// 4 and its partials 1 / 150 a row and split (32 heads).  Within 6% of the best of 10 split counts and both
// forms over 27 batches (1-4000 rows, 10-940 tiles): 1 token at 20000 381 us unsplit, 24 in 32
// splits; 200 rows over 16384 keys 296 unsplit, 104 in 4 (16 columns), 89 in 8 (32); 16 tokens over 4096 keys
// 98 and 48; 6 x 333 rows over 1500 keys 71 unsplit, 75 in 3; 2 x 1000 over 4096 keys 172 and 151 unsplit,
// 130 in 3 (32 columns).
Plan plan_of(const AttnWindowParams& p, const SeqBatch& s, int room) {
  Plan best{1, 1, 1e30};
  for (int qi = 1; qi <= 2; ++qi) {
    const int rb = (64 * qi) >> p.group_shift;
    int nqb[kMaxSeqs], longest = 1;
    int first[kMaxSeqs], last[kMaxSeqs];  // tiles of a sequence's first and last row block
    for (int b = 0; b < s.n; ++b) {
      const int n = s.n_new[b];
      nqb[b] = (n + rb - 1) / rb;
      first[b] = last[b] = 0;
      if (!n) continue;
      const int at = s.start[b];
      first[b] = tile_run(at, at + std::min(rb, n) - 1, p.window, p.n_sinks).count;
      last[b] = tile_run(at + (nqb[b] - 1) * rb, at + n - 1, p.window, p.n_sinks).count;
      longest = std::max({longest, first[b], last[b]});
    }
    const double c1 = qi == 1 ? 1.12 : 1.63, c2 = qi == 1 ? 1.39 : 2.24;
    int tried = 0;
    for (const int n : {1, 2, 3, 4, 5, 6, 8, 10, 12, 16, 20, 24, 32, 40, 48, kAttnWindowMaxSplits}) {
      const int tps = (longest + n - 1) / n;
      if (n > longest || tps == tried) continue;
      tried = tps;
      long long items = 0, part = 0;
      double steps = 0;
      for (int b = 0; b < s.n; ++b) {
        const int k = std::max(1, (std::max(first[b], last[b]) + tps - 1) / tps);
        items += (long long)nqb[b] * k * kKVHeads;
        steps += 0.5 * (first[b] + last[b]) * nqb[b] * kKVHeads;
        if (k > 1) part += (long long)s.n_new[b] * k;
      }
      if (part > room) break;
      const double t = items ? steps / items : 0;  // a workgroup's tiles, on average
      const long long rest = items % 512;
      const double turns = (double)(items / 512) * t * c2 + (rest == 0 ? 0 : rest <= 256 ? t * c1 : t * c2);
      const double cost = std::max(turns, tps * c1) + 3.5 +
                          (part ? 4 + 0.04 * n + part * (kKVHeads << p.group_shift) / (32 * 150.0) : 0);
      if (cost < best.cost) best = Plan{qi, tps, cost};
      else if (items > 1024) break;  // (more of them only cost more)
    }
  }
  return best;
}

}  // namespace

int launch_attn_window(AttnWindowParams p, const SeqBatch& s, void* workspace, hipStream_t st) {
  int rows = 0;
  long long keys = 0;
  for (int b = 0; b < s.n; ++b) {
    rows += s.n_new[b];
    p.start[b] = s.start[b];
    p.row_end[b] = rows;
    keys += std::min(s.start[b] + s.n_new[b], p.window + p.n_sinks + s.n_new[b]);
  }
  if (!rows) return IE_OK;
  const Plan plan = plan_of(p, s, attn_window_part_rows(rows));
  const int rb = (64 * plan.qi) >> p.group_shift;
  int items = 0, part = 0;
  for (int b = 0; b < s.n; ++b) {
    const int n = s.n_new[b], nqb = (n + rb - 1) / rb;
    int tiles = 0;
    if (n)
      tiles = std::max(tile_run(s.start[b], s.start[b] + std::min(rb, n) - 1, p.window, p.n_sinks).count,
                       tile_run(s.start[b] + (nqb - 1) * rb, s.start[b] + n - 1, p.window, p.n_sinks).count);
    p.splits[b] = std::max(1, (tiles + plan.tps - 1) / plan.tps);
    items += nqb * p.splits[b];
    p.item_end[b] = items;
    p.part0[b] = part;
    if (p.splits[b] > 1) part += n * p.splits[b];
  }
  p.n_seqs = s.n;
  // a batch whose keys of all layers exceed the 256 MB cache finds none of them there: such keys, where one
  // workgroup reads them, pass it by (16 tokens over 4096 keys: 55.7 us without, 47.9 with)
  p.nt = keys > 2048;
  p.part = static_cast<float*>(workspace);
  p.part_ml = p.part + (size_t)part * (kKVHeads << p.group_shift) * kHeadDim;
  const dim3 grid(items * kKVHeads), block(256);
  if (plan.qi == 1)
    hipLaunchKernelGGL(attn_window_16_kernel, grid, block, 0, st, p);
  else
    hipLaunchKernelGGL(attn_window_32_kernel, grid, block, 0, st, p);
  IE_CHECK_LAUNCH();
  if (part) {
    hipLaunchKernelGGL(attn_window_merge_kernel, dim3(rows << p.group_shift), dim3(256), 0, st, p);
    IE_CHECK_LAUNCH();
  }
  return IE_OK;
}

}  // namespace ie
