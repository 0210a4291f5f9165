// Attention of ragged chunks of new tokens over the paged K/V cache, with a sliding window and
// sinks (no reference counterpart: the reference attends one sequence, all keys, one plane).
//
// Sequence b's new rows sit at positions start .. start + n_new - 1; the row at position p sees the
// keys j <= p with j > p - window or j < n_sinks whose page is there:
//   o = sum_j softmax_j(q . k_j / sqrt(128)) v_j,  zeros where it sees none.
//
// A workgroup takes one kv head and a block of query columns, a column being a (row, q head of the
// kv head's group): consecutive columns are the group's heads, then the next row, so that a single
// token of a 4-head group fills 4 of a wave's 16 columns and a chunk fills all of them, whatever the
// group.  It walks the 64-key tiles that the block's rows see (a tile is a page: the sink tiles, then the
// window's), each staged once in LDS for all its waves.  Per tile and wave, with
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

// A wave's query columns (lane fr of each group of 16 holds column 16 qi + fr).
template <int QI>
struct Columns {
  bf16x8_t q[QI][4];  // Q^T fragments
  int pos[QI];        // the columns' positions
  f32x4_t o[QI][8];   // unnormalised outputs
  float m[QI];        // running max of the raw scores (the scale is applied inside the exponent)
  f32x4_t l[QI];      // [0]: the running sum (the ones-MFMA's other rows are not rescaled)
};

// The columns over one tile: kb8 the tile's stage, key0 its first key.  MASK applies the window,
// the sinks and the diagonal.  A column may have seen no key so far: its max stays -inf and
// its weights are 0 (the exponent's offset is then taken from a finite stand-in).
template <bool MASK, int QI>
__device__ __forceinline__ void attend_tile(Columns<QI>& c, const char* kb8, int key0, int G,
                                            const uint32_t (&koffs)[4], const uint32_t (&voffs)[8],
                                            int window, int n_sinks) {
  const u32x4_t ones_w = {0x3F803F80u, 0x3F803F80u, 0x3F803F80u, 0x3F803F80u};
  const bf16x8_t ones = __builtin_bit_cast(bf16x8_t, ones_w);
  f32x4_t s[QI][4];
#pragma unroll
  for (int kb = 0; kb < 4; ++kb) {
#pragma unroll
    for (int qi = 0; qi < QI; ++qi) s[qi][kb] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int ks = 0; ks < 4; ++ks) {
      const bf16x8_t a = *reinterpret_cast<const bf16x8_t*>(kb8 + koffs[ks] + kb * 4096);
#pragma unroll
      for (int qi = 0; qi < QI; ++qi)
        s[qi][kb] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, c.q[qi][ks], s[qi][kb], 0, 0, 0);
    }
  }
  bf16x8_t pb[QI][2];
#pragma unroll
  for (int qi = 0; qi < QI; ++qi) {
    float mt = -INFINITY;
#pragma unroll
    for (int kb = 0; kb < 4; ++kb)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        if constexpr (MASK) {
          const int key = key0 + 16 * kb + 4 * G + r;
          const bool seen = key <= c.pos[qi] && (key > c.pos[qi] - window || key < n_sinks);
          if (!seen) s[qi][kb][r] = -INFINITY;
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
      c.l[qi] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(ones, pb[qi][ks2], c.l[qi], 0, 0, 0);
    }
  }
  auto v_frag = [&](int db, int ks2) {
    const char* va = kb8 + voffs[db] + ks2 * 8192;
    const short4_t lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_short4*)va);
    const short4_t hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_short4*)(va + 4096));
    const short4_t both[2] = {lo, hi};
    return __builtin_bit_cast(u32x4_t, both);
  };
  uint32_t bad = 0;
#pragma unroll
  for (int db = 0; db < 8; ++db)
#pragma unroll
    for (int ks2 = 0; ks2 < 2; ++ks2) {
      u32x4_t w = v_frag(db, ks2);
      if constexpr (MASK) {
        // 0 x (infinity or NaN) of a key that the column does not see must stay 0: such values are
        // kept out of the product here and added below to the columns that see them
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
  if constexpr (MASK) {
    if (__builtin_expect(__ballot(bad != 0) != 0, 0)) {
      // 1 where the column's weight is positive x (1 where V is +inf, -inf, NaN), by MFMA
      bf16x8_t seen[QI][2];
#pragma unroll
      for (int qi = 0; qi < QI; ++qi)
#pragma unroll
        for (int ks2 = 0; ks2 < 2; ++ks2) {
          u32x4_t w = __builtin_bit_cast(u32x4_t, pb[qi][ks2]);
#pragma unroll
          for (int e = 0; e < 4; ++e)
            w[e] = (w[e] & 0xFFFFu ? 0x3F80u : 0u) | (w[e] >> 16 ? 0x3F800000u : 0u);
          seen[qi][ks2] = __builtin_bit_cast(bf16x8_t, w);
        }
#pragma unroll
      for (int db = 0; db < 8; ++db)
#pragma unroll
        for (int kind = 0; kind < 3; ++kind) {
          u32x4_t hit[2];
#pragma unroll
          for (int ks2 = 0; ks2 < 2; ++ks2) {
            const u32x4_t w = v_frag(db, ks2);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const auto is = [&](uint32_t h) {
                return kind == 0   ? h == 0x7F80u
                       : kind == 1 ? h == 0xFF80u
                                   : (h & 0x7FFFu) > 0x7F80u;
              };
              hit[ks2][e] = (is(w[e] & 0xFFFFu) ? 0x3F80u : 0u) | (is(w[e] >> 16) ? 0x3F800000u : 0u);
            }
          }
          const float value = kind == 0 ? INFINITY : kind == 1 ? -INFINITY : NAN;
#pragma unroll
          for (int qi = 0; qi < QI; ++qi) {
            f32x4_t n = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int ks2 = 0; ks2 < 2; ++ks2)
              n = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, hit[ks2]),
                                                          seen[qi][ks2], n, 0, 0, 0);
#pragma unroll
            for (int r = 0; r < 4; ++r)
              if (n[r] > 0.f) c.o[qi][db][r] += value;
          }
        }
    }
  }
}

// One tile's loads into a stage (K at stage[0..TC), V at stage[TC..2TC)) by NW waves: this wave's
// groups of 4 rows.
template <int NW>
__device__ __forceinline__ void issue_tile(u32x4_t* stage, __amdgpu_buffer_rsrc_t krs,
                                           __amdgpu_buffer_rsrc_t vrs,
                                           const uint32_t (&voff)[16 / NW], int wave) {
#pragma unroll
  for (int j = 0; j < 16 / NW; ++j) {
    u32x4_t* kd = stage + (wave + NW * j) * 64;
    __builtin_amdgcn_raw_ptr_buffer_load_lds(krs, (lds_void*)kd, 16, voff[j], 0, 0, 0);
    __builtin_amdgcn_raw_ptr_buffer_load_lds(vrs, (lds_void*)(kd + TC), 16, voff[j], 0, 0, 0);
  }
}

template <int QI, int NW>
__global__ __launch_bounds__(64 * NW, 2) void attn_window_kernel(AttnWindowParams p) {
  __shared__ u32x4_t lds0[2 * TC];  // ring stage 0: [K | V][key][16 chunks], 32 KiB
  __shared__ u32x4_t lds1[2 * TC];  // ring stage 1
  constexpr int CW = 16 * QI;       // columns per wave
  constexpr int CB = CW * NW;       // columns per workgroup
  constexpr int NL = 16 / NW;       // 1 KiB loads of K (and V) a wave and tile

  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int fr = lane & 15, G = lane >> 4;
  const int gs = p.group_shift;
  // workgroup -> (sequence, split, row block, kv head): kv heads go round the XCDs, whose L2 then holds
  // the head's keys for the blocks that share them
  const int g = blockIdx.x % kKVHeads, item = blockIdx.x / kKVHeads;
  const int b = __popcll(__ballot(lane < p.n_seqs && p.item_end[lane] <= item));
  const int start = p.start[b], row0 = b ? p.row_end[b - 1] : 0, n_new = p.row_end[b] - row0;
  const int splits = p.splits[b];
  const int local = item - (b ? p.item_end[b - 1] : 0);
  const int rb = CB >> gs;  // rows per workgroup
  const int nqb = (n_new + rb - 1) / rb;
  const int qb = nqb - 1 - local % nqb, split = local / nqb;
  const int r0 = qb * rb, nr = min(rb, n_new - r0);
  const int p0 = start + r0, nkeys = start + n_new;
  const TileRun run = tile_run(p0, p0 + nr - 1, p.window, p.n_sinks);
  const int tps = (run.count + splits - 1) / splits;
  const int i0 = min(run.count, split * tps), i1 = min(run.count, i0 + tps);
  // this wave's rows (positions wp0 .. wp1; none: wp1 < wp0)
  const int wr0 = (wave * CW) >> gs;
  const int wp0 = p0 + wr0, wp1 = p0 + min(nr, wr0 + (CW >> gs)) - 1;

  const int* table = p.block_tables + (size_t)b * p.table_stride;
  // load j of this wave: tile rows 4 (wave + NW j) + lane/16; a lane fills slot lane%16 of its row
  // from chunk (lane%16) ^ swz(row)
  uint32_t voff[NL];
#pragma unroll
  for (int j = 0; j < NL; ++j) {
    const int r = 4 * (wave + NW * j) + G;
    voff[j] = (uint32_t)(r * kRowBytes + ((fr ^ kv_swz(r)) * 16));
  }
  auto tile_of = [&](int i) { return i < run.sinks ? i : run.first + i - run.sinks; };

  // Q^T fragments: c.q[qi][ks] = Q[column][32 ks + 8 G .. +8]; columns past the rows repeat the last row
  Columns<QI> c;
#pragma unroll
  for (int qi = 0; qi < QI; ++qi) {
    const int col = wave * CW + 16 * qi + fr;
    const int r = min(col >> gs, nr - 1);
    c.pos[qi] = p0 + r;
    const size_t at = ((size_t)(row0 + r0 + r) << gs << 3) + ((size_t)g << gs) + (col & ((1 << gs) - 1));
    const u32x4_t* qrow = reinterpret_cast<const u32x4_t*>(p.q + at * kHeadDim);
#pragma unroll
    for (int ks = 0; ks < 4; ++ks) c.q[qi][ks] = __builtin_bit_cast(bf16x8_t, qrow[4 * ks + G]);
  }

#pragma unroll
  for (int qi = 0; qi < QI; ++qi) {
    c.m[qi] = -INFINITY, c.l[qi] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int db = 0; db < 8; ++db) c.o[qi][db] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  }

  const int kr = fr >> 2, dq = fr & 3;
  uint32_t koffs[4], voffs[8];
#pragma unroll
  for (int ks = 0; ks < 4; ++ks) koffs[ks] = (uint32_t)kv_slot(fr, 4 * ks + G) * 16;
#pragma unroll
  for (int db = 0; db < 8; ++db)
    voffs[db] = (uint32_t)(TC + kv_slot(4 * G + kr, 2 * db + (dq >> 1))) * 16 + (dq & 1) * 8;

  // Loads of tile i (page `page`) into a stage; a page outside the pool has no bytes (zeros).
  auto issue = [&](u32x4_t* stage, int i, int page) {
    const bool ok = page >= 0 && page < p.n_pages;
    const size_t base = (size_t)(ok ? page : 0) * kPageElems + (size_t)g * kPageHead;
    const int bytes = __builtin_amdgcn_readfirstlane(
        ok ? min(BKEY, nkeys - tile_of(i) * BKEY) * kRowBytes : 0);
    const __amdgpu_buffer_rsrc_t krs =
        __builtin_amdgcn_make_buffer_rsrc((void*)(p.k + base), 0, bytes, kBufferFlags);
    const __amdgpu_buffer_rsrc_t vrs =
        __builtin_amdgcn_make_buffer_rsrc((void*)(p.v + base), 0, bytes, kBufferFlags);
    issue_tile<NW>(stage, krs, vrs, voff, wave);
  };
  // page of the tile in flight, and of the one after it (loaded a step ahead)
  int page = -1, next = -1;
  if (i0 < i1) {
    page = __builtin_amdgcn_readfirstlane(table[tile_of(i0)]);
    issue(lds0, i0, page);
    next = table[tile_of(min(i0 + 1, i1 - 1))];
  }

  auto step = [&](int i, const u32x4_t* cur, u32x4_t* nxt) {
    // tile i has landed (the only loads in flight) and every wave is done with tile i - 1
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
    const bool there = page >= 0 && page < p.n_pages;
    // tile i + 1 is issued unconditionally: past the last tile it has no bytes
    page = i + 1 < i1 ? __builtin_amdgcn_readfirstlane(next) : -1;
    issue(nxt, i + 1, page);
    next = table[tile_of(min(i + 2, i1 - 1))];
    const int key0 = tile_of(i) * BKEY, last = key0 + BKEY - 1;
    // (wave-uniform) no row of the wave sees the tile / every row sees all of it
    if (!there || wp1 < wp0 || key0 > wp1 || (last <= wp0 - p.window && key0 >= p.n_sinks)) return;
    const char* kb8 = reinterpret_cast<const char*>(cur);
    if (last <= wp0 && (key0 > wp1 - p.window || last < p.n_sinks))
      attend_tile<false, QI>(c, kb8, key0, G, koffs, voffs, p.window, p.n_sinks);
    else
      attend_tile<true, QI>(c, kb8, key0, G, koffs, voffs, p.window, p.n_sinks);
  };
  for (int i = i0; i < i1; i += 2) {
    step(i, lds0, lds1);
    if (i + 1 < i1) step(i + 1, lds1, lds0);
  }

  // ---- c.o[qi][db][r] = O[column 16 qi + fr][d = 16 db + 4 G + r] (unnormalised)
  const int heads = kKVHeads << gs;
#pragma unroll
  for (int qi = 0; qi < QI; ++qi) {
    const int col = wave * CW + 16 * qi + fr, r = col >> gs;
    if (r >= nr) continue;
    const int h = (g << gs) + (col & ((1 << gs) - 1));
    if (splits > 1) {
      // this split's partial, [slot][head][128] and [slot][head](m, l), slots split by split of the
      // sequence's rows
      const size_t slot = ((size_t)p.part0[b] + (size_t)split * n_new + r0 + r) * heads + h;
      float* dst = p.part + slot * kHeadDim + 4 * G;
#pragma unroll
      for (int db = 0; db < 8; ++db) *reinterpret_cast<f32x4_t*>(dst + 16 * db) = c.o[qi][db];
      if (G == 0)
        *reinterpret_cast<float2*>(p.part_ml + 2 * slot) = make_float2(c.m[qi], c.l[qi][0]);
    } else {
      const float inv = c.l[qi][0] == 0.f ? 0.f : 1.0f / c.l[qi][0];
      uint16_t* dst = p.out + ((size_t)(row0 + r0 + r) * heads + h) * kHeadDim;
#pragma unroll
      for (int db = 0; db < 8; ++db) {
        const u32x2_t w = {pack_bf2(c.o[qi][db][0] * inv, c.o[qi][db][1] * inv),
                           pack_bf2(c.o[qi][db][2] * inv, c.o[qi][db][3] * inv)};
        *reinterpret_cast<u32x2_t*>(dst + db * 16 + 4 * G) = w;
      }
    }
  }
}

// Combines the splits of each (row, q head) of the sequences that have them: 32 lanes each, 4
// dims a lane, in split order.  A split without keys for the row (l = 0) is passed over.
__global__ __launch_bounds__(256) void attn_window_merge_kernel(AttnWindowParams p) {
  const int lane = threadIdx.x & 63;
  const int heads = kKVHeads << p.group_shift;
  const int row = blockIdx.x * 8 / heads;  // (8 heads a workgroup: heads is a multiple of 8)
  const int b = __popcll(__ballot(lane < p.n_seqs && p.row_end[lane] <= row));
  const int splits = p.splits[b];
  if (splits < 2) return;
  const int row0 = b ? p.row_end[b - 1] : 0, n_new = p.row_end[b] - row0;
  const int h = blockIdx.x * 8 % heads + (threadIdx.x >> 5), d = (threadIdx.x & 31) * 4;
  const size_t slot0 = ((size_t)p.part0[b] + row - row0) * heads + h, step = (size_t)n_new * heads;
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

constexpr int kSlots = 512;  // workgroups that run at once (two a CU)

}  // namespace

// Partial rows (a row and split) that a workspace for `rows` rows holds.
int attn_window_part_rows(int rows) { return rows >= kAttnWindowPartRows ? 0 : kAttnWindowPartRows; }

size_t attn_window_workspace_bytes(int rows, int heads) {
  return (size_t)attn_window_part_rows(rows) * heads * (kHeadDim + 2) * sizeof(float);
}

int launch_attn_window(AttnWindowParams p, const SeqBatch& s, void* workspace, hipStream_t st) {
  constexpr int QI = 1, NW = 4;
  const int rb = (16 * QI * NW) >> p.group_shift;
  int rows = 0, longest = 0, nqb[kMaxSeqs], tiles[kMaxSeqs];
  for (int b = 0; b < s.n; ++b) {
    const int n = s.n_new[b];
    rows += n;
    p.start[b] = s.start[b];
    p.row_end[b] = rows;
    nqb[b] = (n + rb - 1) / rb;
    tiles[b] = 0;
    // the last block's run is the longest but for rounding to tiles
    if (n) tiles[b] = tile_run(s.start[b] + (nqb[b] - 1) * rb, s.start[b] + n - 1, p.window, p.n_sinks).count;
    longest = std::max(longest, tiles[b]);
  }
  if (!rows) return IE_OK;
  // tiles a split: the least (rounds of the chip) x (a split's tiles + its fixed cost, 2) + the merge
  const int room = workspace ? attn_window_part_rows(rows) : 0;
  int best = std::max(longest, 1);
  double best_cost = 1e30;
  for (int n = 1; n <= kMaxSplits && n <= std::max(longest, 1); ++n) {
    const int tps = (longest + n - 1) / n;
    long long items = 0, part = 0;
    for (int b = 0; b < s.n; ++b) {
      const int k = std::max(1, (tiles[b] + tps - 1) / tps);
      items += (long long)nqb[b] * k * kKVHeads;
      if (k > 1) part += (long long)s.n_new[b] * k;
    }
    if (part > room) break;
    const double cost = (double)((items + kSlots - 1) / kSlots) * (tps + 2) + (part ? 4 + part / 128.0 : 0);
    if (cost < best_cost) best = tps, best_cost = cost;
  }
  int items = 0, part = 0;
  for (int b = 0; b < s.n; ++b) {
    p.splits[b] = std::max(1, (tiles[b] + best - 1) / best);
    items += nqb[b] * p.splits[b];
    p.item_end[b] = items;
    p.part0[b] = part;
    if (p.splits[b] > 1) part += s.n_new[b] * p.splits[b];
  }
  p.n_seqs = s.n;
  p.part = static_cast<float*>(workspace);
  p.part_ml = p.part + (size_t)part * (kKVHeads << p.group_shift) * kHeadDim;
  hipLaunchKernelGGL((attn_window_kernel<QI, NW>), dim3(items * kKVHeads), dim3(64 * NW), 0, st, p);
  IE_CHECK_LAUNCH();
  if (part) {
    hipLaunchKernelGGL(attn_window_merge_kernel, dim3(rows << p.group_shift), dim3(256), 0, st, p);
    IE_CHECK_LAUNCH();
  }
  return IE_OK;
}

}  // namespace ie
