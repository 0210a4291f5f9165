// What the attention kernels over 64-key tiles of the paged cache share (k_attn_window.hip,
// k_attn_shared.hip): a tile's layout in LDS, the products and the softmax of a wave's query
// columns over one tile.
#pragma once

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

// Both halves of a dword as bf16: true where one of them is an infinity or a NaN.
__device__ __forceinline__ uint32_t nonfinite2(uint32_t w) {
  return ((w & 0x7F807F80u) + 0x00800080u) & 0x80008000u;
}

// A wave's query columns: lane fr of each group of 16 holds column fr of each of QI sets.
template <int QI>
struct ColumnState {
  bf16x8_t q[QI][4];  // Q^T fragments: Q[column][32 ks + 8 G .. +8]
  int pos[QI];        // the columns' positions
  f32x4_t o[QI][8];   // unnormalised: [db][r] = O[column][16 db + 4 G + r]
  float m[QI];        // running max of the raw scores (the scale is applied inside the exponent)
  f32x4_t l[QI];      // [0]: the running sum (the ones-MFMA's other rows are not rescaled)

  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int qi = 0; qi < QI; ++qi) {
      m[qi] = -INFINITY, l[qi] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int db = 0; db < 8; ++db) o[qi][db] = f32x4_t{0.f, 0.f, 0.f, 0.f};
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
__device__ __forceinline__ void scores(f32x4_t (&s)[QI][4], const ColumnState<QI>& c, const Frags& f,
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

// Scores of keys that a column does not see to -inf.
template <int QI>
__device__ __forceinline__ void mask(f32x4_t (&s)[QI][4], const ColumnState<QI>& c, int key0, int window, int n_sinks) {
  int first = 4 * (threadIdx.x >> 4 & 3);  // the lane's first key in each 16
  asm volatile("" : "+v"(first));  // (opaque: nothing made of it is kept over the tiles)
#pragma unroll
  for (int qi = 0; qi < QI; ++qi)
#pragma unroll
    for (int kb = 0; kb < 4; ++kb)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int key = key0 + first + 16 * kb + r;
        const bool seen = (key <= c.pos[qi]) & ((key > c.pos[qi] - window) | (key < n_sinks));
        s[qi][kb][r] = seen ? s[qi][kb][r] : -INFINITY;
      }
}

// The scores to weights (bf16, as P^T operands), the outputs and sums so far rescaled.  MASK applies the
// window, the sinks and the diagonal.  A column may have seen no key so far: its max stays -inf and its
// weights are 0 (the exponent's offset is then taken from a finite stand-in).
template <bool MASK, int QI>
__device__ __forceinline__ void weights(bf16x8_t (&pb)[QI][2], ColumnState<QI>& c, f32x4_t (&s)[QI][4],
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

// The same as weights, rescaling only where a column's maximum has grown: in most tiles of a long run none has (8192 rows
// over 4096 8-bit keys 673 -> 621 us).  (A reference that stays until the scores outgrow it by 2^8 saves 3% more, but the largest
// weight is then rounded as all others are, where it is an exact 1 here: 0.0023 of error in place of 0.0020.)
template <bool MASK, int QI>
__device__ __forceinline__ void weights_grown(bf16x8_t (&pb)[QI][2], ColumnState<QI>& c,
                                             f32x4_t (&s)[QI][4], int key0, int window, int n_sinks) {
  if constexpr (MASK) mask(s, c, key0, window, n_sinks);
  float mn[QI];
  bool moved = false;
#pragma unroll
  for (int qi = 0; qi < QI; ++qi) {
    float mt = -INFINITY;
#pragma unroll
    for (int kb = 0; kb < 4; ++kb)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        mt = fmaxf(mt, s[qi][kb][r]);
      }
    mt = xor32_max(xor16_max(mt));
    mn[qi] = fmaxf(c.m[qi], mt);
    moved |= mn[qi] != c.m[qi];
  }
  if (__ballot(moved) != 0) {
#pragma unroll
    for (int qi = 0; qi < QI; ++qi) {
      const float nb = -fmaxf(mn[qi], -3.0e38f) * kScoreScale;
      // (m = -inf: 0; exactly 1 for a column that stays, whatever its neighbours do)
      const float alpha =
          mn[qi] != c.m[qi] ? __builtin_amdgcn_exp2f(fmaf(c.m[qi], kScoreScale, nb)) : 1.0f;
      c.m[qi] = mn[qi];
#pragma unroll
      for (int db = 0; db < 8; ++db) c.o[qi][db] *= alpha;
      c.l[qi][0] *= alpha;
    }
  }
#pragma unroll
  for (int qi = 0; qi < QI; ++qi) {
    const float nb = -fmaxf(mn[qi], -3.0e38f) * kScoreScale;
#pragma unroll
    for (int kb = 0; kb < 4; ++kb)
#pragma unroll
      for (int r = 0; r < 4; ++r)
        s[qi][kb][r] = __builtin_amdgcn_exp2f(fmaf(s[qi][kb][r], kScoreScale, nb));
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

// o += V^T . P^T and the sums, of a tile.  MASK: 0 x (an infinity or NaN) of a key that a column does not see must
// stay 0: such values are kept out of the product and added to the columns that see them.
// AHEAD: the fragments of so many groups of 16 dims are read ahead of their products (0: as the compiler likes).
template <bool MASK, int AHEAD = 0, int QI>
__device__ __forceinline__ void values(ColumnState<QI>& c, const bf16x8_t (&pb)[QI][2], const Frags& f,
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
  if constexpr (!MASK && AHEAD > 0) {
    // (0x100: LDS reads, 0x8: MFMAs; the sums' come first)
    __builtin_amdgcn_sched_group_barrier(0x100, 4 * AHEAD, 0);
    __builtin_amdgcn_sched_group_barrier(0x8, 2 * QI, 0);
#pragma unroll
    for (int db = 0; db < 8; ++db) {
      if (db + AHEAD < 8) __builtin_amdgcn_sched_group_barrier(0x100, 4, 0);
      __builtin_amdgcn_sched_group_barrier(0x8, 2 * QI, 0);
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
// How the rows at positions wp0 .. wp1 see the tile of keys from key0 on.
enum Sight { kNone, kSome, kAll };
__device__ __forceinline__ Sight sight(int key0, int wp0, int wp1, int window, int n_sinks) {
  const int last = key0 + BKEY - 1;
  if (wp1 < wp0 || key0 > wp1 || (last <= wp0 - window && key0 >= n_sinks)) return kNone;
  return last <= wp0 && (key0 > wp1 - window || last < n_sinks) ? kAll : kSome;
}

}  // namespace

}  // namespace ie
