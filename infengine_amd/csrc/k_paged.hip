// What a server does to the paged K/V cache between its attention calls: the norms and rotation of
// new queries and keys with the append of their K/V rows, forks of sequences, and compaction of
// the pool (no reference counterparts: the reference holds one sequence in one plane).  All are
// byte movers.
#include <algorithm>

#include "ie_kernels.h"

namespace ie {

namespace {

// ---------------------------------------------------------------- norms, rotation, append
// q' = rot(q * rsqrt(mean(q^2) + 1e-5) * w), the same for k (without a weight no norm), v as it
// is; in fp32, rounded once.  16 lanes a head, 8 dims each; dim j and its partner j + 64 are 8
// lanes apart.  A workgroup takes a row: GROUPS of 16 heads, the last one K and V.  A lane keeps its dims'
// angles and weights over its heads (a workgroup for 16 heads, each with its own loads of the
// angles, 64 bytes a lane beside 16 of the row, took 24.4 us for 4214 normed rows of 48 heads; this one
// 18.8, 5.6 TB/s read and written, bound by them; one token of 16 sequences 5.7-6.4, the launch).
template <int GROUPS>
__global__ __launch_bounds__(256) void qk_norm_rope_kernel(QkNormRopeParams p) {
  const int tid = threadIdx.x, lane = tid & 63, li = tid & 15, hg = tid >> 4;
  const int row = blockIdx.x;
  // (the sequences' arguments in one go, a lane each)
  const int row_end = p.row_end[lane], start = p.start[lane];
  const u32x4_t* src = reinterpret_cast<const u32x4_t*>(p.qkv + (size_t)row * p.qkv_stride) + tid;
  u32x4_t x[GROUPS];
#pragma unroll
  for (int j = 0; j < GROUPS; ++j) x[j] = ld_stream(src + 256 * j);
  const u32x4_t none = {0, 0, 0, 0};
  const u32x4_t wq = p.q_norm ? reinterpret_cast<const u32x4_t*>(p.q_norm)[li] : none;
  const u32x4_t wk = p.k_norm ? reinterpret_cast<const u32x4_t*>(p.k_norm)[li] : none;
  const int b = __popcll(__ballot(lane < p.n_seqs && row_end <= row));
  const int before = b ? __builtin_amdgcn_readlane(row_end, max(b - 1, 0)) : 0;
  const int pos = __builtin_amdgcn_readlane(start, b) + row - before;
  const int page = p.block_tables[(size_t)b * p.table_stride + pos / kPagePos];
  const float4* c4 = reinterpret_cast<const float4*>(p.rope_cos + (size_t)pos * 64 + 8 * (li & 7));
  const float4* s4 = reinterpret_cast<const float4*>(p.rope_sin + (size_t)pos * 64 + 8 * (li & 7));
  const float4 ca = c4[0], cb = c4[1], sa = s4[0], sb = s4[1];
  const float c[8] = {ca.x, ca.y, ca.z, ca.w, cb.x, cb.y, cb.z, cb.w};
  const float s[8] = {sa.x, sa.y, sa.z, sa.w, sb.x, sb.y, sb.z, sb.w};
#pragma unroll
  for (int j = 0; j < GROUPS; ++j) {
    const bool is_q = j < GROUPS - 1, is_v = !is_q && hg >= kKVHeads;
    float v[8], t[8];
#pragma unroll
    for (int e = 0; e < 4; ++e) v[2 * e] = bf_lo(x[j][e]), v[2 * e + 1] = bf_hi(x[j][e]);
    if (is_q ? p.q_norm : p.k_norm) {
      const u32x4_t wv = is_q ? wq : wk;
      float ss = 0.f;
#pragma unroll
      for (int e = 0; e < 8; ++e) ss = fmaf(v[e], v[e], ss);
      const float r = rsqrtf(row16_sum(ss) * (1.0f / kHeadDim) + kRmsEps);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        v[2 * e] *= r * bf_lo(wv[e]);
        v[2 * e + 1] *= r * bf_hi(wv[e]);
      }
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float other = dpp_f<0x128>(v[e]);  // row_ror 8: the partner dim
      t[e] = li < 8 ? rope_lo(v[e], other, c[e], s[e]) : rope_hi(other, v[e], c[e], s[e]);
    }
    u32x4_t y;
#pragma unroll
    for (int e = 0; e < 4; ++e) y[e] = pack_bf2(t[2 * e], t[2 * e + 1]);
    if (is_q) {
      reinterpret_cast<u32x4_t*>(p.q_out + (size_t)row * p.heads * kHeadDim)[256 * j + tid] = y;
    } else if (page >= 0 && page < p.n_pages) {
      uint16_t* dst = (is_v ? p.v : p.k) + (size_t)page * kPageElems +
                      ((size_t)(hg & (kKVHeads - 1)) * kPagePos + pos % kPagePos) * kHeadDim;
      reinterpret_cast<u32x4_t*>(dst)[li] = is_v ? x[j] : y;
    }
  }
}

// ---------------------------------------------------------------- fork
// The forks in groups that copy the same positions of the same row (continuations of one prompt).
struct ForkParams {
  uint16_t* pages;
  int* tables;
  int n_pages, stride;
  int src[kMaxSeqs], n_pos[kMaxSeqs], end[kMaxSeqs];  // by group; `end`: one past its last fork
  int dst[kMaxSeqs], page[kMaxSeqs];                  // by fork
};
constexpr int kPlanes = kLayers * 2 * kKVHeads;  // [64][128] planes of a page
constexpr int kPlanePieces = (int)(kPageHead / 8);  // 16-byte pieces of a plane
static_assert(kPlanes >= kMaxSeqs, "a workgroup for every table row of a group");

// blockIdx.x: a plane, blockIdx.y: a group.  The first n_pos % 64 positions of the plane in the source's
// last page are read once and written to every fork's page; the first workgroups also write a table
// row each.  Bound by the stores: 16 forks of 58 positions, 122 MB written, take 21.7 us, 5.6 TB/s of them (with a
// copy per fork 31; a nontemporal fill of as much 22); four forks of one short prompt 5.6-6.0, the launch.
__global__ __launch_bounds__(256) void kv_fork_kernel(ForkParams p) {
  const int g = blockIdx.y, plane = blockIdx.x;
  const int first = g ? p.end[g - 1] : 0, end = p.end[g];
  const int full = p.n_pos[g] / kPagePos, part = p.n_pos[g] % kPagePos;
  const int* from = p.tables + (size_t)p.src[g] * p.stride;
  if (first + plane < end) {
    int* to = p.tables + (size_t)p.dst[first + plane] * p.stride;
    for (int i = threadIdx.x; i < p.stride; i += 256)
      to[i] = i < full ? from[i] : i == full && part ? p.page[first + plane] : -1;
  }
  if (!part) return;
  const int src = from[full];
  if (src < 0 || src >= p.n_pages) return;
  const int n = part * (kHeadDim / 8);
  const size_t at = (size_t)plane * kPlanePieces + threadIdx.x;
  u32x4_t v[kPlanePieces / 256];
#pragma unroll
  for (int u = 0; u < kPlanePieces / 256; ++u)
    v[u] = reinterpret_cast<const u32x4_t*>(p.pages + (size_t)src * kPageElems)[at + min(256 * u, n - 1)];
  for (int f = first; f < end; ++f) {
    u32x4_t* d = reinterpret_cast<u32x4_t*>(p.pages + (size_t)p.page[f] * kPageElems) + at;
#pragma unroll
    for (int u = 0; u < kPlanePieces / 256; ++u)
      if ((int)threadIdx.x + 256 * u < n) __builtin_nontemporal_store(v[u], d + 256 * u);
  }
}

// ---------------------------------------------------------------- compaction
struct CompactParams {
  uint16_t* pages;
  const int* tables;
  int* new_tables;
  int* remap;
  int* counts;   // live pages, moved pages
  int* holes;    // [n_pages] free ids below the live count, ascending
  int* movers;   // [n_pages] live ids from it on, ascending
  int n_rows, n_pages, stride, window, n_sinks;
  int len[kMaxSeqs];
};
constexpr int kPlanThreads = 1024;

// Entry i of a row of n positions is still needed (n = 0: the sequence is over).
__device__ __forceinline__ bool entry_kept(const CompactParams& p, int n, int i) {
  if (n == 0) return false;
  return i * kPagePos < p.n_sinks || (i + 1) * kPagePos > n - p.window + 1 ||
         i >= (n + kPagePos - 1) / kPagePos;
}

// One workgroup: marks the pages that the kept entries name in an LDS bitmap, ranks them, pairs the
// live ids >= the live count with the free ids below it in ascending order, and writes the
// remapped tables.  4.5 us for 4 or 8 rows of up to 63 entries: a chain of barriers and dependent loads, small beside
// the moves; the call takes 18 us for 64 rows of 128 entries, 51 of 512 and 187 of 2048 where nothing moves: 1024
// entries a step, twice.
__global__ __launch_bounds__(kPlanThreads) void kv_compact_plan_kernel(CompactParams p) {
  constexpr int kWords = kCompactMaxPages / 64, kPer = kWords / kPlanThreads;
  __shared__ unsigned long long live[kWords];
  __shared__ int before[kWords];  // live pages in the words before
  __shared__ int wsum[kPlanThreads / 64];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  for (int w = tid; w < kWords; w += kPlanThreads) live[w] = 0;
  __syncthreads();
  const int entries = p.n_rows * p.stride;
  for (int e = tid; e < entries; e += kPlanThreads) {
    const int row = e / p.stride, page = p.tables[e];
    if (page >= 0 && page < p.n_pages && entry_kept(p, p.len[row], e - row * p.stride))
      atomicOr(&live[page >> 6], 1ull << (page & 63));
  }
  __syncthreads();
  int own = 0;
#pragma unroll
  for (int k = 0; k < kPer; ++k) own += __popcll(live[tid * kPer + k]);
  int inc = own;
#pragma unroll
  for (int s = 1; s < 64; s <<= 1) {
    const int v = __shfl_up(inc, s, 64);
    if (lane >= s) inc += v;
  }
  if (lane == 63) wsum[wave] = inc;
  __syncthreads();
  int total = 0;
  for (int w = 0; w < kPlanThreads / 64; ++w) {
    if (w < wave) inc += wsum[w];
    total += wsum[w];
  }
  int at = inc - own;
#pragma unroll
  for (int k = 0; k < kPer; ++k) {
    before[tid * kPer + k] = at;
    at += __popcll(live[tid * kPer + k]);
  }
  __syncthreads();
  const auto rank = [&](int page) {  // live pages below `page`
    const int w = page >> 6;
    return before[w] + __popcll(live[w] & ((1ull << (page & 63)) - 1));
  };
  // (total <= n_pages; rank(n_pages) needs no word past the last when n_pages is the limit)
  const int below = total < kCompactMaxPages ? rank(total) : total;
  const int moved = total - below;
  for (int page = tid; page < p.n_pages; page += kPlanThreads) {
    const bool is = live[page >> 6] >> (page & 63) & 1;
    const int r = rank(page);
    if (page < total && !is) p.holes[page - r] = page;
    if (page >= total && is) p.movers[r - below] = page;
  }
  __syncthreads();
  for (int page = tid; page < p.n_pages; page += kPlanThreads) {
    const bool is = live[page >> 6] >> (page & 63) & 1;
    p.remap[page] = !is ? -1 : page < total ? page : p.holes[rank(page) - below];
  }
  if (tid == 0) p.counts[0] = total, p.counts[1] = moved;
  __syncthreads();
  for (int e = tid; e < entries; e += kPlanThreads) {
    const int row = e / p.stride, page = p.tables[e];
    const bool kept = page >= 0 && page < p.n_pages && entry_kept(p, p.len[row], e - row * p.stride);
    p.new_tables[e] = kept ? p.remap[page] : -1;
  }
}

constexpr int kMoveBytes = 64 << 10;  // of a page, a workgroup at a time

// Moves the pages: sources are ids >= the live count, destinations free ids below it.  Bound by HBM: 17 pages of 8 MiB
// 47 us, 6.0 TB/s read and written, 83 252, 5.5 (a nontemporal copy of as much 5.5-5.7 and 5.1-5.2).
__global__ __launch_bounds__(256) void kv_compact_move_kernel(CompactParams p) {
  constexpr int kParts = (int)(kPageElems * 2 / kMoveBytes), kEach = kMoveBytes / 16 / 256;
  const int total = p.counts[1] * kParts;
  for (int i = blockIdx.x; i < total; i += gridDim.x) {
    const int k = i / kParts, part = i % kParts;
    const size_t at = (size_t)part * (kMoveBytes / 16) + threadIdx.x;
    const u32x4_t* s = reinterpret_cast<const u32x4_t*>(p.pages + (size_t)p.movers[k] * kPageElems) + at;
    u32x4_t* d = reinterpret_cast<u32x4_t*>(p.pages + (size_t)p.holes[k] * kPageElems) + at;
    u32x4_t v[kEach];
#pragma unroll
    for (int e = 0; e < kEach; ++e) v[e] = ld_stream(s + e * 256);
#pragma unroll
    for (int e = 0; e < kEach; ++e) __builtin_nontemporal_store(v[e], d + e * 256);
  }
}

}  // namespace

int launch_qk_norm_rope(QkNormRopeParams p, const SeqBatch& s, hipStream_t st) {
  int rows = 0;
  for (int b = 0; b < s.n; ++b) {
    p.start[b] = s.start[b];
    p.row_end[b] = rows += s.n_new[b];
  }
  if (!rows) return IE_OK;
  p.n_seqs = s.n;
  const dim3 grid(rows), block(256);
  if (p.heads == 16)
    hipLaunchKernelGGL((qk_norm_rope_kernel<2>), grid, block, 0, st, p);
  else if (p.heads == 32)
    hipLaunchKernelGGL((qk_norm_rope_kernel<3>), grid, block, 0, st, p);
  else
    hipLaunchKernelGGL((qk_norm_rope_kernel<5>), grid, block, 0, st, p);
  IE_CHECK_LAUNCH();
  return IE_OK;
}

int launch_kv_fork(int n_forks, const int* src_rows, const int* dst_rows, const int* n_pos,
                   const int* new_pages, uint16_t* pages, int n_pages, int* tables, int stride,
                   hipStream_t st) {
  ForkParams p{};
  p.pages = pages;
  p.tables = tables;
  p.n_pages = n_pages;
  p.stride = stride;
  int groups = 0, n = 0;
  bool done[kMaxSeqs] = {};
  for (int f = 0; f < n_forks; ++f) {
    if (done[f]) continue;
    p.src[groups] = src_rows[f];
    p.n_pos[groups] = n_pos[f];
    for (int i = f; i < n_forks; ++i) {
      if (src_rows[i] != src_rows[f] || n_pos[i] != n_pos[f]) continue;
      done[i] = true;
      p.dst[n] = dst_rows[i];
      p.page[n++] = new_pages[i];
    }
    p.end[groups++] = n;
  }
  hipLaunchKernelGGL(kv_fork_kernel, dim3(kPlanes, groups), dim3(256), 0, st, p);
  IE_CHECK_LAUNCH();
  return IE_OK;
}

size_t kv_compact_workspace_bytes(int n_pages) { return 2 * (size_t)n_pages * sizeof(int); }

int launch_kv_compact(int n_rows, const int* seq_lens, int window, int n_sinks, uint16_t* pages,
                      int n_pages, const int* tables, int stride, int* new_tables, int* remap,
                      int* counts, void* workspace, hipStream_t st) {
  CompactParams p{};
  p.pages = pages;
  p.tables = tables;
  p.new_tables = new_tables;
  p.remap = remap;
  p.counts = counts;
  p.holes = static_cast<int*>(workspace);
  p.movers = p.holes + n_pages;
  p.n_rows = n_rows;
  p.n_pages = n_pages;
  p.stride = stride;
  p.window = window;
  p.n_sinks = n_sinks;
  for (int r = 0; r < n_rows; ++r) p.len[r] = seq_lens[r];
  hipLaunchKernelGGL(kv_compact_plan_kernel, dim3(1), dim3(kPlanThreads), 0, st, p);
  hipLaunchKernelGGL(kv_compact_move_kernel, dim3(2048), dim3(256), 0, st, p);
  IE_CHECK_LAUNCH();
  return IE_OK;
}

}  // namespace ie
