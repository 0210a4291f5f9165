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
// lanes apart.  A workgroup takes 16 heads of one row.
__global__ __launch_bounds__(256) void qk_norm_rope_kernel(QkNormRopeParams p) {
  const int tid = threadIdx.x, lane = tid & 63, li = tid & 15;
  const int row = blockIdx.x, head = blockIdx.y * 16 + (tid >> 4);
  const int b = __popcll(__ballot(lane < p.n_seqs && p.row_end[lane] <= row));
  const int pos = p.start[b] + row - (b ? p.row_end[b - 1] : 0);
  const u32x4_t x = *reinterpret_cast<const u32x4_t*>(p.qkv + (size_t)row * p.qkv_stride +
                                                      (size_t)head * kHeadDim + 8 * li);
  const bool is_q = head < p.heads, is_v = head >= p.heads + kKVHeads;
  u32x4_t y = x;
  if (!is_v) {
    float v[8];
#pragma unroll
    for (int e = 0; e < 4; ++e) v[2 * e] = bf_lo(x[e]), v[2 * e + 1] = bf_hi(x[e]);
    const uint16_t* w = is_q ? p.q_norm : p.k_norm;
    if (w) {
      const u32x4_t wv = *reinterpret_cast<const u32x4_t*>(w + 8 * li);
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
    const float4* c4 = reinterpret_cast<const float4*>(p.rope_cos + (size_t)pos * 64 + 8 * (li & 7));
    const float4* s4 = reinterpret_cast<const float4*>(p.rope_sin + (size_t)pos * 64 + 8 * (li & 7));
    const float4 ca = c4[0], cb = c4[1], sa = s4[0], sb = s4[1];
    const float c[8] = {ca.x, ca.y, ca.z, ca.w, cb.x, cb.y, cb.z, cb.w};
    const float s[8] = {sa.x, sa.y, sa.z, sa.w, sb.x, sb.y, sb.z, sb.w};
    float t[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float other = dpp_f<0x128>(v[e]);  // row_ror 8: the partner dim
      t[e] = li < 8 ? rope_lo(v[e], other, c[e], s[e]) : rope_hi(other, v[e], c[e], s[e]);
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) y[e] = pack_bf2(t[2 * e], t[2 * e + 1]);
  }
  uint16_t* dst;
  if (is_q) {
    dst = p.q_out + ((size_t)row * p.heads + head) * kHeadDim;
  } else {
    const int page = p.block_tables[(size_t)b * p.table_stride + pos / kPagePos];
    if (page < 0 || page >= p.n_pages) return;
    const int kvh = (head - p.heads) & (kKVHeads - 1);
    dst = (is_v ? p.v : p.k) + (size_t)page * kPageElems +
          ((size_t)kvh * kPagePos + pos % kPagePos) * kHeadDim;
  }
  *reinterpret_cast<u32x4_t*>(dst + 8 * li) = y;
}

// ---------------------------------------------------------------- fork
struct ForkParams {
  uint16_t* pages;
  int* tables;
  int n_pages, stride;
  int src[kMaxSeqs], dst[kMaxSeqs], n_pos[kMaxSeqs], page[kMaxSeqs];
};
constexpr int kPlanes = kLayers * 2 * kKVHeads;  // [64][128] planes of a page

// blockIdx.y: the fork.  The first n_pos % 64 positions of the source's last page, plane by plane;
// the first workgroup also writes the table row.
__global__ __launch_bounds__(256) void kv_fork_kernel(ForkParams p) {
  const int f = blockIdx.y, full = p.n_pos[f] / kPagePos, part = p.n_pos[f] % kPagePos;
  const int* from = p.tables + (size_t)p.src[f] * p.stride;
  if (blockIdx.x == 0) {
    int* to = p.tables + (size_t)p.dst[f] * p.stride;
    for (int i = threadIdx.x; i < p.stride; i += 256)
      to[i] = i < full ? from[i] : i == full && part ? p.page[f] : -1;
  }
  if (!part) return;
  const int src = from[full];
  if (src < 0 || src >= p.n_pages) return;
  const u32x4_t* s = reinterpret_cast<const u32x4_t*>(p.pages + (size_t)src * kPageElems);
  u32x4_t* d = reinterpret_cast<u32x4_t*>(p.pages + (size_t)p.page[f] * kPageElems);
  const int n = part * (kHeadDim / 8);  // 16-byte pieces a plane
  for (int i = blockIdx.x * 256 + threadIdx.x; i < n * kPlanes; i += gridDim.x * 256) {
    const int at = i / n * (kPagePos * kHeadDim / 8) + i % n;
    d[at] = s[at];
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
// remapped tables.
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

// Moves the pages: sources are ids >= the live count, destinations free ids below it.
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
  p.rows = rows;
  hipLaunchKernelGGL(qk_norm_rope_kernel, dim3(rows, (p.heads + 2 * kKVHeads) / 16), dim3(256), 0, st, p);
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
  for (int f = 0; f < n_forks; ++f) {
    p.src[f] = src_rows[f];
    p.dst[f] = dst_rows[f];
    p.n_pos[f] = n_pos[f];
    p.page[f] = new_pages[f];
  }
  hipLaunchKernelGGL(kv_fork_kernel, dim3(128, n_forks), dim3(256), 0, st, p);
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
