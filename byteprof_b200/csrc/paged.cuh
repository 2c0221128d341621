// Shared by the paged-attention kernels: the arguments, the cut of the work into units, and the partial
// results that the join kernel adds up.
//
// Sequence s has rows [q_start[s], q_start[s + 1]) of q and kv_len[s] cached positions, its last row at
// position kv_len[s] - 1; row t of it sees the positions up to its own. The g = nh / nkv query heads that share a
// kv head are rows of one matrix: packed row i of (s, kv head h) is token i / g, head h * g + i % g. An item is
// (s, h, one tile of 16 packed rows) with few rows, (s, h, two tiles of 128 / g whole tokens) with many; a unit is one
// block of keys of an item (many rows: an item has kSetup units more). Units are numbered over all items in the
// order s, h, tile, key block, and CTA c of G takes the units [c * share, (c + 1) * share): every CTA has the same
// number of units whatever the lengths are, and the lengths are read on the device, so that a captured graph
// serves every length. An item that lies in one CTA's share is written out by it; otherwise each CTA leaves its
// part (running maximum, sum, unnormalised output; fp32) in the workspace, in slot 2 c + 1 if the item starts in
// its share and 2 c if it started before, and names the item that it leaves unfinished; the join kernel merges the
// parts in CTA order.
#pragma once

#include <cuda.h>

#include "bp_common.cuh"

namespace bp {

constexpr unsigned kPagedFull = 0xffffffffu;

struct PagedArgs {
  const __nv_bfloat16* q;
  long long ldq;
  const __nv_bfloat16* kp;
  const __nv_bfloat16* vp;
  int num_pages, page_log2;
  const int* pages;
  long long ld_pages;
  int max_pages;
  const int* q_start;
  const int* kv_len;
  int seqs, rows, nh, nkv, g, hd;
  float scale_log2;  // softmax scale * log2(e)
  __nv_bfloat16* out;
  long long ldo;
  float* part_o;     // [2 G, tile rows, hd]
  float* part_ml;    // [2 G, tile rows, 2]
  int4* split;       // [G]: the item that starts in a CTA's share and goes on behind it
  int G;
  int min_share;
  int tile_tokens;   // many rows: tokens per tile
};

__device__ __forceinline__ float pg_ex2(float v) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}

// Non-negative a / b; 64-bit division is a call of some 100 instructions, and hardly any count here needs it.
__device__ __forceinline__ long long quotient(long long a, long long b) {
  if (((a | b) >> 32) == 0) return static_cast<uint32_t>(a) / static_cast<uint32_t>(b);
  return a / b;
}

// What is not 0 in a 16-byte piece of 8 bf16 values that holds an Inf or NaN (0 * x is 0 for every finite x).
__device__ __forceinline__ uint32_t not_finite8(const uint4 v) {
  const uint32_t* w = &v.x;
  uint32_t acc = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) asm("fma.rn.bf16x2 %0, %1, %2, %0;" : "+r"(acc) : "r"(w[i]), "r"(0u));
  return acc;
}

// CTAs' equal shares of `total` units.
__device__ __forceinline__ long long share_of(const PagedArgs& a, long long total) {
  const long long s = quotient(total + a.G - 1, a.G);
  return s > a.min_share ? s : a.min_share;
}

// What CTA c leaves for the join kernel: the item that starts in its share and whose parts end in CTA `last` (> c), as
// (sequence, kv head or group of heads, tile, last); last = c: none.
__device__ __forceinline__ void leave_split(const PagedArgs& a, int seq, int head, int tile, int last) {
  a.split[blockIdx.x] = make_int4(seq, head, tile, last);
}

// Values that some rows of a tile do not see. Their weight is 0, but 0 * Inf and 0 * NaN are not: where a block holds
// positions behind the first that a row of the tile does not see, values that are not finite are taken as 0, and the rows that do
// see them give NaN, as for a page that is not there. Only positions of the call's own rows can be of that kind, so this
// costs next to nothing.

// A sequence as the kernels see it: rows clipped to the call's, cached length clipped to the table's.
struct PagedSeq {
  int first, n;       // rows [first, first + n) of q
  int kv;             // cached positions
  int bad;            // the lowest position beyond the table (INT_MAX: none)
  long long pos0;     // position of row `first`
};
__device__ __forceinline__ PagedSeq paged_seq(const PagedArgs& a, int s) {
  PagedSeq r;
  const int b = a.q_start[s], e = a.q_start[s + 1], kv = a.kv_len[s];
  const int b0 = b > 0 ? b : 0, e0 = e < a.rows ? e : a.rows;
  r.first = b0;
  r.n = e0 > b0 ? e0 - b0 : 0;
  // A table may name pages again and again, so it may be longer than any cache: positions from kMaxPos on lie past it (the
  // key counters are 32 bits and run up to a block behind the last key).
  constexpr long long kMaxPos = 0x7fffff00;
  const long long table = static_cast<long long>(a.max_pages) << a.page_log2, cap = table < kMaxPos ? table : kMaxPos;
  r.kv = kv < 0 ? 0 : (kv < cap ? kv : static_cast<int>(cap));
  r.bad = kv > cap ? r.kv : 0x7fffffff;
  r.pos0 = static_cast<long long>(kv) - (static_cast<long long>(e) - b) + (b0 - b);
  return r;
}

// Tensor maps of the cache (paged_attn.cu).
int paged_maps(const PagedArgs& a, int box_rows, CUtensorMap* tk, CUtensorMap* tv);

// The kernel for many rows (paged_attn_tc.cu): scratch bytes, and the launch (a's G, min_share and parts are set there).
size_t paged_tc_workspace_bytes(int hd);
int launch_paged_tc(PagedArgs a, void* workspace, cudaStream_t stream);

}  // namespace bp
