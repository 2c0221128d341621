// Attention of new tokens over a paged cache (bp_paged_attention): the kernel for a few rows per kv head, and the
// kernel that joins split rows. (Many rows: paged_attn_tc.cu.)
//
// Reference: GlobalStep.step attends one position at a time over a StaticCache (byteprof/optim/bolmo.py:100-136).
//
//   out[t, h] = sum_j p_j v_j / sum_j p_j over the positions j up to row t's own, p_j = exp(scale q.k_j - m), one pass
//   over the keys with the running maximum m and sum; rows that see nothing give zeros.
//
// Few rows (single tokens, drafts, grouped heads of one token): memory bound, the keys and values are read once.
// A unit is 64 keys x one tile of 16 packed rows; each of the 4 warps takes 16 of the 64 keys, straight from
// global memory into the pieces that its threads hand to mma.sync: the head dimension is summed in an order that lets a thread
// read 16 consecutive bytes of a key (the same order for q), and the output's columns are numbered so that a
// thread reads 16 consecutive bytes of a value row. No shared memory, no barrier in the loop. The tensor core
// does 16 rows for the price of one here; 16 rows at HBM speed need a tenth of what mma.sync can do, so tcgen05 has
// nothing to add. P is rounded to bf16 for the second product (its relative error, 2^-9 at most, averages out over
// the keys; the sum l adds the unrounded fp32 values).
#include "paged.cuh"
#include "skinny_internal.h"
#include "sm100.cuh"

namespace bp {
namespace {

constexpr int kRows = 16;   // packed rows per tile
constexpr int kKeys = 64;   // keys per unit
constexpr int kWarps = 4;
constexpr int kSlotRows = kWarps * kRows;  // rows of a part: up to 4 heads of a tile
constexpr int kThreads = 32 * kWarps;
constexpr float kLazy = 8.0f;  // the running maximum moves when a score exceeds it by this much (log2 units)

__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t a0, const uint32_t a1, const uint32_t a2,
                                         const uint32_t a3, const uint32_t b0, const uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  const __nv_bfloat162 p = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&p);
}

// Units of sequence s: every tile of a sequence counts the whole cached length (the rows of a few new tokens see
// all but the last few keys).
struct FewUnits {
  int tiles, per;  // row tiles per kv head, units per item
  long long all;
};
// `hp`: kv heads per CTA (below).
__device__ __forceinline__ FewUnits few_units(const PagedArgs& a, const PagedSeq& q, int hp) {
  FewUnits u;
  u.tiles = static_cast<int>((static_cast<long long>(q.n) * a.g + kRows - 1) / kRows);
  u.per = q.kv > kKeys ? (q.kv + kKeys - 1) / kKeys : 1;
  u.all = static_cast<long long>(a.nkv / hp) * u.tiles * u.per;
  return u;
}

// How many kv heads the warps of a CTA take side by side over the same keys (the other warps take other keys). A key's
// heads lie next to each other, so 4 at a time read 1 KB of DRAM in one go instead of 256 bytes here and the rest some
// other time (head_dim 128); with too few units for that, the heads go to CTAs of their own. `one`: units at one head per CTA.
__device__ __forceinline__ int heads_per_cta(const PagedArgs& a, long long one) {
  if (a.nkv % 4 == 0 && one >= 16LL * a.G) return 4;
  if (a.nkv % 2 == 0 && one >= 8LL * a.G) return 2;
  return 1;
}

__device__ __forceinline__ long long share_of(const PagedArgs& a, long long total) {
  const long long s = (total + a.G - 1) / a.G;
  return s > a.min_share ? s : a.min_share;
}

// Sum of the units of all sequences, and (for the sequence holding unit `u`) that sequence and the units before it.
// Every thread of the CTA calls it; `sm` is scratch.
struct Located {
  int s;
  long long before;
};
__device__ long long total_units(const PagedArgs& a, long long* sm) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  long long t = 0;
  for (int s = threadIdx.x; s < a.seqs; s += kThreads) t += few_units(a, paged_seq(a, s), 1).all;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) t += __shfl_xor_sync(kPagedFull, t, o);
  if (lane == 0) sm[warp] = t;
  __syncthreads();
  t = 0;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) t += sm[w];
  __syncthreads();
  return t;
}
__device__ Located locate(const PagedArgs& a, long long u, int hp, long long* sm) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  long long base = 0;
  for (int s0 = 0; s0 < a.seqs; s0 += kThreads) {
    const int s = s0 + threadIdx.x;
    const long long mine = s < a.seqs ? few_units(a, paged_seq(a, s), hp).all : 0;
    long long pre = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long v = __shfl_up_sync(kPagedFull, pre, o);
      if (lane >= o) pre += v;
    }
    if (lane == 31) sm[warp] = pre;
    if (threadIdx.x == 0) sm[kWarps] = -1;
    __syncthreads();
    long long off = base, sum = 0;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      if (w < warp) off += sm[w];
      sum += sm[w];
    }
    pre += off - mine;  // units before s
    if (mine > 0 && u >= pre && u < pre + mine) {
      sm[kWarps] = s;
      sm[kWarps + 1] = pre;
    }
    __syncthreads();
    const long long hit = sm[kWarps], before = sm[kWarps + 1];
    __syncthreads();
    if (hit >= 0) return {static_cast<int>(hit), before};
    base += sum;
  }
  return {-1, 0};
}

// Each warp has a ring of kStages units of its 16 keys and values; a thread copies exactly the 16-byte pieces that it
// will read itself, piece i of lane l at [i][l], so that its own wait_group is all the synchronisation there is.
constexpr int kStages = 3;
template <int HD>
struct FewSmem {
  static constexpr int kPieces = 2 * (HD / 32) + 4 * (HD / 64);  // of the keys, then of the values
  union {
    uint4 ring[kWarps][kStages][kPieces][32];
    struct {
      float o[kWarps][kRows][HD + 4];
      float m[kWarps][kRows], l[kWarps][kRows];
    };
  };
  long long scan[kWarps + 2];
};

// 16 bytes global -> shared, zeros when !ok (nothing is read then).
__device__ __forceinline__ void copy16(uint32_t dst, const void* src, bool ok) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(ok ? 16 : 0) : "memory");
}

// Pages of a warp's 16 keys of a unit: of keys base.. and base + 8.. (a page holds at least 8 positions and base is a
// multiple of 16).
__device__ __forceinline__ void find_pages(const PagedArgs& a, const int* table, int base, int kv, int (&page)[2]) {
#pragma unroll
  for (int i = 0; i < 2; ++i) page[i] = base + 8 * i < kv ? __ldg(table + ((base + 8 * i) >> a.page_log2)) : 0;
}

// Requests the keys base + 8 i + lane / 4, dims 32 c + 8 (lane % 4) .., and the values base + 2 (lane % 4) + {0, 1, 8, 9},
// dims 64 h + 8 (lane / 4) .. Past the end they are zero (what lies there may be NaN, and p = 0 would not hide it). `bad`:
// the lowest position whose page is not in the pool.
template <int HD>
__device__ __forceinline__ void request(const PagedArgs& a, const int (&page)[2], int base, int kv, int h, int lane, uint32_t dst,
                                        int& bad) {
  const long long ld = static_cast<long long>(a.nkv) * HD;
  const int in_page = base & ((1 << a.page_log2) - 1);
  long long row[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int key = base + 8 * i;
    const bool have = page[i] >= 0 && page[i] < a.num_pages;
    if (!have && key < kv) bad = key < bad ? key : bad;
    row[i] = !have || key >= kv ? -1
                                : (static_cast<long long>(page[i]) << a.page_log2) + (a.page_log2 == 3 ? 0 : in_page + 8 * i);
  }
  dst += lane * 16;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int j = lane >> 2;
    const bool ok = row[i] >= 0 && base + 8 * i + j < kv;
    const __nv_bfloat16* p = a.kp + ((ok ? row[i] + j : 0) * ld + h * HD + (lane & 3) * 8);
#pragma unroll
    for (int c = 0; c < HD / 32; ++c) copy16(dst + (i * (HD / 32) + c) * 512, p + 32 * c, ok);
  }
  dst += 2 * (HD / 32) * 512;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int j = 2 * (lane & 3) + (i & 1);
    const bool ok = row[i >> 1] >= 0 && base + 8 * (i >> 1) + j < kv;
    const __nv_bfloat16* p = a.vp + ((ok ? row[i >> 1] + j : 0) * ld + h * HD + (lane >> 2) * 8);
#pragma unroll
    for (int hh = 0; hh < HD / 64; ++hh) copy16(dst + (i * (HD / 64) + hh) * 512, p + 64 * hh, ok);
  }
}

template <int HD>
__global__ void __launch_bounds__(kThreads, 2) paged_few_kernel(const PagedArgs a) {
  extern __shared__ __align__(16) uint8_t smem_raw[];
  FewSmem<HD>& sm = *reinterpret_cast<FewSmem<HD>*>(smem_raw);
  pdl_launch_dependents();
  pdl_wait_prior_grids();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const long long one = total_units(a, sm.scan);
  const int hp = heads_per_cta(a, one), hl = warp % hp, part = warp / hp, step = kKeys / hp;
  const long long total = one / hp;
  const long long share = share_of(a, total);
  long long u = blockIdx.x * share;
  const long long u1 = u + share < total ? u + share : total;
  if (u >= u1) return;
  const Located at = locate(a, u, hp, sm.scan);
  int s = at.s;
  long long before = at.before;
  PagedSeq seq = paged_seq(a, s);
  FewUnits fu = few_units(a, seq, hp);
  while (true) {
    // the segment of this item in the CTA's share
    const long long rel = u - before;
    const int item = static_cast<int>(rel / fu.per), off = static_cast<int>(rel % fu.per);
    const int h = item / fu.tiles * hp + hl, tile = item % fu.tiles;
    const int end = static_cast<int>(fu.per - off < u1 - u ? fu.per : off + (u1 - u));
    const int* table = a.pages + static_cast<long long>(s) * a.ld_pages;

    // q as the A operand: rows lane / 4 and lane / 4 + 8 of the tile, dims 32 c + 8 (lane % 4) ..
    const int nrows = seq.n * a.g;  // packed rows of the sequence
    uint4 qa[HD / 32], qb[HD / 32];
    long long pos[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int r = tile * kRows + (lane >> 2) + 8 * i;
      const bool ok = r < nrows;
      const int tok = ok ? r / a.g : 0;
      const __nv_bfloat16* p = a.q + (seq.first + tok) * a.ldq + (h * a.g + (ok ? r % a.g : 0)) * HD + (lane & 3) * 8;
      pos[i] = ok ? seq.pos0 + tok : -1;
#pragma unroll
      for (int c = 0; c < HD / 32; ++c) {
        const uint4 v = ok ? ldg16(p + 32 * c) : make_uint4(0, 0, 0, 0);
        if (i == 0) qa[c] = v; else qb[c] = v;
      }
    }
    float o[HD / 8][4];
#pragma unroll
    for (int j = 0; j < HD / 8; ++j) o[j][0] = o[j][1] = o[j][2] = o[j][3] = 0.0f;
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f};
    int bad = seq.bad;

    // the ring is kStages units ahead, the pages one more
    uint4(*ring)[FewSmem<HD>::kPieces][32] = sm.ring[warp];
    int page[2];
    const int s0 = off * hp, s1 = end * hp;  // steps of `step` keys of the segment, 16 of them this warp's
#pragma unroll
    for (int st = 0; st < kStages; ++st) {
      const int base = (s0 + st) * step + part * 16;
      if (s0 + st < s1) {
        find_pages(a, table, base, seq.kv, page);
        request<HD>(a, page, base, seq.kv, h, lane, smem_addr(ring[st]), bad);
      }
      cp_async_commit();
    }
    find_pages(a, table, (s0 + kStages) * step + part * 16, s0 + kStages < s1 ? seq.kv : 0, page);
    int st = 0;
    for (int b = s0; b < s1; ++b) {
      const int base = b * step + part * 16;
      cp_async_wait<kStages - 1>();
      const uint4* kr = &ring[st][0][lane];
      const uint4* vr = &ring[st][2 * (HD / 32)][lane];
      float sc[2][4];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        sc[i][0] = sc[i][1] = sc[i][2] = sc[i][3] = 0.0f;
#pragma unroll
        for (int c = 0; c < HD / 32; ++c) {
          const uint4 k = kr[(i * (HD / 32) + c) * 32];
          mma16816(sc[i], qa[c].x, qb[c].x, qa[c].y, qb[c].y, k.x, k.y);
          mma16816(sc[i], qa[c].z, qb[c].z, qa[c].w, qb[c].w, k.z, k.w);
        }
      }
      // scores in log2 units, hidden keys -inf; sc[i][2 r + e] is row r (of the thread's two), key base + 8 i + 2 (lane % 4) + e
      float mx[2] = {-INFINITY, -INFINITY};
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int key = base + 8 * i + 2 * (lane & 3) + (e & 1);
          sc[i][e] = key <= pos[e >> 1] && key < seq.kv ? sc[i][e] * a.scale_log2 : -INFINITY;
          mx[e >> 1] = fmaxf(mx[e >> 1], sc[i][e]);
        }
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        mx[r] = fmaxf(mx[r], __shfl_xor_sync(kPagedFull, mx[r], 1));
        mx[r] = fmaxf(mx[r], __shfl_xor_sync(kPagedFull, mx[r], 2));
      }
      // the maximum moves only when it must: p stays below 2^kLazy, which neither fp32 nor bf16 minds
      if (__any_sync(kPagedFull, mx[0] > m[0] + kLazy || mx[1] > m[1] + kLazy)) {
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const float mn = fmaxf(m[r], mx[r]);
          const float f = m[r] == -INFINITY ? 0.0f : pg_ex2(m[r] - mn);
          m[r] = mn;
          l[r] *= f;
#pragma unroll
          for (int j = 0; j < HD / 8; ++j) {
            o[j][2 * r] *= f;
            o[j][2 * r + 1] *= f;
          }
        }
      }
      float p[2][4];
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float mr = m[e >> 1] == -INFINITY ? 0.0f : m[e >> 1];
          p[i][e] = pg_ex2(sc[i][e] - mr);
          l[e >> 1] += p[i][e];
        }
      const uint32_t a0 = pack2(p[0][0], p[0][1]), a1 = pack2(p[0][2], p[0][3]), a2 = pack2(p[1][0], p[1][1]),
                     a3 = pack2(p[1][2], p[1][3]);
#pragma unroll
      for (int hh = 0; hh < HD / 64; ++hh) {
        const uint4 v0 = vr[(0 * (HD / 64) + hh) * 32], v1 = vr[(1 * (HD / 64) + hh) * 32], v2 = vr[(2 * (HD / 64) + hh) * 32],
                    v3 = vr[(3 * (HD / 64) + hh) * 32];
        const uint32_t* w0 = &v0.x;
        const uint32_t* w1 = &v1.x;
        const uint32_t* w2 = &v2.x;
        const uint32_t* w3 = &v3.x;
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          mma16816(o[8 * hh + 2 * w], a0, a1, a2, a3, __byte_perm(w0[w], w1[w], 0x5410), __byte_perm(w2[w], w3[w], 0x5410));
          mma16816(o[8 * hh + 2 * w + 1], a0, a1, a2, a3, __byte_perm(w0[w], w1[w], 0x7632),
                   __byte_perm(w2[w], w3[w], 0x7632));
        }
      }
      if (b + kStages < s1) request<HD>(a, page, base + kStages * step, seq.kv, h, lane, smem_addr(ring[st]), bad);
      cp_async_commit();
      find_pages(a, table, base + (kStages + 1) * step, b + kStages + 1 < s1 ? seq.kv : 0, page);
      st = st + 1 == kStages ? 0 : st + 1;
    }
    // the 4 warps' parts meet in shared memory (the rings' memory: every warp is through with its own)
    cp_async_wait<0>();
    __syncthreads();
    bad = __reduce_min_sync(kPagedFull, bad);
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      l[r] += __shfl_xor_sync(kPagedFull, l[r], 1);
      l[r] += __shfl_xor_sync(kPagedFull, l[r], 2);
      const int row = (lane >> 2) + 8 * r;
      if ((lane & 3) == 0) {
        sm.m[warp][row] = m[r];
        sm.l[warp][row] = pos[r] >= bad ? __int_as_float(0x7fc00000) : l[r];
      }
#pragma unroll
      for (int hh = 0; hh < HD / 64; ++hh)
#pragma unroll
        for (int e = 0; e < 2; ++e) {  // column 2 (lane % 4) + e of tile j is dim 64 hh + 8 column + j
          float* d = &sm.o[warp][row][64 * hh + (2 * (lane & 3) + e) * 8];
          *reinterpret_cast<float4*>(d) = make_float4(o[8 * hh][2 * r + e], o[8 * hh + 1][2 * r + e], o[8 * hh + 2][2 * r + e],
                                                      o[8 * hh + 3][2 * r + e]);
          *reinterpret_cast<float4*>(d + 4) = make_float4(o[8 * hh + 4][2 * r + e], o[8 * hh + 5][2 * r + e],
                                                          o[8 * hh + 6][2 * r + e], o[8 * hh + 7][2 * r + e]);
        }
    }
    __syncthreads();
    const bool whole = off == 0 && end == fu.per;
    const int slot = 2 * blockIdx.x + (off == 0 ? 1 : 0);
    constexpr int kPer = HD / 8;  // dims per thread: 8 threads per row
    for (int j = 0; j < hp; ++j) {  // warps j, j + hp, .. hold parts of head j
      const int row = tid / 8, d0 = (tid % 8) * kPer, hj = item / fu.tiles * hp + j;
      const int r = tile * kRows + row;
      if (r < nrows) {
        float mm = -INFINITY, ll = 0.0f, acc[kPer];
        for (int w = j; w < kWarps; w += hp) mm = fmaxf(mm, sm.m[w][row]);
#pragma unroll
        for (int d = 0; d < kPer; ++d) acc[d] = 0.0f;
        for (int w = j; w < kWarps; w += hp) {
          const float f = sm.m[w][row] == -INFINITY ? 0.0f : pg_ex2(sm.m[w][row] - mm);
          ll += f == 0.0f && !isnan(sm.l[w][row]) ? 0.0f : f * sm.l[w][row];
#pragma unroll
          for (int d = 0; d < kPer; ++d) acc[d] = fmaf(f, sm.o[w][row][d0 + d], acc[d]);
        }
        if (whole) {
          const float inv = ll == 0.0f ? 0.0f : 1.0f / ll;
          uint32_t w[kPer / 2];
#pragma unroll
          for (int d = 0; d < kPer / 2; ++d) w[d] = pack2(acc[2 * d] * inv, acc[2 * d + 1] * inv);
          __nv_bfloat16* dst = a.out + (seq.first + r / a.g) * a.ldo + (hj * a.g + r % a.g) * HD + d0;
#pragma unroll
          for (int d = 0; d < kPer / 8; ++d)
            reinterpret_cast<uint4*>(dst)[d] = make_uint4(w[4 * d], w[4 * d + 1], w[4 * d + 2], w[4 * d + 3]);
        } else {
          const size_t at = static_cast<size_t>(slot) * kSlotRows + j * kRows + row;
          float* dst = a.part_o + at * HD + d0;
#pragma unroll
          for (int d = 0; d < kPer / 4; ++d)
            reinterpret_cast<float4*>(dst)[d] = make_float4(acc[4 * d], acc[4 * d + 1], acc[4 * d + 2], acc[4 * d + 3]);
          if (d0 == 0) reinterpret_cast<float2*>(a.part_ml)[at] = make_float2(mm, ll);
        }
      }
    }
    u += end - off;
    if (u >= u1) break;
    __syncthreads();  // sm.o is written again
    if (u - before >= fu.all) {  // on to the next sequence that has rows
      before += fu.all;
      do {
        ++s;
        seq = paged_seq(a, s);
      } while (seq.n == 0);
      fu = few_units(a, seq, hp);
    }
  }
}

// Joins the parts of the split items: one CTA per (row, head).
template <int HD>
__global__ void __launch_bounds__(kThreads) paged_few_join_kernel(const PagedArgs a) {
  __shared__ float sm_l[kWarps];
  __shared__ float sm_o[kWarps][HD];
  __shared__ long long scan[kWarps + 2];
  __shared__ int found[1];
  pdl_launch_dependents();
  pdl_wait_prior_grids();
  const int t = blockIdx.x, head = blockIdx.y, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  // the row's sequence, the units before it, and the total
  long long before = 0, total = 0;
  if (tid == 0) found[0] = -1;
  __syncthreads();
  for (int s = tid; s < a.seqs; s += kThreads) {
    const PagedSeq q = paged_seq(a, s);
    const long long n = few_units(a, q, 1).all;
    total += n;
    if (q.first + q.n <= t) before += n;
    if (q.n > 0 && t >= q.first && t < q.first + q.n) found[0] = s;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    before += __shfl_xor_sync(kPagedFull, before, o);
    total += __shfl_xor_sync(kPagedFull, total, o);
  }
  if (lane == 0) scan[warp] = before;
  __syncthreads();
  before = scan[0] + scan[1] + scan[2] + scan[3];
  __syncthreads();
  if (lane == 0) scan[warp] = total;
  __syncthreads();
  total = scan[0] + scan[1] + scan[2] + scan[3];
  const int s = found[0];
  if (s < 0) return;
  const PagedSeq q = paged_seq(a, s);
  const int hp = heads_per_cta(a, total), h = head / a.g;
  const FewUnits fu = few_units(a, q, hp);
  const long long share = share_of(a, total / hp);
  const int pr = (t - q.first) * a.g + head % a.g;
  const long long a0 = before / hp + (static_cast<long long>(h / hp) * fu.tiles + pr / kRows) * fu.per;
  const int c0 = static_cast<int>(a0 / share), c1 = static_cast<int>((a0 + fu.per - 1) / share);
  if (c0 == c1) return;
  const int row = h % hp * kRows + pr % kRows;
  constexpr int kPer = HD / 32;
  const float2* ml = reinterpret_cast<const float2*>(a.part_ml);
  float m = -INFINITY;
  for (int c = c0 + lane; c <= c1; c += 32) m = fmaxf(m, ml[static_cast<size_t>(2 * c + (c == c0)) * kSlotRows + row].x);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(kPagedFull, m, o));
  float l = 0.0f, acc[kPer];
#pragma unroll
  for (int j = 0; j < kPer; ++j) acc[j] = 0.0f;
#pragma unroll 4
  for (int c = c0 + warp; c <= c1; c += kWarps) {
    const size_t at = static_cast<size_t>(2 * c + (c == c0)) * kSlotRows + row;
    const float2 p = ml[at];
    const float f = p.x == -INFINITY ? 0.0f : pg_ex2(p.x - m);
    l += f == 0.0f && !isnan(p.y) ? 0.0f : f * p.y;
    const float* src = a.part_o + at * HD + lane * kPer;
#pragma unroll
    for (int j = 0; j < kPer; ++j) acc[j] = fmaf(f, src[j], acc[j]);
  }
  if (lane == 0) sm_l[warp] = l;
#pragma unroll
  for (int j = 0; j < kPer; ++j) sm_o[warp][lane * kPer + j] = acc[j];
  __syncthreads();
  if (tid < HD) {
    float v = 0.0f;
    l = 0.0f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      l += sm_l[w];
      v += sm_o[w][tid];
    }
    a.out[t * a.ldo + head * HD + tid] = __float2bfloat16_rn(l == 0.0f ? 0.0f : v / l);
  }
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

constexpr int kCtasPerSm = 2;

// Up to 32 packed rows per sequence and kv head on average (the lengths themselves are on the device): two tiles of the
// 16-row kernel, which then reads each key twice; the other kernel pads to 128
// and takes groups of up to 128 heads.
bool few_rows(int rows, int seqs, int g) { return static_cast<long long>(rows) * g <= 32LL * seqs || g > 128; }

int few_grid() { return kCtasPerSm * tc_sm_count(); }

template <int HD>
cudaError_t launch_few(const PagedArgs& a, cudaStream_t s) {
  static bool ready[64] = {false};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64 || !ready[dev]) {
    const cudaError_t e = cudaFuncSetAttribute(paged_few_kernel<HD>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                               static_cast<int>(sizeof(FewSmem<HD>)));
    if (e != cudaSuccess) return e;
    if (dev >= 0 && dev < 64) ready[dev] = true;
  }
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[2];
  cfg.gridDim = dim3(a.G);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = sizeof(FewSmem<HD>);
  cfg.stream = s;
  set_launch_attrs(cfg, attr);
  cudaError_t e = cudaLaunchKernelEx(&cfg, paged_few_kernel<HD>, a);
  if (e != cudaSuccess) return e;
  cfg.gridDim = dim3(a.rows, a.nh);
  cfg.dynamicSmemBytes = 0;
  return cudaLaunchKernelEx(&cfg, paged_few_join_kernel<HD>, a);
}

}  // namespace
}  // namespace bp

extern "C" size_t bp_paged_attention_workspace_bytes(int rows, int seqs, int nh, int nkv, int head_dim) {
  using namespace bp;
  if (rows <= 0 || seqs <= 0 || nkv <= 0 || nh < nkv || head_dim <= 0) return 0;
  return few_rows(rows, seqs, nh / nkv) ? static_cast<size_t>(2 * few_grid()) * kSlotRows * (head_dim + 2) * sizeof(float)
                                        : paged_tc_workspace_bytes(head_dim);
}

extern "C" int bp_paged_attention(const void* q, long long ldq, const void* k_pages, const void* v_pages, int num_pages,
                                  int page_size, const int32_t* pages, long long ld_pages, int max_pages,
                                  const int32_t* q_start, const int32_t* kv_len, int seqs, int rows, int nh, int nkv,
                                  int head_dim, float scale, void* out, long long ldo, void* workspace,
                                  size_t workspace_bytes, void* stream) {
  using namespace bp;
  clear_error();
  if (seqs < 0 || rows < 0 || num_pages < 0 || max_pages < 0)
    return fail(BP_ERR_INVALID_ARGUMENT, "negative size (seqs=%d rows=%d num_pages=%d max_pages=%d)", seqs, rows,
                num_pages, max_pages);
  if (nkv < 1 || nh < nkv || nh % nkv != 0 || nh > 1024)
    return fail(BP_ERR_INVALID_ARGUMENT, "nh=%d must be a multiple of nkv=%d (at most 1024 heads)", nh, nkv);
  if (head_dim != 64 && head_dim != 128)
    return fail(BP_ERR_UNSUPPORTED, "paged attention supports head_dim 64 and 128 (got %d)", head_dim);
  if (page_size < 8 || page_size > 256 || (page_size & (page_size - 1)) != 0)
    return fail(BP_ERR_UNSUPPORTED, "page_size must be a power of two from 8 to 256 (got %d)", page_size);
  if (rows > (1 << 20)) return fail(BP_ERR_UNSUPPORTED, "paged attention takes at most 2^20 rows per call (got %d)", rows);
  if (static_cast<long long>(num_pages) * page_size > 0x7fffffffLL - 256)
    return fail(BP_ERR_UNSUPPORTED, "the cache holds at most 2^31 positions (got %d pages of %d)", num_pages, page_size);
  if (rows == 0 || seqs == 0) return BP_OK;
  if (num_pages < 1) return fail(BP_ERR_INVALID_ARGUMENT, "a cache of no pages");
  if (q == nullptr || pages == nullptr || q_start == nullptr || kv_len == nullptr || k_pages == nullptr ||
      v_pages == nullptr || out == nullptr)
    return fail(BP_ERR_INVALID_ARGUMENT, "a pointer argument is NULL");
  if (ldq < static_cast<long long>(nh) * head_dim || ldo < static_cast<long long>(nh) * head_dim || ld_pages < max_pages)
    return fail(BP_ERR_INVALID_ARGUMENT, "row strides must cover a row of q, of out and of the page table");
  if (!(scale > 0.0f) || scale > 1e30f) return fail(BP_ERR_INVALID_ARGUMENT, "scale must be positive and finite");
  if (!aligned16(q) || !aligned16(out) || !aligned16(k_pages) || !aligned16(v_pages) || ldq % 8 != 0 || ldo % 8 != 0)
    return fail(BP_ERR_MISALIGNED, "paged_attention needs 16-byte aligned bases and row strides multiples of 8");
  int st = require_sm100();
  if (st != BP_OK) return st;
  const size_t need = bp_paged_attention_workspace_bytes(rows, seqs, nh, nkv, head_dim);
  if (workspace == nullptr || workspace_bytes < need)
    return fail(BP_ERR_INVALID_ARGUMENT, "paged_attention needs a workspace of %zu bytes (got %zu)", need, workspace_bytes);
  if ((reinterpret_cast<uintptr_t>(workspace) & 255u) != 0)
    return fail(BP_ERR_MISALIGNED, "workspace must be 256-byte aligned");
  int lg = 3;
  while ((1 << lg) < page_size) ++lg;
  PagedArgs a{};
  a.q = static_cast<const __nv_bfloat16*>(q);
  a.ldq = ldq;
  a.kp = static_cast<const __nv_bfloat16*>(k_pages);
  a.vp = static_cast<const __nv_bfloat16*>(v_pages);
  a.num_pages = num_pages;
  a.page_log2 = lg;
  a.pages = pages;
  a.ld_pages = ld_pages;
  a.max_pages = max_pages;
  a.q_start = q_start;
  a.kv_len = kv_len;
  a.seqs = seqs;
  a.rows = rows;
  a.nh = nh;
  a.nkv = nkv;
  a.g = nh / nkv;
  a.hd = head_dim;
  a.scale_log2 = scale * 1.4426950408889634f;
  a.out = static_cast<__nv_bfloat16*>(out);
  a.ldo = ldo;
  if (!few_rows(rows, seqs, a.g)) {
    st = launch_paged_tc(a, workspace, static_cast<cudaStream_t>(stream));
    return st != BP_OK ? st : check_launch("paged_attention");
  }
  a.G = few_grid();
  a.min_share = 1;
  a.part_o = static_cast<float*>(workspace);
  a.part_ml = a.part_o + static_cast<size_t>(2 * a.G) * kSlotRows * head_dim;
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  const cudaError_t e = head_dim == 128 ? launch_few<128>(a, s) : launch_few<64>(a, s);
  if (e != cudaSuccess) return fail(BP_ERR_CUDA, "paged_attention launch: %s", cudaGetErrorString(e));
  return check_launch("paged_attention");
}
