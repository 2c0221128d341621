// Attention of new tokens over a paged cache (bp_paged_attention): the kernel for a few rows per kv head, and the
// kernel that joins split rows. (Many rows: paged_attn_tc.cu.)
//
// Reference: GlobalStep.step attends one position at a time over a StaticCache (byteprof/optim/bolmo.py:100-136).
//
//   out[t, h] = sum_j p_j v_j / sum_j p_j over the positions j up to row t's own, p_j = exp(scale q.k_j - m), one pass
//   over the keys with the running maximum m and sum; rows that see nothing give zeros.
//
// Few rows (single tokens, drafts, grouped heads of one token): memory bound, the keys and values are read once.
// A unit is 64 keys x one tile of 16 packed rows. One warp finds the pages and loads the keys and values by TMA (16 rows
// of 64 dims a box, 128-byte swizzle) into a ring of 3 steps of 32 KB, two CTAs per SM; four warps take 16 keys each
// of a step. The 16-byte pieces that a thread reads from the swizzled tiles are its mma.sync operands as they are: the
// head dimension is summed in an order that lets a thread use 8 consecutive values of a key (the same order for q),
// keys and output columns are numbered so that the 8 lanes of a shared-memory phase touch all banks. The tensor core
// does 16 rows for the price of one here; 16 rows at HBM speed need a tenth of what mma.sync can do, so tcgen05 has
// nothing to add. P is rounded to bf16 for the second product (its relative error, 2^-8 at most, averages out over
// the keys; the sum l adds the unrounded fp32 values).
// 64 streams of up to 8192 keys, 32 heads of 128 over 8: 185 to 191 us for 1.13 GB, 5.9 to 6.1 TB/s, where registers filled
// straight from global memory, one unit ahead, took 225; 5 drafted tokens over 30001 keys 51 us (4.8 TB/s), one token over
// 1025 10.1 (latency: the cut, one trip through the ring, the join).
#include <cudaTypedefs.h>

#include <algorithm>

#include "paged.cuh"
#include "skinny_internal.h"
#include "sm100.cuh"

namespace bp {
namespace {

constexpr int kRows = 16;   // packed rows per tile
constexpr int kKeys = 64;   // keys per unit
constexpr int kWarps = 4;   // that compute; one more loads
constexpr int kSlotRows = kWarps * kRows;  // rows of a part: up to 4 heads of a tile
constexpr int kThreads = 32 * (kWarps + 1);
constexpr int kMathThreads = 32 * kWarps;
constexpr int kStages = 3;
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
  u.tiles = (q.n * a.g + kRows - 1) / kRows;  // at most 2^30 rows
  u.per = q.kv > kKeys ? (q.kv + kKeys - 1) / kKeys : 1;
  u.all = static_cast<long long>(a.nkv >> (hp >> 1)) * u.tiles * u.per;  // (hp: 1, 2 or 4)
  return u;
}

// How many kv heads the warps of a CTA take side by side over the same keys (the other warps take other keys). A key's
// heads lie next to each other, so 4 at a time read 1 KB of DRAM in one go instead of 256 bytes here and the rest some
// other time (head_dim 128); with too few units for that, the heads go to CTAs of their own. `one`: units at one head per CTA.
// Measured with 1, 2 and 4 heads fixed: 64 streams of up to 8192 keys (117 G units) 193, 192 and 185 us; 5 tokens over 30001
// keys (25 G) 50, 60 and 78; one token over 1025 (1 G) 9.5, 13.4 and 19.5.
__device__ __forceinline__ int heads_per_cta(const PagedArgs& a, long long one) {
  if (a.nkv % 4 == 0 && one >= 64LL * a.G) return 4;
  if (a.nkv % 2 == 0 && one >= 32LL * a.G) return 2;
  return 1;
}

constexpr int kScan = kThreads / 32;
// Sum of the units of all sequences, and (for the sequence holding unit `u`) that sequence and the units before it.
// Every thread of the CTA calls it; `sm` is scratch.
struct Located {
  int s;
  long long before;
};
__device__ long long total_units(const PagedArgs& a, long long* sm) {
  if (a.seqs == 1) return few_units(a, paged_seq(a, 0), 1).all;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  long long t = 0;
  for (int s = threadIdx.x; s < a.seqs; s += kThreads) t += few_units(a, paged_seq(a, s), 1).all;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) t += __shfl_xor_sync(kPagedFull, t, o);
  if (lane == 0) sm[warp] = t;
  __syncthreads();
  t = 0;
#pragma unroll
  for (int w = 0; w < kThreads / 32; ++w) t += sm[w];
  __syncthreads();
  return t;
}
__device__ Located locate(const PagedArgs& a, long long u, int hp, long long* sm) {
  if (a.seqs == 1) return {0, 0};
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
    if (threadIdx.x == 0) sm[kScan] = -1;
    __syncthreads();
    long long off = base, sum = 0;
#pragma unroll
    for (int w = 0; w < kScan; ++w) {
      if (w < warp) off += sm[w];
      sum += sm[w];
    }
    pre += off - mine;  // units before s
    if (mine > 0 && u >= pre && u < pre + mine) {
      sm[kScan] = s;
      sm[kScan + 1] = pre;
    }
    __syncthreads();
    const long long hit = sm[kScan], before = sm[kScan + 1];
    __syncthreads();
    if (hit >= 0) return {static_cast<int>(hit), before};
    base += sum;
  }
  return {-1, 0};
}

template <int HD>
struct FewSmem {
  static constexpr int kWarpTile = kRows * HD * 2;             // 16 keys (or values) of a warp
  static constexpr int kStageBytes = 2 * kWarps * kWarpTile;   // [warp][K, V][64 dims][16 rows][128 bytes]
  uint8_t ring[kStages][kStageBytes];
  float o[kWarps][kRows][64];
  float m[kWarps][kRows], l[kWarps][kRows];
  uint64_t full[kStages], empty[kStages];
  int bad[kStages];
  int abort;
  long long scan[kScan + 2];
};

// A CTA's walk over its units: one segment (a range of units of one item) at a time.
struct FewWalk {
  PagedSeq q;
  FewUnits fu;
  int s, item, off, end;
  long long before, u, u1;
  __device__ __forceinline__ void segment() {
    const long long rel = u - before;
    item = static_cast<int>(quotient(rel, fu.per));
    off = static_cast<int>(rel - static_cast<long long>(item) * fu.per);
    end = static_cast<int>(fu.per - off < u1 - u ? fu.per : off + (u1 - u));
  }
  __device__ __forceinline__ void start(const PagedArgs& a, const Located& at, int hp, long long first, long long last) {
    s = at.s;
    before = at.before;
    u = first;
    u1 = last;
    q = paged_seq(a, s);
    fu = few_units(a, q, hp);
    segment();
  }
  __device__ __forceinline__ bool next(const PagedArgs& a, int hp) {
    u += end - off;
    if (u >= u1) return false;
    if (u - before >= fu.all) {  // on to the next sequence that has rows
      before += fu.all;
      do {
        ++s;
        q = paged_seq(a, s);
      } while (q.n == 0);
      fu = few_units(a, q, hp);
    }
    segment();
    return true;
  }
};

// Rows `lo` and up of a warp's V tile (keys base + lo ..), by that warp: pieces that are not finite become 0, those past the
// sequence's end too; the first key that had one (INT_MAX: none).
template <int HD>
__device__ __forceinline__ int hide_not_finite(uint8_t* vt, int lo, int base, int lane) {
  constexpr int kPer = HD / 8, kU = 4;  // pieces of a row, in flight
  int lost = 0x7fffffff;
#pragma unroll 1
  for (int c0 = lane; c0 < (kRows - lo) * kPer; c0 += 32 * kU) {
    uint4 x[kU];
    auto at = [&](int u) {
      const int c = c0 + 32 * u, piece = c % kPer;
      return reinterpret_cast<uint4*>(vt + (piece >> 3) * (kRows * 128) + (lo + c / kPer) * 128 + (piece & 7) * 16);
    };
#pragma unroll
    for (int u = 0; u < kU; ++u) x[u] = c0 + 32 * u < (kRows - lo) * kPer ? *at(u) : make_uint4(0, 0, 0, 0);
#pragma unroll
    for (int u = 0; u < kU; ++u)
      if (not_finite8(x[u]) != 0) {
        *at(u) = make_uint4(0, 0, 0, 0);
        lost = min(lost, base + lo + (c0 + 32 * u) / kPer);
      }
  }
  fence_async_shared();  // the slot is refilled by TMA
  __syncwarp();
  return __reduce_min_sync(kPagedFull, lost);
}

template <int HD>
__global__ void __launch_bounds__(kThreads, 2)
    paged_few_kernel(const __grid_constant__ CUtensorMap tk, const __grid_constant__ CUtensorMap tv, const PagedArgs a) {
  using S = FewSmem<HD>;
  extern __shared__ uint8_t smem_raw[];
  // The kernel has no static shared memory, so the dynamic part starts behind the first 1024 bytes, aligned for the
  // swizzle; room to align it would cost the second CTA on the SM.
  if ((smem_addr(smem_raw) & 1023u) != 0) {
    if (threadIdx.x == 0) atomicOr(&g_bp_device_errors, BP_DEVERR_TIMEOUT);
    return;
  }
  S& sm = *reinterpret_cast<S*>(smem_raw);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  if (tid == 0) {
    for (int i = 0; i < kStages; ++i) {
      mbar_init(&sm.full[i], 1);
      mbar_init(&sm.empty[i], kWarps);
    }
    sm.abort = 0;
    mbar_fence_init();
    tma_prefetch_desc(&tk);
    tma_prefetch_desc(&tv);
  }
  pdl_launch_dependents();
  pdl_wait_prior_grids();
  volatile int* abort = &sm.abort;
  __syncthreads();  // the barriers are initialised
  const long long one = total_units(a, sm.scan);
  const int hp = heads_per_cta(a, one), step = kKeys / hp;
  const long long total = one >> (hp >> 1);
  const long long share = share_of(a, total), u0 = blockIdx.x * share;
  const long long u1 = u0 + share < total ? u0 + share : total;
  if (u0 >= u1) {
    if (tid == 0) leave_split(a, 0, 0, 0, blockIdx.x);
    return;
  }
  const Located at = locate(a, u0, hp, sm.scan);
  FewWalk w;
  w.start(a, at, hp, u0, u1);

  if (warp == kWarps) {
    // ---- pages and TMA: one box per lane ----
    const int box = min(1 << a.page_log2, kRows), per = kRows / box;  // rows of a box, boxes per 16 keys
    const int boxes = 2 * kWarps * (HD / 64) * per, none = a.num_pages << a.page_log2;
    // lane: (key or value, 64 dims, warp, rows of its 16)
    const int sub = lane % per, wi = lane / per % kWarps, half = lane / (per * kWarps) % (HD / 64), kv = lane / (per * kWarps * (HD / 64));
    const int hl = wi % hp, part = wi / hp;
    const uint32_t at_off = static_cast<uint32_t>(((wi * 2 + kv) * (HD / 64) + half) * kRows * 128 + sub * box * 128);
    int n = 0;  // steps issued
    bool ok = true;
    int4 open = make_int4(0, 0, 0, blockIdx.x);
    do {
      if (w.off == 0 && w.end < w.fu.per)
        open = make_int4(w.s, w.item / w.fu.tiles, w.item % w.fu.tiles,
                         blockIdx.x + static_cast<int>(quotient(w.fu.per - w.end + share - 1, share)));
      const int* table = a.pages + static_cast<long long>(w.s) * a.ld_pages;
      const int h = w.item / w.fu.tiles * hp + hl;
      const int s1 = w.end * hp;
      // pages one step ahead of their use
      int key = w.off * hp * step + part * kRows + sub * box;
      int page = lane < boxes && key < w.q.kv ? table[key >> a.page_log2] : -1;
      for (int b = w.off * hp; b < s1; ++b, ++n) {
        int row = none, bad = w.q.bad;
        if (key < w.q.kv && lane < boxes) {
          if (page >= 0 && page < a.num_pages)
            row = (page << a.page_log2) + (key & ((1 << a.page_log2) - 1));
          else
            bad = min(bad, key);
        }
        bad = __reduce_min_sync(kPagedFull, bad);
        key += step;
        page = b + 1 < s1 && lane < boxes && key < w.q.kv ? table[key >> a.page_log2] : -1;
        const int st = n % kStages;
        int go = 1;
        if (lane == 0) {
          if (n >= kStages) go = mbar_wait(&sm.empty[st], static_cast<uint32_t>((n / kStages) + 1) & 1u, abort);
          if (go) {
            sm.bad[st] = bad;
            mbar_arrive_expect_tx(&sm.full[st], S::kStageBytes);
          }
        }
        ok = __shfl_sync(kPagedFull, go, 0) != 0;
        if (!ok) break;
        if (lane < boxes) tma_load_3d(sm.ring[st] + at_off, kv == 0 ? &tk : &tv, &sm.full[st], half * 64, row, h);
        __syncwarp();
      }
    } while (ok && w.next(a, hp));
    if (lane == 0) leave_split(a, open.x, open.y | hp << 24, open.z, open.w);
    if (lane == 0)  // no copy is in flight when the CTA ends
      for (int st = 0; st < kStages && st < n; ++st) {
        const unsigned long long t0 = globaltimer();
        while (!mbar_try_wait(&sm.full[st], static_cast<uint32_t>((n - 1 - st) / kStages) & 1u)) {
          if (globaltimer() - t0 > kWaitLimitNs) {
            atomicOr(&g_bp_device_errors, BP_DEVERR_TIMEOUT);
            break;
          }
        }
      }
    __syncwarp();
    return;
  }

  const int hl = warp % hp, part = warp / hp, c4 = lane & 3, l4 = lane >> 2;
  const int kperm = (l4 >> 1) + 4 * (l4 & 1);  // the key (of 8) behind MMA column l4, and the dims' chunk behind output column l4
  int n = 0;
  do {
    const int h = w.item / w.fu.tiles * hp + hl, tile = w.item % w.fu.tiles;
    // q as the A operand: rows lane / 4 and lane / 4 + 8 of the tile, dims 32 c + 8 (lane % 4) ..
    const int nrows = w.q.n * a.g;  // packed rows of the sequence
    uint4 qa[HD / 32], qb[HD / 32];
    long long pos[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int r = tile * kRows + l4 + 8 * i;
      const bool ok = r < nrows;
      const int tok = ok ? r / a.g : 0;
      const __nv_bfloat16* p = a.q + (w.q.first + tok) * a.ldq + (h * a.g + (ok ? r % a.g : 0)) * HD + c4 * 8;
      pos[i] = ok ? w.q.pos0 + tok : -1;
#pragma unroll
      for (int c = 0; c < HD / 32; ++c) {
        const uint4 v = ok ? ld16(p + 32 * c) : make_uint4(0, 0, 0, 0);
        if (i == 0) qa[c] = v; else qb[c] = v;
      }
    }
    float o[HD / 8][4];
#pragma unroll
    for (int j = 0; j < HD / 8; ++j) o[j][0] = o[j][1] = o[j][2] = o[j][3] = 0.0f;
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f};
    int bad = w.q.bad;
    // cached positions that every row of the tile sees
    const int all_see = static_cast<int>(max(min(w.q.pos0 + tile * kRows / a.g + 1, static_cast<long long>(w.q.kv)), 0LL));
    bool dead = false;
    for (int b = w.off * hp; b < w.end * hp; ++b, ++n) {
      const int base = b * step + part * kRows, st = n % kStages;
      const bool ok = mbar_wait(&sm.full[st], static_cast<uint32_t>(n / kStages) & 1u, abort);
      if (!__all_sync(kPagedFull, ok)) {
        dead = true;
        break;
      }
      bad = min(bad, sm.bad[st]);
      // piece (row, chunk) of a tile is at row * 128 + (chunk ^ (row & 7)) * 16
      const uint8_t* kt = sm.ring[st] + warp * 2 * S::kWarpTile;
      uint8_t* vt = sm.ring[st] + (warp * 2 + 1) * S::kWarpTile;
      if (base + kRows > all_see) bad = min(bad, hide_not_finite<HD>(vt, max(all_see - base, 0), base, lane));
      float sc[2][4];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        sc[i][0] = sc[i][1] = sc[i][2] = sc[i][3] = 0.0f;
#pragma unroll
        for (int c = 0; c < HD / 32; ++c) {
          const int chunk = (c & 1) * 4 + c4;
          const uint4 k = *reinterpret_cast<const uint4*>(kt + (c >> 1) * (kRows * 128) + (8 * i + kperm) * 128 + ((chunk ^ kperm) * 16));
          mma16816(sc[i], qa[c].x, qb[c].x, qa[c].y, qb[c].y, k.x, k.y);
          mma16816(sc[i], qa[c].z, qb[c].z, qa[c].w, qb[c].w, k.z, k.w);
        }
      }
      // scores in log2 units, hidden keys -inf; sc[i][2 r + e] is row r (of the thread's two), key base + 8 i + lane % 4 + 4 e
      float mx[2] = {-INFINITY, -INFINITY};
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int key = base + 8 * i + c4 + 4 * (e & 1);
          sc[i][e] = key <= pos[e >> 1] && key < w.q.kv ? sc[i][e] * a.scale_log2 : -INFINITY;
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
      // values of the keys lane % 4 + {0, 4, 8, 12}, dims 64 hh + 8 perm(lane / 4) ..
#pragma unroll
      for (int hh = 0; hh < HD / 64; ++hh) {
        uint4 v[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int row = c4 + 4 * i;
          v[i] = *reinterpret_cast<const uint4*>(vt + hh * (kRows * 128) + row * 128 + ((kperm ^ (row & 7)) * 16));
        }
        const uint32_t* w0 = &v[0].x;
        const uint32_t* w1 = &v[1].x;
        const uint32_t* w2 = &v[2].x;
        const uint32_t* w3 = &v[3].x;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          mma16816(o[8 * hh + 2 * j], a0, a1, a2, a3, __byte_perm(w0[j], w1[j], 0x5410), __byte_perm(w2[j], w3[j], 0x5410));
          mma16816(o[8 * hh + 2 * j + 1], a0, a1, a2, a3, __byte_perm(w0[j], w1[j], 0x7632), __byte_perm(w2[j], w3[j], 0x7632));
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&sm.empty[st]);
    }
    if (named_barrier_or(1, kMathThreads, dead)) return;  // (all four warps are in the same segment)
    // the warps' parts meet in shared memory, 64 dims at a time
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      l[r] += __shfl_xor_sync(kPagedFull, l[r], 1);
      l[r] += __shfl_xor_sync(kPagedFull, l[r], 2);
      if (c4 == 0) {
        sm.m[warp][l4 + 8 * r] = m[r];
        sm.l[warp][l4 + 8 * r] = pos[r] >= bad ? __int_as_float(0x7fc00000) : l[r];
      }
    }
    const bool whole = w.off == 0 && w.end == w.fu.per;
    const int slot = 2 * blockIdx.x + (w.off == 0 ? 1 : 0);
#pragma unroll
    for (int hh = 0; hh < HD / 64; ++hh) {
#pragma unroll
      for (int r = 0; r < 2; ++r)
#pragma unroll
        for (int e = 0; e < 2; ++e) {  // column 2 (lane % 4) + e of tile j is dim 64 hh + 8 (lane % 4 + 4 e) + j
          float* d = &sm.o[warp][l4 + 8 * r][(c4 + 4 * e) * 8];
          *reinterpret_cast<float4*>(d) = make_float4(o[8 * hh][2 * r + e], o[8 * hh + 1][2 * r + e], o[8 * hh + 2][2 * r + e],
                                                      o[8 * hh + 3][2 * r + e]);
          *reinterpret_cast<float4*>(d + 4) = make_float4(o[8 * hh + 4][2 * r + e], o[8 * hh + 5][2 * r + e],
                                                          o[8 * hh + 6][2 * r + e], o[8 * hh + 7][2 * r + e]);
        }
      __syncwarp();
      named_barrier_sync(1, kMathThreads);
      const int row = tid / 8, d0 = (tid % 8) * 8, r = tile * kRows + row;  // 8 threads per row, 8 dims each
      for (int j = 0; j < hp && r < nrows; ++j) {  // warps j, j + hp, .. hold parts of head j
        const int hj = w.item / w.fu.tiles * hp + j;
        float mm = -INFINITY, ll = 0.0f, acc[8];
        for (int wi = j; wi < kWarps; wi += hp) mm = fmaxf(mm, sm.m[wi][row]);
#pragma unroll
        for (int d = 0; d < 8; ++d) acc[d] = 0.0f;
        for (int wi = j; wi < kWarps; wi += hp) {
          const float f = sm.m[wi][row] == -INFINITY ? 0.0f : pg_ex2(sm.m[wi][row] - mm);
          ll += f == 0.0f && !isnan(sm.l[wi][row]) ? 0.0f : f * sm.l[wi][row];
#pragma unroll
          for (int d = 0; d < 8; ++d) acc[d] = fmaf(f, sm.o[wi][row][d0 + d], acc[d]);
        }
        if (whole) {
          const float inv = ll == 0.0f ? 0.0f : 1.0f / ll;
          __nv_bfloat16* dst = a.out + (w.q.first + r / a.g) * a.ldo + (hj * a.g + r % a.g) * HD + hh * 64 + d0;
          *reinterpret_cast<uint4*>(dst) = make_uint4(pack2(acc[0] * inv, acc[1] * inv), pack2(acc[2] * inv, acc[3] * inv),
                                                      pack2(acc[4] * inv, acc[5] * inv), pack2(acc[6] * inv, acc[7] * inv));
        } else {
          const size_t at_row = static_cast<size_t>(slot) * kSlotRows + j * kRows + row;
          float* dst = a.part_o + at_row * HD + hh * 64 + d0;
          reinterpret_cast<float4*>(dst)[0] = make_float4(acc[0], acc[1], acc[2], acc[3]);
          reinterpret_cast<float4*>(dst)[1] = make_float4(acc[4], acc[5], acc[6], acc[7]);
          if (hh == 0 && d0 == 0) reinterpret_cast<float2*>(a.part_ml)[at_row] = make_float2(mm, ll);
        }
      }
      __syncwarp();
      named_barrier_sync(1, kMathThreads);  // sm.o is written again
    }
  } while (w.next(a, hp));
}

// Joins the item that CTA c left unfinished: block (c, y) takes its rows y, y + gridDim.y, .. (a row of 64: 4 heads of 16),
// the parts of a row dealt to its 4 warps.
constexpr int kJoinY = 8;  // at most
template <int HD>
__global__ void __launch_bounds__(kMathThreads) paged_few_join_kernel(const PagedArgs a) {
  __shared__ float sm_l[kWarps];
  __shared__ float sm_o[kWarps][HD];
  pdl_launch_dependents();
  pdl_wait_prior_grids();
  const int c0 = blockIdx.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int4 open = a.split[c0];
  const int c1 = open.w;
  if (c1 <= c0) return;
  const PagedSeq q = paged_seq(a, open.x);
  const int hp = open.y >> 24, h0 = (open.y & 0xffffff) * hp, nrows = q.n * a.g - open.z * kRows;  // packed rows of the tile
  const int live = min(nrows, kRows);
  constexpr int kPer = HD / 32;
  const float2* ml = reinterpret_cast<const float2*>(a.part_ml);
  for (int k = blockIdx.y; k < hp * live; k += gridDim.y) {
    const int j = k / live, pr = open.z * kRows + k % live, row = j * kRows + k % live;
    float m = -INFINITY;
    for (int c = c0 + lane; c <= c1; c += 32) m = fmaxf(m, ml[static_cast<size_t>(2 * c + (c == c0)) * kSlotRows + row].x);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(kPagedFull, m, o));
    float l = 0.0f, acc[kPer];
#pragma unroll
    for (int d = 0; d < kPer; ++d) acc[d] = 0.0f;
#pragma unroll 4
    for (int c = c0 + warp; c <= c1; c += kWarps) {
      const size_t at = static_cast<size_t>(2 * c + (c == c0)) * kSlotRows + row;
      const float2 p = ml[at];
      const float f = p.x == -INFINITY ? 0.0f : pg_ex2(p.x - m);
      l += f == 0.0f && !isnan(p.y) ? 0.0f : f * p.y;
      const float* src = a.part_o + at * HD + lane * kPer;
#pragma unroll
      for (int d = 0; d < kPer; ++d) acc[d] = fmaf(f, src[d], acc[d]);
    }
    if (lane == 0) sm_l[warp] = l;
#pragma unroll
    for (int d = 0; d < kPer; ++d) sm_o[warp][lane * kPer + d] = acc[d];
    __syncthreads();
    if (tid < HD) {
      float v = 0.0f;
      l = 0.0f;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        l += sm_l[w];
        v += sm_o[w][tid];
      }
      a.out[static_cast<long long>(q.first + pr / a.g) * a.ldo + ((h0 + j) * a.g + pr % a.g) * HD + tid] =
          __float2bfloat16_rn(l == 0.0f ? 0.0f : v / l);
    }
    __syncthreads();
  }
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

constexpr int kCtasPerSm = 2;

// Up to 32 packed rows per sequence and kv head on average (the lengths themselves are on the device): two tiles of the
// 16-row kernel, which then reads each key twice; the other kernel pads to 128 and takes groups of up to 128 heads.
// 64 sequences over 2048 keys, 8 kv heads of 128: 16 packed rows take 108 us here and 223 there, 32 take 197 and 220, 40
// take 278 and 220. The rule knows the average alone, so that a call of unequal sequences goes wholly to one kernel: 63 single
// tokens over 2048 to 8192 keys with a chunk of 449 rows over 4545 (32 heads over 8) take 429 us here, with one of 450 rows
// 405 there, and 205 and 65 in two calls. A chunk's tiles of 16 rows each read all its keys here.
bool few_rows(int rows, int seqs, int g) { return static_cast<long long>(rows) * g <= 32LL * seqs || g > 128; }

int few_grid() { return kCtasPerSm * tc_sm_count(); }

template <int HD>
int launch_few(const PagedArgs& a, cudaStream_t s) {
  static bool ready[64] = {false};
  constexpr size_t smem = sizeof(FewSmem<HD>);
  static_assert(2 * (smem + 1024) <= 228 * 1024, "two CTAs per SM");
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64 || !ready[dev]) {
    const cudaError_t e = cudaFuncSetAttribute(paged_few_kernel<HD>, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem));
    if (e != cudaSuccess) return fail(BP_ERR_CUDA, "cudaFuncSetAttribute(smem %zu): %s", smem, cudaGetErrorString(e));
    if (dev >= 0 && dev < 64) ready[dev] = true;
  }
  CUtensorMap tk, tv;
  const int ps = 1 << a.page_log2;
  int st = paged_maps(a, ps < kRows ? ps : kRows, &tk, &tv);
  if (st != BP_OK) return st;
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[2];
  cfg.gridDim = dim3(a.G);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  set_launch_attrs(cfg, attr);
  cudaError_t e = cudaLaunchKernelEx(&cfg, paged_few_kernel<HD>, tk, tv, a);
  if (e == cudaSuccess) {
    cfg.gridDim = dim3(a.G, static_cast<unsigned>(std::min<long long>(static_cast<long long>(a.rows) * a.g, kJoinY)));
    cfg.blockDim = dim3(kMathThreads);
    cfg.dynamicSmemBytes = 0;
    e = cudaLaunchKernelEx(&cfg, paged_few_join_kernel<HD>, a);
  }
  if (e != cudaSuccess) return fail(BP_ERR_CUDA, "paged_attention launch (few rows): %s", cudaGetErrorString(e));
  return BP_OK;
}

}  // namespace
}  // namespace bp

extern "C" size_t bp_paged_attention_workspace_bytes(int rows, int seqs, int nh, int nkv, int head_dim) {
  using namespace bp;
  if (rows <= 0 || seqs <= 0 || nkv <= 0 || nh < nkv || head_dim <= 0) return 0;
  return few_rows(rows, seqs, nh / nkv) ? static_cast<size_t>(2 * few_grid()) * kSlotRows * (head_dim + 2) * sizeof(float) +
                                              few_grid() * sizeof(int4)
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
  if (q == nullptr || (pages == nullptr && max_pages > 0) || q_start == nullptr || kv_len == nullptr || k_pages == nullptr ||
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
  a.split = reinterpret_cast<int4*>(a.part_ml + static_cast<size_t>(2 * a.G) * kSlotRows * 2);
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  st = head_dim == 128 ? launch_few<128>(a, s) : launch_few<64>(a, s);
  return st != BP_OK ? st : check_launch("paged_attention");
}

namespace bp {
BP_DEFINE_DEVICE_ERROR_READER(read_device_errors_paged_few)

// Maps of the cache's keys and values: [64 dims, box_rows positions, one kv head] at (dim, page * page_size + row, head).
int paged_maps(const PagedArgs& a, int box_rows, CUtensorMap* tk, CUtensorMap* tv) {
  const uint64_t dims[3] = {static_cast<uint64_t>(a.hd), static_cast<uint64_t>(a.num_pages) << a.page_log2, static_cast<uint64_t>(a.nkv)};
  const uint64_t strides[2] = {static_cast<uint64_t>(a.nkv) * a.hd * 2, static_cast<uint64_t>(a.hd) * 2};
  const uint32_t box[3] = {64, static_cast<uint32_t>(box_rows), 1};
  const int st = tc_encode(tk, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, a.kp, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B,
                           CU_TENSOR_MAP_L2_PROMOTION_L2_256B);
  if (st != BP_OK) return st;
  return tc_encode(tv, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, a.vp, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B,
                   CU_TENSOR_MAP_L2_PROMOTION_L2_256B);
}
}  // namespace bp
