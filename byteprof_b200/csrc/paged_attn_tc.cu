// Attention of many new rows over a paged cache on the 5th-generation tensor cores (bp_paged_attention's kernel for
// prompts and chunks; few rows: paged_attn.cu).
//
//   S = q K^T, p = exp2(scale S - m), O += p V, l += sum p, out = O / l: one pass over the keys per tile of rows.
//
//  * An item is two tiles of 128 rows (128 / g tokens with their g heads each) of one sequence and kv head, a unit is 128
//    keys of it (paged.cuh); CTAs take equal ranges of units, whatever the lengths.
//  * Warp 0 finds the pages and loads K and V tiles by TMA, one box per page (page rows are strided by the kv heads):
//    the 128-byte swizzled tile serves as K (K-major) and as V (keys are the second product's K dimension: MN-major).
//    A page that is not there is fetched from behind the pool, which TMA fills with zeros.
//  * Warp 1 issues the MMAs of both tiles in turn: S0, S1, then per key block P0 V, S0', P1 V, S1', so that one
//    tile's softmax runs under the other's products. S (fp32), P (bf16, over S) and O (fp32) live in TMEM.
//  * Warp 2 waits for the V tile of the block and the K tile of the next one in the issuing thread's place, and looks
//    through the values that some row does not see, behind the sequence's end too: what is not finite becomes 0.
//  * Two warpgroups do the softmax, one thread per row: twice through its 128 scores in TMEM, for the maximum and for exp2
//    and P, masked only where a row's limit lies in the block. The running maximum moves only when a score exceeds it by
//    2^8: then O is rescaled in TMEM by the same threads, which is rare after the first block. P is rounded to bf16
//    (2^-8 of each p at most), the sum adds the unrounded fp32 values.
//
// A block of two tiles takes 2048 clocks of MMA (head_dim 128) and 2048 of exp2, each behind the other within a tile; it
// takes 3300 (a chunk of 4096 rows over 20480 keys, 16 heads of 128: 840 to 920 us with the GPU's power cap, 874 TFLOP/s of visible
// keys at 1.73 GHz) to 3800 clocks (9 prompts of 6151 tokens, 32 heads of 64: 94.6 us), and an item about 5000 more: bound by the
// hand-overs between the softmax warps and the issuing thread (about 1300 clocks a block and tile), not by either unit.
// Measured and not kept: exp2 partly as a polynomial on the FMA pipes (910 us and more), one pass over the scores with the
// block before's maximum (907), an issuing thread per tile (1069 against 890 then), a block's columns in one unrolled
// piece (instruction fetch: 110 us of 870), per-chunk masks (900), the next item's first scores behind this item's last
// product (876, and 100 for the prompts), P in columns of its own at head_dim 64 and the next scores in front of the product
// with V (prompts 97), all 128 scores loaded at once for the maximum (848, prompts 97), the next chunk's scores loaded
// ahead (925, prompts 104), a row's softmax over two threads (894, prompts 101). The chunk's time is what back-to-back
// launches leave of the clock: one launch by itself takes 755. Looking for values that are not finite (warp 2) costs the prompts
// 1.3 us and the chunk nothing, in a short rolled loop; unrolled it cost 3.6, for instruction fetch.
#include <cudaTypedefs.h>

#include "paged.cuh"
#include "skinny_internal.h"
#include "sm100.cuh"

namespace bp {
namespace {

constexpr int kTile = 128;                // rows per tile, keys per unit
constexpr int kItemRows = 2 * kTile;
constexpr int kSlots = 4;                 // K and V tiles in the ring (two blocks)
constexpr int kThreads = 384;
constexpr int kWarps = kThreads / 32;
constexpr int kSmWarp0 = 4;               // softmax warpgroups: warps 4..7 (tile 0) and 8..11 (tile 1)
constexpr int kBadRing = 16;
constexpr float kLazy = 8.0f;
constexpr int kScanSeqs = 512;
constexpr uint32_t kBase = 1024;          // shared-memory address of the tiles
// register split: launched with 168 per thread (64512), 4 warps keep 120, 8 warps take 192: 64512
constexpr int kRegsLaunch = 168, kRegsLow = 120, kRegsHigh = 192;
static_assert(128 * kRegsLow + 256 * kRegsHigh <= kThreads * kRegsLaunch, "register split");

// 32 lanes x 32 TMEM columns into registers, not waited for.
__device__ __forceinline__ void tmem_ld32_nowait(uint32_t taddr, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
        "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
        "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr)
      : "memory");
}
// 32 lanes x 16 registers into TMEM columns (complete at tmem_st_wait).
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t* r) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
               "%15, %16};" ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]),
               "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
               : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// D[tmem] (+)= A[tmem] . B[smem], bf16, fp32 accumulator.
__device__ __forceinline__ void umma_f16_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t b_desc, uint32_t idesc,
                                            uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
      ::"r"(d_tmem), "r"(a_tmem), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}

// umma_desc_sw128 of a constant address.
__host__ __device__ constexpr uint64_t umma_desc_at(uint32_t saddr) {
  return static_cast<uint64_t>((saddr >> 4) & 0x3FFFu) | (1ull << 16) | (static_cast<uint64_t>(1024 >> 4) << 32) | (1ull << 46) |
         (2ull << 61);
}
// MN-major operand with 128-byte swizzling: 64 values of N per 128-byte row, one row per k, 8-row groups 1024 bytes
// apart, the next 64 values of N `lbo` bytes away.
__host__ __device__ constexpr uint64_t umma_desc_mn_at(uint32_t saddr, uint32_t lbo) {
  return umma_desc_at(saddr) - (1ull << 16) + (static_cast<uint64_t>(lbo >> 4) << 16);
}

// ---- the cut of the work ----------------------------------------------------------------------------------
// A tile holds the g heads of 128 / g tokens (g <= 128; the few rows left over idle), an item two tiles.
__device__ __forceinline__ int tile_tokens(const PagedArgs& a) { return a.tile_tokens; }  // kTile / g
__device__ __forceinline__ int item_tiles(const PagedArgs& a, int n) { return (n + 2 * tile_tokens(a) - 1) / (2 * tile_tokens(a)); }
// Blocks of 128 keys that the tokens up to `last` (exclusive) of a sequence see.
__device__ __forceinline__ int blocks_of(const PagedSeq& q, int last) {
  long long vis = q.pos0 + last;
  if (vis > q.kv) vis = q.kv;
  return vis <= 0 ? 0 : static_cast<int>((static_cast<uint32_t>(vis) + kTile - 1) / kTile);
}
// An item's units: its blocks (at least one) and kSetup more, what loading q, filling the pipeline and storing cost
// (about 1.5 blocks' time: 9 prompts of 6151 tokens take 96.0 us at 1 and 94.4 at 2, a chunk of 4096 over 20480 the same).
constexpr int kSetup = 2;
__device__ __forceinline__ int item_units(const PagedArgs& a, const PagedSeq& q, int tile) {
  return kSetup + max(1, blocks_of(q, min(q.n, (tile + 1) * 2 * tile_tokens(a))));
}

struct Scan {
  long long units[kScanSeqs];  // of one kv head, per sequence of the block at hand
  long long warp_sum[kWarps], before;
  int seq;
};

// A CTA's start: the sequence of its first unit, that unit's place behind the sequence's first, the units of one of its
// kv heads, and how many units are the CTA's (0: none).
struct Start {
  long long share, rel, head, count;
  int seq;
};

// Up to 32 sequences: every warp finds it by itself, 32 / seqs lanes per sequence (with the barriers of the cut for
// more, and the join kernel searching for its items, 9 prompts took 110 us instead of 96).
__device__ __forceinline__ Start find_start_few(const PagedArgs& a) {
  const int lane = threadIdx.x & 31;
  int lanes = 32;
  while (lanes * a.seqs > 32) lanes >>= 1;
  const int seq = lane / lanes, sub = lane % lanes;
  long long u = 0;
  if (seq < a.seqs) {
    const PagedSeq q = paged_seq(a, seq);
    const int nt = item_tiles(a, q.n);
    for (int t = sub; t < nt; t += lanes) u += item_units(a, q, t);
  }
  for (int o = lanes / 2; o > 0; o >>= 1) u += __shfl_xor_sync(kPagedFull, u, o);
  const long long mine = sub == 0 ? u * a.nkv : 0;
  long long pre = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long v = __shfl_up_sync(kPagedFull, pre, o);
    if (lane >= o) pre += v;
  }
  const long long total = __shfl_sync(kPagedFull, pre, 31);
  Start st;
  st.share = share_of(a, total);
  const long long u0 = blockIdx.x * st.share;
  st.count = total - u0 < st.share ? total - u0 : st.share;
  const unsigned hit = __ballot_sync(kPagedFull, mine > 0 && u0 >= pre - mine && u0 < pre);
  const int src = hit != 0 ? __ffs(hit) - 1 : 0;
  st.seq = src / lanes;
  st.rel = u0 - __shfl_sync(kPagedFull, pre - mine, src);
  st.head = __shfl_sync(kPagedFull, u, src);
  return st;
}

// units[] of the sequences s0 .. s0 + kScanSeqs: 8 lanes per sequence; called by all threads, ends with a barrier.
__device__ __noinline__ void scan_units(const PagedArgs& a, Scan& sc, int s0) {
  const int count = min(kScanSeqs, a.seqs - s0), sub = threadIdx.x & 7;
  for (int i = threadIdx.x / 8; i - (threadIdx.x & 31) / 8 < count; i += kThreads / 8) {
    long long u = 0;
    if (i < count) {
      const PagedSeq q = paged_seq(a, s0 + i);
      const int nt = item_tiles(a, q.n);
      for (int t = sub; t < nt; t += 8) u += item_units(a, q, t);
    }
#pragma unroll
    for (int o = 4; o > 0; o >>= 1) u += __shfl_xor_sync(kPagedFull, u, o);
    if (i < count && sub == 0) sc.units[i] = u;
  }
  __syncthreads();
}

// Any number of sequences; all threads.
__device__ __noinline__ Start find_start_many(const PagedArgs& a, Scan& sc) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  long long total = 0;
  for (int s0 = 0; s0 < a.seqs; s0 += kScanSeqs) {
    scan_units(a, sc, s0);
    const int count = min(kScanSeqs, a.seqs - s0);
    for (int i = threadIdx.x; i < count; i += kThreads) total += sc.units[i];
    if (s0 + kScanSeqs < a.seqs) __syncthreads();
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(kPagedFull, total, o);
  if (lane == 0) sc.warp_sum[warp] = total;
  __syncthreads();
  total = 0;
  for (int w = 0; w < kWarps; ++w) total += sc.warp_sum[w];
  total *= a.nkv;
  Start st;
  st.share = share_of(a, total);
  const long long u = blockIdx.x * st.share;
  st.count = total - u < st.share ? total - u : st.share;
  st.seq = 0;
  st.rel = 0;
  st.head = 1;
  if (st.count <= 0) return st;  // (the same for the whole CTA)
  long long base = 0;
  for (int s0 = 0; s0 < a.seqs; s0 += kScanSeqs) {
    if (a.seqs > kScanSeqs) scan_units(a, sc, s0);
    const int count = min(kScanSeqs, a.seqs - s0);
    if (threadIdx.x < 32) {
      long long run = base;
      int hit = -1;
      long long hit_before = 0;
      for (int i0 = 0; i0 < count; i0 += 32) {
        const long long mine = i0 + lane < count ? sc.units[i0 + lane] * a.nkv : 0;
        long long pre = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const long long v = __shfl_up_sync(kPagedFull, pre, o);
          if (lane >= o) pre += v;
        }
        const long long start = run + pre - mine;
        const unsigned m = __ballot_sync(kPagedFull, mine > 0 && u >= start && u < start + mine);
        if (m != 0) {
          const int src = __ffs(m) - 1;
          hit = i0 + src;
          hit_before = __shfl_sync(kPagedFull, start, src);
          break;
        }
        run += __shfl_sync(kPagedFull, pre, 31);
      }
      if (lane == 0) {
        sc.seq = hit;
        sc.before = hit >= 0 ? hit_before : run;
      }
    }
    __syncthreads();
    if (sc.seq >= 0) {
      st.seq = s0 + sc.seq;
      st.rel = u - sc.before;
      st.head = sc.units[sc.seq];
      return st;
    }
    base = sc.before;
    __syncthreads();
  }
  return st;
}

// A CTA's walk over its units: one segment (a range of key blocks of one item) at a time. Every role walks by itself.
struct Walk {
  PagedSeq q;
  int s, h, tile, tiles;
  int off, end, per;        // the segment's blocks, the item's
  int blocks[2];            // what each tile sees of the item
  int rest;                 // the item's units behind the segment
  long long left;           // units of the CTA after this segment

  __device__ __forceinline__ void enter(const PagedArgs& a) {
    q = paged_seq(a, s);
    tiles = item_tiles(a, q.n);
  }
  // the units [v0, v1) of the item are the CTA's
  __device__ __forceinline__ void segment(const PagedArgs& a, int v0, int v1) {
    const int t0 = tile * 2 * tile_tokens(a), t1 = t0 + tile_tokens(a);
    blocks[0] = blocks_of(q, min(q.n, t1));
    blocks[1] = q.n > t1 ? blocks_of(q, min(q.n, t1 + tile_tokens(a))) : 0;
    off = max(v0 - kSetup, 0);
    end = max(v1 - kSetup, 0);
  }
  // False: nothing to do.
  __device__ bool start(const PagedArgs& a, const Start& st) {
    const long long rel = st.rel, head = st.head, count = st.count;
    s = st.seq;
    enter(a);
    h = static_cast<int>(quotient(rel, head));
    long long r = rel - h * head;
    int n;
    for (tile = 0;; ++tile) {
      n = item_units(a, q, tile);
      if (r < n) break;
      r -= n;
    }
    per = n - kSetup;
    const int v0 = static_cast<int>(r), v1 = static_cast<int>(n - v0 < count ? n : v0 + count);
    segment(a, v0, v1);
    rest = n - v1;
    left = count - (v1 - v0);
    return off < end || next(a);
  }
  __device__ bool next(const PagedArgs& a) {
    while (left > 0) {
      if (++tile == tiles) {
        tile = 0;
        if (++h == a.nkv) {
          h = 0;
          do {
            ++s;
            enter(a);
          } while (q.n == 0);
        }
      }
      const int n = item_units(a, q, tile), v1 = static_cast<int>(n < left ? n : left);
      per = n - kSetup;
      segment(a, 0, v1);
      rest = n - v1;
      left -= v1;
      if (off < end) return true;  // (the share may end in an item's setup: nothing of it is done here)
    }
    return false;
  }
  // Cached positions that every row of the item sees: the first ones.
  __device__ __forceinline__ int all_see(const PagedArgs& a) const {
    return static_cast<int>(max(min(q.pos0 + static_cast<long long>(tile) * 2 * tile_tokens(a) + 1, static_cast<long long>(q.kv)), 0LL));
  }
  // blocks [off, until(i)) of the segment are tile i's
  __device__ __forceinline__ int until(int i) const { return min(end, blocks[i]); }
  // Blocks [off, used()) of the segment are loaded: `end`, but none of an item whose rows see nothing. A block that neither
  // tile uses may not be in the ring: no product would hold warp 2, which clears values in it, and its slot's refill together.
  __device__ __forceinline__ int used() const { return min(end, max(blocks[0], blocks[1])); }
};

template <int HD>
struct Smem {
  static constexpr int kTileBytes = kTile * HD * 2;
  uint8_t q[2][kTileBytes];
  uint8_t kv[kSlots][kTileBytes];
  uint64_t full[kSlots], empty[2], q_full[2], q_done[2], s_full[2], p_full[2], o_done[2], mma_done;
  int bad[kBadRing];
  int2 lost[2][2];  // per tile, for its segments in turn: (segment, first position whose value was taken out)
  uint32_t tmem_base;
  int abort;
  Scan scan;
};

__device__ __forceinline__ void wait_drain(uint64_t* bar, uint32_t parity) {
  const unsigned long long t0 = globaltimer();
  while (!mbar_try_wait(bar, parity)) {
    if (globaltimer() - t0 > kWaitLimitNs) {
      atomicOr(&g_bp_device_errors, BP_DEVERR_TIMEOUT);
      return;
    }
  }
}

// Two fp32 values in a register pair, and arithmetic on both at once.
__device__ __forceinline__ uint64_t f32x2(float lo, float hi) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ float f32x2_lo(uint64_t v) { return __uint_as_float(static_cast<uint32_t>(v)); }
__device__ __forceinline__ float f32x2_hi(uint64_t v) { return __uint_as_float(static_cast<uint32_t>(v >> 32)); }
__device__ __forceinline__ uint64_t fma_f32x2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t add_f32x2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}

__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  const __nv_bfloat162 p = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&p);
}

// Rows `lo` and up of a V tile (keys base + lo ..), by one warp: pieces that are not finite become 0, those past the
// sequence's end too; the first key that had one (INT_MAX: none). 32 rows a step from the step that holds `lo`: rows before it
// are seen by all, and what is found there is right for all.
template <int HD>
__device__ __noinline__ int hide_not_finite(uint8_t* v, int lo, int base, int lane) {
  constexpr int kU = 4;
  int lost = 0x7fffffff;
  uint4* t = reinterpret_cast<uint4*>(v) + lane;
#pragma unroll 1
  for (int c = (lo & ~31) * 8; c < kTile * 8 * (HD / 64); c += 32 * kU) {  // (pieces; 64 dims behind the others)
    if (HD > 64 && c == kTile * 8) c += (lo & ~31) * 8;
    uint32_t any = 0;
#pragma unroll
    for (int u = 0; u < kU; ++u) any |= not_finite8(t[c + 32 * u]);
    if (any == 0) continue;
#pragma unroll 1
    for (int u = 0; u < kU; ++u)
      if (not_finite8(t[c + 32 * u]) != 0) {
        t[c + 32 * u] = make_uint4(0, 0, 0, 0);
        lost = min(lost, base + (c + lane) / 8 % kTile + 4 * u);
      }
  }
  lost = __reduce_min_sync(kPagedFull, lost);
  if (lost != 0x7fffffff) fence_async_shared();  // the product reads them
  __syncwarp();
  return lost;
}

constexpr int kChunk = 32;
// N scores of a row; the columns from `lim` on are hidden when `masked`.
template <int N>
__device__ __forceinline__ void load_scores(uint32_t taddr, uint32_t (&x)[N], bool masked, int lim) {
#pragma unroll
  for (int c = 0; c < N; c += 32) tmem_ld32_nowait(taddr + c, x + c);
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
  for (int c = 0; c < N; ++c) asm volatile("" : "+r"(x[c]));  // no use moves above the wait
  if (masked) {
#pragma unroll
    for (int c = 0; c < N; ++c) x[c] = c < lim ? x[c] : 0xff800000u;
  }
}

template <int HD>
__global__ void __launch_bounds__(kThreads, 1)
    paged_tc_kernel(const __grid_constant__ CUtensorMap tq, const __grid_constant__ CUtensorMap tk,
                    const __grid_constant__ CUtensorMap tv, const PagedArgs a) {
  constexpr int kHalf = kTile * 128;  // bytes of 64 head dimensions of a tile
  constexpr int kTileBytes = Smem<HD>::kTileBytes;
  extern __shared__ uint8_t smem_raw[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  // The kernel has no static shared memory, so the dynamic part starts in the first 1024 bytes, and its tiles at kBase.
  if (smem_addr(smem_raw) > kBase) {
    if (threadIdx.x == 0) atomicOr(&g_bp_device_errors, BP_DEVERR_TIMEOUT);
    return;
  }
  Smem<HD>& s = *reinterpret_cast<Smem<HD>*>(smem_raw + (kBase - smem_addr(smem_raw)));
  if (threadIdx.x == 0) {
    for (int i = 0; i < kSlots; ++i) mbar_init(&s.full[i], 1);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&s.empty[i], 1);
      mbar_init(&s.q_full[i], 1);
      mbar_init(&s.q_done[i], 1);
      mbar_init(&s.s_full[i], 1);
      mbar_init(&s.p_full[i], 5);  // 4 softmax warps and warp 2
      mbar_init(&s.o_done[i], 1);
      s.lost[i][0] = s.lost[i][1] = make_int2(-1, 0);
    }
    mbar_init(&s.mma_done, 1);
    s.abort = 0;
    mbar_fence_init();
    tma_prefetch_desc(&tq);
    tma_prefetch_desc(&tk);
    tma_prefetch_desc(&tv);
  }
  if (warp == 1) {
    tmem_alloc(&s.tmem_base, 512);
    tmem_relinquish();
  }
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  pdl_launch_dependents();
  pdl_wait_prior_grids();
  constexpr uint32_t tmem = 0;  // all 512 columns are this CTA's
  volatile int* abort = &s.abort;

  const Start st = a.seqs <= 32 ? find_start_few(a) : find_start_many(a, s.scan);
  const bool work = st.count > 0;
  if (!work && threadIdx.x == 0) leave_split(a, 0, 0, 0, blockIdx.x);

  if (warp < kSmWarp0) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegsLow));
    if (warp == 0 && work) {
      // ---- pages and TMA: K(b), V(b) per block, alternating in the ring; q behind a segment's first K ----
      Walk w;
      const int rows_per = min(1 << a.page_log2, kTile), np = kTile / rows_per;  // rows and boxes per block
      const int mask = (1 << a.page_log2) - 1, none = a.num_pages << a.page_log2;
      const uint32_t q_bytes = static_cast<uint32_t>(tile_tokens(a) * a.g) * (HD * 2);
      int t = 0, issued = 0;      // blocks, ring tiles
      uint32_t qn[2] = {0, 0};    // q tiles loaded
      bool ok = true;
      int4 open = make_int4(0, 0, 0, blockIdx.x);
      for (bool more = w.start(a, st); more && ok; more = w.next(a)) {
        if (w.off == 0 && w.rest > 0)
          open = make_int4(w.s, w.h, w.tile, blockIdx.x + static_cast<int>(quotient(w.rest + st.share - 1, st.share)));
        const int* table = a.pages + static_cast<long long>(w.s) * a.ld_pages;
        for (int b = w.off; b < w.used() && ok; ++b, ++t) {
          const int key = b * kTile + lane * rows_per;
          int row = none, bad = w.q.bad;
          if (lane < np && key < w.q.kv) {
            const int page = table[key >> a.page_log2];
            if (page >= 0 && page < a.num_pages)
              row = (page << a.page_log2) + (key & mask);
            else
              bad = min(bad, key);
          }
          bad = __reduce_min_sync(kPagedFull, bad);
          if (lane == 0) s.bad[t % kBadRing] = bad;
          for (int kv = 0; kv < 2 && ok; ++kv, ++issued) {
            const int slot = issued % kSlots;
            int go = 1;
            if (lane == 0) {
              // the slot's last tile, K(t - 2) or V(t - 2), was freed with pair t - 2 or t - 1 (pair p: V(p - 1) and K(p))
              if (t >= 2) {
                const int pair = t - 2 + kv;
                go = mbar_wait(&s.empty[pair & 1], static_cast<uint32_t>(pair >> 1) & 1u, abort);
              }
              if (go) mbar_arrive_expect_tx(&s.full[slot], kTileBytes);
            }
            ok = __shfl_sync(kPagedFull, go, 0) != 0;
            if (!ok) break;
            if (lane < np) {
#pragma unroll
              for (int c = 0; c < HD / 64; ++c)
                tma_load_3d(s.kv[slot] + c * kHalf + lane * rows_per * 128, kv == 0 ? &tk : &tv, &s.full[slot], c * 64, row, w.h);
            }
            __syncwarp();
            if (kv == 0 && b == w.off) {
              if (lane == 0) {
                for (int i = 0; i < 2 && go; ++i) {
                  if (w.until(i) <= w.off) continue;
                  if (qn[i] > 0) go = mbar_wait(&s.q_done[i], (qn[i] + 1) & 1u, abort);  // its last scores are issued
                  if (!go) break;
                  ++qn[i];
                  mbar_arrive_expect_tx(&s.q_full[i], q_bytes);
                  for (int c = 0; c < HD / 64; ++c)
                    tma_load_3d(s.q[i] + c * kHalf, &tq, &s.q_full[i], c * 64, w.h * a.g,
                                w.q.first + (2 * w.tile + i) * tile_tokens(a));
                }
              }
              ok = __shfl_sync(kPagedFull, go, 0) != 0;
            }
          }
        }
      }
      if (lane == 0) {
        leave_split(a, open.x, open.y, open.z, open.w);
        for (int i = 0; i < kSlots && i < issued; ++i) wait_drain(&s.full[i], static_cast<uint32_t>((issued - 1 - i) / kSlots) & 1u);
        for (int i = 0; i < 2; ++i)
          if (qn[i] > 0) wait_drain(&s.q_full[i], (qn[i] + 1) & 1u);
      }
    } else if (warp == 1 && work) {
      // ---- MMA: one thread, from wait to wait as short as it can be written ----
      if (lane == 0) {
        constexpr uint32_t idesc_s = umma_idesc_bf16(kTile, kTile);
        constexpr uint32_t idesc_o = umma_idesc_bf16(kTile, HD) | (1u << 16);  // B is MN-major
        // Block number `blk` of the CTA has K in slot 0 or 2 and V in slot 1 or 3. The two cases are written out and the
        // shared memory starts at a known address, so that every descriptor and barrier is a constant of the kernel:
        // one that is computed has to be moved to uniform registers for each MMA.
        constexpr uint64_t dq = umma_desc_at(kBase), dk = umma_desc_at(kBase + 2 * kTileBytes),
                           dv = umma_desc_mn_at(kBase + 2 * kTileBytes, kHalf);
        constexpr int kT = kTileBytes >> 4;
        auto scores_of = [&](int i, int slot) {
          const uint64_t da = dq + i * kT, db = dk + slot * kT;
#pragma unroll
          for (int k = 0; k < HD / 16; ++k) {
            constexpr int kNext = kHalf >> 4;
            umma_f16(tmem + i * kTile, da + (k / 4) * kNext + (k % 4) * 2, db + (k / 4) * kNext + (k % 4) * 2, idesc_s, k > 0 ? 1u : 0u);
          }
          umma_commit(&s.s_full[i]);
        };
        auto scores = [&](int i, int blk) {
          if (blk & 1)
            scores_of(i, 2);
          else
            scores_of(i, 0);
        };
        auto output_of = [&](int i, int slot, uint32_t more) {
#pragma unroll
          for (int k = 0; k < kTile / 16; ++k)
            umma_f16_ts(tmem + 2 * kTile + i * kTile, tmem + i * kTile + k * 8, dv + slot * kT + k * (2048 >> 4), idesc_o,
                        k > 0 ? 1u : more);
        };
        auto output = [&](int i, int blk, uint32_t more) {
          if (blk & 1)
            output_of(i, 3, more);
          else
            output_of(i, 1, more);
        };
        Walk w;
        int blk = 0;  // blocks so far: K of block blk is tile 2 blk of the ring, V tile 2 blk + 1
        uint32_t seg[2] = {0, 0}, pn[2] = {0, 0};  // phases: q_full and p_full per tile
        bool ok = true;
        for (bool on = w.start(a, st); on && ok; on = w.next(a)) {
          const int un[2] = {w.until(0), w.until(1)};
          if (w.used() <= w.off) continue;
#pragma unroll
          for (int i = 0; i < 2; ++i)
            if (un[i] > w.off) ok = ok && mbar_wait(&s.q_full[i], seg[i]++ & 1u, abort);
          ok = ok && mbar_wait(&s.full[(2 * blk) & 3], (blk >> 1) & 1, abort);
          if (!ok) break;
          tc_fence_after_sync();
#pragma unroll
          for (int i = 0; i < 2; ++i)
            if (un[i] > w.off) {
              scores(i, blk);
              if (w.off + 1 == un[i]) umma_commit(&s.q_done[i]);
            }
          umma_commit(&s.empty[blk & 1]);  // pair blk: the V before and this K
          for (int b = w.off; b < w.end; ++b, ++blk) {
            const bool more = b + 1 < w.end;
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              if (b < un[i] && ok) {
                ok = mbar_wait(&s.p_full[i], pn[i]++ & 1u, abort);  // P, and (through warp 2) this block's V and the next K
                if (!ok) break;
                tc_fence_after_sync();
                output(i, blk, b > w.off ? 1u : 0u);
                if (b + 1 < un[i]) {
                  scores(i, blk + 1);  // (its completion is also that of the product before)
                  if (b + 2 == un[i]) umma_commit(&s.q_done[i]);
                } else {
                  umma_commit(&s.o_done[i]);
                }
              }
            }
            if (!ok) break;
            if (more) umma_commit(&s.empty[(blk + 1) & 1]);
          }
        }
        umma_commit(&s.mma_done);
        wait_drain(&s.mma_done, 0);
      }
    } else if (warp == 2 && work) {
      // ---- the fifth arrival at p_full: V of the block and K of the next have landed. A wait costs the issuing thread
      // some 100 clocks in which the tensor cores run dry, so it has one per product. Values that a row does not see, and
      // those past a sequence's end, may be NaN, which p = 0 does not hide: they are taken out here (paged.cuh).
      Walk w;
      int blk = 0, segs[2] = {0, 0};  // blocks, and segments of each tile, so far
      uint32_t pn[2] = {0, 0};
      bool ok = true;
      auto wait = [&](uint64_t* bar, uint32_t parity) {
        int go = 1;
        if (lane == 0) go = mbar_wait(bar, parity, abort);
        __syncwarp();
        return __all_sync(kPagedFull, go != 0) != 0;
      };
      for (bool on = w.start(a, st); on && ok; on = w.next(a)) {
        const int un[2] = {w.until(0), w.until(1)}, all_see = w.all_see(a);
        for (int b = w.off; b < w.used() && ok; ++b, ++blk) {
          ok = wait(&s.full[(2 * blk + 1) & 3], (blk >> 1) & 1);
          int lost = 0x7fffffff;
          if (ok && all_see < (b + 1) * kTile)
            lost = hide_not_finite<HD>(s.kv[(2 * blk + 1) & 3], max(all_see - b * kTile, 0), b * kTile, lane);
          if (ok && b + 1 < w.end) ok = wait(&s.full[(2 * blk + 2) & 3], ((blk + 1) >> 1) & 1);
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            if (b >= un[i] || !ok) continue;
            if (pn[i] > 0) ok = wait(&s.p_full[i], (pn[i] + 1) & 1u);  // the phase before is complete
            ++pn[i];
            // With that phase the tile's softmax group is in its segment before this one at the earliest, whose place is the other.
            if (ok && lane == 0 && lost < w.q.kv) {
              int2& e = s.lost[i][segs[i] & 1];
              e = make_int2(segs[i], e.x == segs[i] ? min(e.y, lost) : lost);
            }
            if (ok && lane == 0) mbar_arrive(&s.p_full[i]);
          }
        }
#pragma unroll
        for (int i = 0; i < 2; ++i) segs[i] += un[i] > w.off ? 1 : 0;
      }
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegsHigh));
    if (work) {
      // ---- softmax: one thread per packed row ----
      const int i = (warp - kSmWarp0) / 4, r = threadIdx.x & (kTile - 1);
      const uint32_t lanes = static_cast<uint32_t>(32 * (warp & 3)) << 16;
      const uint32_t ts = tmem + lanes + i * kTile, to = tmem + lanes + 2 * kTile + i * kTile;
      const float sc = a.scale_log2;
      Walk w;
      int n = 0, t0 = 0;  // blocks of this tile so far; blocks of the CTA before the segment
      uint32_t segs = 0;  // segments of this tile so far
      bool ok = true;
      const int rt = r / a.g, rh = r % a.g;
      for (bool on = w.start(a, st); on && ok; on = w.next(a)) {
        const int until = w.until(i), token = (2 * w.tile + i) * tile_tokens(a) + rt;
        const bool live = rt < tile_tokens(a) && token < w.q.n;
        const int tok = live ? token : 0, head = w.h * a.g + rh;
        float m = -INFINITY, l = 0.0f;
        int bad = w.q.bad;
        const long long pos = live ? w.q.pos0 + tok : -1;
        const long long vis = pos + 1 < w.q.kv ? pos + 1 : w.q.kv;  // visible keys
        if (until > w.off) {
          for (int b = w.off; b < until; ++b, ++n) {
            ok = mbar_wait(&s.s_full[i], static_cast<uint32_t>(n) & 1u, abort);
            if (!__all_sync(kPagedFull, ok)) {
              ok = false;
              break;
            }
            tc_fence_after_sync();
            bad = min(bad, s.bad[(t0 + b - w.off) % kBadRing]);
            const long long lim = vis - static_cast<long long>(b) * kTile;
            const bool masked = __any_sync(kPagedFull, lim < kTile);
            const int lim32 = lim > kTile ? kTile : (lim < 0 ? 0 : static_cast<int>(lim));
            // Twice through the scores, kChunk columns at a time in rolled loops: they come from TMEM again faster than the
            // code of 128 unrolled columns comes from the instruction cache (a second copy of it cost 110 us of 870).
            float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll 1
            for (int c = 0; c < kTile; c += kChunk) {
              uint32_t x[kChunk];
              load_scores<kChunk>(ts + c, x, masked, lim32 - c);
#pragma unroll
              for (int j = 0; j < kChunk; j += 8)
#pragma unroll
                for (int k = 0; k < 4; ++k) mx[k] = fmaxf(fmaxf(mx[k], __uint_as_float(x[j + k])), __uint_as_float(x[j + 4 + k]));
            }
            const float top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * sc;
            if (__any_sync(kPagedFull, top > m + kLazy)) {
              const float mn = fmaxf(m, top), f = m == -INFINITY ? 0.0f : pg_ex2(m - mn);
              m = mn;
              l *= f;
              if (b > w.off) {  // O holds the blocks before (s_full came after their last product), under the old maximum
#pragma unroll 1
                for (int c = 0; c < HD; c += 16) {
                  float o[16];
                  uint32_t v[16];
                  tmem_ld_32x32b_x16(to + c, o);
#pragma unroll
                  for (int j = 0; j < 16; ++j) v[j] = __float_as_uint(o[j] * f);
                  tmem_st16(to + c, v);
                }
              }
            }
            const float neg = m == -INFINITY ? 0.0f : -m;
            const uint64_t sc2 = f32x2(sc, sc), neg2 = f32x2(neg, neg);
            uint64_t sum2[2] = {0, 0};
#pragma unroll 1
            for (int c = 0; c < kTile; c += kChunk) {  // P goes over scores that have been read
              uint32_t x[kChunk], p[kChunk / 2];
              load_scores<kChunk>(ts + c, x, masked, lim32 - c);
#pragma unroll
              for (int j = 0; j < kChunk / 2; ++j) {
                const uint64_t y = fma_f32x2(f32x2(__uint_as_float(x[2 * j]), __uint_as_float(x[2 * j + 1])), sc2, neg2);
                const uint64_t e = f32x2(pg_ex2(f32x2_lo(y)), pg_ex2(f32x2_hi(y)));
                sum2[j & 1] = add_f32x2(sum2[j & 1], e);
                p[j] = pack2(f32x2_lo(e), f32x2_hi(e));
              }
              tmem_st16(ts + c / 2, p);
            }
            l += (f32x2_lo(sum2[0]) + f32x2_hi(sum2[0])) + (f32x2_lo(sum2[1]) + f32x2_hi(sum2[1]));
            tmem_st_wait();
            tc_fence_before_sync();
            __syncwarp();
            if (lane == 0) mbar_arrive(&s.p_full[i]);
          }
          if (!ok) break;
          ok = mbar_wait(&s.o_done[i], segs & 1u, abort) && mbar_wait(&s.p_full[i], static_cast<uint32_t>(n - 1) & 1u, abort);
          if (!__all_sync(kPagedFull, ok)) break;  // (p_full, long complete, orders what warp 2 left before its arrival)
          tc_fence_after_sync();
          const int2 lost = s.lost[i][segs & 1];
          if (lost.x == static_cast<int>(segs)) bad = min(bad, lost.y);
          ++segs;
        }
        if (pos >= bad) l = __int_as_float(0x7fc00000);
        const bool any = until > w.off, whole = w.off == 0 && w.end == w.per;
        if (whole) {
          const float inv = l == 0.0f ? 0.0f : 1.0f / l;
          __nv_bfloat16* dst = a.out + static_cast<long long>(w.q.first + tok) * a.ldo + head * HD;
#pragma unroll 1
          for (int c = 0; c < HD; c += 32) {
            uint32_t o[32];
            __syncwarp();  // (dead rows store nothing, and the load is the whole warp's)
            if (any)
              tmem_ld_32x32b_x32(to + c, o);
            else
#pragma unroll
              for (int j = 0; j < 32; ++j) o[j] = 0;
            if (live) {
#pragma unroll
              for (int j = 0; j < 4; ++j) {
                uint32_t v[4];
#pragma unroll
                for (int e = 0; e < 4; ++e)
                  v[e] = pack2(__uint_as_float(o[8 * j + 2 * e]) * inv, __uint_as_float(o[8 * j + 2 * e + 1]) * inv);
                *reinterpret_cast<uint4*>(dst + c + 8 * j) = make_uint4(v[0], v[1], v[2], v[3]);
              }
            }
          }
        } else {
          const size_t at = static_cast<size_t>(2 * blockIdx.x + (w.off == 0 ? 1 : 0)) * kItemRows + i * kTile + r;
          float* dst = a.part_o + at * HD;
          if (any) {
#pragma unroll 1
            for (int c = 0; c < HD; c += 32) {
              uint32_t o[32];
              __syncwarp();
              tmem_ld_32x32b_x32(to + c, o);
              if (live) {
#pragma unroll
                for (int j = 0; j < 8; ++j)
                  *reinterpret_cast<uint4*>(dst + c + 4 * j) = make_uint4(o[4 * j], o[4 * j + 1], o[4 * j + 2], o[4 * j + 3]);
              }
            }
          }
          if (live) reinterpret_cast<float2*>(a.part_ml)[at] = make_float2(any ? m : -INFINITY, l);
        }
        tc_fence_before_sync();
        t0 += w.used() - w.off;
      }
    }
  }
  tc_fence_before_sync();
  cta_teardown_barrier();
  if (warp == 1) {
    tc_fence_after_sync();
    tmem_dealloc(tmem, 512);
  }
}

// Joins the item that CTA c left unfinished: block (c, rows / 32), one warp per 4 rows.
constexpr int kJoinThreads = 256;
template <int HD>
__global__ void __launch_bounds__(kJoinThreads) paged_tc_join_kernel(const PagedArgs a) {
  pdl_launch_dependents();
  pdl_wait_prior_grids();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, c = blockIdx.x;
  const int4 open = a.split[c];
  const int c1 = open.w, h = open.y, tile = open.z;
  if (c1 <= c) return;
  const PagedSeq q = paged_seq(a, open.x);
  const float2* ml = reinterpret_cast<const float2*>(a.part_ml);
  constexpr int kPer = HD / 32;
  for (int k = 0; k < 4; ++k) {
    const int row = blockIdx.y * 32 + warp * 4 + k;
    const int rt = (row % kTile) / a.g, token = (2 * tile + row / kTile) * tile_tokens(a) + rt;
    if (rt >= tile_tokens(a) || token >= q.n) continue;
    float m = -INFINITY;
    for (int d = c + lane; d <= c1; d += 32) m = fmaxf(m, ml[static_cast<size_t>(2 * d + (d == c)) * kItemRows + row].x);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(kPagedFull, m, o));
    float l = 0.0f, acc[kPer];
#pragma unroll
    for (int j = 0; j < kPer; ++j) acc[j] = 0.0f;
#pragma unroll 4
    for (int d = c; d <= c1; ++d) {
      const size_t at = static_cast<size_t>(2 * d + (d == c)) * kItemRows + row;
      const float2 p = ml[at];
      if (p.x == -INFINITY) {  // nothing seen there: no output was left (a NaN sum still counts)
        if (isnan(p.y)) l = p.y;
        continue;
      }
      const float f = pg_ex2(p.x - m);
      l = fmaf(f, p.y, l);
      const float* src = a.part_o + at * HD + lane * kPer;
#pragma unroll
      for (int j = 0; j < kPer; ++j) acc[j] = fmaf(f, src[j], acc[j]);
    }
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    __nv_bfloat16* dst = a.out + static_cast<long long>(q.first + token) * a.ldo + (h * a.g + (row % kTile) % a.g) * HD + lane * kPer;
#pragma unroll
    for (int j = 0; j < kPer; j += 2) *reinterpret_cast<uint32_t*>(dst + j) = pack2(acc[j] * inv, acc[j + 1] * inv);
  }
}

template <int HD>
int launch(PagedArgs a, cudaStream_t stream) {
  static bool ready[64] = {false};
  constexpr size_t smem = sizeof(Smem<HD>) + 1024;
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64 || !ready[dev]) {
    cudaFuncAttributes at;
    cudaError_t e = cudaFuncGetAttributes(&at, paged_tc_kernel<HD>);
    if (e == cudaSuccess && at.numRegs < kRegsLaunch)  // the register split would wait for registers that are not there
      return fail(BP_ERR_UNSUPPORTED, "paged attention was built with %d registers per thread, %d expected", at.numRegs, kRegsLaunch);
    if (e == cudaSuccess)
      e = cudaFuncSetAttribute(paged_tc_kernel<HD>, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem));
    if (e != cudaSuccess) return fail(BP_ERR_CUDA, "cudaFuncSetAttribute(smem %zu): %s", smem, cudaGetErrorString(e));
    if (dev >= 0 && dev < 64) ready[dev] = true;
  }
  const int ps = 1 << a.page_log2;
  CUtensorMap tq, tk, tv;
  const uint64_t qdims[3] = {HD, static_cast<uint64_t>(a.nh), static_cast<uint64_t>(a.rows)};
  const uint64_t qstrides[2] = {HD * 2, static_cast<uint64_t>(a.ldq) * 2};
  const uint32_t qbox[3] = {64, static_cast<uint32_t>(a.g), static_cast<uint32_t>(kTile / a.g)};
  int st = tc_encode(&tq, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, a.q, qdims, qstrides, qbox, CU_TENSOR_MAP_SWIZZLE_128B,
                     CU_TENSOR_MAP_L2_PROMOTION_L2_128B);
  if (st != BP_OK) return st;
  st = paged_maps(a, ps < kTile ? ps : kTile, &tk, &tv);
  if (st != BP_OK) return st;
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[2];
  cfg.gridDim = dim3(a.G);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  set_launch_attrs(cfg, attr);
  cudaError_t e = cudaLaunchKernelEx(&cfg, paged_tc_kernel<HD>, tq, tk, tv, a);
  if (e == cudaSuccess && a.G > 1) {
    cfg.gridDim = dim3(a.G - 1, kItemRows / 32);
    cfg.blockDim = dim3(kJoinThreads);
    cfg.dynamicSmemBytes = 0;
    e = cudaLaunchKernelEx(&cfg, paged_tc_join_kernel<HD>, a);
  }
  if (e != cudaSuccess) return fail(BP_ERR_CUDA, "paged_attention launch (many rows): %s", cudaGetErrorString(e));
  return BP_OK;
}

}  // namespace

size_t paged_tc_workspace_bytes(int hd) {
  return static_cast<size_t>(2 * tc_sm_count()) * kItemRows * (hd + 2) * sizeof(float) + tc_sm_count() * sizeof(int4);
}

int launch_paged_tc(PagedArgs a, void* workspace, cudaStream_t stream) {
  a.G = tc_sm_count();
  a.min_share = 4;  // a part costs its write and its join
  a.part_o = static_cast<float*>(workspace);
  a.part_ml = a.part_o + static_cast<size_t>(2 * a.G) * kItemRows * a.hd;
  a.split = reinterpret_cast<int4*>(a.part_ml + static_cast<size_t>(2 * a.G) * kItemRows * 2);
  a.tile_tokens = kTile / a.g;
  return a.hd == 128 ? launch<128>(a, stream) : launch<64>(a, stream);
}

BP_DEFINE_DEVICE_ERROR_READER(read_device_errors_paged)

}  // namespace bp
