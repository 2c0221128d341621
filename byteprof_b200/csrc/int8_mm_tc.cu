// The 8-bit integer product on the 5th-generation tensor cores (kind::i8, int32 accumulators in TMEM), for the
// entry point in int8_mm.cu: y[m, n] = x_scale[m] * w_scale[n] * sum_k x[m, k] w[n, k] (+ bias[n]).
//
//  * One warp loads 128-byte K slices of both operands by TMA (128-byte swizzle, zero fill past M, N and K) into a
//    ring, one thread issues the MMAs, four warps drain the accumulators, scale and store.
//  * Many rows (kSwap = false): 128 tokens are the MMA's M, kBN channels its N. With enough tiles for the GPU the
//    grid is persistent and two accumulators alternate, so that a tile's epilogue runs under the next tile's
//    MMAs.
//  * Few rows (kSwap = true): the weights are the MMA's M (128 channels) and the tokens its N, in tiles of 16 or 32.
//  * Few tiles: the S CTAs of a cluster split a tile's K; their int32 partials meet in distributed shared memory
//    (the ring's memory, free by then), each CTA finishing 128 / S of the tile's lanes. Integer sums do not depend
//    on the order, so all forms give the same bits as the CUDA-core kernel.
#include <cudaTypedefs.h>

#include "int8_mm.h"
#include "skinny_internal.h"
#include "sm100.cuh"

namespace bp {
namespace {

constexpr int kBM = 128;
constexpr int kBK = 128;  // K bytes per stage: one 128-byte swizzle row
constexpr int kThreads = 192;
constexpr int kEpiWarp0 = 2;
constexpr int kEpiThreads = 128;
constexpr int kMaxSplit = 8;

// Two CTAs fit an SM (shared memory, TMEM, registers): one's prologue and epilogue run under the other's loads, and under
// programmatic dependent launch the next kernel's. With one CTA and twice the stages every launch exposed its own:
// 8.5 us for one row of 2048 -> 8192, whose weights take 2.6 us.
template <int kBN, bool kFuse>
struct Cfg {
  static constexpr int kStageBytes = (kBM + (kFuse ? 0 : kBN)) * kBK;
  static constexpr int kStages = kFuse ? 4 : kBN >= 128 ? 3 : 5;
  static constexpr int kRingBytes = kStages * kStageBytes;
  // in cluster mode the ring's memory holds the partials: S x kBN / 4 x (128 / S + 1) x 16 bytes
  static_assert(kRingBytes >= 4 * kBN * (kBM + kMaxSplit), "partials");
  static constexpr uint32_t kTmemCols = 2 * kBN < 32 ? 32 : 2 * kBN;
};

template <int kBN, bool kFuse>
struct Smem {
  uint8_t ring[Cfg<kBN, kFuse>::kRingBytes];  // 1024-byte aligned stages: A rows, then B rows
  float ws[2][kBN];                           // w_scale and bias of the tile's channels (kSwap: x_scale of its tokens)
  float bias[2][kBN];
  float lane_scale[2][kBM];                   // cluster mode: the scales (kSwap: and biases) of the tile's lanes
  uint64_t full[Cfg<kBN, kFuse>::kStages], empty[Cfg<kBN, kFuse>::kStages], tfull[2], tempty[2], mma_done, quantized;
  uint32_t tmem_base;
  int abort;
  float row_scale[16];  // kFuse
  uint32_t red[16];
};

template <int kBN, bool kFuse>
constexpr size_t smem_bytes() { return (sizeof(Smem<kBN, kFuse>) + 1023) / 1024 * 1024 + 1024; }

constexpr size_t kFuseBytes = 32 * 1024;  // the quantized tokens of a CTA's K range (kFuse)

struct Part {
  int ta, tb;   // tiles along the MMA's M and N
  int kb;       // K blocks
  int S;        // CTAs per tile (cluster), 1: persistent
  int grid;
};

// K blocks of the longest range of the split.
inline int fuse_blocks(const Part& p) { return (p.kb + p.S - 1) / p.S; }

__device__ __forceinline__ void wait_drain(uint64_t* bar, uint32_t parity) {
  const unsigned long long t0 = globaltimer();
  while (!mbar_try_wait(bar, parity)) {
    if (globaltimer() - t0 > kWaitLimitNs) {
      atomicOr(&g_bp_device_errors, BP_DEVERR_TIMEOUT);
      return;
    }
  }
}

// Tile order: 8 tiles along the MMA's M for each step along N, so that the CTAs at work share rows of both operands.
__device__ __forceinline__ void tile_of(const Part& p, int t, int& ia, int& ib) {
  constexpr int kGroup = 8;
  const int per = kGroup * p.tb, g = t / per, r = t - g * per;
  const int h = min(kGroup, p.ta - g * kGroup);
  ia = g * kGroup + r % h;
  ib = r / h;
}

__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  const __nv_bfloat162 p = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&p);
}

__device__ __forceinline__ void store1(const Int8Args& a, long long m, int n, float v) {
  if (a.y_f32)
    static_cast<float*>(a.y)[m * a.ldy + n] = v;
  else
    static_cast<__nv_bfloat16*>(a.y)[m * a.ldy + n] = __float2bfloat16_rn(v);
}

// Lane l's v[k] becomes lane k's v[l].
__device__ __forceinline__ void transpose32(float (&v)[32], int lane) {
#pragma unroll
  for (int s = 16; s > 0; s >>= 1) {
    const bool up = (lane & s) != 0;
#pragma unroll
    for (int i = 0; i < 32; ++i) {
      if (i & s) continue;
      const float got = __shfl_xor_sync(0xffffffffu, up ? v[i] : v[i | s], s);
      v[i] = up ? got : v[i];
      v[i | s] = up ? v[i | s] : got;
    }
  }
}

// A thread's row of a tile: kBN int32 columns of its TMEM lane -> scaled values of row m, columns n0 .. ; `drained` is
// called once when the accumulator has been read. Where the rows are not aligned, or end within 32 columns, the warp stores
// its 32 rows one after the other, 32 columns at a time (each thread its own row, value by value: 100 x 2048 -> 8191 in
// 40 us instead of 23).
template <int kBN, typename F>
__device__ __forceinline__ void drain_rows(const Int8Args& a, uint32_t src, long long m, int n0, const float* ws,
                                           const float* bias, int vec, F drained) {
  const float sx = m < a.M ? a.x_scale[m] : 0.0f;
#pragma unroll 1
  for (int c = 0; c < kBN; c += 32) {
    uint32_t raw[32];
    __syncwarp();  // (the lanes' stores below differ, and the load is the whole warp's)
    tmem_ld_32x32b_x32(src + c, raw);
    if (c + 32 == kBN) drained();
    const int n = n0 + c;
    float v[32];
#pragma unroll
    for (int j = 0; j < 32; ++j) v[j] = int8_value(a, static_cast<int>(raw[j]), sx, ws[c + j], bias[c + j]);
    if (vec && n + 32 <= a.N) {
      if (m >= a.M) {
        // a row past the end: nothing to store
      } else if (a.y_f32) {
        float4* d = reinterpret_cast<float4*>(static_cast<float*>(a.y) + m * a.ldy + n);
#pragma unroll
        for (int j = 0; j < 8; ++j) d[j] = make_float4(v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]);
      } else {
        uint4* d = reinterpret_cast<uint4*>(static_cast<__nv_bfloat16*>(a.y) + m * a.ldy + n);
#pragma unroll
        for (int j = 0; j < 4; ++j)
          d[j] = make_uint4(pack2(v[8 * j], v[8 * j + 1]), pack2(v[8 * j + 2], v[8 * j + 3]),
                            pack2(v[8 * j + 4], v[8 * j + 5]), pack2(v[8 * j + 6], v[8 * j + 7]));
      }
    } else {
      const int lane = threadIdx.x & 31;
      transpose32(v, lane);
#pragma unroll
      for (int k = 0; k < 32; ++k)
        if (m - lane + k < a.M && n + lane < a.N) store1(a, m - lane + k, n + lane, v[k]);
    }
  }
}

// Adds the S partials of L rows (m0 ..) of a tile and stores them; `red` is [S][kBN / 4][L + 1] groups of 4 columns; sx
// holds the rows' scales, ws and bias the columns'.
template <int kBN>
__device__ __forceinline__ void finish_rows(const Int8Args& a, const int4* red, int S, int L, long long m0, int n0, int vec,
                                            int threads, const float* sx, const float* ws, const float* bias) {
#pragma unroll 2
  for (int i = threadIdx.x; i < L * (kBN / 4); i += threads) {
    const int c4 = i % (kBN / 4), ll = i / (kBN / 4), n = n0 + 4 * c4;
    const long long m = m0 + ll;
    if (m >= a.M || n >= a.N) continue;
    int4 acc = make_int4(0, 0, 0, 0);
    for (int src = 0; src < S; ++src) {
      const int4 v = red[(src * (kBN / 4) + c4) * (L + 1) + ll];
      acc.x += v.x, acc.y += v.y, acc.z += v.z, acc.w += v.w;
    }
    const int* av = &acc.x;
    float v[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = int8_value(a, av[j], sx[ll], ws[4 * c4 + j], bias[4 * c4 + j]);
    if (vec && n + 4 <= a.N) {
      if (a.y_f32)
        *reinterpret_cast<float4*>(static_cast<float*>(a.y) + m * a.ldy + n) = make_float4(v[0], v[1], v[2], v[3]);
      else
        *reinterpret_cast<uint2*>(static_cast<__nv_bfloat16*>(a.y) + m * a.ldy + n) = make_uint2(pack2(v[0], v[1]), pack2(v[2], v[3]));
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (n + j < a.N) store1(a, m, n + j, v[j]);
    }
  }
}

// The K blocks [k0, k1) of the tokens' rows in 8 bits, as the MMA reads them: [block][kBN rows][128 bytes], 128-byte
// swizzle, zeros past K. Called by `n` threads (whole warps, not all of the CTA).
template <int kBN>
__device__ __forceinline__ void quantize_range(const Int8Args& a, const __nv_bfloat16* x, long long ldx, uint8_t* dst, int k0, int k1,
                                               float* row_scale, uint32_t* red, int tid, int n) {
  const int chunks = a.K / 8;  // K is a multiple of 8
  if (tid < 16) red[tid] = 0;
  __syncwarp();
  named_barrier_sync(1, n);
  constexpr int kU = 8;  // loads in flight
  for (int i0 = tid; i0 - (tid & 31) < a.M * chunks; i0 += kU * n) {
    uint4 v[kU];
    int row[kU];
#pragma unroll
    for (int u = 0; u < kU; ++u) {
      const int i = i0 + u * n;
      row[u] = i / chunks;
      v[u] = row[u] < a.M ? ld16(x + row[u] * ldx + (i - row[u] * chunks) * 8) : make_uint4(0, 0, 0, 0);
    }
#pragma unroll
    for (int u = 0; u < kU; ++u) {
      const uint32_t mx = abs_max8(v[u], 0);
      const int first = __shfl_sync(0xffffffffu, row[u], 0);
      if (__all_sync(0xffffffffu, row[u] == first)) {
        const uint32_t all = __reduce_max_sync(0xffffffffu, mx);
        if ((tid & 31) == 0 && first < a.M) atomicMax(&red[first], all);
      } else if (row[u] < a.M) {
        atomicMax(&red[row[u]], mx);
      }
    }
  }
  __syncwarp();
  named_barrier_sync(1, n);
  if (tid < a.M) row_scale[tid] = red[tid] >= 0x7f800000u ? __uint_as_float(0x7fc00000u) : int8_row_scale(red[tid]);
  // the MMA's columns past M read what lies here and nobody reads them
  const int span = (k1 - k0) * 16;  // 8-value pieces of a row
  for (int r = 0; r < a.M; ++r) {
    const bool bad = red[r] >= 0x7f800000u;
    const float s = int8_row_scale(red[r]), inv = 1.0f / s;
    for (int i = tid; i < span; i += n) {
      const int b = i / 16, c = i % 16, k = (k0 + b) * kBK + c * 8;
      const uint2 v = k < a.K && !bad ? q8(ld16(x + r * ldx + k), s, inv) : make_uint2(0, 0);
      *reinterpret_cast<uint2*>(dst + b * kBN * kBK + r * kBK + (((c / 2) ^ (r & 7)) * 16) + (c & 1) * 8) = v;
    }
  }
  __syncwarp();
  named_barrier_sync(1, n);  // row_scale is visible to the epilogue
}

// kFuse (kSwap, one or two tokens): x is bf16 and every CTA quantizes its K range of it itself, while the weights stream:
// one launch instead of two, where launches are most of the time. The rows' maxima need all of K, which is little
// then (int8_fused_supported).
template <int kBN, bool kSwap, bool kCluster, bool kFuse>
__global__ void __launch_bounds__(kThreads, 2)
    int8_mm_tc_kernel(const __grid_constant__ CUtensorMap ta, const __grid_constant__ CUtensorMap tb, const Int8Args a,
                      const Part p, const int vec, const __nv_bfloat16* xb, const long long ldxb) {
  using C = Cfg<kBN, kFuse>;
  constexpr int kStages = C::kStages;
  extern __shared__ uint8_t smem_raw[];
  Smem<kBN, kFuse>& s = *reinterpret_cast<Smem<kBN, kFuse>*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  uint8_t* fused = reinterpret_cast<uint8_t*>(&s) + (sizeof(Smem<kBN, kFuse>) + 1023) / 1024 * 1024;  // kFuse: [K block][kBN][128]
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = kCluster ? blockIdx.y : 0;
  const int t0 = blockIdx.x, step = kCluster ? 1 << 30 : p.grid, tiles = p.ta * p.tb;
  const int k0 = kCluster ? static_cast<int>(static_cast<long long>(rank) * p.kb / p.S) : 0;
  const int k1 = kCluster ? static_cast<int>(static_cast<long long>(rank + 1) * p.kb / p.S) : p.kb;

  if (threadIdx.x == 0) {
    for (int i = 0; i < kStages; ++i) {
      mbar_init(&s.full[i], 1);
      mbar_init(&s.empty[i], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&s.tfull[b], 1);
      mbar_init(&s.tempty[b], kEpiThreads);
    }
    mbar_init(&s.mma_done, 1);
    s.abort = 0;
    mbar_fence_init();
    tma_prefetch_desc(&ta);
    if (!kFuse) tma_prefetch_desc(&tb);
    mbar_init(&s.quantized, kThreads - 32);
    mbar_fence_init();
  }
  if (warp == 1) {
    tmem_alloc(&s.tmem_base, C::kTmemCols);
    tmem_relinquish();
  }
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  pdl_launch_dependents();
  pdl_wait_prior_grids();  // both operands may come from the kernel before (the quantizer makes either)
  const uint32_t tmem = s.tmem_base;
  volatile int* abort = &s.abort;

  if (warp == 0) {
    if (lane == 0) {
      int i = 0;
      bool ok = true;
      for (int t = t0; t < tiles && ok; t += step) {
        int ia, ib;
        tile_of(p, t, ia, ib);
        for (int kb = k0; kb < k1; ++kb, ++i) {
          const int st = i % kStages;
          if (i >= kStages && !mbar_wait(&s.empty[st], static_cast<uint32_t>((i / kStages) + 1) & 1u, abort)) {
            ok = false;
            break;
          }
          uint8_t* dst = s.ring + st * C::kStageBytes;
          mbar_arrive_expect_tx(&s.full[st], kFuse ? kBM * kBK : C::kStageBytes);
          tma_load_2d(dst, &ta, &s.full[st], kb * kBK, ia * kBM);
          if (!kFuse) tma_load_2d(dst + kBM * kBK, &tb, &s.full[st], kb * kBK, ib * kBN);
        }
      }
      for (int st = 0; st < kStages && st < i; ++st)  // the last copy issued into each stage has landed
        wait_drain(&s.full[st], static_cast<uint32_t>((i - 1 - st) / kStages) & 1u);
    }
  } else if (kFuse) {
    quantize_range<kBN>(a, xb, ldxb, fused, k0, k1, s.row_scale, s.red, threadIdx.x - 32, kThreads - 32);
    fence_async_shared();
    mbar_arrive(&s.quantized);
  }
  if (warp == 1) {
    if (lane == 0) {
      if (kFuse) mbar_wait(&s.quantized, 0, abort);
      constexpr uint32_t idesc = umma_idesc_s8(kBM, kBN);
      // descriptors of the first stage; the others are address differences away (in units of 16 bytes)
      const uint64_t ring = umma_desc_sw128(smem_addr(s.ring)), planes = kFuse ? umma_desc_sw128(smem_addr(fused)) : 0;
      int i = 0, it = 0;
      bool ok = true;
      for (int t = t0; t < tiles && ok; t += step, ++it) {
        const int buf = it & 1;
        if (it >= 2 && !mbar_wait(&s.tempty[buf], static_cast<uint32_t>((it >> 1) + 1) & 1u, abort)) break;
        tc_fence_after_sync();
        const uint32_t dacc = tmem + static_cast<uint32_t>(buf * kBN);
        for (int kb = k0; kb < k1; ++kb, ++i) {
          const int st = i % kStages;
          if (!mbar_wait(&s.full[st], static_cast<uint32_t>(i / kStages) & 1u, abort)) {
            ok = false;
            break;
          }
          tc_fence_after_sync();
          const uint64_t da = ring + st * (C::kStageBytes >> 4),
                         db = kFuse ? planes + (kb - k0) * (kBN * kBK >> 4) : da + (kBM * kBK >> 4);
#pragma unroll
          for (int kk = 0; kk < kBK / 32; ++kk) umma_i8(dacc, da + 2 * kk, db + 2 * kk, idesc, (kb > k0 || kk > 0) ? 1u : 0u);
          umma_commit(&s.empty[st]);
        }
        if (ok) umma_commit(&s.tfull[buf]);
      }
      umma_commit(&s.mma_done);
      wait_drain(&s.mma_done, 0);
    }
  } else if (!kCluster && warp >= kEpiWarp0) {
    const int q = warp & 3, r = 32 * q + lane, et = threadIdx.x - 32 * kEpiWarp0;
    int it = 0;
    for (int t = t0; t < tiles; t += step, ++it) {
      const int buf = it & 1;
      int ia, ib;
      tile_of(p, t, ia, ib);
      if (kSwap) {
        for (int j = et; j < kBN; j += kEpiThreads) s.ws[buf][j] = ib * kBN + j >= a.M ? 0.0f : kFuse ? s.row_scale[j] : a.x_scale[ib * kBN + j];
      } else {
        for (int j = et; j < kBN; j += kEpiThreads) {
          const int n = ib * kBN + j;
          s.ws[buf][j] = n < a.N ? int8_w_scale(a, n) : 0.0f;
          s.bias[buf][j] = n < a.N ? int8_bias(a, n) : 0.0f;
        }
      }
      const bool ok = mbar_wait(&s.tfull[buf], static_cast<uint32_t>(it >> 1) & 1u, abort);
      __syncwarp();
      if (named_barrier_or(1, kEpiThreads, !ok)) break;  // (also: the scales above are visible)
      tc_fence_after_sync();
      const uint32_t src = tmem + (static_cast<uint32_t>(32 * q) << 16) + static_cast<uint32_t>(buf * kBN);
      if (kSwap) {
        const int n = ia * kBM + r;
        const float sw = n < a.N ? int8_w_scale(a, n) : 0.0f, bias = n < a.N ? int8_bias(a, n) : 0.0f;
#pragma unroll 1
        for (int c = 0; c < kBN; c += 16) {
          float raw[16];
          __syncwarp();
          tmem_ld_32x32b_x16(src + c, raw);
          if (c + 16 == kBN) {
            tc_fence_before_sync();
            mbar_arrive(&s.tempty[buf]);
          }
          if (n < a.N) {
#pragma unroll
            for (int j = 0; j < 16; ++j) {
              const int m = ib * kBN + c + j;
              if (m < a.M) store1(a, m, n, int8_value(a, __float_as_int(raw[j]), s.ws[buf][c + j], sw, bias));
            }
          }
        }
      } else {
        const long long m = static_cast<long long>(ia) * kBM + r;
        drain_rows<kBN>(a, src, m, ib * kBN, s.ws[buf], s.bias[buf], vec, [&] {
          tc_fence_before_sync();
          mbar_arrive(&s.tempty[buf]);
        });
      }
    }
  }

  if constexpr (kCluster) {
    // one tile per cluster. The scales are fetched under the MMAs
    int ia, ib;
    tile_of(p, t0, ia, ib);
    if (warp >= kEpiWarp0) {
      const int et = threadIdx.x - 32 * kEpiWarp0;
      if (kSwap) {
        const int n = ia * kBM + et;
        s.lane_scale[0][et] = n < a.N ? int8_w_scale(a, n) : 0.0f;
        s.lane_scale[1][et] = n < a.N ? int8_bias(a, n) : 0.0f;
        if (et < kBN) s.ws[0][et] = ib * kBN + et >= a.M ? 0.0f : kFuse ? s.row_scale[et & 15] : a.x_scale[ib * kBN + et];
      } else {
        const long long m = static_cast<long long>(ia) * kBM + et;
        s.lane_scale[0][et] = m < a.M ? a.x_scale[m] : 0.0f;
        for (int j = et; j < kBN; j += kEpiThreads) {
          const int n = ib * kBN + j;
          s.ws[0][j] = n < a.N ? int8_w_scale(a, n) : 0.0f;
          s.bias[0][j] = n < a.N ? int8_bias(a, n) : 0.0f;
        }
      }
    }
    // the partials go through the ring's memory: every CTA's MMAs have read it ...
    if (warp >= kEpiWarp0 && !mbar_wait(&s.tfull[0], 0, abort)) *abort = 1;
    __syncwarp();
    cluster_sync_unaligned();
    const int S = p.S, L = kBM / S;
    if (warp >= kEpiWarp0) {
      tc_fence_after_sync();
      const int q = warp & 3, r = 32 * q + lane, own = r / L, ll = r % L;
      const uint32_t dst = mapa_shared(smem_addr(s.ring), static_cast<uint32_t>(own));
      const uint32_t src = tmem + (static_cast<uint32_t>(32 * q) << 16);
#pragma unroll 1
      for (int c = 0; c < kBN; c += 16) {
        float raw[16];
        tmem_ld_32x32b_x16(src + c, raw);
#pragma unroll
        for (int j = 0; j < 4; ++j)
          asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(
                           dst + static_cast<uint32_t>(((rank * (kBN / 4) + c / 4 + j) * (L + 1) + ll) * 16)),
                       "f"(raw[4 * j]), "f"(raw[4 * j + 1]), "f"(raw[4 * j + 2]), "f"(raw[4 * j + 3])
                       : "memory");
      }
      tc_fence_before_sync();
    }
    cluster_sync_unaligned();  // ... and every partial has landed
    if (!*abort) {
      const int4* red = reinterpret_cast<const int4*>(s.ring);
      if (kSwap) {
#pragma unroll 2
        for (int i = threadIdx.x; i < L * kBN; i += kThreads) {
          const int ll = i % L, j = i / L, n = ia * kBM + rank * L + ll, m = ib * kBN + j;
          if (m >= a.M || n >= a.N) continue;
          int acc = 0;
          for (int src = 0; src < S; ++src)
            acc += reinterpret_cast<const int*>(red + (src * (kBN / 4) + j / 4) * (L + 1) + ll)[j & 3];
          store1(a, m, n, int8_value(a, acc, s.ws[0][j], s.lane_scale[0][rank * L + ll], s.lane_scale[1][rank * L + ll]));
        }
      } else {
        finish_rows<kBN>(a, red, S, L, static_cast<long long>(ia) * kBM + rank * L, ib * kBN, vec, kThreads,
                         s.lane_scale[0] + rank * L, s.ws[0], s.bias[0]);
      }
    }
  }

  tc_fence_before_sync();
  cta_teardown_barrier();
  if (warp == 1) {
    tc_fence_after_sync();
    tmem_dealloc(tmem, C::kTmemCols);
  }
}

template <int kBN, bool kSwap, bool kCluster, bool kFuse>
int launch(const Int8Args& a, const Part& p, cudaStream_t stream, const __nv_bfloat16* xb = nullptr, long long ldxb = 0) {
  auto* kern = int8_mm_tc_kernel<kBN, kSwap, kCluster, kFuse>;
  constexpr size_t smem_max = smem_bytes<kBN, kFuse>() + (kFuse ? kFuseBytes : 0);
  const size_t smem = smem_bytes<kBN, kFuse>() + (kFuse ? static_cast<size_t>(fuse_blocks(p)) * kBN * kBK : 0);
  static bool ready[64] = {false};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64 || !ready[dev]) {
    const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                               static_cast<int>(smem_max));
    if (e != cudaSuccess) return fail(BP_ERR_CUDA, "cudaFuncSetAttribute(smem %zu): %s", smem_max, cudaGetErrorString(e));
    if (dev >= 0 && dev < 64) ready[dev] = true;
  }
  const int8_t* A = kSwap ? a.w : a.x;
  const int8_t* B = kSwap ? a.x : a.w;
  CUtensorMap ta, tb;
  int st = tc_encode_2d(&ta, CU_TENSOR_MAP_DATA_TYPE_UINT8, A, a.K, kSwap ? a.N : a.M, kSwap ? a.ldw : a.ldx, kBK, kBM,
                        CU_TENSOR_MAP_L2_PROMOTION_L2_256B);
  if (st != BP_OK) return st;
  if (kFuse) {
    tb = ta;
  } else {
    st = tc_encode_2d(&tb, CU_TENSOR_MAP_DATA_TYPE_UINT8, B, a.K, kSwap ? a.M : a.N, kSwap ? a.ldx : a.ldw, kBK, kBN,
                      CU_TENSOR_MAP_L2_PROMOTION_L2_256B);
    if (st != BP_OK) return st;
  }
  const int es = a.y_f32 ? 4 : 2;
  const int vec = reinterpret_cast<uintptr_t>(a.y) % 16 == 0 && (a.ldy * es) % 16 == 0;
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[2];
  cfg.gridDim = kCluster ? dim3(p.ta * p.tb, p.S) : dim3(p.grid);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  set_launch_attrs(cfg, attr, kCluster ? p.S : 1);
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kern, ta, tb, a, p, vec, xb, ldxb);
  if (e != cudaSuccess)
    return fail(BP_ERR_CUDA, "int8_mm launch (M=%d N=%d K=%d BN=%d S=%d): %s", a.M, a.N, a.K, kBN, p.S, cudaGetErrorString(e));
  return BP_OK;
}

template <int kBN, bool kSwap>
Part partition(const Int8Args& a) {
  Part p;
  p.ta = ((kSwap ? a.N : a.M) + kBM - 1) / kBM;
  p.tb = ((kSwap ? a.M : a.N) + kBN - 1) / kBN;
  p.kb = (a.K + kBK - 1) / kBK;
  p.S = 1;
  const long long tiles = static_cast<long long>(p.ta) * p.tb;
  p.grid = static_cast<int>(tiles < 2 * tc_sm_count() ? tiles : 2 * tc_sm_count());
  return p;
}

// Few tiles for the GPU: the 8 or 4 CTAs of a cluster share a tile's K. Meeting in distributed shared memory costs 3 to
// 5 us, so a split has to save more (one row, weights cold: 8192 -> 2048 takes 22.5 us whole, 10.5 in 4, 8.7 in 8;
// 8192 -> 8192 23 whole, 16.5 in 4; 2048 -> 8192 8.7 whole, 8.9 in 4; two CTAs gained nowhere).
template <int kBN, bool kSwap>
Part split_partition(const Int8Args& a) {
  Part p = partition<kBN, kSwap>(a);
  const long long ctas = 2 * tc_sm_count(), tiles = static_cast<long long>(p.ta) * p.tb;
  if (tiles * 8 <= ctas && p.kb >= 8)
    p.S = 8;
  else if (tiles * 4 <= ctas && p.kb >= 32)
    p.S = 4;
  return p;
}

template <int kBN, bool kFuse>
int launch_swap(const Int8Args& a, cudaStream_t stream, const __nv_bfloat16* xb = nullptr, long long ldxb = 0) {
  const Part p = split_partition<kBN, true>(a);
  return p.S > 1 ? launch<kBN, true, true, kFuse>(a, p, stream, xb, ldxb) : launch<kBN, true, false, kFuse>(a, p, stream, xb, ldxb);
}

// ---- many rows: pairs of CTAs -------------------------------------------------------------------------
// A 256 x 256 tile per pair (cta_group::2): each CTA loads 128 tokens and 128 channels per K slice for the MMA work
// for which a CTA by itself loads 128 and 256. The tile sizes are set by that: the operands come from L2, and
// with 48 KB per CTA and K slice the L2 delivers them at 10 TB/s while the tensor cores wait two thirds of the time
// (8192 x 2048 -> 16384: 318 us).
// Eight warps drain: four take the tile's first 128 channels, four the others, each group in two steps of 64 channels
// through 16 KB of shared memory and a TMA store (bf16). A warp that stores its lanes' rows straight from registers
// needs 32 transactions per instruction, and one group of four warps took longer than the tile's MMAs at K = 2048.
struct PairSmem {
  static constexpr int kStages = 5;
  static constexpr int kStageBytes = 2 * kBM * kBK;
  uint8_t ring[kStages * kStageBytes];  // 128 token rows, then 128 channel rows, per stage
  uint8_t out[2][kBM * 128];            // per group: 128 rows x 64 bf16, 128-byte swizzle
  float ws[2][256], bias[2][256];
  uint64_t full[kStages], empty[kStages], tfull[2], tempty[2], mma_done;
  uint32_t tmem_base;
  int abort;
};
constexpr int kPairN = 256;
constexpr int kPairEpi = 256;
constexpr int kPairThreads = 32 * kEpiWarp0 + kPairEpi;

// vec: y's rows are 16-byte aligned, and in bf16 end at 16 bytes: stored through `ty`, a map of y in 64 x 128 boxes
__global__ void __launch_bounds__(kPairThreads, 1) __cluster_dims__(2, 1, 1)
    int8_mm_pair_kernel(const __grid_constant__ CUtensorMap ta, const __grid_constant__ CUtensorMap tb,
                        const __grid_constant__ CUtensorMap ty, const Int8Args a, const Part p, const int vec) {
  constexpr int kStages = PairSmem::kStages;
  extern __shared__ uint8_t smem_raw[];
  PairSmem& s = *reinterpret_cast<PairSmem*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = static_cast<int>(cluster_ctarank());
  const int t0 = blockIdx.x / 2, step = p.grid / 2, tiles = p.ta * p.tb;

  if (threadIdx.x == 0) {
    for (int i = 0; i < kStages; ++i) {
      mbar_init(&s.full[i], 1);
      mbar_init(&s.empty[i], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&s.tfull[b], 1);
      mbar_init(&s.tempty[b], 2 * kPairEpi);
    }
    mbar_init(&s.mma_done, 1);
    s.abort = 0;
    mbar_fence_init();
    tma_prefetch_desc(&ta);
    tma_prefetch_desc(&tb);
  }
  if (warp == 1) tmem_alloc_pair(&s.tmem_base, 512);
  tc_fence_before_sync();
  __syncthreads();
  cluster_sync_unaligned();  // the peer's barriers are initialised before anything arrives on them
  tc_fence_after_sync();
  pdl_launch_dependents();
  pdl_wait_prior_grids();
  const uint32_t tmem = s.tmem_base;
  volatile int* abort = &s.abort;

  if (warp == 0) {
    if (lane == 0) {
      int i = 0;
      bool ok = true;
      for (int t = t0; t < tiles && ok; t += step) {
        int ia, ib;
        tile_of(p, t, ia, ib);
        for (int kb = 0; kb < p.kb; ++kb, ++i) {
          const int st = i % kStages;
          if (i >= kStages && !mbar_wait(&s.empty[st], static_cast<uint32_t>((i / kStages) + 1) & 1u, abort)) {
            ok = false;
            break;
          }
          uint8_t* dst = s.ring + st * PairSmem::kStageBytes;
          const uint32_t bar = mapa_shared(smem_addr(&s.full[st]), 0);  // the leader's barrier counts both CTAs' bytes
          if (rank == 0) mbar_arrive_expect_tx(&s.full[st], 2 * PairSmem::kStageBytes);
          tma_load_2d_pair(dst, &ta, bar, kb * kBK, ia * 2 * kBM + rank * kBM);
          tma_load_2d_pair(dst + kBM * kBK, &tb, bar, kb * kBK, ib * kPairN + rank * (kPairN / 2));
        }
      }
      if (rank == 0)
        for (int st = 0; st < kStages && st < i; ++st) wait_drain(&s.full[st], static_cast<uint32_t>((i - 1 - st) / kStages) & 1u);
    }
  } else if (warp == 1) {
    if (lane == 0 && rank == 0) {
      constexpr uint32_t idesc = umma_idesc_s8(2 * kBM, kPairN);
      const uint64_t ring = umma_desc_sw128(smem_addr(s.ring));
      int i = 0, it = 0;
      bool ok = true;
      for (int t = t0; t < tiles && ok; t += step, ++it) {
        const int buf = it & 1;
        if (it >= 2 && !mbar_wait(&s.tempty[buf], static_cast<uint32_t>((it >> 1) + 1) & 1u, abort)) break;
        tc_fence_after_sync();
        const uint32_t dacc = tmem + static_cast<uint32_t>(buf * kPairN);
        for (int kb = 0; kb < p.kb; ++kb, ++i) {
          const int st = i % kStages;
          if (!mbar_wait(&s.full[st], static_cast<uint32_t>(i / kStages) & 1u, abort)) {
            ok = false;
            break;
          }
          tc_fence_after_sync();
          const uint64_t da = ring + st * (PairSmem::kStageBytes >> 4), db = da + (kBM * kBK >> 4);
#pragma unroll
          for (int kk = 0; kk < kBK / 32; ++kk) umma_i8_pair(dacc, da + 2 * kk, db + 2 * kk, idesc, (kb > 0 || kk > 0) ? 1u : 0u);
          umma_commit_pair(&s.empty[st]);
        }
        if (ok) umma_commit_pair(&s.tfull[buf]);
      }
      umma_commit_pair(&s.mma_done);
      wait_drain(&s.mma_done, 0);
    }
  } else {
    const int q = warp & 3, r = 32 * q + lane, et = threadIdx.x - 32 * kEpiWarp0, grp = et / 128;
    uint8_t* stage = s.out[grp];
    int it = 0;
    for (int t = t0; t < tiles; t += step, ++it) {
      const int buf = it & 1;
      int ia, ib;
      tile_of(p, t, ia, ib);
      {
        const int n = ib * kPairN + et;
        s.ws[buf][et] = n < a.N ? int8_w_scale(a, n) : 0.0f;
        s.bias[buf][et] = n < a.N ? int8_bias(a, n) : 0.0f;
      }
      const bool ok = mbar_wait(&s.tfull[buf], static_cast<uint32_t>(it >> 1) & 1u, abort);
      __syncwarp();
      if (named_barrier_or(1, kPairEpi, !ok)) break;
      tc_fence_after_sync();
      const int c0 = grp * 128;
      const uint32_t src = tmem + (static_cast<uint32_t>(32 * q) << 16) + static_cast<uint32_t>(buf * kPairN + c0);
      const uint32_t done = mapa_shared(smem_addr(&s.tempty[buf]), 0);
      const int m0 = (ia * 2 + rank) * kBM;
      auto drained = [&] {
        tc_fence_before_sync();
        mbar_arrive_cluster(done);
      };
      if (a.y_f32) {
        drain_rows<128>(a, src, static_cast<long long>(m0) + r, ib * kPairN + c0, s.ws[buf] + c0, s.bias[buf] + c0, vec, drained);
        continue;
      }
      const float sx = m0 + r < a.M ? a.x_scale[m0 + r] : 0.0f;
#pragma unroll 1
      for (int h = 0; h < 2; ++h) {
        if (et % 128 == 0) tma_store_wait<false>();  // the store before has read the buffer
        __syncwarp();
        named_barrier_sync(2 + grp, 128);
#pragma unroll
        for (int c = 0; c < 64; c += 32) {
          uint32_t raw[32];
          tmem_ld_32x32b_x32(src + h * 64 + c, raw);
          if (h == 1 && c == 32) drained();
          const float* ws = s.ws[buf] + c0 + h * 64 + c;
          const float* bias = s.bias[buf] + c0 + h * 64 + c;
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            float v[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = int8_value(a, static_cast<int>(raw[8 * j + e]), sx, ws[8 * j + e], bias[8 * j + e]);
            *reinterpret_cast<uint4*>(stage + r * 128 + (((c / 8 + j) ^ (r & 7)) * 16)) =
                make_uint4(pack2(v[0], v[1]), pack2(v[2], v[3]), pack2(v[4], v[5]), pack2(v[6], v[7]));
          }
        }
        fence_async_shared();
        named_barrier_sync(2 + grp, 128);
        const int n0 = ib * kPairN + c0 + h * 64;
        if (vec) {
          if (et % 128 == 0) {
            tma_store_2d(&ty, stage, n0, m0);
            tma_store_commit();
          }
          continue;
        }
        // Rows that TMA cannot store: a warp writes its 32 rows one after the other, 64 bytes in a row at a time (straight from
        // registers each of 32 rows gets 2 bytes at a time: 4000 x 512 -> 50001 took 1912 us instead of 316).
        const int rows = min(32, a.M - m0 - 32 * q), cols = a.N - n0;
        __nv_bfloat16* y = static_cast<__nv_bfloat16*>(a.y) + static_cast<long long>(m0 + 32 * q) * a.ldy + n0;
#pragma unroll 4
        for (int k = 0; k < rows; ++k) {
          const uint8_t* row = stage + (32 * q + k) * 128;
#pragma unroll
          for (int cc = lane; cc < 64; cc += 32)
            if (cc < cols) y[k * a.ldy + cc] = *reinterpret_cast<const __nv_bfloat16*>(row + (((cc / 8) ^ (k & 7)) * 16) + cc % 8 * 2);
        }
      }
    }
    if (et % 128 == 0) tma_store_wait<true>();
    // The leader's commits arrive in both CTAs, in order: the peer may not end (and give up its shared memory) before the
    // last one has reached it. Waited for here, behind the tiles, where it is due.
    if (rank != 0 && et == 0) wait_drain(&s.mma_done, 0);
  }
  tc_fence_before_sync();
  cta_teardown_barrier();
  cluster_sync_unaligned();  // the leader's MMAs have read the peer's memory, every copy has landed in both
  if (warp == 1) {
    tc_fence_after_sync();
    tmem_dealloc_pair(tmem, 512);
  }
}

Part pair_partition(const Int8Args& a) {
  Part p;
  p.ta = (a.M + 2 * kBM - 1) / (2 * kBM);
  p.tb = (a.N + kPairN - 1) / kPairN;
  p.kb = (a.K + kBK - 1) / kBK;
  p.S = 1;
  const long long pairs = tc_sm_count() / 2, tiles = static_cast<long long>(p.ta) * p.tb;
  p.grid = static_cast<int>(2 * (tiles < pairs ? tiles : pairs));
  return p;
}

int launch_pair(const Int8Args& a, const Part& p, cudaStream_t stream) {
  static bool ready[64] = {false};
  constexpr size_t smem = sizeof(PairSmem) + 1024;
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64 || !ready[dev]) {
    const cudaError_t e = cudaFuncSetAttribute(int8_mm_pair_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem));
    if (e != cudaSuccess) return fail(BP_ERR_CUDA, "cudaFuncSetAttribute(smem %zu): %s", smem, cudaGetErrorString(e));
    if (dev >= 0 && dev < 64) ready[dev] = true;
  }
  CUtensorMap ta, tb;
  int st = tc_encode_2d(&ta, CU_TENSOR_MAP_DATA_TYPE_UINT8, a.x, a.K, a.M, a.ldx, kBK, kBM, CU_TENSOR_MAP_L2_PROMOTION_L2_256B);
  if (st != BP_OK) return st;
  st = tc_encode_2d(&tb, CU_TENSOR_MAP_DATA_TYPE_UINT8, a.w, a.K, a.N, a.ldw, kBK, kBM, CU_TENSOR_MAP_L2_PROMOTION_L2_256B);
  if (st != BP_OK) return st;
  const int es = a.y_f32 ? 4 : 2;
  // A TMA store does not end within 16 bytes: with N = 159 bf16 in rows of 160 it wrote the column behind the block, too. Such
  // results are stored a row at a time.
  const int vec = reinterpret_cast<uintptr_t>(a.y) % 16 == 0 && (a.ldy * es) % 16 == 0 && (a.y_f32 || a.N % 8 == 0);
  CUtensorMap ty = ta;
  if (vec && !a.y_f32) {
    st = tc_encode_2d(&ty, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, a.y, a.N, a.M, a.ldy * 2, 64, kBM, CU_TENSOR_MAP_L2_PROMOTION_NONE);
    if (st != BP_OK) return st;
  }
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[2];
  cfg.gridDim = dim3(p.grid);
  cfg.blockDim = dim3(kPairThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  set_launch_attrs(cfg, attr);
  const cudaError_t e = cudaLaunchKernelEx(&cfg, int8_mm_pair_kernel, ta, tb, ty, a, p, vec);
  if (e != cudaSuccess) return fail(BP_ERR_CUDA, "int8_mm launch (pairs, M=%d N=%d K=%d): %s", a.M, a.N, a.K, cudaGetErrorString(e));
  return BP_OK;
}

}  // namespace

bool int8_mm_tc_supported(const Int8Args& a) {
  return a.K > 0 && a.ldx % 16 == 0 && a.ldw % 16 == 0 && reinterpret_cast<uintptr_t>(a.x) % 16 == 0 &&
         reinterpret_cast<uintptr_t>(a.w) % 16 == 0;
}

int launch_int8_mm_tc(const Int8Args& a, cudaStream_t stream) {
  // Up to 64 tokens: the weights as the MMA's rows (8 tokens of 2048 -> 2048 take 10.0 us, 14.6 with the tokens as rows; 64 of
  // 8192 -> 2048 15.8 and 18.4, of 2048 -> 8192 16.5 and 16.8).
  if (a.M <= 16) return launch_swap<16, false>(a, stream);
  if (a.M <= 64) return launch_swap<32, false>(a, stream);
  // Both forms stream 256 operand rows per CTA and K slice at the rate of the L2, about 0.4 us a slice, and what differs is
  // how many slices an SM has to take, waves included; meeting in a cluster costs a split about ten slices
  // (2048 x 2048 -> 16384: 53 us in pairs, 72 in single CTAs; 509 x 8192 -> 2048: 26 in pairs, 18 split in 4).
  const Part p = pair_partition(a);
  const long long sms = tc_sm_count(), pt = static_cast<long long>(p.ta) * p.tb;
  if (pt > (1 << 28)) return fail(BP_ERR_UNSUPPORTED, "int8_mm: too many tiles (M=%d N=%d)", a.M, a.N);
  const Part o = split_partition<128, false>(a);
  const long long ot = static_cast<long long>(o.ta) * o.tb;
  const long long pair_cost = (2 * pt + sms - 1) / sms * p.kb;
  const long long one_cost = (ot * o.S + sms - 1) / sms * ((o.kb + o.S - 1) / o.S) + (o.S > 1 ? 10 : 0);
  if (a.M > kBM && pair_cost <= one_cost) return launch_pair(a, p, stream);
  return o.S > 1 ? launch<128, false, true, false>(a, o, stream) : launch<128, false, false, false>(a, o, stream);
}

// Each CTA quantizes the tokens of its whole K range, so this pays for a row or two: one row of 2048 -> 8192 takes 10.8 us
// (13.1 in two kernels), of 8192 -> 2048 10.7 (11.7); 2 rows of 2048 -> 8192 12.0 (13.2), of 4096 -> 4096 11.2 (11.1), 3 of
// 2048 -> 8192 13.2 (13.3), 4 14.2 (13.4).
bool int8_fused_supported(const Int8Args& a, const void* x, long long ldx) {
  if (a.M > 2 || a.K % 8 != 0 || static_cast<long long>(a.M) * a.K > 8192 || ldx % 8 != 0 || a.ldw % 16 != 0 ||
      reinterpret_cast<uintptr_t>(x) % 16 != 0 || reinterpret_cast<uintptr_t>(a.w) % 16 != 0)
    return false;
  return static_cast<size_t>(fuse_blocks(split_partition<16, true>(a))) * 16 * kBK <= kFuseBytes;
}

int launch_int8_fused(const Int8Args& a, const __nv_bfloat16* x, long long ldx, cudaStream_t stream) {
  return launch_swap<16, true>(a, stream, x, ldx);
}

BP_DEFINE_DEVICE_ERROR_READER(read_device_errors_int8mm)

}  // namespace bp
