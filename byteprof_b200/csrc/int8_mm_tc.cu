// The 8-bit integer product on the 5th-generation tensor cores (kind::i8, int32 accumulators in TMEM), for the
// entry point in int8_mm.cu: y[m, n] = x_scale[m] * w_scale[n] * sum_k x[m, k] w[n, k] (+ bias[n]).
//
//  * One warp loads 128-byte K slices of both operands by TMA (128-byte swizzle, zero fill past M, N and K) into a
//    ring, one thread issues the MMAs, four warps drain the accumulators, scale and store.
//  * Many rows (kSwap = false): 128 tokens are the MMA's M, kBN channels its N. With enough tiles for the GPU the
//    grid is persistent and two accumulators alternate, so that a tile's epilogue runs under the next tile's
//    MMAs.
//  * Few rows (kSwap = true): the weights are the MMA's M (128 channels) and the tokens its N, padded to 16, 32 or
//    64: the weights stream once, whatever the number of tokens.
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

template <int kBN>
struct Cfg {
  static constexpr int kStageBytes = (kBM + kBN) * kBK;
  static constexpr int kStages = kBN >= 256 ? 4 : kBN >= 128 ? 6 : 8;
  // in cluster mode the ring's memory holds the partials: S x kBN / 4 x (128 / S + 1) x 16 bytes
  static constexpr int kRedBytes = kMaxSplit * (kBN / 4) * (kBM / kMaxSplit + 1) * 16;
  static constexpr int kRingBytes = kStages * kStageBytes > kRedBytes ? kStages * kStageBytes : kRedBytes;
  static constexpr uint32_t kTmemCols = 2 * kBN < 32 ? 32 : 2 * kBN;
};

template <int kBN>
struct Smem {
  uint8_t ring[Cfg<kBN>::kRingBytes];  // 1024-byte aligned stages: A rows, then B rows
  float ws[2][256];                    // w_scale and bias of the tile's channels (kSwap = false), or x_scale (kSwap)
  float bias[2][256];
  uint64_t full[Cfg<kBN>::kStages], empty[Cfg<kBN>::kStages], tfull[2], tempty[2], mma_done;
  uint32_t tmem_base;
  int abort;
};

template <int kBN>
constexpr size_t smem_bytes() { return sizeof(Smem<kBN>) + 1024; }

struct Part {
  int ta, tb;   // tiles along the MMA's M and N
  int kb;       // K blocks
  int S;        // CTAs per tile (cluster), 1: persistent
  int grid;
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

// A thread's row of a tile: kBN int32 columns of its TMEM lane -> scaled values of row m, columns n0 .. ; `drained` is
// called once when the accumulator has been read.
template <int kBN, typename F>
__device__ __forceinline__ void drain_rows(const Int8Args& a, uint32_t src, long long m, int n0, const float* ws,
                                           const float* bias, int vec, F drained) {
  const float sx = m < a.M ? a.x_scale[m] : 0.0f;
#pragma unroll 1
  for (int c = 0; c < kBN; c += 32) {
    uint32_t raw[32];
    tmem_ld_32x32b_x32(src + c, raw);
    if (c + 32 == kBN) drained();
    if (m >= a.M) continue;
    const int n = n0 + c;
    if (vec && n + 32 <= a.N) {
      float v[32];
#pragma unroll
      for (int j = 0; j < 32; ++j) v[j] = int8_value(a, static_cast<int>(raw[j]), sx, ws[c + j], bias[c + j]);
      if (a.y_f32) {
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
#pragma unroll
      for (int j = 0; j < 32; ++j)
        if (n + j < a.N) store1(a, m, n + j, int8_value(a, static_cast<int>(raw[j]), sx, ws[c + j], bias[c + j]));
    }
  }
}

template <int kBN, bool kSwap, bool kCluster>
__global__ void __launch_bounds__(kThreads, 1)
    int8_mm_tc_kernel(const __grid_constant__ CUtensorMap ta, const __grid_constant__ CUtensorMap tb, const Int8Args a,
                      const Part p, const int vec) {
  using C = Cfg<kBN>;
  constexpr int kStages = C::kStages;
  extern __shared__ uint8_t smem_raw[];
  Smem<kBN>& s = *reinterpret_cast<Smem<kBN>*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
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
    tma_prefetch_desc(&tb);
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
          mbar_arrive_expect_tx(&s.full[st], C::kStageBytes);
          tma_load_2d(dst, &ta, &s.full[st], kb * kBK, ia * kBM);
          tma_load_2d(dst + kBM * kBK, &tb, &s.full[st], kb * kBK, ib * kBN);
        }
      }
      for (int st = 0; st < kStages && st < i; ++st)  // the last copy issued into each stage has landed
        wait_drain(&s.full[st], static_cast<uint32_t>((i - 1 - st) / kStages) & 1u);
    }
  } else if (warp == 1) {
    if (lane == 0) {
      constexpr uint32_t idesc = umma_idesc_s8(kBM, kBN);
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
          const uint32_t ab = smem_addr(s.ring + st * C::kStageBytes), bb = ab + kBM * kBK;
#pragma unroll
          for (int kk = 0; kk < kBK / 32; ++kk)
            umma_i8(dacc, umma_desc_sw128(ab + 32 * kk), umma_desc_sw128(bb + 32 * kk), idesc, (kb > k0 || kk > 0) ? 1u : 0u);
          umma_commit(&s.empty[st]);
        }
        if (ok) umma_commit(&s.tfull[buf]);
      }
      umma_commit(&s.mma_done);
      wait_drain(&s.mma_done, 0);
    }
  } else if (!kCluster) {
    const int q = warp & 3, r = 32 * q + lane, et = threadIdx.x - 32 * kEpiWarp0;
    int it = 0;
    for (int t = t0; t < tiles; t += step, ++it) {
      const int buf = it & 1;
      int ia, ib;
      tile_of(p, t, ia, ib);
      if (kSwap) {
        for (int j = et; j < kBN; j += kEpiThreads) s.ws[buf][j] = ib * kBN + j < a.M ? a.x_scale[ib * kBN + j] : 0.0f;
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
    // one tile per cluster. The partials go through the ring's memory: every CTA's MMAs have read it ...
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
      int ia, ib;
      tile_of(p, t0, ia, ib);
      const int4* red = reinterpret_cast<const int4*>(s.ring);
      if (kSwap) {
        for (int i = threadIdx.x; i < L * kBN; i += kThreads) {
          const int ll = i % L, j = i / L, n = ia * kBM + rank * L + ll, m = ib * kBN + j;
          if (m >= a.M || n >= a.N) continue;
          int acc = 0;
          for (int src = 0; src < S; ++src)
            acc += reinterpret_cast<const int*>(red + (src * (kBN / 4) + j / 4) * (L + 1) + ll)[j & 3];
          store1(a, m, n, int8_value(a, acc, a.x_scale[m], int8_w_scale(a, n), int8_bias(a, n)));
        }
      } else {
        for (int i = threadIdx.x; i < L * (kBN / 4); i += kThreads) {
          const int c4 = i % (kBN / 4), ll = i / (kBN / 4), n = ib * kBN + 4 * c4;
          const long long m = static_cast<long long>(ia) * kBM + rank * L + ll;
          if (m >= a.M || n >= a.N) continue;
          int4 acc = make_int4(0, 0, 0, 0);
          for (int src = 0; src < S; ++src) {
            const int4 v = red[(src * (kBN / 4) + c4) * (L + 1) + ll];
            acc.x += v.x, acc.y += v.y, acc.z += v.z, acc.w += v.w;
          }
          const int* av = &acc.x;
          const float sx = a.x_scale[m];
          float v[4];
#pragma unroll
          for (int j = 0; j < 4; ++j)
            v[j] = n + j < a.N ? int8_value(a, av[j], sx, int8_w_scale(a, n + j), int8_bias(a, n + j)) : 0.0f;
          if (vec && n + 4 <= a.N) {
            if (a.y_f32)
              *reinterpret_cast<float4*>(static_cast<float*>(a.y) + m * a.ldy + n) = make_float4(v[0], v[1], v[2], v[3]);
            else
              *reinterpret_cast<uint2*>(static_cast<__nv_bfloat16*>(a.y) + m * a.ldy + n) =
                  make_uint2(pack2(v[0], v[1]), pack2(v[2], v[3]));
          } else {
#pragma unroll
            for (int j = 0; j < 4; ++j)
              if (n + j < a.N) store1(a, m, n + j, v[j]);
          }
        }
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

template <int kBN, bool kSwap, bool kCluster>
int launch(const Int8Args& a, const Part& p, cudaStream_t stream) {
  auto* kern = int8_mm_tc_kernel<kBN, kSwap, kCluster>;
  static bool ready[64] = {false};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64 || !ready[dev]) {
    const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                               static_cast<int>(smem_bytes<kBN>()));
    if (e != cudaSuccess) return fail(BP_ERR_CUDA, "cudaFuncSetAttribute(smem %zu): %s", smem_bytes<kBN>(), cudaGetErrorString(e));
    if (dev >= 0 && dev < 64) ready[dev] = true;
  }
  const int8_t* A = kSwap ? a.w : a.x;
  const int8_t* B = kSwap ? a.x : a.w;
  CUtensorMap ta, tb;
  int st = tc_encode_2d(&ta, CU_TENSOR_MAP_DATA_TYPE_UINT8, A, a.K, kSwap ? a.N : a.M, kSwap ? a.ldw : a.ldx, kBK, kBM,
                        CU_TENSOR_MAP_L2_PROMOTION_L2_256B);
  if (st != BP_OK) return st;
  st = tc_encode_2d(&tb, CU_TENSOR_MAP_DATA_TYPE_UINT8, B, a.K, kSwap ? a.M : a.N, kSwap ? a.ldx : a.ldw, kBK, kBN,
                    CU_TENSOR_MAP_L2_PROMOTION_L2_256B);
  if (st != BP_OK) return st;
  const int es = a.y_f32 ? 4 : 2;
  const int vec = reinterpret_cast<uintptr_t>(a.y) % 16 == 0 && (a.ldy * es) % 16 == 0;
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[2];
  cfg.gridDim = kCluster ? dim3(p.ta * p.tb, p.S) : dim3(p.grid);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem_bytes<kBN>();
  cfg.stream = stream;
  set_launch_attrs(cfg, attr, kCluster ? p.S : 1);
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kern, ta, tb, a, p, vec);
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
  p.grid = static_cast<int>(tiles < tc_sm_count() ? tiles : tc_sm_count());
  return p;
}

// Few tiles for the GPU: the CTAs of a cluster share a tile's K.
template <int kBN, bool kSwap>
int launch_split(const Int8Args& a, cudaStream_t stream) {
  Part p = partition<kBN, kSwap>(a);
  const int sms = tc_sm_count(), tiles = p.ta * p.tb;
  while (p.S < kMaxSplit && static_cast<long long>(tiles) * p.S * 2 <= sms && p.S * 2 <= p.kb) p.S *= 2;
  return p.S > 1 ? launch<kBN, kSwap, true>(a, p, stream) : launch<kBN, kSwap, false>(a, p, stream);
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

// vec: 0: y's rows are not 16-byte aligned; 1: they are (fp32); 2: bf16 through `ty`, a map of y in 64 x 128 boxes
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
          const uint32_t ab = smem_addr(s.ring + st * PairSmem::kStageBytes), bb = ab + kBM * kBK;
#pragma unroll
          for (int kk = 0; kk < kBK / 32; ++kk)
            umma_i8_pair(dacc, umma_desc_sw128(ab + 32 * kk), umma_desc_sw128(bb + 32 * kk), idesc,
                         (kb > 0 || kk > 0) ? 1u : 0u);
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
      if (vec != 2) {
        drain_rows<128>(a, src, static_cast<long long>(m0) + r, ib * kPairN + c0, s.ws[buf] + c0, s.bias[buf] + c0, vec, drained);
        continue;
      }
      const float sx = m0 + r < a.M ? a.x_scale[m0 + r] : 0.0f;
#pragma unroll 1
      for (int h = 0; h < 2; ++h) {
        if (et % 128 == 0) tma_store_wait<false>();  // the store before has read the buffer
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
        if (et % 128 == 0) {
          tma_store_2d(&ty, stage, ib * kPairN + c0 + h * 64, m0);
          tma_store_commit();
        }
      }
    }
    if (et % 128 == 0) tma_store_wait<true>();
  }
  tc_fence_before_sync();
  __syncthreads();
  cluster_sync_unaligned();  // the leader's MMAs have read the peer's memory, every copy has landed in both
  if (warp == 1) {
    tc_fence_after_sync();
    tmem_dealloc_pair(tmem, 512);
  }
}

int launch_pair(const Int8Args& a, cudaStream_t stream) {
  static bool ready[64] = {false};
  constexpr size_t smem = sizeof(PairSmem) + 1024;
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64 || !ready[dev]) {
    const cudaError_t e = cudaFuncSetAttribute(int8_mm_pair_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem));
    if (e != cudaSuccess) return fail(BP_ERR_CUDA, "cudaFuncSetAttribute(smem %zu): %s", smem, cudaGetErrorString(e));
    if (dev >= 0 && dev < 64) ready[dev] = true;
  }
  Part p;
  p.ta = (a.M + 2 * kBM - 1) / (2 * kBM);
  p.tb = (a.N + kPairN - 1) / kPairN;
  p.kb = (a.K + kBK - 1) / kBK;
  p.S = 1;
  const int pairs = tc_sm_count() / 2, tiles = p.ta * p.tb;
  p.grid = 2 * (tiles < pairs ? tiles : pairs);
  CUtensorMap ta, tb;
  int st = tc_encode_2d(&ta, CU_TENSOR_MAP_DATA_TYPE_UINT8, a.x, a.K, a.M, a.ldx, kBK, kBM, CU_TENSOR_MAP_L2_PROMOTION_L2_256B);
  if (st != BP_OK) return st;
  st = tc_encode_2d(&tb, CU_TENSOR_MAP_DATA_TYPE_UINT8, a.w, a.K, a.N, a.ldw, kBK, kBM, CU_TENSOR_MAP_L2_PROMOTION_L2_256B);
  if (st != BP_OK) return st;
  const int es = a.y_f32 ? 4 : 2;
  int vec = reinterpret_cast<uintptr_t>(a.y) % 16 == 0 && (a.ldy * es) % 16 == 0;
  CUtensorMap ty = ta;
  if (vec && !a.y_f32) {
    st = tc_encode_2d(&ty, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, a.y, a.N, a.M, a.ldy * 2, 64, kBM, CU_TENSOR_MAP_L2_PROMOTION_NONE);
    if (st != BP_OK) return st;
    vec = 2;
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
  if (a.M <= 16) return launch_split<16, true>(a, stream);
  if (a.M <= 32) return launch_split<32, true>(a, stream);
  if (a.M <= 64) return launch_split<64, true>(a, stream);
  const long long tiles = static_cast<long long>((a.M + kBM - 1) / kBM) * ((a.N + 255) / 256);
  if (tiles > (1 << 29)) return fail(BP_ERR_UNSUPPORTED, "int8_mm: too many tiles (M=%d N=%d)", a.M, a.N);
  if (tiles >= tc_sm_count()) return launch_pair(a, stream);
  return launch_split<128, false>(a, stream);
}

BP_DEFINE_DEVICE_ERROR_READER(read_device_errors_int8mm)

}  // namespace bp
