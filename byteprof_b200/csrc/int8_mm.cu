// Product in 8-bit integers with a scale for each token and channel: the rows' quantizer
// (bp_quantize_rows_int8), the entry point of the product (bp_int8_mm) and the CUDA-core kernel for operands the
// tensor-core kernel (int8_mm_tc.cu) cannot load.
//
// Reference: Int8Linear at more than one row dequantizes its weights and calls F.linear
// (byteprof/quant/integrate.py:40-49); byteprof has no product of quantized activations.
//
//   s_m = max(max_k |x_mk| / 127, 1e-12), q_mk = rint(x_mk / s_m);  y_mn = s_m * ws_n * sum_k q_mk w_nk (+ bias_n).
// The sum is exact (int32: 131071 products of -128 and -128 fit); the division is correctly rounded, so every implementation that does
// the same gets the same integers. A row holding Inf or NaN gets a NaN scale (and so a NaN row of y).
#include "bp_common.cuh"
#include "int8_mm.h"
#include "skinny_internal.h"

namespace bp {
namespace {

constexpr unsigned kFull = 0xffffffffu;

// ---- quantizer ------------------------------------------------------------------------------------------
// A team of threads per row: one warp up to 2048 values (8 rows per CTA and no barrier: with a CTA per row the
// barrier and the single load in flight per thread held 8192 x 2048 at 23 us), else the CTA. Each thread keeps up to 8
// chunks of 8 values in registers between the maximum and the rounding.
constexpr int kQThreads = 256;
constexpr int kQCache = 8;

template <int kTeam>
__device__ __forceinline__ uint32_t team_max(uint32_t m, uint32_t* red) {
  m = __reduce_max_sync(kFull, m);
  if (kTeam > 32) {
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = m;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kQThreads / 32; ++w) m = max(m, red[w]);
  }
  return m;
}

// kVec: rows are 16-byte aligned and K a multiple of 8 (q rows 8-byte aligned).
template <bool kVec, int kTeam>
__global__ void __launch_bounds__(kQThreads) quantize_rows_kernel(const __nv_bfloat16* x, long long ldx, int8_t* q,
                                                                  long long ldq, float* scale, int M, int K) {
  __shared__ uint32_t red[kQThreads / 32];
  pdl_launch_dependents();
  pdl_wait_prior_grids();
  const int tid = threadIdx.x % kTeam, row = blockIdx.x * (kQThreads / kTeam) + threadIdx.x / kTeam;
  if (row >= M) return;  // whole teams
  const __nv_bfloat16* xr = x + row * ldx;
  int8_t* qr = q + row * ldq;
  const int chunks = K / 8;
  uint32_t m = 0;
  uint4 keep[kQCache];
  if (kVec) {
#pragma unroll
    for (int i = 0; i < kQCache; ++i) {
      const int c = tid + i * kTeam;
      keep[i] = c < chunks ? ld16(xr + c * 8) : make_uint4(0, 0, 0, 0);
    }
#pragma unroll
    for (int i = 0; i < kQCache; ++i) m = abs_max8(keep[i], m);
    for (int c = tid + kQCache * kTeam; c < chunks; c += kTeam) m = abs_max8(ld16(xr + c * 8), m);
  } else {
    for (int k = tid; k < K; k += kTeam) m = max(m, __float_as_uint(__bfloat162float(xr[k])) & 0x7fffffffu);
  }
  m = team_max<kTeam>(m, red);
  const bool bad = m >= 0x7f800000u;
  const float s = int8_row_scale(m);
  const float inv = 1.0f / s;
  if (tid == 0) scale[row] = bad ? __uint_as_float(0x7fc00000u) : s;
  if (kVec) {
#pragma unroll
    for (int i = 0; i < kQCache; ++i) {
      const int c = tid + i * kTeam;
      if (c < chunks) *reinterpret_cast<uint2*>(qr + c * 8) = bad ? make_uint2(0, 0) : q8(keep[i], s, inv);
    }
    for (int c = tid + kQCache * kTeam; c < chunks; c += kTeam)
      *reinterpret_cast<uint2*>(qr + c * 8) = bad ? make_uint2(0, 0) : q8(ld16(xr + c * 8), s, inv);
  } else {
    for (int k = tid; k < K; k += kTeam) qr[k] = bad ? 0 : static_cast<int8_t>(q1(__bfloat162float(xr[k]), s, inv));
  }
}

// ---- the CUDA-core product: any alignment, any K --------------------------------------------------------
constexpr int kT = 64;      // rows and channels per CTA
constexpr int kKB = 64;     // K per step
constexpr int kLd = kKB / 4 + 1;

// Bytes k .. k + 3 of a row (zero past K).
__device__ __forceinline__ int load4(const int8_t* row, int k, int K) {
  int v = 0;
#pragma unroll
  for (int j = 0; j < 4; ++j)
    if (k + j < K) v |= (static_cast<int>(row[k + j]) & 0xff) << (8 * j);
  return v;
}

__global__ void __launch_bounds__(256) int8_mm_dp4a_kernel(const Int8Args a) {
  __shared__ int xs[kT][kLd], ws[kT][kLd];
  pdl_launch_dependents();
  pdl_wait_prior_grids();
  const int tid = threadIdx.x, tx = tid % 16, ty = tid / 16;
  const int n0 = blockIdx.x * kT;
  for (long long m0 = static_cast<long long>(blockIdx.y) * kT; m0 < a.M; m0 += static_cast<long long>(gridDim.y) * kT) {
    int acc[4][4] = {};
    for (int k0 = 0; k0 < a.K; k0 += kKB) {
      for (int i = tid; i < kT * (kKB / 4); i += 256) {
        const int r = i / (kKB / 4), c = i % (kKB / 4);
        xs[r][c] = m0 + r < a.M ? load4(a.x + (m0 + r) * a.ldx, k0 + 4 * c, a.K) : 0;
        ws[r][c] = n0 + r < a.N ? load4(a.w + static_cast<long long>(n0 + r) * a.ldw, k0 + 4 * c, a.K) : 0;
      }
      __syncthreads();
#pragma unroll
      for (int c = 0; c < kKB / 4; ++c) {
        int xv[4], wv[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          xv[i] = xs[ty + 16 * i][c];
          wv[i] = ws[tx + 16 * i][c];
        }
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int j = 0; j < 4; ++j) acc[i][j] = __dp4a(xv[i], wv[j], acc[i][j]);
      }
      __syncthreads();
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const long long m = m0 + ty + 16 * i;
      if (m >= a.M) continue;
      const float sx = a.x_scale[m];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int n = n0 + tx + 16 * j;
        if (n >= a.N) continue;
        const float v = int8_value(a, acc[i][j], sx, int8_w_scale(a, n), int8_bias(a, n));
        if (a.y_f32)
          static_cast<float*>(a.y)[m * a.ldy + n] = v;
        else
          static_cast<__nv_bfloat16*>(a.y)[m * a.ldy + n] = __float2bfloat16_rn(v);
      }
    }
  }
}

bool aligned(const void* p, uintptr_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

// The product's argument checks (before any device work for empty problems); x is int8 or, fused, bf16.
int check_mm(const void* x, uintptr_t x_align, long long ldx, const void* x_scale, const int8_t* w, long long ldw,
             const void* w_scale, int w_scale_dtype, const void* bias, const void* y, long long ldy, int y_dtype, int M, int N,
             int K) {
  if (M < 0 || N < 0 || K < 0) return fail(BP_ERR_INVALID_ARGUMENT, "negative size (M=%d N=%d K=%d)", M, N, K);
  if (y_dtype != BP_DTYPE_BF16 && y_dtype != BP_DTYPE_F32)
    return fail(BP_ERR_INVALID_ARGUMENT, "output dtype %d is not bf16 or fp32", y_dtype);
  if (w_scale_dtype != BP_DTYPE_BF16 && w_scale_dtype != BP_DTYPE_F32)
    return fail(BP_ERR_INVALID_ARGUMENT, "weight-scale dtype %d is not bf16 or fp32", w_scale_dtype);
  if (M == 0 || N == 0) return BP_OK;
  if (y == nullptr || x_scale == nullptr || w_scale == nullptr || (K > 0 && (x == nullptr || w == nullptr)))
    return fail(BP_ERR_INVALID_ARGUMENT, "a pointer argument is NULL");
  if (ldx < K || ldw < K || ldy < N) return fail(BP_ERR_INVALID_ARGUMENT, "row strides must cover a row");
  if (K > 131071) return fail(BP_ERR_UNSUPPORTED, "K = %d: the int32 sums hold K up to 131071", K);
  if (!aligned(x, x_align) || !aligned(y, y_dtype == BP_DTYPE_F32 ? 4 : 2) || !aligned(x_scale, 4) ||
      !aligned(w_scale, w_scale_dtype == BP_DTYPE_F32 ? 4 : 2) || !aligned(bias, 2))
    return fail(BP_ERR_MISALIGNED, "y, the scales and bias need their elements' alignment");
  return require_sm100();
}

}  // namespace
}  // namespace bp

extern "C" int bp_quantize_rows_int8(const void* x, long long ldx, int8_t* q, long long ldq, float* scale, int M, int K,
                                     void* stream) {
  using namespace bp;
  clear_error();
  if (M < 0 || K < 0) return fail(BP_ERR_INVALID_ARGUMENT, "negative size (M=%d K=%d)", M, K);
  if (M == 0) return BP_OK;
  if (scale == nullptr || (K > 0 && (x == nullptr || q == nullptr)))
    return fail(BP_ERR_INVALID_ARGUMENT, "x, q or scale is NULL");
  if (ldx < K || ldq < K) return fail(BP_ERR_INVALID_ARGUMENT, "row strides must be >= K");
  if (!aligned(x, 2) || !aligned(scale, 4)) return fail(BP_ERR_MISALIGNED, "x and scale need their elements' alignment");
  int st = require_sm100();
  if (st != BP_OK) return st;
  const bool vec = K % 8 == 0 && ldx % 8 == 0 && ldq % 8 == 0 && aligned(x, 16) && aligned(q, 8);
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[2];
  const bool warp_rows = K <= 2048;
  cfg.gridDim = dim3(warp_rows ? (M + kQThreads / 32 - 1) / (kQThreads / 32) : M);
  cfg.blockDim = dim3(kQThreads);
  cfg.stream = static_cast<cudaStream_t>(stream);
  set_launch_attrs(cfg, attr);
  const cudaError_t e = cudaLaunchKernelEx(&cfg,
                                           vec ? (warp_rows ? quantize_rows_kernel<true, 32> : quantize_rows_kernel<true, kQThreads>)
                                               : (warp_rows ? quantize_rows_kernel<false, 32> : quantize_rows_kernel<false, kQThreads>),
                                           static_cast<const __nv_bfloat16*>(x), ldx, q, ldq, scale, M, K);
  if (e != cudaSuccess) return fail(BP_ERR_CUDA, "quantize_rows_int8 launch: %s", cudaGetErrorString(e));
  return check_launch("quantize_rows_int8");
}

extern "C" size_t bp_int8_linear_workspace_bytes(int M, int K) {
  if (M <= 0 || K < 0) return 0;
  return (static_cast<size_t>(M) * 4 + 255) / 256 * 256 + static_cast<size_t>(M) * ((static_cast<size_t>(K) + 15) / 16 * 16);
}

extern "C" int bp_int8_linear(const void* x, long long ldx, const int8_t* w, long long ldw, const void* w_scale,
                              int w_scale_dtype, const void* bias, void* y, long long ldy, int y_dtype, int M, int N,
                              int K, void* workspace, size_t workspace_bytes, void* stream) {
  using namespace bp;
  clear_error();
  if (M > 0 && K >= 0) {
    const size_t need = bp_int8_linear_workspace_bytes(M, K);
    if (workspace == nullptr || workspace_bytes < need)
      return fail(BP_ERR_INVALID_ARGUMENT, "int8_linear needs a workspace of %zu bytes (got %zu)", need, workspace_bytes);
    if (!aligned(workspace, 256)) return fail(BP_ERR_MISALIGNED, "workspace must be 256-byte aligned");
  }
  if (M > 0 && N > 0 && K > 0) {
    const Int8Args a{nullptr, 0, nullptr, w, ldw, w_scale, w_scale_dtype == BP_DTYPE_F32,
                     static_cast<const __nv_bfloat16*>(bias), y, ldy, y_dtype == BP_DTYPE_F32, M, N, K};
    if (int8_fused_supported(a, x, ldx)) {
      int st = check_mm(x, 16, ldx, workspace, w, ldw, w_scale, w_scale_dtype, bias, y, ldy, y_dtype, M, N, K);
      if (st != BP_OK) return st;
      st = launch_int8_fused(a, static_cast<const __nv_bfloat16*>(x), ldx, static_cast<cudaStream_t>(stream));
      return st != BP_OK ? st : check_launch("int8_linear");
    }
  }
  const long long ldq = (static_cast<long long>(K) + 15) / 16 * 16;
  float* scale = static_cast<float*>(workspace);
  int8_t* q = static_cast<int8_t*>(workspace) + (static_cast<size_t>(M > 0 ? M : 0) * 4 + 255) / 256 * 256;
  const int st = bp_quantize_rows_int8(x, ldx, q, ldq, scale, M, K, stream);
  if (st != BP_OK) return st;
  return bp_int8_mm(q, ldq, scale, w, ldw, w_scale, w_scale_dtype, bias, y, ldy, y_dtype, M, N, K, stream);
}

extern "C" int bp_int8_mm(const int8_t* x, long long ldx, const float* x_scale, const int8_t* w, long long ldw,
                          const void* w_scale, int w_scale_dtype, const void* bias, void* y, long long ldy, int y_dtype,
                          int M, int N, int K, void* stream) {
  using namespace bp;
  clear_error();
  int st = check_mm(x, 1, ldx, x_scale, w, ldw, w_scale, w_scale_dtype, bias, y, ldy, y_dtype, M, N, K);
  if (st != BP_OK) return st;
  if (M == 0 || N == 0) return BP_OK;
  const Int8Args a{x, ldx, x_scale, w, ldw, w_scale, w_scale_dtype == BP_DTYPE_F32, static_cast<const __nv_bfloat16*>(bias),
                   y, ldy, y_dtype == BP_DTYPE_F32, M, N, K};
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (int8_mm_tc_supported(a)) {
    st = launch_int8_mm_tc(a, s);
    return st != BP_OK ? st : check_launch("int8_mm");
  }
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[2];
  const int my = (M + kT - 1) / kT;
  cfg.gridDim = dim3((N + kT - 1) / kT, my < 65535 ? my : 65535);
  cfg.blockDim = dim3(256);
  cfg.stream = s;
  set_launch_attrs(cfg, attr);
  const cudaError_t e = cudaLaunchKernelEx(&cfg, int8_mm_dp4a_kernel, a);
  if (e != cudaSuccess) return fail(BP_ERR_CUDA, "int8_mm launch (M=%d N=%d K=%d): %s", M, N, K, cudaGetErrorString(e));
  return check_launch("int8_mm");
}
