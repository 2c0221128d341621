// The paged cache's writer: q, k, v rows of new positions -> RMSNorm of q and k over their widths, rotary
// embedding, k and v into the cache's pages, q to its own tensor (bp_paged_append).
//
// Reference: GlobalStep.step writes one position at a time into a StaticCache (byteprof/optim/bolmo.py:
// 100-136); here any number of rows of any number of sequences go in one launch.
//
//   q' = rope(q * inv_q * wq), k' = rope(k * inv_k * wk), inv = 1 / sqrt(mean(x^2) + eps); fp32 until the one
//   rounding to bf16 of what is stored; v is copied.
//
// Memory bound: (nh + 2 nkv) head_dim values read and written once per row. One CTA per row: both halves of a
// rotated pair sit in one thread (8 + 8 values), the row is read a second time behind the two sums (from
// L1: a row is 12-24 KB).
#include "bp_common.cuh"

namespace bp {
namespace {

constexpr int kThreads = 256;
constexpr unsigned kFull = 0xffffffffu;

struct AppendArgs {
  const __nv_bfloat16* qkv;
  long long ldqkv;
  const __nv_bfloat16* qw;
  const __nv_bfloat16* kw;
  const float* cos_t;
  const float* sin_t;
  int max_pos;
  const int* pages;
  long long ld_pages;
  int max_pages;
  const int* q_start;
  const int* kv_len;
  int seqs;
  __nv_bfloat16* kp;
  __nv_bfloat16* vp;
  int num_pages, page_log2;
  int nh, nkv, hd;
  float eps;
  __nv_bfloat16* q_out;
  long long ldq;
};

__device__ __forceinline__ void unpack8(const uint4 v, float (&f)[8]) {
  f[0] = bf16lo(v.x); f[1] = bf16hi(v.x); f[2] = bf16lo(v.y); f[3] = bf16hi(v.y);
  f[4] = bf16lo(v.z); f[5] = bf16hi(v.z); f[6] = bf16lo(v.w); f[7] = bf16hi(v.w);
}

__device__ __forceinline__ uint4 pack8(const float (&f)[8]) {
  uint4 r;
  uint32_t* w = &r.x;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const __nv_bfloat162 p = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
    w[i] = *reinterpret_cast<const uint32_t*>(&p);
  }
  return r;
}

// One rotated pair of 8-value chunks (dims c..c+7 and c+hd/2..) of a head.
__device__ __forceinline__ void norm_rope8(const __nv_bfloat16* x, const __nv_bfloat16* w, float inv, const float* cs,
                                           const float* sn, int half, __nv_bfloat16* y) {
  float a[8], b[8];
  unpack8(*reinterpret_cast<const uint4*>(x), a);
  unpack8(*reinterpret_cast<const uint4*>(x + half), b);
  if (w != nullptr) {
    float wa[8], wb[8];
    unpack8(ldg16(w), wa);
    unpack8(ldg16(w + half), wb);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      a[j] = a[j] * inv * wa[j];
      b[j] = b[j] * inv * wb[j];
    }
  }
  if (cs != nullptr) {
    float c[8], s[8];
    *reinterpret_cast<uint4*>(c) = ldg16(cs);
    *reinterpret_cast<uint4*>(c + 4) = ldg16(cs + 4);
    *reinterpret_cast<uint4*>(s) = ldg16(sn);
    *reinterpret_cast<uint4*>(s + 4) = ldg16(sn + 4);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float p = a[j] * c[j] - b[j] * s[j];
      b[j] = b[j] * c[j] + a[j] * s[j];
      a[j] = p;
    }
  }
  *reinterpret_cast<uint4*>(y) = pack8(a);
  *reinterpret_cast<uint4*>(y + half) = pack8(b);
}

__device__ __forceinline__ float sum_sq8(const uint4 v, float acc) {
  float f[8];
  unpack8(v, f);
#pragma unroll
  for (int j = 0; j < 8; ++j) acc = fmaf(f[j], f[j], acc);
  return acc;
}

__global__ void __launch_bounds__(kThreads) paged_append_kernel(const AppendArgs a) {
  __shared__ float red[2][kThreads / 32];
  pdl_launch_dependents();
  pdl_wait_prior_grids();
  const int t = blockIdx.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  // the row's sequence: the number of sequences that end at or before it
  int s = 0;
  for (int i = lane; i < a.seqs; i += 32) s += a.q_start[i + 1] <= t;
  s = __reduce_add_sync(kFull, s);
  if (s >= a.seqs) return;  // behind the last sequence
  const int first = a.q_start[s], end = a.q_start[s + 1];
  if (t < first) return;
  const long long pos = static_cast<long long>(a.kv_len[s]) - (end - first) + (t - first);
  bool ok = pos >= 0 && (pos >> a.page_log2) < a.max_pages && (a.cos_t == nullptr || pos < a.max_pos);
  int page = -1;
  if (ok) page = a.pages[s * a.ld_pages + (pos >> a.page_log2)];
  ok = page >= 0 && page < a.num_pages;

  const int half = a.hd / 2, qn = a.nh * a.hd, kn = a.nkv * a.hd, per = half / 8;  // chunk pairs per head
  const __nv_bfloat16* x = a.qkv + static_cast<long long>(t) * a.ldqkv;
  __nv_bfloat16* qo = a.q_out + static_cast<long long>(t) * a.ldq;
  if (!ok) {  // a position outside the tables or the cache: NaN, and no cache row is touched
    const uint4 nan4 = make_uint4(0x7fc07fc0u, 0x7fc07fc0u, 0x7fc07fc0u, 0x7fc07fc0u);
    for (int c = tid * 8; c < qn; c += kThreads * 8) *reinterpret_cast<uint4*>(qo + c) = nan4;
    return;
  }
  float sq = 0.0f, sk = 0.0f;
  if (a.qw != nullptr)
    for (int c = tid * 8; c < qn; c += kThreads * 8) sq = sum_sq8(*reinterpret_cast<const uint4*>(x + c), sq);
  if (a.kw != nullptr)
    for (int c = tid * 8; c < kn; c += kThreads * 8) sk = sum_sq8(*reinterpret_cast<const uint4*>(x + qn + c), sk);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    sq += __shfl_xor_sync(kFull, sq, o);
    sk += __shfl_xor_sync(kFull, sk, o);
  }
  if (lane == 0) {
    red[0][warp] = sq;
    red[1][warp] = sk;
  }
  __syncthreads();
  sq = sk = 0.0f;
#pragma unroll
  for (int w = 0; w < kThreads / 32; ++w) {
    sq += red[0][w];
    sk += red[1][w];
  }
  const float inv_q = 1.0f / sqrtf(sq / qn + a.eps), inv_k = 1.0f / sqrtf(sk / kn + a.eps);
  const long long row = (static_cast<long long>(page) << a.page_log2) + (pos & ((1 << a.page_log2) - 1));
  __nv_bfloat16* ko = a.kp + row * kn;
  __nv_bfloat16* vo = a.vp + row * kn;
  const float* cs = a.cos_t == nullptr ? nullptr : a.cos_t + pos * half;
  const float* sn = a.cos_t == nullptr ? nullptr : a.sin_t + pos * half;
  const int nq = a.nh * per, nk = a.nkv * per;
  for (int u = tid; u < nq + 2 * nk; u += kThreads) {
    if (u < nq + nk) {
      const bool is_q = u < nq;
      const int v = is_q ? u : u - nq;
      const int c = (v % per) * 8, d = (v / per) * a.hd + c;
      const __nv_bfloat16* w = is_q ? a.qw : a.kw;
      norm_rope8(x + (is_q ? 0 : qn) + d, w == nullptr ? nullptr : w + d, is_q ? inv_q : inv_k,
                 cs == nullptr ? nullptr : cs + c, cs == nullptr ? nullptr : sn + c, half, (is_q ? qo : ko) + d);
    } else {
      const int d = (u - nq - nk) * 16;
      const uint4* src = reinterpret_cast<const uint4*>(x + qn + kn + d);
      uint4* dst = reinterpret_cast<uint4*>(vo + d);
      const uint4 v0 = src[0], v1 = src[1];
      dst[0] = v0;
      dst[1] = v1;
    }
  }
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

}  // namespace
}  // namespace bp

extern "C" int bp_paged_append(const void* qkv, long long ldqkv, const void* q_norm_w, const void* k_norm_w,
                               const float* cos_t, const float* sin_t, int max_pos, const int32_t* pages,
                               long long ld_pages, int max_pages, const int32_t* q_start, const int32_t* kv_len,
                               int seqs, int rows, void* k_pages, void* v_pages, int num_pages, int page_size, int nh,
                               int nkv, int head_dim, float eps, void* q_out, long long ldq, void* stream) {
  using namespace bp;
  clear_error();
  if (seqs < 0 || rows < 0 || num_pages < 0 || max_pages < 0)
    return fail(BP_ERR_INVALID_ARGUMENT, "negative size (seqs=%d rows=%d num_pages=%d max_pages=%d)", seqs, rows,
                num_pages, max_pages);
  if (nkv < 1 || nh < nkv || nh % nkv != 0 || nh > 1024)
    return fail(BP_ERR_INVALID_ARGUMENT, "nh=%d must be a multiple of nkv=%d (at most 1024 heads)", nh, nkv);
  if (head_dim != 64 && head_dim != 128)
    return fail(BP_ERR_UNSUPPORTED, "the paged cache supports head_dim 64 and 128 (got %d)", head_dim);
  if (page_size < 8 || page_size > 256 || (page_size & (page_size - 1)) != 0)
    return fail(BP_ERR_UNSUPPORTED, "page_size must be a power of two from 8 to 256 (got %d)", page_size);
  if (rows == 0 || seqs == 0) return BP_OK;
  if (qkv == nullptr || pages == nullptr || q_start == nullptr || kv_len == nullptr || k_pages == nullptr ||
      v_pages == nullptr || q_out == nullptr || (cos_t == nullptr) != (sin_t == nullptr) ||
      (q_norm_w == nullptr) != (k_norm_w == nullptr))
    return fail(BP_ERR_INVALID_ARGUMENT, "a pointer is NULL (cos_t / sin_t and the norm weights: both or neither)");
  if (ldqkv < static_cast<long long>(nh + 2 * nkv) * head_dim || ldq < static_cast<long long>(nh) * head_dim ||
      ld_pages < max_pages)
    return fail(BP_ERR_INVALID_ARGUMENT, "row strides must cover a row of qkv, of q_out and of the page table");
  if (!aligned16(qkv) || !aligned16(q_out) || !aligned16(k_pages) || !aligned16(v_pages) || !aligned16(q_norm_w) ||
      !aligned16(k_norm_w) || !aligned16(cos_t) || !aligned16(sin_t) || ldqkv % 8 != 0 || ldq % 8 != 0)
    return fail(BP_ERR_MISALIGNED, "paged_append needs 16-byte aligned bases and row strides multiples of 8");
  int st = require_sm100();
  if (st != BP_OK) return st;
  int lg = 3;
  while ((1 << lg) < page_size) ++lg;
  AppendArgs a{static_cast<const __nv_bfloat16*>(qkv), ldqkv, static_cast<const __nv_bfloat16*>(q_norm_w),
               static_cast<const __nv_bfloat16*>(k_norm_w), cos_t, sin_t, max_pos, pages, ld_pages, max_pages, q_start,
               kv_len, seqs, static_cast<__nv_bfloat16*>(k_pages), static_cast<__nv_bfloat16*>(v_pages), num_pages, lg,
               nh, nkv, head_dim, eps, static_cast<__nv_bfloat16*>(q_out), ldq};
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[2];
  cfg.gridDim = dim3(rows);
  cfg.blockDim = dim3(kThreads);
  cfg.stream = static_cast<cudaStream_t>(stream);
  set_launch_attrs(cfg, attr);
  const cudaError_t e = cudaLaunchKernelEx(&cfg, paged_append_kernel, a);
  if (e != cudaSuccess) return fail(BP_ERR_CUDA, "paged_append launch: %s", cudaGetErrorString(e));
  return check_launch("paged_append");
}
