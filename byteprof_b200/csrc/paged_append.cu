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
// rotated pair sit in one thread (8 + 8 values). A thread requests its first kKeep pairs before it looks up where the
// row belongs and keeps them in registers until the two sums are known (6144 values a row; what is beyond is read a
// second time). 4099 rows of 32 + 2 x 8 heads of 128: 21.5 us for 101 MB, 4.7 TB/s; reading everything twice,
// behind the lookup, took 32. One row: 3.1 us, the lookup's and the row's latency.
#include "bp_common.cuh"

namespace bp {
namespace {

constexpr int kThreads = 128;
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

// Two fp32 values in a register pair, and arithmetic on both at once.
__device__ __forceinline__ uint64_t f32x2(float lo, float hi) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t wide(uint32_t w) { return f32x2(bf16lo(w), bf16hi(w)); }
__device__ __forceinline__ uint32_t narrow(uint64_t v) {
  const __nv_bfloat162 p = __floats2bfloat162_rn(__uint_as_float(static_cast<uint32_t>(v)), __uint_as_float(static_cast<uint32_t>(v >> 32)));
  return *reinterpret_cast<const uint32_t*>(&p);
}

// The 8 angles of a pair of chunks.
struct Angles {
  uint64_t c[4], s[4];
  __device__ __forceinline__ void load(const float* cs, const float* sn) {
    const float4 c0 = __ldg(reinterpret_cast<const float4*>(cs)), c1 = __ldg(reinterpret_cast<const float4*>(cs) + 1);
    const float4 s0 = __ldg(reinterpret_cast<const float4*>(sn)), s1 = __ldg(reinterpret_cast<const float4*>(sn) + 1);
    c[0] = f32x2(c0.x, c0.y), c[1] = f32x2(c0.z, c0.w), c[2] = f32x2(c1.x, c1.y), c[3] = f32x2(c1.z, c1.w);
    s[0] = f32x2(s0.x, s0.y), s[1] = f32x2(s0.z, s0.w), s[2] = f32x2(s1.x, s1.y), s[3] = f32x2(s1.z, s1.w);
  }
};

// One rotated pair of 8-value chunks (dims c..c+7 and c+hd/2..) of a head.
__device__ __forceinline__ void norm_rope8(const uint4 xa, const uint4 xb, const __nv_bfloat16* w, float inv, const Angles* ang,
                                           int half, __nv_bfloat16* y) {
  const uint32_t* pa = &xa.x;
  const uint32_t* pb = &xb.x;
  uint4 wa = make_uint4(0, 0, 0, 0), wb = wa, ya, yb;
  if (w != nullptr) {
    wa = ldg16(w);
    wb = ldg16(w + half);
  }
  const uint32_t* qa = &wa.x;
  const uint32_t* qb = &wb.x;
  uint32_t* ra = &ya.x;
  uint32_t* rb = &yb.x;
  const uint64_t inv2 = f32x2(inv, inv), minus = f32x2(-1.0f, -1.0f);
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    uint64_t a = wide(pa[j]), b = wide(pb[j]);
    if (w != nullptr) {
      a = mul2(mul2(a, inv2), wide(qa[j]));
      b = mul2(mul2(b, inv2), wide(qb[j]));
    }
    if (ang != nullptr) {
      const uint64_t p = fma2(mul2(b, ang->s[j]), minus, mul2(a, ang->c[j]));
      b = fma2(a, ang->s[j], mul2(b, ang->c[j]));
      a = p;
    }
    ra[j] = narrow(a);
    rb[j] = narrow(b);
  }
  *reinterpret_cast<uint4*>(y) = ya;
  *reinterpret_cast<uint4*>(y + half) = yb;
}

__device__ __forceinline__ uint64_t sum_sq8(const uint4 v, uint64_t acc) {
  const uint32_t* w = &v.x;
#pragma unroll
  for (int j = 0; j < 4; ++j) acc = fma2(wide(w[j]), wide(w[j]), acc);
  return acc;
}

constexpr int kKeep = 3;  // pairs that a thread keeps

template <int HD>
__global__ void __launch_bounds__(kThreads, 7) paged_append_kernel(const AppendArgs a) {
  __shared__ float red[2][kThreads / 32];
  pdl_launch_dependents();
  pdl_wait_prior_grids();
  const int t = blockIdx.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  constexpr int half = HD / 2, per = half / 8;  // pairs per head
  const int qn = a.nh * HD, kn = a.nkv * HD;
  const int nq = a.nh * per, nk = a.nkv * per, all = nq + 2 * nk;                   // pairs of q, k and (plain 16 values) v
  const __nv_bfloat16* x = a.qkv + static_cast<long long>(t) * a.ldqkv;
  // pair u: its first chunk's place in the row, and the second's distance
  auto place = [&](unsigned u) -> int { return u < static_cast<unsigned>(nq + nk) ? (u / per) * HD + u % per * 8 : qn + kn + (u - nq - nk) * 16; };
  auto apart = [&](unsigned u) { return u < static_cast<unsigned>(nq + nk) ? half : 8; };
  uint4 keep[kKeep][2];
#pragma unroll
  for (int i = 0; i < kKeep; ++i) {
    const int u = tid + i * kThreads;
    if (u < all) {
      keep[i][0] = ld16(x + place(u));
      keep[i][1] = ld16(x + place(u) + apart(u));
    }
  }
  // the row's sequence: the number of sequences that end at or before it
  int s = 0, first, end, len;
  if (a.seqs <= 32) {  // bounds and lengths in one go, a lane each
    const int mine = lane < a.seqs ? a.q_start[lane + 1] : 0x7fffffff, my_len = lane < a.seqs ? a.kv_len[lane] : 0;
    const int zero = a.q_start[0];
    s = __popc(__ballot_sync(kFull, mine <= t));
    if (s >= a.seqs) return;  // behind the last sequence
    end = __shfl_sync(kFull, mine, s);
    first = s == 0 ? zero : __shfl_sync(kFull, mine, s - 1);
    len = __shfl_sync(kFull, my_len, s);
  } else {
    for (int i = lane; i < a.seqs; i += 32) s += a.q_start[i + 1] <= t;
    s = __reduce_add_sync(kFull, s);
    if (s >= a.seqs) return;
    first = a.q_start[s];
    end = a.q_start[s + 1];
    len = a.kv_len[s];
  }
  if (t < first) return;
  const long long pos = static_cast<long long>(len) - (end - first) + (t - first);
  constexpr long long kMaxPos = 0x7fffff00;  // as far as the attention goes (paged.cuh)
  bool ok = pos >= 0 && pos < kMaxPos && (pos >> a.page_log2) < a.max_pages && (a.cos_t == nullptr || pos < a.max_pos);
  int page = -1;
  if (ok) page = a.pages[s * a.ld_pages + (pos >> a.page_log2)];
  ok = page >= 0 && page < a.num_pages;

  __nv_bfloat16* qo = a.q_out + static_cast<long long>(t) * a.ldq;
  if (!ok) {  // a position outside the tables or the cache: NaN, and no cache row is touched
    const uint4 nan4 = make_uint4(0x7fc07fc0u, 0x7fc07fc0u, 0x7fc07fc0u, 0x7fc07fc0u);
    for (int c = tid * 8; c < qn; c += kThreads * 8) *reinterpret_cast<uint4*>(qo + c) = nan4;
    return;
  }
  // a thread's pairs are all at the same dims of their heads (kThreads is a multiple of the pairs per head)
  static_assert(kThreads % per == 0, "angles");
  Angles ang;
  if (a.cos_t != nullptr) ang.load(a.cos_t + pos * half + tid % per * 8, a.sin_t + pos * half + tid % per * 8);
  float sq = 0.0f, sk = 0.0f;
  if (a.qw != nullptr) {
    uint64_t sq2 = 0, sk2 = 0;
    auto add = [&](int u, const uint4 c0, const uint4 c1) {
      if (u < nq)
        sq2 = sum_sq8(c1, sum_sq8(c0, sq2));
      else if (u < nq + nk)
        sk2 = sum_sq8(c1, sum_sq8(c0, sk2));
    };
#pragma unroll
    for (int i = 0; i < kKeep; ++i)
      if (tid + i * kThreads < all) add(tid + i * kThreads, keep[i][0], keep[i][1]);
    for (int u = tid + kKeep * kThreads; u < nq + nk; u += kThreads) add(u, ld16(x + place(u)), ld16(x + place(u) + half));
    sq = __uint_as_float(static_cast<uint32_t>(sq2)) + __uint_as_float(static_cast<uint32_t>(sq2 >> 32));
    sk = __uint_as_float(static_cast<uint32_t>(sk2)) + __uint_as_float(static_cast<uint32_t>(sk2 >> 32));
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
  }
  const float inv_q = 1.0f / sqrtf(sq / qn + a.eps), inv_k = 1.0f / sqrtf(sk / kn + a.eps);
  const long long row = (static_cast<long long>(page) << a.page_log2) + (pos & ((1 << a.page_log2) - 1));
  __nv_bfloat16* ko = a.kp + row * kn;
  __nv_bfloat16* vo = a.vp + row * kn;
  auto put = [&](int u, const uint4 c0, const uint4 c1) {
    if (u < nq + nk) {
      const bool is_q = u < nq;
      const int d = place(u) - (is_q ? 0 : qn);
      const __nv_bfloat16* w = is_q ? a.qw : a.kw;
      norm_rope8(c0, c1, w == nullptr ? nullptr : w + d, is_q ? inv_q : inv_k, a.cos_t == nullptr ? nullptr : &ang,
                 half, (is_q ? qo : ko) + d);
    } else {
      uint4* dst = reinterpret_cast<uint4*>(vo + (u - nq - nk) * 16);
      dst[0] = c0;
      dst[1] = c1;
    }
  };
#pragma unroll
  for (int i = 0; i < kKeep; ++i)
    if (tid + i * kThreads < all) put(tid + i * kThreads, keep[i][0], keep[i][1]);
  for (int u = tid + kKeep * kThreads; u < all; u += kThreads) put(u, ld16(x + place(u)), ld16(x + place(u) + apart(u)));
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
  if (qkv == nullptr || (pages == nullptr && max_pages > 0) || q_start == nullptr || kv_len == nullptr || k_pages == nullptr ||
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
  const cudaError_t e = head_dim == 128 ? cudaLaunchKernelEx(&cfg, paged_append_kernel<128>, a)
                                         : cudaLaunchKernelEx(&cfg, paged_append_kernel<64>, a);
  if (e != cudaSuccess) return fail(BP_ERR_CUDA, "paged_append launch: %s", cudaGetErrorString(e));
  return check_launch("paged_append");
}
