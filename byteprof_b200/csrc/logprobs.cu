// Log probabilities of given tokens with the entropy of each row and its top alternatives, in one pass over
// the logits (bp_token_logprobs).
//
// Reference: byteprof's bits-per-byte evaluation takes log_softmax of every row and gathers the given byte
// (byteprof/evaluate.py:122-166), several passes over [rows, vocab].
//
//   m = max x, R = sum over all but one instance of the maximum of exp(x - m), T = sum exp(x - m) (m - x):
//   lse = m + log1p(R), logprob = x_id - lse, entropy = log1p(R) + T / (1 + R).
// R leaves the maximum's own term (1) out, so a row whose probability is all on one token keeps the small
// rest that 1 + R would round away. A thread sets its largest value so far aside without a branch: of (largest,
// new value) the smaller one goes into the sums, taken relative to a reference that moves only when the largest
// exceeds it by kLazy. (Moving it with every new maximum costs a rescale whenever any of 32 lanes has one, which is
// at nearly every vector of a row.) Two parts merge as (m1 >= m2, f = exp(m2 - m1)):
//   R = R1 + f (1 + R2), T = T1 + f (T2 + (m1 - m2)(1 + R2)).
// All of it in fp32, over short chains (a thread's share).
//
// Top alternatives: of 32 groups of threads the largest value that each saw is sorted; the `top`-th of them is a lower
// bound of the row's `top`-th value. The few threads that saw anything of that size (about `top`) have their share read
// once more, by a whole warp each; what reaches the bound goes into the warp's buffer as 64-bit keys (value, then lower
// index), and 32 keys are sorted and merged at once (20 steps of a bitonic network). So the pass over the logits carries
// nothing for them but the maximum that it has anyway. (Comparing every vector with a bound taken from the first 8192
// values cost 27 us of 94 for 1500 rows of 100352 with 5 alternatives, since some 60 values of a row reach it.)
//
// Bound by the instructions of the pass (about 14 per pair of values, two of them exp2, which alone take 35 us) and by
// memory: 1500 rows of 100352 in bf16 take 58 to 60 us (5.1 TB/s), 69 to 76 us with 5 alternatives; one row on a cluster of 8
// CTAs 4.8, with 5 alternatives 8.2 and with 20 10.3 to 13 us. Where the bound says nothing (fewer values above -inf than
// alternatives, or equal values throughout) every value is offered: one row 69 us, 1500 rows 570. A row goes to a warp, a CTA
// or a cluster of up to 8 CTAs (launch), merged in a fixed order (deterministic).
#include <float.h>

#include "bp_common.cuh"
#include "skinny_internal.h"
#include "sm100.cuh"

namespace bp {
namespace {

constexpr unsigned kFull = 0xffffffffu;
constexpr float kLog2e = 1.4426950408889634f;
constexpr int kMaxTop = 32;
constexpr int kWarpRowThreads = 256;  // 8 rows per CTA
constexpr int kMaxCluster = 8;

__device__ __forceinline__ float ex2(float v) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float min_nan(float a, float b) {
  float r;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

__device__ __forceinline__ uint32_t max_nan2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
__device__ __forceinline__ uint32_t min_nan2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("min.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
// Two fp32 values in a register pair, and arithmetic on both at once.
__device__ __forceinline__ uint64_t f32x2(float lo, float hi) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ float x2_lo(uint64_t v) { return __uint_as_float(static_cast<uint32_t>(v)); }
__device__ __forceinline__ float x2_hi(uint64_t v) { return __uint_as_float(static_cast<uint32_t>(v >> 32)); }
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
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}

constexpr float kLazy = 4.0f;

// The largest values so far of a thread's even and odd elements, set aside; `swap` returns what goes into the sums.
template <typename T>
struct Aside;
template <>
struct Aside<float> {
  float a = -INFINITY, b = -INFINITY;
  __device__ __forceinline__ uint64_t swap(float x, float y) {
    const uint64_t lo = f32x2(min_nan(a, x), min_nan(b, y));
    a = max_nan(a, x);
    b = max_nan(b, y);
    return lo;
  }
  __device__ __forceinline__ float even() const { return a; }
  __device__ __forceinline__ float odd() const { return b; }
  __device__ __forceinline__ float largest() const { return fmaxf(a, b); }
};
template <>
struct Aside<__nv_bfloat16> {
  uint32_t p = 0xff80ff80u;
  __device__ __forceinline__ uint64_t swap(uint32_t w) {
    const uint32_t lo = min_nan2(p, w);
    p = max_nan2(p, w);
    return f32x2(bf16lo(lo), bf16hi(lo));
  }
  __device__ __forceinline__ float even() const { return bf16lo(p); }
  __device__ __forceinline__ float odd() const { return bf16hi(p); }
  __device__ __forceinline__ float largest() const { return fmaxf(bf16lo(p), bf16hi(p)); }
};

// A thread's running sums over what is not set aside, even and odd elements apart: s = sum exp(x - ref),
// t = sum exp(x - ref)(ref - x).
template <typename T>
struct Run {
  Aside<T> top;
  float ref = -FLT_MAX;
  uint64_t s = 0, t = 0;
  __device__ __forceinline__ void add(uint64_t lo) {
    const uint64_t d = fma2(lo, f32x2(-1.0f, -1.0f), f32x2(ref, ref)), y = mul2(d, f32x2(-kLog2e, -kLog2e));
    const uint64_t e = f32x2(ex2(x2_lo(y)), ex2(x2_hi(y)));
    s = add2(s, e);
    t = fma2(e, f32x2(fminf(x2_lo(d), 1e30f), fminf(x2_hi(d), 1e30f)), t);  // -inf: e = 0, and 0 * inf would be NaN
  }
  // before values up to vm are added
  __device__ __forceinline__ void make_room(float vm) {
    if (vm > ref + kLazy) move(vm);
  }
  __device__ __forceinline__ void move(float to) {
    const float f = ex2((ref - to) * kLog2e);
    const uint64_t f2 = f32x2(f, f);
    t = f == 0.0f ? 0 : mul2(fma2(s, f32x2(to - ref, to - ref), t), f2);
    s = mul2(s, f2);
    ref = to;
  }
};

// A finished part: R and T as above, relative to m; m = -inf: nothing, NaN: a NaN was seen.
struct Stat {
  float m, r, t;
  template <typename T>
  __device__ __forceinline__ void from(Run<T> a) {
    const float e = a.top.even(), o = a.top.odd();
    const float mx = fmaxf(e, o);
    r = t = 0.0f;
    if (mx > -INFINITY) a.move(mx);  // both sums relative to the larger of the two set aside
    const float lo = fminf(e, o), f = mx > -INFINITY && lo > -INFINITY ? ex2((lo - mx) * kLog2e) : 0.0f;
    m = max_nan(e, o);
    if (mx > -INFINITY) {
      r = x2_lo(a.s) + x2_hi(a.s) + f;  // the smaller one joins the rest
      t = x2_lo(a.t) + x2_hi(a.t) + (f > 0.0f ? f * (mx - lo) : 0.0f);
    }
  }
  __device__ __forceinline__ void merge(float m2, float r2, float t2) {
    if (m2 > m) {
      const float a = m, b = r, c = t;
      m = m2, r = r2, t = t2;
      m2 = a, r2 = b, t2 = c;
    }
    const float f = m2 == m ? (m2 > -INFINITY ? 1.0f : 0.0f) : ex2((m2 - m) * kLog2e);
    if (f > 0.0f) {
      r += f * (1.0f + r2);
      t += f * (t2 + (m - m2) * (1.0f + r2));
    }
    m = max_nan(m, m2);
  }
};

// ---- top alternatives -------------------------------------------------------------------------------------
// Keys in torch's order: NaN is the largest value, the lower index wins among equals (and -0 equals 0). 0: none.
__device__ __forceinline__ uint32_t ordered(float x) {
  x += 0.0f;
  const uint32_t u = __float_as_uint(x);
  return isnan(x) ? 0xffffffffu : u ^ (static_cast<int>(u) < 0 ? 0xffffffffu : 0x80000000u);
}
__device__ __forceinline__ float from_ordered(uint32_t o) { return __uint_as_float(o & 0x80000000u ? o ^ 0x80000000u : ~o); }
__device__ __forceinline__ unsigned long long key_of(float x, int i) {
  return static_cast<unsigned long long>(ordered(x)) << 32 | ~static_cast<uint32_t>(i);
}
__device__ __forceinline__ float key_value(unsigned long long k) { return from_ordered(static_cast<uint32_t>(k >> 32)); }
__device__ __forceinline__ int key_index(unsigned long long k) { return static_cast<int>(~static_cast<uint32_t>(k)); }

// (K: 64-bit keys, or the ordered values alone)
template <typename K>
__device__ __forceinline__ K exchange(K k, int lane, int stride, bool down) {
  const K o = __shfl_xor_sync(kFull, k, stride);
  return ((lane & stride) == 0) == down ? (k > o ? k : o) : (k < o ? k : o);
}
// The larger 32 of two lists sorted downwards across the lanes, sorted.
template <typename K>
__device__ __forceinline__ K merge_sorted(K a, K b, int lane) {
  const K r = __shfl_sync(kFull, b, 31 - lane);
  K k = a > r ? a : r;
#pragma unroll
  for (int s = 16; s > 0; s >>= 1) k = exchange(k, lane, s, true);
  return k;
}
template <typename K>
__device__ __forceinline__ K sort_down(K k, int lane) {
#pragma unroll
  for (int size = 2; size <= 32; size <<= 1)
#pragma unroll
    for (int s = size >> 1; s > 0; s >>= 1) k = exchange(k, lane, s, (lane & size) == 0 || size == 32);
  return k;
}

constexpr int kBuf = 64;  // a warp's candidates: up to 31 waiting and 32 more
// A warp's alternatives, in shared memory (they are touched a few times per row).
struct TopList {
  unsigned long long list[32];  // the best so far, sorted; used when `sorted`
  unsigned long long buf[kBuf];
  unsigned long long thr;       // the last wanted entry
  int waiting, sorted;
  __device__ __forceinline__ void init(int lane) {
    list[lane] = 0;
    if (lane == 0) thr = 0, waiting = sorted = 0;
    __syncwarp();
  }
  // every lane offers one value (or none)
  __device__ __forceinline__ void offer(float x, int ix, bool valid, int top, int lane) {
    const unsigned long long k = valid ? key_of(x, ix) : 0;
    const bool in = k > thr;
    const int have = waiting;
    __syncwarp();
    const unsigned mask = __ballot_sync(kFull, in);
    if (mask == 0) return;
    if (in) buf[have + __popc(mask & ((1u << lane) - 1))] = k;
    if (lane == 0) waiting = have + __popc(mask);
    __syncwarp();
    if (have + __popc(mask) >= 32) flush(have + __popc(mask), top, lane);
  }
  __device__ __noinline__ void flush(int have, int top, int lane) {
    const unsigned long long k = lane < have ? buf[lane] : 0, rest = 32 + lane < have ? buf[32 + lane] : 0;
    const unsigned long long best = merge_sorted(list[lane], sort_down(k, lane), lane);
    __syncwarp();
    list[lane] = best;
    buf[lane] = rest;
    if (lane == top - 1) thr = best;
    if (lane == 0) waiting = have > 32 ? have - 32 : 0, sorted = 1;
    __syncwarp();
  }
};

template <typename T>
struct Vec;
template <>
struct Vec<float> {
  static constexpr int N = 4;
  using Raw = float4;
  __device__ static __forceinline__ Raw load(const float* p) { return __ldcs(reinterpret_cast<const float4*>(p)); }
  __device__ static __forceinline__ Raw fill(float x) { return make_float4(x, -INFINITY, -INFINITY, -INFINITY); }
  __device__ static __forceinline__ float one(const float* p) { return *p; }
  __device__ static __forceinline__ float at(const Raw& v, int j) { return j == 0 ? v.x : j == 1 ? v.y : j == 2 ? v.z : v.w; }
  using Max = float;
  __device__ static __forceinline__ Max largest(const Raw& v) { return fmaxf(fmaxf(v.x, v.y), fmaxf(v.z, v.w)); }
  __device__ static __forceinline__ Max larger(Max a, Max b) { return fmaxf(a, b); }
  __device__ static __forceinline__ float value(Max m) { return m; }
  __device__ static __forceinline__ void add(const Raw& v, Run<float>& r) {
    r.add(r.top.swap(v.x, v.y));
    r.add(r.top.swap(v.z, v.w));
  }
};
template <>
struct Vec<__nv_bfloat16> {
  static constexpr int N = 8;
  using Raw = uint4;
  __device__ static __forceinline__ Raw load(const __nv_bfloat16* p) { return __ldcs(reinterpret_cast<const uint4*>(p)); }
  __device__ static __forceinline__ Raw fill(float x) {
    return make_uint4(0xff800000u | __float_as_uint(x) >> 16, 0xff80ff80u, 0xff80ff80u, 0xff80ff80u);
  }
  __device__ static __forceinline__ float one(const __nv_bfloat16* p) { return __bfloat162float(*p); }
  __device__ static __forceinline__ float at(const Raw& v, int j) {
    const uint32_t w = j < 4 ? (j < 2 ? v.x : v.y) : (j < 6 ? v.z : v.w);
    return j & 1 ? bf16hi(w) : bf16lo(w);
  }
  using Max = __nv_bfloat162;
  __device__ static __forceinline__ Max largest(const Raw& v) {
    const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&v);
    return __hmax2(__hmax2(h[0], h[1]), __hmax2(h[2], h[3]));
  }
  __device__ static __forceinline__ Max larger(Max a, Max b) { return __hmax2(a, b); }
  __device__ static __forceinline__ float value(Max m) { return fmaxf(__low2float(m), __high2float(m)); }
  __device__ static __forceinline__ void add(const Raw& v, Run<__nv_bfloat16>& r) {
    r.add(r.top.swap(v.x));
    r.add(r.top.swap(v.y));
    r.add(r.top.swap(v.z));
    r.add(r.top.swap(v.w));
  }
};

// U vectors of a thread, -inf where it has none.
template <typename T, int U>
__device__ __forceinline__ void take(const typename Vec<T>::Raw (&v)[U], Run<T>& run) {
  typename Vec<T>::Max mx = Vec<T>::largest(v[0]);
#pragma unroll
  for (int u = 1; u < U; ++u) mx = Vec<T>::larger(mx, Vec<T>::largest(v[u]));
  run.make_room(Vec<T>::value(mx));
#pragma unroll
  for (int u = 0; u < U; ++u) Vec<T>::add(v[u], run);
}

// Offers what of the lanes' vectors (elements at, at + 1, ..; `valid` of them) reaches thr_v; the new thr_v.
template <typename T>
__device__ __forceinline__ float candidates(const typename Vec<T>::Raw& v, int at, int valid, float thr_v, int top, int lane, TopList* tl) {
  unsigned hits = 0;
#pragma unroll
  for (int j = 0; j < Vec<T>::N; ++j) hits |= (j < valid && Vec<T>::at(v, j) >= thr_v ? 1u : 0u) << j;
  if (!__any_sync(kFull, hits != 0)) return thr_v;
  while (__any_sync(kFull, hits != 0)) {
    const int j = __ffs(hits) - 1;
    float x = 0.0f;
#pragma unroll
    for (int i = 0; i < Vec<T>::N; ++i) x = i == j ? Vec<T>::at(v, i) : x;
    tl->offer(x, at + j, hits != 0, top, lane);
    hits &= hits - 1;
  }
  const unsigned long long thr = tl->thr;
  return thr != 0 ? fmaxf(thr_v, key_value(thr)) : thr_v;  // (the bound stays until the list reaches it)
}

// A lower bound of the `top`-th largest value of a row part from its threads' largest values (vm): the largest of each of
// 32 groups of threads, sorted; `top` of them reach its entry top - 1.
template <int kTeamWarps>
__device__ __forceinline__ float bound_of(float vm, int top, int lane, int warp, uint32_t* groups) {
  uint32_t k = vm == vm ? ordered(vm) : 0u;  // (a NaN maximum counts as nothing: a bound may only be too low)
  if (kTeamWarps > 1) {
#pragma unroll
    for (int o = kTeamWarps / 2; o > 0; o >>= 1) k = max(k, __shfl_xor_sync(kFull, k, o));
    if (lane % kTeamWarps == 0) groups[warp * (32 / kTeamWarps) + lane / kTeamWarps] = k;
    __syncthreads();
    k = groups[lane];
  }
  const uint32_t b = __shfl_sync(kFull, sort_down(k, lane), top - 1);
  return b == 0 ? -INFINITY : from_ordered(b);
}

// Elements [lo, hi) of a row by kTeamWarps warps, thread `tid` of them.
template <typename T, int kTeamWarps>
__device__ __forceinline__ void scan(const T* x, int lo, int hi, int tid, Run<T>& run, TopList* tl, int top, uint32_t* groups) {
  constexpr int N = Vec<T>::N, n = kTeamWarps * 32;
  constexpr int U = 4;
  using Raw = typename Vec<T>::Raw;
  const int lane = tid & 31, warp = tid >> 5;
  const int mis = static_cast<int>((reinterpret_cast<uintptr_t>(x + lo) & 15u) / sizeof(T));
  int a0 = lo + (mis == 0 ? 0 : N - mis);  // the first aligned element
  if (a0 > hi) a0 = hi;
  const int nv = (hi - a0) / N;
  const int a1 = a0 + nv * N;
  const Raw none = Vec<T>::fill(-INFINITY);
  Raw f[U];
  int v = tid;
#pragma unroll
  for (int u = 0; u < U; ++u) f[u] = v + u * n < nv ? Vec<T>::load(x + a0 + (v + u * n) * N) : none;
  for (; v + (2 * U - 1) * n < nv; v += U * n) {
    Raw g[U];  // the next ones
#pragma unroll
    for (int u = 0; u < U; ++u) g[u] = Vec<T>::load(x + a0 + (v + (U + u) * n) * N);
    take<T, U>(f, run);
#pragma unroll
    for (int u = 0; u < U; ++u) f[u] = g[u];
  }
  for (; v < nv; v += U * n) {
    take<T, U>(f, run);
#pragma unroll
    for (int u = 0; u < U; ++u) f[u] = v + (U + u) * n < nv ? Vec<T>::load(x + a0 + (v + (U + u) * n) * N) : none;
  }
  // single values before and behind the aligned part: fewer than 2 N, one per lane of the first warp
  const int head = a0 - lo, singles = head + hi - a1;
  const int single_at = tid < head ? lo + tid : a1 + tid - head;
  if (tid < singles) {
    const Raw one[1] = {Vec<T>::fill(Vec<T>::one(x + single_at))};
    take<T, 1>(one, run);
  }
  if (top > 0) {
    tl->init(lane);
    const float vm = run.top.largest();
    float thr_v = bound_of<kTeamWarps>(vm, top, lane, warp, groups);
    for (unsigned lanes = __ballot_sync(kFull, vm >= thr_v); lanes != 0; lanes &= lanes - 1) {
      const int src = __ffs(lanes) - 1;  // this lane's share once more, by the whole warp
      if (warp == 0 && src < singles) {
        const int at = src < head ? lo + src : a1 + src - head;
        thr_v = candidates<T>(Vec<T>::fill(Vec<T>::one(x + at)), at, lane == 0 ? 1 : 0, thr_v, top, lane, tl);
      }
      for (int w = warp * 32 + src; w < nv; w += 32 * n) {
        const int mine = w + lane * n;
        const Raw r = mine < nv ? Vec<T>::load(x + a0 + mine * N) : none;
        thr_v = candidates<T>(r, a0 + mine * N, mine < nv ? N : 0, thr_v, top, lane, tl);
      }
    }
  }
}

struct LpArgs {
  const void* logits;
  long long ld;
  const long long* ids;
  float* lp;
  float* ent;
  float* top_lp;
  long long* top_id;
  int rows, vocab, top;
};

// The full row once more with every value compared: rows holding NaN, whose vector maxima do not show it.
template <typename T>
__device__ __noinline__ void rescan_top(const T* x, int vocab, TopList* tl, int top, int lane) {
  tl->init(lane);
  for (int b = 0; b < vocab; b += 32) {
    const bool valid = b + lane < vocab;
    tl->offer(valid ? Vec<T>::one(x + b + lane) : 0.0f, b + lane, valid, top, lane);
  }
  tl->flush(tl->waiting, top, lane);
}

// The row's results, by one warp that holds its merged state and best alternatives (sorted across the lanes).
template <typename T>
__device__ __forceinline__ void finish(const LpArgs& a, int row, const T* x, Stat st, unsigned long long best, TopList* tl, int lane) {
  const float nan = __int_as_float(0x7fc00000);
  st.m = __shfl_sync(kFull, st.m, 0);  // one lane's merge order, so that all results of a row agree
  st.r = __shfl_sync(kFull, st.r, 0);
  st.t = __shfl_sync(kFull, st.t, 0);
  const float lr = log1pf(st.r);
  const bool bad = !(fabsf(st.m) < INFINITY);  // NaN or +inf in the row, or nothing above -inf
  if (lane == 0) {
    const long long id = a.ids == nullptr ? -1 : a.ids[row];
    if (a.lp != nullptr)
      a.lp[row] = bad || id < 0 || id >= a.vocab ? nan : (Vec<T>::one(x + id) - st.m) - lr;
    a.ent[row] = bad ? nan : lr + st.t / (1.0f + st.r);
  }
  if (a.top > 0) {
    if (bad) {
      rescan_top(x, a.vocab, tl, a.top, lane);
      best = tl->list[lane];
    }
    if (lane < a.top) {
      a.top_lp[static_cast<long long>(row) * a.top + lane] = bad ? nan : (key_value(best) - st.m) - lr;
      a.top_id[static_cast<long long>(row) * a.top + lane] = key_index(best);
    }
  }
}

__device__ __forceinline__ void warp_merge(Stat& st) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const float m = __shfl_xor_sync(kFull, st.m, o), r = __shfl_xor_sync(kFull, st.r, o), t = __shfl_xor_sync(kFull, st.t, o);
    st.merge(m, r, t);
  }
}

// The best of the lists and waiting candidates of kWarps warps, sorted across the lanes: by one warp.
template <int kWarps>
__device__ __forceinline__ unsigned long long gather(const TopList* tl, int lane) {
  unsigned long long best = 0;
  int total = 0, mine = lane < kWarps ? tl[lane].waiting : 0;
  unsigned lists = __ballot_sync(kFull, lane < kWarps && tl[lane].sorted);
  for (; lists != 0; lists &= lists - 1) best = merge_sorted(best, tl[__ffs(lists) - 1].list[lane], lane);
  int before = mine;  // candidates of the warps before
#pragma unroll
  for (int o = 1; o < kWarps; o <<= 1) {
    const int w = __shfl_up_sync(kFull, before, o);
    if (lane >= o) before += w;
  }
  total = __shfl_sync(kFull, before, kWarps - 1);
  before -= mine;
  for (int c = 0; c < total; c += 32) {
    int w = 0, at = c + lane;
#pragma unroll
    for (int i = 1; i < kWarps; ++i)
      if (c + lane >= __shfl_sync(kFull, before, i)) w = i;
    at -= __shfl_sync(kFull, before, w);
    best = merge_sorted(best, sort_down(c + lane < total ? tl[w].buf[at] : 0ull, lane), lane);
  }
  return best;
}

template <typename T>
__global__ void __launch_bounds__(kWarpRowThreads) logprobs_warp_kernel(const LpArgs a) {
  __shared__ TopList lists[kWarpRowThreads / 32];
  pdl_launch_dependents();
  pdl_wait_prior_grids();
  const int lane = threadIdx.x & 31, row = blockIdx.x * (kWarpRowThreads / 32) + (threadIdx.x >> 5);
  if (row >= a.rows) return;
  const T* x = static_cast<const T*>(a.logits) + row * a.ld;
  TopList* tl = &lists[threadIdx.x >> 5];
  Run<T> run;
  Stat st;
  scan<T, 1>(x, 0, a.vocab, lane, run, tl, a.top, nullptr);
  st.from(run);
  warp_merge(st);
  __syncwarp();
  finish(a, row, x, st, a.top > 0 ? gather<1>(tl, lane) : 0ull, tl, lane);
}

template <typename T, int kRowThreads>
__global__ void __launch_bounds__(kRowThreads, kRowThreads == 512 ? 1 : 1024 / kRowThreads) logprobs_row_kernel(const LpArgs a) {
  constexpr int kWarps = kRowThreads / 32;
  __shared__ float sm[kWarps], sr[kWarps], stt[kWarps];
  __shared__ uint32_t groups[32];
  __shared__ TopList lists[kWarps];
  __shared__ float cm[kMaxCluster], cr[kMaxCluster], ct[kMaxCluster];  // the leader's slots, one per CTA
  __shared__ unsigned long long cl[kMaxCluster][32];
  pdl_launch_dependents();
  if (gridDim.y > 1) asm volatile("barrier.cluster.arrive.relaxed;" ::: "memory");  // this CTA has started
  pdl_wait_prior_grids();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int C = gridDim.y, rank = blockIdx.y, row = blockIdx.x;  // the cluster is gridDim.y CTAs along y
  const T* x = static_cast<const T*>(a.logits) + row * a.ld;
  const int part = (a.vocab + C - 1) / C;
  const int lo = rank * part < a.vocab ? rank * part : a.vocab, hi = lo + part < a.vocab ? lo + part : a.vocab;
  Run<T> run;
  Stat st;
  scan<T, kWarps>(x, lo, hi, tid, run, &lists[warp], a.top, groups);
  st.from(run);
  warp_merge(st);
  if (lane == 0) sm[warp] = st.m, sr[warp] = st.r, stt[warp] = st.t;
  __syncthreads();
  unsigned long long best = 0;
  if (warp == 0) {
    st.m = -INFINITY, st.r = st.t = 0.0f;
    if (lane < kWarps) st.m = sm[lane], st.r = sr[lane], st.t = stt[lane];
    warp_merge(st);
    if (a.top > 0) best = gather<kWarps>(lists, lane);
  }
  if (C > 1) {
    asm volatile("barrier.cluster.wait.acquire;" ::: "memory");  // every CTA has started: its memory can be written
    if (warp == 0) {
      if (lane == 0) {
        asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(mapa_shared(smem_addr(&cm[rank]), 0)), "f"(st.m) : "memory");
        asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(mapa_shared(smem_addr(&cr[rank]), 0)), "f"(st.r) : "memory");
        asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(mapa_shared(smem_addr(&ct[rank]), 0)), "f"(st.t) : "memory");
      }
      asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(mapa_shared(smem_addr(&cl[rank][lane]), 0)), "l"(best) : "memory");
    }
    cluster_sync_unaligned();  // every CTA's slot written and visible to the leader
    if (rank != 0) return;
    if (warp == 0) {
      st.m = -INFINITY, st.r = st.t = 0.0f;
      if (lane < C) st.m = cm[lane], st.r = cr[lane], st.t = ct[lane];
      warp_merge(st);
      if (a.top > 0)
        for (int c = 1; c < C; ++c) best = merge_sorted(best, cl[c][lane], lane);
    }
  }
  if (warp == 0) finish(a, row, x, st, best, lists, lane);
}

template <typename T>
cudaError_t launch(const LpArgs& a, cudaStream_t s) {
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[2];
  cfg.stream = s;
  // Many rows (4 per SM): short ones a warp each (what a row costs beside its values, sorting and merging above all, is
  // paid by one warp, and rows do not wait for one another: 4096 rows of 4096 take 19 us, 28 on 4 warps each, 47 on 8),
  // long ones by as many warps as keep the SMs full (4096 rows of 16384: 44 us on 4 warps, 59 on 8; 1500 of 100352: 75 on
  // 4, 70 on 8, 122 on 16; a warp each 178). Few rows: 16 warps in each of up to 8 CTAs, a warp only where there is
  // nothing to split.
  const bool many = a.rows >= 4 * tc_sm_count();
  if (a.vocab <= (many ? 8192 : 1024)) {
    cfg.gridDim = dim3((a.rows + kWarpRowThreads / 32 - 1) / (kWarpRowThreads / 32));
    cfg.blockDim = dim3(kWarpRowThreads);
    set_launch_attrs(cfg, attr);
    return cudaLaunchKernelEx(&cfg, logprobs_warp_kernel<T>, a);
  }
  int C = 1;
  while (C < kMaxCluster && a.rows * C < tc_sm_count() && a.vocab / (2 * C) >= 4096) C *= 2;
  const int threads = many && a.vocab <= 32768 ? 128 : C == 1 ? 256 : 512;
  cfg.gridDim = dim3(a.rows, C);
  cfg.blockDim = dim3(threads);
  set_launch_attrs(cfg, attr, C);
  if (threads == 128) return cudaLaunchKernelEx(&cfg, logprobs_row_kernel<T, 128>, a);
  return threads == 256 ? cudaLaunchKernelEx(&cfg, logprobs_row_kernel<T, 256>, a)
                        : cudaLaunchKernelEx(&cfg, logprobs_row_kernel<T, 512>, a);
}

}  // namespace
}  // namespace bp

extern "C" int bp_token_logprobs(const void* logits, long long ld, int dtype, const int64_t* ids, float* logprob,
                                 float* entropy, float* top_logprob, int64_t* top_id, int rows, int vocab, int top,
                                 void* stream) {
  using namespace bp;
  clear_error();
  if (rows < 0 || vocab < 0) return fail(BP_ERR_INVALID_ARGUMENT, "negative size (rows=%d vocab=%d)", rows, vocab);
  if (dtype != BP_DTYPE_BF16 && dtype != BP_DTYPE_F32)
    return fail(BP_ERR_INVALID_ARGUMENT, "logits dtype %d is not bf16 or fp32", dtype);
  if (top < 0 || top > kMaxTop || top > vocab)
    return fail(BP_ERR_INVALID_ARGUMENT, "top must be 0..%d and at most vocab (got %d of %d)", kMaxTop, top, vocab);
  if (rows == 0) return BP_OK;
  if (vocab == 0) return fail(BP_ERR_INVALID_ARGUMENT, "rows of an empty vocabulary have no distribution");
  if (logits == nullptr || entropy == nullptr || (ids == nullptr) != (logprob == nullptr) ||
      (top > 0 && (top_logprob == nullptr || top_id == nullptr)))
    return fail(BP_ERR_INVALID_ARGUMENT, "a pointer is NULL (ids and logprob: both or neither)");
  if (ld < vocab) return fail(BP_ERR_INVALID_ARGUMENT, "ld must be >= vocab");
  if (vocab > (1 << 30)) return fail(BP_ERR_UNSUPPORTED, "vocab %d is above 2^30", vocab);
  const uintptr_t es = dtype == BP_DTYPE_F32 ? 4 : 2;
  if (reinterpret_cast<uintptr_t>(logits) % es != 0 || (reinterpret_cast<uintptr_t>(ids) & 7u) != 0 ||
      (reinterpret_cast<uintptr_t>(top_id) & 7u) != 0)
    return fail(BP_ERR_MISALIGNED, "logits, ids and top_id need their elements' alignment");
  int st = require_sm100();
  if (st != BP_OK) return st;
  LpArgs a{logits, ld, reinterpret_cast<const long long*>(ids), logprob, entropy, top_logprob,
           reinterpret_cast<long long*>(top_id), rows, vocab, top};
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  const cudaError_t e = dtype == BP_DTYPE_F32 ? launch<float>(a, s) : launch<__nv_bfloat16>(a, s);
  if (e != cudaSuccess) return fail(BP_ERR_CUDA, "token_logprobs launch: %s", cudaGetErrorString(e));
  return check_launch("token_logprobs");
}
