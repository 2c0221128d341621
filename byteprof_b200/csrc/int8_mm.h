// Shared by the kernels of the 8-bit integer product (int8_mm.cu, int8_mm_tc.cu).
#pragma once

#include "bp_common.cuh"

namespace bp {

struct Int8Args {
  const int8_t* x;       // [M, K], row stride ldx
  long long ldx;
  const float* x_scale;  // [M]
  const int8_t* w;       // [N, K], row stride ldw
  long long ldw;
  const void* w_scale;   // [N], fp32 or bf16
  int w_scale_f32;
  const __nv_bfloat16* bias;  // [N] or NULL
  void* y;               // [M, N], fp32 or bf16, row stride ldy
  long long ldy;
  int y_f32;
  int M, N, K;
};

__device__ __forceinline__ float int8_w_scale(const Int8Args& a, int n) {
  return a.w_scale_f32 ? static_cast<const float*>(a.w_scale)[n]
                       : __bfloat162float(static_cast<const __nv_bfloat16*>(a.w_scale)[n]);
}
__device__ __forceinline__ float int8_bias(const Int8Args& a, int n) {
  return a.bias == nullptr ? 0.0f : __bfloat162float(a.bias[n]);
}
// The one formula of all kernels, so that they agree to the last bit: the integer sum as fp32 (one rounding above
// 2^24), the token's scale, the channel's, the bias.
__device__ __forceinline__ float int8_value(const Int8Args& a, int acc, float sx, float sw, float bias) {
  const float v = __fmul_rn(__fmul_rn(static_cast<float>(acc), sx), sw);
  return a.bias == nullptr ? v : __fadd_rn(v, bias);
}

// ---- the rows' quantizer, shared with the kernel that quantizes its own few rows ------------------------
__device__ __forceinline__ uint32_t abs_max8(const uint4 v, uint32_t m) {
  const uint32_t* w = &v.x;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    m = max(m, (w[i] << 16) & 0x7fffffffu);
    m = max(m, w[i] & 0x7fff0000u);
  }
  return m;
}

// rint(x / s) with the division correctly rounded, in the low byte. x / s is within 2^-16 of x * inv (|x / s| < 128, inv
// is off by half a step: 2^-17 in all), so only a product that close to a half-integer needs the division itself. Adding
// 1.5 * 2^23 rounds to an integer, to even between two, and leaves it in the low bits: conversions and rint run at a
// quarter of the rate and were the quantizer's busiest pipe.
__device__ __forceinline__ uint32_t q1(float x, float s, float inv) {
  constexpr float kMagic = 12582912.0f;
  float t = fmaf(x, inv, kMagic);
  const float off = fmaf(x, inv, kMagic - t);
  if (fabsf(fabsf(off) - 0.5f) < 0x1p-16f) t = kMagic + __fdiv_rn(x, s);
  return __float_as_uint(t);
}

__device__ __forceinline__ uint32_t q4(float a, float b, float c, float d, float s, float inv) {
  return __byte_perm(__byte_perm(q1(a, s, inv), q1(b, s, inv), 0x0040), __byte_perm(q1(c, s, inv), q1(d, s, inv), 0x0040), 0x5410);
}

__device__ __forceinline__ uint2 q8(const uint4 v, float s, float inv) {
  return make_uint2(q4(bf16lo(v.x), bf16hi(v.x), bf16lo(v.y), bf16hi(v.y), s, inv),
                    q4(bf16lo(v.z), bf16hi(v.z), bf16lo(v.w), bf16hi(v.w), s, inv));
}

// 127 levels to either side; the bits of |x|'s maximum tell Inf and NaN.
__device__ __forceinline__ float int8_row_scale(uint32_t max_bits) {
  return fmaxf(__fdiv_rn(__uint_as_float(max_bits), 127.0f), 1e-12f);
}

// The tensor-core kernel (int8_mm_tc.cu): 16-byte aligned operands with row strides multiples of 16, K > 0.
bool int8_mm_tc_supported(const Int8Args& a);
int launch_int8_mm_tc(const Int8Args& a, cudaStream_t stream);

// The same with the quantizer inside, for one or two rows of 16-byte aligned bf16 x (a.x and a.x_scale unused).
bool int8_fused_supported(const Int8Args& a, const void* x, long long ldx);
int launch_int8_fused(const Int8Args& a, const __nv_bfloat16* x, long long ldx, cudaStream_t stream);

}  // namespace bp
