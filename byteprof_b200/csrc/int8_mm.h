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

// rint(x / s) with the division correctly rounded. The product with 1 / s is within 2^-22 of the quotient (relative;
// |quotient| < 128: 2^-15 absolute), so only a product that close to a half-integer needs the division itself.
__device__ __forceinline__ int q1(float x, float s, float inv) {
  const float y = x * inv;
  float r = rintf(y);
  if (fabsf(fabsf(y - r) - 0.5f) < 1e-4f) r = rintf(__fdiv_rn(x, s));
  return static_cast<int>(r);
}

__device__ __forceinline__ uint32_t q4(float a, float b, float c, float d, float s, float inv) {
  return (q1(a, s, inv) & 0xff) | ((q1(b, s, inv) & 0xff) << 8) | ((q1(c, s, inv) & 0xff) << 16) |
         (static_cast<uint32_t>(q1(d, s, inv)) << 24);
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
