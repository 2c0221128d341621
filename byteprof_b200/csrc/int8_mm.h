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

// The tensor-core kernel (int8_mm_tc.cu): 16-byte aligned operands with row strides multiples of 16, K > 0.
bool int8_mm_tc_supported(const Int8Args& a);
int launch_int8_mm_tc(const Int8Args& a, cudaStream_t stream);

}  // namespace bp
