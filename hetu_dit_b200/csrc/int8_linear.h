// What the two kernels of the linear layer over 8-bit integers share.
#pragma once
#include "host_common.h"
#include "ptx_sm100.cuh"

namespace hdit {

// Sums in fp32 with both scales and the bias; both kernels round in this order, so that they give the same bits.
__device__ __forceinline__ float2 int8_value2(int sum0, int sum1, float row_scale, float2 col_scale, float2 bias) {
  return fma2(mul2(make_float2(static_cast<float>(sum0), static_cast<float>(sum1)), both(row_scale)), col_scale, bias);
}

// GELU, tanh approximation, tanh on the special-function unit (within 2^-11 of its result, as in the 16-bit layers)
__device__ __forceinline__ float2 int8_gelu2(float2 x) {
  const float2 k = both(0.7978845608028654f), c = both(0.7978845608028654f * 0.044715f);
  const float2 u = mul2(x, fma2(mul2(x, x), c, k));
  float2 t;
  asm("tanh.approx.f32 %0, %1;" : "=f"(t.x) : "f"(u.x));
  asm("tanh.approx.f32 %0, %1;" : "=f"(t.y) : "f"(u.y));
  const float2 h = mul2(x, both(0.5f));
  return fma2(h, t, h);
}

// int8_linear_few.cu
constexpr int kInt8FewRows = 8;
bool int8_linear_few_takes(const hdit_int8_linear_args* a);
bool int8_linear_few_pays(const hdit_int8_linear_args* a);       // against tiles
bool int8_linear_few_quantizes(const hdit_int8_linear_args* a);  // brings 16-bit rows into 8 bits by itself
int int8_linear_few(const hdit_int8_linear_args* a);             // checked arguments

}  // namespace hdit
