// What the two kernels of the linear layer over 8-bit integers share.
#pragma once
#include "host_common.h"

namespace hdit {

// A sum in fp32 with both scales and the bias; every kernel rounds in this order, so that all of them give the same bits.
__device__ __forceinline__ float int8_value(int sum, float row_scale, float col_scale, float bias) {
  return fmaf(static_cast<float>(sum) * row_scale, col_scale, bias);
}

// int8_linear_few.cu
constexpr int kInt8FewRows = 8;
bool int8_linear_few_takes(const hdit_int8_linear_args* a);
bool int8_linear_few_quantizes(const hdit_int8_linear_args* a);  // brings 16-bit rows into 8 bits by itself
int int8_linear_few(const hdit_int8_linear_args* a);             // checked arguments

}  // namespace hdit
