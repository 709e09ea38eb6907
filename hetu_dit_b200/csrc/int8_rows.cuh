// A row of values as 8-bit integers with one scale:  s = max|y| / 127,  q = y / s rounded to the nearest integer, ties to
// even. What quantize_rows, ln_modulate_int8 and the group norm with 8-bit rows share.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

namespace hdit {
namespace {

// A row whose largest magnitude is below this counts as zero (s = 0, q = 0): 127 / max stays finite and max / 127 normal.
// Infinities and NaN have larger bit patterns than every number; a row that holds one gets s = NaN and q = 0, so that
// whatever is computed from the row is NaN.
constexpr uint32_t kInt8RowTiny = 0x0D800000u;  // 2^-100
constexpr uint32_t kInt8RowInf = 0x7F800000u;

struct Int8Scale {
  float scale, inv;  // value of one step, steps per unit
};

// From the bits of max|y| (as unsigned integers magnitudes order like their values, and NaN is above all).
__device__ __forceinline__ Int8Scale int8_scale(uint32_t top_bits) {
  if (top_bits >= kInt8RowInf) return {__uint_as_float(0x7FC00000u), 0.f};
  if (top_bits < kInt8RowTiny) return {0.f, 0.f};
  const float top = __uint_as_float(top_bits);
  return {__fdiv_rn(top, 127.f), __fdiv_rn(127.f, top)};
}

// Adding 1.5 * 2^23 rounds to the nearest integer, ties to even, and leaves it in the low bits as two's complement; the
// low bytes of four of them are packed.
__device__ __forceinline__ uint32_t int8_pack4(float a, float b, float c, float d) {
  const uint32_t ua = __float_as_uint(__fadd_rn(a, 12582912.f)), ub = __float_as_uint(__fadd_rn(b, 12582912.f));
  const uint32_t uc = __float_as_uint(__fadd_rn(c, 12582912.f)), ud = __float_as_uint(__fadd_rn(d, 12582912.f));
  return __byte_perm(__byte_perm(ua, ub, 0x0040), __byte_perm(uc, ud, 0x0040), 0x5410);
}

// v / s for a 16-bit v, exact at the borders between two integers. 254 v - (2 n + 1) max is a whole number of units in the
// last place of v (v <= max), so 127 v / max is n + 1/2 or at least 2^-19 of its size away from it (v has at most 11 bits);
// v * inv is within 2^-22.9 of the quotient. Rounding to 20 bits moves it by 2^-20 at most: that restores n + 1/2 (8 bits)
// exactly and brings nothing else onto it or across.
__device__ __forceinline__ float int8_steps_of_16bit(float v, float inv) {
  return __uint_as_float((__float_as_uint(__fmul_rn(v, inv)) + 8u) & ~15u);
}

template <bool FP16>
__device__ __forceinline__ float2 int8_unpack2(uint32_t u) {
  if constexpr (FP16) return __half22float2(*reinterpret_cast<const __half2*>(&u));
  else return make_float2(__uint_as_float(u << 16), __uint_as_float(u & 0xFFFF0000u));
}

// Eight elements from column c on of a row of dim; what lies behind the row's end reads as 0. vec: the row starts on a
// 16-byte boundary.
__device__ __forceinline__ uint4 int8_load8(const uint16_t* row, int c, int dim, bool vec) {
  if (vec && c + 8 <= dim) return *reinterpret_cast<const uint4*>(row + c);
  uint32_t e[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) e[i] = c + i < dim ? row[c + i] : 0u;
  return make_uint4(e[0] | (e[1] << 16), e[2] | (e[3] << 16), e[4] | (e[5] << 16), e[6] | (e[7] << 16));
}

// Eight bytes to column c (a multiple of 8) of a row of dim that starts on a 16-byte boundary.
__device__ __forceinline__ void int8_store8(int8_t* row, int c, int dim, uint2 v) {
  if (c + 8 <= dim) {
    *reinterpret_cast<uint2*>(row + c) = v;
  } else {
    for (int i = 0; i < 8 && c + i < dim; ++i) row[c + i] = static_cast<int8_t>((i < 4 ? v.x >> (8 * i) : v.y >> (8 * (i - 4))) & 0xFFu);
  }
}

constexpr int kRowThreads = 256;  // of a CTA that works on rows

// TEAM threads of a CTA that share a row; all teams of the CTA make the same calls.
template <int TEAM>
struct Team {
  static constexpr int kWarps = TEAM / 32;
  float* red;  // one float per warp of the CTA
  __device__ __forceinline__ uint32_t max(uint32_t v) const {
    v = __reduce_max_sync(0xffffffffu, v);
    if constexpr (kWarps > 1) {
      uint32_t* r = reinterpret_cast<uint32_t*>(red);
      __syncthreads();
      if ((threadIdx.x & 31) == 0) r[threadIdx.x >> 5] = v;
      __syncthreads();
      v = 0;
      const int w0 = threadIdx.x / TEAM * kWarps;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) v = v > r[w0 + w] ? v : r[w0 + w];
    }
    return v;
  }
  __device__ __forceinline__ float sum(float v) const {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    if constexpr (kWarps > 1) {
      __syncthreads();
      if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
      __syncthreads();
      v = 0.f;
      const int w0 = threadIdx.x / TEAM * kWarps;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) v += red[w0 + w];
    }
    return v;
  }
};

}  // namespace
}  // namespace hdit
