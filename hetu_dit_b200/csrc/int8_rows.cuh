// A row of values as 8-bit integers with one scale:  s = max|y| / 127,  q = y / s rounded to the nearest integer, ties to
// even. What quantize_rows, ln_modulate_int8 and the group norm with 8-bit rows share.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "ptx_sm100.cuh"

namespace hdit {
namespace {

// A row whose largest magnitude is below this counts as zero (s = 0, q = 0): 127 / max stays finite and max / 127 normal.
// Infinities and NaN have larger bit patterns than every number; a row that holds one gets s = NaN and q = 0, so that
// whatever is computed from the row is NaN.
constexpr uint32_t kInt8RowTiny = 0x0D800000u;  // 2^-100
constexpr uint32_t kInt8RowInf = 0x7F800000u;

struct Int8Scale {
  uint32_t top_bits;  // of max|y|; as unsigned integers magnitudes order like their values, and NaN is above all
  float inv;          // steps per unit; 0: the row is all zeros
};

__device__ __forceinline__ Int8Scale int8_scale(uint32_t top_bits) {
  return {top_bits, top_bits >= kInt8RowInf || top_bits < kInt8RowTiny ? 0.f : __fdiv_rn(127.f, __uint_as_float(top_bits))};
}
// The row's scale, for the one thread that writes it.
__device__ __forceinline__ float int8_step(const Int8Scale& s) {
  if (s.top_bits >= kInt8RowInf) return __uint_as_float(0x7FC00000u);
  return s.inv == 0.f ? 0.f : __fdiv_rn(__uint_as_float(s.top_bits), 127.f);
}

constexpr float kInt8Round = 1.5f * 8388608.f;

// Adding 1.5 * 2^23 rounds to the nearest integer, ties to even, and leaves it in the low bits as two's complement; the low
// bytes of four of them are packed.
__device__ __forceinline__ uint32_t int8_bytes(float2 a, float2 b) {
  return __byte_perm(__byte_perm(__float_as_uint(a.x), __float_as_uint(a.y), 0x0040), __byte_perm(__float_as_uint(b.x), __float_as_uint(b.y), 0x0040), 0x5410);
}

// v / s for a 16-bit v, exact at the borders between two integers. 254 v - (2 n + 1) max is a whole number of units in the
// last place of v (v <= max), so 127 v / max is n + 1/2 or at least 2^-19 of its size away from it (v has at most 11 bits);
// v * inv is within 2^-24 of the quotient. The sum below is v * inv rounded to 20 bits (Dekker's splitting: both terms are
// multiples of 16 units of the quotient's last place, the second one rounds the exact difference), which moves it by 2^-20 at
// most: that restores n + 1/2 (8 bits) exactly and brings nothing else onto it or across. inv17 = 17 * inv. Operations
// on two values an instruction; on the bits, (bits + 8) & ~15 behind the product, it would take the integer pipe twice, which the
// packing needs.
__device__ __forceinline__ float2 int8_steps_of_16bit(float2 v, float inv, float inv17) {
  const float2 p = mul2(v, both(inv17));
  return add2(p, fma2(v, both(inv), make_float2(-p.x, -p.y)));
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

// The same eight elements of a row that starts anywhere, in two steps: the two 16-byte blocks that hold them, then their bits moved
// into place, so that nothing waits for the loads in between. lo, hi: the first element of all rows and the end of the last one. A
// block that reaches outside (the first one of the first row, the last ones of the last row) is put together from the elements; what
// lies between rows may be read, and goes no further.
struct Int8Blocks {
  uint4 a, b;
};
__device__ __forceinline__ Int8Blocks int8_load_blocks(const uint16_t* row, int c, int dim, const uint16_t* lo, const uint16_t* hi) {
  const uintptr_t at = reinterpret_cast<uintptr_t>(row + c);
  const uint16_t* const base = reinterpret_cast<const uint16_t*>(at & ~static_cast<uintptr_t>(15));
  const int skip = static_cast<int>(at & 15) >> 1, live = min(8, dim - c);
  const bool second = skip + live > 8;
  Int8Blocks r{make_uint4(0, 0, 0, 0), make_uint4(0, 0, 0, 0)};
  if (base >= lo && base + (second ? 16 : 8) <= hi) {
    r.a = *reinterpret_cast<const uint4*>(base);
    if (second) r.b = *reinterpret_cast<const uint4*>(base + 8);
  } else {
    uint32_t* u = reinterpret_cast<uint32_t*>(&r);
#pragma unroll
    for (int e = 0; e < 16; ++e)
      if (e >= skip && e < skip + live) u[e >> 1] |= static_cast<uint32_t>(base[e]) << (16 * (e & 1));
  }
  return r;
}
__device__ __forceinline__ uint4 int8_from_blocks(const Int8Blocks& r, const uint16_t* row, int c, int dim) {
  const int skip = static_cast<int>(reinterpret_cast<uintptr_t>(row) & 15) >> 1;  // of the row: c is a multiple of 8
  uint32_t w[8] = {r.a.x, r.a.y, r.a.z, r.a.w, r.b.x, r.b.y, r.b.z, r.b.w};
#pragma unroll
  for (int i = 0; i < 6; ++i) w[i] = skip & 4 ? w[i + 2] : w[i];
#pragma unroll
  for (int i = 0; i < 5; ++i) w[i] = skip & 2 ? w[i + 1] : w[i];
#pragma unroll
  for (int i = 0; i < 4; ++i) w[i] = __funnelshift_r(w[i], w[i + 1], (skip & 1) * 16);
  if (c + 8 > dim) {
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = c + 2 * i + 1 < dim ? w[i] : c + 2 * i < dim ? w[i] & 0xFFFFu : 0u;
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

constexpr int kRowThreads = 256;  // of a CTA that works on rows

// TEAM threads of a CTA that share a row. A reduction over several warps has one barrier, of the team: each has places of its
// own, and the barriers of the others stand between its reads and its next row's writes (where there are no others, the rows'
// parity picks the places).
template <int TEAM, int THREADS = kRowThreads>
struct Team {
  static constexpr int kWarps = TEAM / 32;
  float (*red)[THREADS / 32];
  __device__ __forceinline__ void sync() const { asm volatile("bar.sync %0, %1;" ::"r"(1 + threadIdx.x / TEAM), "n"(TEAM) : "memory"); }
  __device__ __forceinline__ uint32_t max(uint32_t v, int slot) const {
    if constexpr (TEAM < 32) {
#pragma unroll
      for (int o = TEAM / 2; o > 0; o >>= 1) v = ::max(v, __shfl_xor_sync(0xffffffffu, v, o));
      return v;
    }
    v = __reduce_max_sync(0xffffffffu, v);
    if constexpr (kWarps > 1) {
      uint32_t* r = reinterpret_cast<uint32_t*>(red[slot]);
      if ((threadIdx.x & 31) == 0) r[threadIdx.x >> 5] = v;
      sync();
      v = 0;
      const int w0 = threadIdx.x / TEAM * kWarps;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) v = v > r[w0 + w] ? v : r[w0 + w];
    }
    return v;
  }
  __device__ __forceinline__ float sum(float v, int slot) const {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    if constexpr (kWarps > 1) {
      if ((threadIdx.x & 31) == 0) red[slot][threadIdx.x >> 5] = v;
      sync();
      v = 0.f;
      const int w0 = threadIdx.x / TEAM * kWarps;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) v += red[slot][w0 + w];
    }
    return v;
  }
};

// Eight 16-bit values to column c of the row, which is on an 8-byte boundary; zeros where the row has no step (an infinity
// times 0 is none). TAIL: the row may end before, and what lies behind it stays as it was.
template <bool FP16, bool TAIL>
__device__ __forceinline__ void int8_put8(int8_t* row, int c, int dim, const Int8Scale& s, float inv17, const uint4& raw) {
  const uint32_t* u = reinterpret_cast<const uint32_t*>(&raw);
  float2 t[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) t[i] = add2(int8_steps_of_16bit(int8_unpack2<FP16>(u[i]), s.inv, inv17), both(kInt8Round));
  uint2 v = make_uint2(int8_bytes(t[0], t[1]), int8_bytes(t[2], t[3]));
  if (s.inv == 0.f) v = make_uint2(0, 0);
  if (!TAIL || c + 8 <= dim) {
    *reinterpret_cast<uint2*>(row + c) = v;
  } else {
    for (int i = 0; c + i < dim; ++i) row[c + i] = static_cast<int8_t>((i < 4 ? v.x >> (8 * i) : v.y >> (8 * (i - 4))) & 0xFFu);
  }
}

// The same for fp32 values: product with inv and rounding to an integer in one operation.
__device__ __forceinline__ void int8_put8_of(int8_t* row, int c, const Int8Scale& s, const float2 (&y)[4]) {
  float2 t[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) t[i] = fma2(y[i], both(s.inv), both(kInt8Round));
  uint2 v = make_uint2(int8_bytes(t[0], t[1]), int8_bytes(t[2], t[3]));
  if (s.inv == 0.f) v = make_uint2(0, 0);
  *reinterpret_cast<uint2*>(row + c) = v;
}

// Larger of two magnitudes, NaN if one is: the compiler's fmaxf() drops a NaN.
__device__ __forceinline__ float max_magnitude(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(fabsf(b)));
  return r;
}

}  // namespace
}  // namespace hdit
