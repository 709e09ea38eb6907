// Rows of 16-bit values as 8-bit integers with a scale for each row (int8_rows.cuh), as they are or after
// LayerNorm + modulation:
//   quantize_rows    : y = x
//   ln_modulate_int8 : y = LayerNorm(x) * (1 + scale[b]) + shift[b]      (no affine, biased variance)
// One pass: a row stays in the registers of its threads between the read and the write, as the 16-bit values that were
// read (half the registers of fp32 ones). y is not rounded to 16 bits in between. Bound by memory: 2 bytes read and 1
// written per element.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include "host_common.h"
#include "int8_rows.cuh"

namespace hdit {
namespace {

struct RowsParams {
  const uint16_t* x;
  const uint16_t* shift;  // ln_modulate_int8 only
  const uint16_t* scale;
  int8_t* q;
  float* q_scale;
  long long rows, rows_per_batch, x_batch_stride, x_row_stride, q_row_stride, mod_batch_stride;
  int dim;
  float eps;
  bool vec;  // 16-byte loads of x (and of shift, scale) are aligned
};

// TEAM threads hold a row of at most TEAM * NCH * 8 elements. Rows are taken in the same order by all teams of a CTA, so
// that a team without a row still meets the others' barriers.
template <bool FP16, int TEAM, int NCH, bool LN>
__global__ void __launch_bounds__(kRowThreads) int8_rows_kernel(const __grid_constant__ RowsParams p) {
  grid_dependency_release();
  grid_dependency_wait();
  __shared__ float red[kRowThreads / 32];
  const Team<TEAM> team{red};
  constexpr int kTeams = kRowThreads / TEAM;
  const int lane = threadIdx.x % TEAM;
  const long long step = static_cast<long long>(gridDim.x) * kTeams;
  for (long long row0 = static_cast<long long>(blockIdx.x) * kTeams; row0 < p.rows; row0 += step) {
    const long long row = row0 + threadIdx.x / TEAM;
    const bool live = row < p.rows;
    const long long b = live ? row / p.rows_per_batch : 0;
    const uint16_t* xr = p.x + (live ? b * p.x_batch_stride + (row - b * p.rows_per_batch) * p.x_row_stride : 0);
    uint4 raw[NCH];
#pragma unroll
    for (int c = 0; c < NCH; ++c) {
      const int col = (c * TEAM + lane) * 8;
      raw[c] = live && col < p.dim ? int8_load8(xr, col, p.dim, p.vec) : make_uint4(0, 0, 0, 0);
    }
    if constexpr (!LN) {
      // magnitudes of two 16-bit values at a time, as integers
      uint32_t top2 = 0;
#pragma unroll
      for (int c = 0; c < NCH; ++c) {
        const uint32_t* u = reinterpret_cast<const uint32_t*>(&raw[c]);
#pragma unroll
        for (int i = 0; i < 4; ++i) top2 = __vmaxu2(top2, u[i] & 0x7FFF7FFFu);
      }
      const uint32_t top16 = team.max((top2 & 0xFFFFu) > (top2 >> 16) ? top2 & 0xFFFFu : top2 >> 16);
      const Int8Scale s = int8_scale(__float_as_uint(int8_unpack2<FP16>(top16).x));
      if (live) {
#pragma unroll
        for (int c = 0; c < NCH; ++c) {
          const int col = (c * TEAM + lane) * 8;
          const uint32_t* u = reinterpret_cast<const uint32_t*>(&raw[c]);
          float t[8];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float2 v = int8_unpack2<FP16>(u[i]);
            t[2 * i] = int8_steps_of_16bit(v.x, s.inv);
            t[2 * i + 1] = int8_steps_of_16bit(v.y, s.inv);
          }
          if (s.inv == 0.f) {  // infinities and NaN times 0
#pragma unroll
            for (int i = 0; i < 8; ++i) t[i] = 0.f;
          }
          if (col < p.dim)
            int8_store8(p.q + row * p.q_row_stride, col, p.dim, make_uint2(int8_pack4(t[0], t[1], t[2], t[3]), int8_pack4(t[4], t[5], t[6], t[7])));
        }
        if (lane == 0) p.q_scale[row] = s.scale;
      }
    } else {
      float sum = 0.f;
#pragma unroll
      for (int c = 0; c < NCH; ++c) {
        const uint32_t* u = reinterpret_cast<const uint32_t*>(&raw[c]);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float2 v = int8_unpack2<FP16>(u[i]);
          sum += v.x + v.y;
        }
      }
      const float mean = team.sum(sum) / static_cast<float>(p.dim);
      float sq = 0.f;
#pragma unroll
      for (int c = 0; c < NCH; ++c) {
        const uint32_t* u = reinterpret_cast<const uint32_t*>(&raw[c]);
        if ((c * TEAM + lane) * 8 < p.dim) {  // dim is a multiple of 8
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float2 v = int8_unpack2<FP16>(u[i]);
            sq = fmaf(v.x - mean, v.x - mean, sq);
            sq = fmaf(v.y - mean, v.y - mean, sq);
          }
        }
      }
      const float rstd = rsqrtf(team.sum(sq) / static_cast<float>(p.dim) + p.eps);
      float y[NCH][8];
      uint32_t top = 0;
#pragma unroll
      for (int c = 0; c < NCH; ++c) {
        const int col = (c * TEAM + lane) * 8;
        const uint32_t* u = reinterpret_cast<const uint32_t*>(&raw[c]);
        if (col < p.dim) {
          const uint4 sh4 = int8_load8(p.shift + b * p.mod_batch_stride, col, p.dim, p.vec);
          const uint4 sc4 = int8_load8(p.scale + b * p.mod_batch_stride, col, p.dim, p.vec);
          const uint32_t* sh = reinterpret_cast<const uint32_t*>(&sh4);
          const uint32_t* sc = reinterpret_cast<const uint32_t*>(&sc4);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float2 v = int8_unpack2<FP16>(u[i]), h = int8_unpack2<FP16>(sh[i]), g = int8_unpack2<FP16>(sc[i]);
            y[c][2 * i] = fmaf((v.x - mean) * rstd, 1.f + g.x, h.x);
            y[c][2 * i + 1] = fmaf((v.y - mean) * rstd, 1.f + g.y, h.y);
          }
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const uint32_t m = __float_as_uint(y[c][i]) & 0x7FFFFFFFu;
            top = top > m ? top : m;
          }
        }
      }
      const Int8Scale s = int8_scale(team.max(top));
      if (live) {
#pragma unroll
        for (int c = 0; c < NCH; ++c) {
          const int col = (c * TEAM + lane) * 8;
          if (col < p.dim) {
            float t[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) t[i] = s.inv == 0.f ? 0.f : y[c][i] * s.inv;
            int8_store8(p.q + row * p.q_row_stride, col, p.dim, make_uint2(int8_pack4(t[0], t[1], t[2], t[3]), int8_pack4(t[4], t[5], t[6], t[7])));
          }
        }
        if (lane == 0) p.q_scale[row] = s.scale;
      }
    }
  }
}

// Rows longer than the registers of a CTA hold: read twice, the second time from the caches.
template <bool FP16>
__global__ void __launch_bounds__(kRowThreads) int8_long_rows_kernel(const __grid_constant__ RowsParams p) {
  grid_dependency_release();
  grid_dependency_wait();
  __shared__ float red[kRowThreads / 32];
  const Team<kRowThreads> team{red};
  for (long long row = blockIdx.x; row < p.rows; row += gridDim.x) {
    const long long b = row / p.rows_per_batch;
    const uint16_t* xr = p.x + b * p.x_batch_stride + (row - b * p.rows_per_batch) * p.x_row_stride;
    uint32_t top2 = 0;
    for (int col = threadIdx.x * 8; col < p.dim; col += kRowThreads * 8) {
      const uint4 raw = int8_load8(xr, col, p.dim, p.vec);
      const uint32_t* u = reinterpret_cast<const uint32_t*>(&raw);
#pragma unroll
      for (int i = 0; i < 4; ++i) top2 = __vmaxu2(top2, u[i] & 0x7FFF7FFFu);
    }
    const uint32_t top16 = team.max((top2 & 0xFFFFu) > (top2 >> 16) ? top2 & 0xFFFFu : top2 >> 16);
    const Int8Scale s = int8_scale(__float_as_uint(int8_unpack2<FP16>(top16).x));
    for (int col = threadIdx.x * 8; col < p.dim; col += kRowThreads * 8) {
      const uint4 raw = int8_load8(xr, col, p.dim, p.vec);
      const uint32_t* u = reinterpret_cast<const uint32_t*>(&raw);
      float t[8];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 v = int8_unpack2<FP16>(u[i]);
        t[2 * i] = s.inv == 0.f ? 0.f : int8_steps_of_16bit(v.x, s.inv);
        t[2 * i + 1] = s.inv == 0.f ? 0.f : int8_steps_of_16bit(v.y, s.inv);
      }
      int8_store8(p.q + row * p.q_row_stride, col, p.dim, make_uint2(int8_pack4(t[0], t[1], t[2], t[3]), int8_pack4(t[4], t[5], t[6], t[7])));
    }
    if (threadIdx.x == 0) p.q_scale[row] = s.scale;
  }
}

template <bool FP16, int TEAM, int NCH, bool LN>
cudaError_t launch_rows(const RowsParams& p, cudaStream_t st) {
  constexpr int kTeams = kRowThreads / TEAM;
  long long blocks = (p.rows + kTeams - 1) / kTeams;
  if (blocks > 148LL * 8) blocks = 148LL * 8;
  return launch_overlapped(int8_rows_kernel<FP16, TEAM, NCH, LN>, dim3(static_cast<unsigned>(blocks)), dim3(kRowThreads), 0, st, 1, p);
}

template <bool FP16, bool LN>
cudaError_t launch_any(const RowsParams& p, cudaStream_t st) {
  const int chunks = (p.dim + 7) / 8;
  if (chunks <= 32) return launch_rows<FP16, 32, 1, LN>(p, st);
  if (chunks <= 64) return launch_rows<FP16, 32, 2, LN>(p, st);
  if (chunks <= 128) return launch_rows<FP16, 32, 4, LN>(p, st);
  if (chunks <= 192) return launch_rows<FP16, 32, 6, LN>(p, st);
  if (chunks <= 256) return launch_rows<FP16, 128, 2, LN>(p, st);
  if (chunks <= 384) return launch_rows<FP16, 128, 3, LN>(p, st);
  if (chunks <= 512) return launch_rows<FP16, 256, 2, LN>(p, st);
  if (chunks <= 768) return launch_rows<FP16, 256, 3, LN>(p, st);
  if (chunks <= 1024) return launch_rows<FP16, 256, 4, LN>(p, st);
  if constexpr (!LN) {
    if (chunks <= 1536) return launch_rows<FP16, 256, 6, false>(p, st);
    if (chunks <= 2048) return launch_rows<FP16, 256, 8, false>(p, st);
    const long long blocks = p.rows < 148LL * 8 ? p.rows : 148LL * 8;
    return launch_overlapped(int8_long_rows_kernel<FP16>, dim3(static_cast<unsigned>(blocks)), dim3(kRowThreads), 0, st, 1, p);
  }
  return cudaErrorInvalidValue;
}

bool misaligned(const void* p, int64_t stride) { return (reinterpret_cast<uintptr_t>(p) & 15) != 0 || stride % 8 != 0; }

int check_rows(int dtype, const void* x, const void* q, const void* scale, int64_t rows, int64_t dim, int64_t rows_per_batch,
               int64_t q_row_stride) {
  if (dtype != HDIT_BF16 && dtype != HDIT_FP16) return set_error(HDIT_ERR_BAD_ARG, "dtype must be bf16 or fp16");
  if (rows < 0 || dim <= 0 || rows_per_batch <= 0) return set_error(HDIT_ERR_BAD_ARG, "bad sizes");
  if (rows > 0 && (x == nullptr || q == nullptr || scale == nullptr)) return set_error(HDIT_ERR_BAD_ARG, "null x / q / scale");
  if (dim > 0x3fffffffLL) return set_error(HDIT_ERR_TOO_LARGE, "row length must fit 30 bits");
  if ((reinterpret_cast<uintptr_t>(q) & 15) != 0 || q_row_stride % 16 != 0 || q_row_stride < dim)
    return set_error(HDIT_ERR_SHAPE, "8-bit rows need a 16-byte aligned pointer and a row stride that is a multiple of 16 and covers a row");
  if ((reinterpret_cast<uintptr_t>(scale) & 3) != 0 || (reinterpret_cast<uintptr_t>(x) & 1) != 0)
    return set_error(HDIT_ERR_SHAPE, "x / scale not aligned to their elements");
  return HDIT_OK;
}

}  // namespace
}  // namespace hdit

extern "C" int hdit_quantize_rows(int32_t dtype, const void* x, void* q, float* scale, int64_t rows, int64_t dim,
                                  int64_t rows_per_batch, int64_t x_batch_stride, int64_t x_row_stride, int64_t q_row_stride,
                                  void* stream) {
  using namespace hdit;
  const int rc = check_rows(dtype, x, q, scale, rows, dim, rows_per_batch, q_row_stride);
  if (rc != HDIT_OK || rows == 0) return rc;
  RowsParams p{static_cast<const uint16_t*>(x), nullptr, nullptr, static_cast<int8_t*>(q), scale, rows, rows_per_batch, x_batch_stride,
               x_row_stride, q_row_stride, 0, static_cast<int>(dim), 0.f, !misaligned(x, x_row_stride) && x_batch_stride % 8 == 0};
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  HDIT_CUDA_OK((dtype == HDIT_FP16 ? launch_any<true, false>(p, st) : launch_any<false, false>(p, st)));
  return HDIT_OK;
}

extern "C" int hdit_ln_modulate_int8(int32_t dtype, const void* x, const void* shift, const void* scale, void* q, float* q_scale,
                                     int64_t rows, int64_t dim, int64_t rows_per_batch, int64_t x_batch_stride,
                                     int64_t x_row_stride, int64_t q_row_stride, int64_t mod_batch_stride, float eps, void* stream) {
  using namespace hdit;
  const int rc = check_rows(dtype, x, q, q_scale, rows, dim, rows_per_batch, q_row_stride);
  if (rc != HDIT_OK) return rc;
  if (dim % 8 != 0 || dim > 8192) return set_error(HDIT_ERR_SHAPE, "row length must be a multiple of 8 and at most 8192");
  if (rows == 0) return HDIT_OK;
  if (shift == nullptr || scale == nullptr) return set_error(HDIT_ERR_BAD_ARG, "null shift / scale");
  if (((reinterpret_cast<uintptr_t>(shift) | reinterpret_cast<uintptr_t>(scale)) & 1) != 0)
    return set_error(HDIT_ERR_SHAPE, "shift / scale not aligned to their elements");
  const bool vec = !misaligned(x, x_row_stride) && x_batch_stride % 8 == 0 && !misaligned(shift, mod_batch_stride) && !misaligned(scale, mod_batch_stride);
  RowsParams p{static_cast<const uint16_t*>(x), static_cast<const uint16_t*>(shift), static_cast<const uint16_t*>(scale),
               static_cast<int8_t*>(q), q_scale, rows, rows_per_batch, x_batch_stride, x_row_stride, q_row_stride, mod_batch_stride,
               static_cast<int>(dim), eps, vec};
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  HDIT_CUDA_OK((dtype == HDIT_FP16 ? launch_any<true, true>(p, st) : launch_any<false, true>(p, st)));
  return HDIT_OK;
}
