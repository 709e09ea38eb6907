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

#include <type_traits>

#include "host_common.h"
#include "int8_rows.cuh"

namespace hdit {
namespace {

constexpr int kMaxNormDim = 8192;

struct RowsParams {
  const uint16_t* x;
  const uint16_t* x_end;  // the end of the last row
  const uint16_t* shift;  // ln_modulate_int8 only
  const uint16_t* scale;
  int8_t* q;
  float* q_scale;
  long long batches, rows_per_batch, x_batch_stride, x_row_stride, q_row_stride, mod_batch_stride;
  int dim;
  float eps;
  bool mod_vec;  // shift and scale of a batch entry start on 16-byte boundaries
};

// CTAs that are to fit an SM beside one another
constexpr int rows_ctas(int nch, bool ln, bool vec) { return ln || !vec ? (nch <= 2 ? 4 : nch <= 4 ? 3 : 2) : nch <= 4 ? 4 : 2; }

// TEAM threads hold a row of at most TEAM * NCH * 8 elements as the 16-bit values that were read, and have the next row on its
// way while they work on one. What a row costs beside its elements (reductions, divisions, addresses) is paid by every warp of
// the team, so a thread has up to 32 elements: with eight a thread 8192 x 1536 with the norm took 28 us, with a warp to a row, 128
// registers and no row ahead 20, in this form 11. Rows that start anywhere come as 16-byte blocks whose bits are moved into place (VEC
// false without LN). Modulation vectors wait in shared memory as fp32 (1 + scale, shift); a CTA stays with
// one batch entry at a time.
template <bool FP16, int TEAM, int NCH, bool LN, bool VEC>
__global__ void __launch_bounds__(kRowThreads, rows_ctas(NCH, LN, VEC)) int8_rows_kernel(const __grid_constant__ RowsParams p) {
  grid_dependency_release();
  grid_dependency_wait();
  // 1 + scale, then shift: first the lower four columns of every chunk, then the upper four, so that the lanes' 16 bytes lie
  // side by side
  extern __shared__ float4 mods[];
  __shared__ float red[3][kRowThreads / 32];
  const Team<TEAM> team{red};
  constexpr int kTeams = kRowThreads / TEAM;
  const int col0 = static_cast<int>(threadIdx.x % TEAM) * 8;
  const long long first = static_cast<long long>(blockIdx.x) * kTeams + threadIdx.x / TEAM, step = static_cast<long long>(gridDim.x) * kTeams;
  const float inv_dim = 1.f / static_cast<float>(p.dim);
  const int chunks = p.dim / 8;
  int turn = 0;  // goes on from entry to entry: without the norm no other barrier stands between the last row of one and the first of the next
  for (long long b = blockIdx.y; b < p.batches; b += gridDim.y) {
    const uint16_t* xr = p.x + b * p.x_batch_stride + first * p.x_row_stride;
    const long long row0 = b * p.rows_per_batch;
    constexpr bool kBlocks = !LN && !VEC;
    using Next = std::conditional_t<kBlocks, Int8Blocks, uint4>;
    Next next[NCH];
    auto fetch = [&] {
#pragma unroll
      for (int c = 0; c < NCH; ++c) {
        next[c] = Next{};
        if (col0 + c * TEAM * 8 >= p.dim) continue;
        if constexpr (kBlocks) next[c] = int8_load_blocks(xr, col0 + c * TEAM * 8, p.dim, p.x, p.x_end);
        else next[c] = int8_load8(xr, col0 + c * TEAM * 8, p.dim, VEC);
      }
    };
    if (first < p.rows_per_batch) fetch();
    if constexpr (LN) {
      __syncthreads();
      for (int k = threadIdx.x; k < chunks; k += kRowThreads) {
        const uint4 g4 = int8_load8(p.scale + b * p.mod_batch_stride, k * 8, p.dim, p.mod_vec), a4 = int8_load8(p.shift + b * p.mod_batch_stride, k * 8, p.dim, p.mod_vec);
        const uint32_t* g = reinterpret_cast<const uint32_t*>(&g4);
        const uint32_t* a = reinterpret_cast<const uint32_t*>(&a4);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const float2 g0 = int8_unpack2<FP16>(g[2 * h]), g1 = int8_unpack2<FP16>(g[2 * h + 1]);
          const float2 a0 = int8_unpack2<FP16>(a[2 * h]), a1 = int8_unpack2<FP16>(a[2 * h + 1]);
          mods[h * chunks + k] = make_float4(1.f + g0.x, 1.f + g0.y, 1.f + g1.x, 1.f + g1.y);
          mods[(2 + h) * chunks + k] = make_float4(a0.x, a0.y, a1.x, a1.y);
        }
      }
      __syncthreads();
    }
    for (long long r = first; r < p.rows_per_batch; r += step, turn ^= 1) {
      uint4 raw[NCH];
#pragma unroll
      for (int c = 0; c < NCH; ++c) {
        if constexpr (kBlocks) raw[c] = int8_from_blocks(next[c], xr, col0 + c * TEAM * 8, p.dim);
        else raw[c] = next[c];
      }
      xr += step * p.x_row_stride;
      if (r + step < p.rows_per_batch) fetch();
      int8_t* const qr = p.q + (row0 + r) * p.q_row_stride;
      Int8Scale s;
      if constexpr (!LN) {
        // magnitudes of two 16-bit values at a time, as integers
        uint32_t top2 = 0;
#pragma unroll
        for (int c = 0; c < NCH; ++c) {
          const uint32_t* u = reinterpret_cast<const uint32_t*>(&raw[c]);
#pragma unroll
          for (int i = 0; i < 4; ++i) top2 = __vmaxu2(top2, u[i] & 0x7FFF7FFFu);
        }
        const uint32_t top16 = team.max((top2 & 0xFFFFu) > (top2 >> 16) ? top2 & 0xFFFFu : top2 >> 16, turn);
        s = int8_scale(__float_as_uint(int8_unpack2<FP16>(top16).x));
        const float inv17 = 17.f * s.inv;
#pragma unroll
        for (int c = 0; c < NCH; ++c) {
          if (col0 + c * TEAM * 8 >= p.dim) continue;
          int8_put8<FP16, !VEC>(qr, col0 + c * TEAM * 8, p.dim, s, inv17, raw[c]);
        }
      } else {
        float2 y[NCH][4];  // x, its distance from the mean, the result
        float2 sum = both(0.f);
#pragma unroll
        for (int c = 0; c < NCH; ++c) {
          const uint32_t* u = reinterpret_cast<const uint32_t*>(&raw[c]);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            y[c][i] = int8_unpack2<FP16>(u[i]);
            sum = add2(sum, y[c][i]);
          }
        }
        const float mean = team.sum(sum.x + sum.y, 0) * inv_dim;
        float2 sq = both(0.f);
#pragma unroll
        for (int c = 0; c < NCH; ++c)
          if (col0 + c * TEAM * 8 < p.dim) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              y[c][i] = add2(y[c][i], both(-mean));
              sq = fma2(y[c][i], y[c][i], sq);
            }
          }
        const float rstd = rsqrtf(team.sum(sq.x + sq.y, 1) * inv_dim + p.eps);
        float top = 0.f;
#pragma unroll
        for (int c = 0; c < NCH; ++c) {
          const int col = col0 + c * TEAM * 8;
          if (col >= p.dim) continue;
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const float4 g = mods[h * chunks + (col >> 3)], a = mods[(2 + h) * chunks + (col >> 3)];
            float2* v = &y[c][2 * h];
            v[0] = fma2(mul2(v[0], both(rstd)), make_float2(g.x, g.y), make_float2(a.x, a.y));
            v[1] = fma2(mul2(v[1], both(rstd)), make_float2(g.z, g.w), make_float2(a.z, a.w));
          }
#pragma unroll
          for (int i = 0; i < 4; ++i) top = max_magnitude(max_magnitude(top, y[c][i].x), y[c][i].y);
        }
        s = int8_scale(team.max(__float_as_uint(top) & 0x7FFFFFFFu, 2));
#pragma unroll
        for (int c = 0; c < NCH; ++c)
          if (col0 + c * TEAM * 8 < p.dim) int8_put8_of(qr, col0 + c * TEAM * 8, s, y[c]);
      }
      if (col0 == 0) p.q_scale[row0 + r] = int8_step(s);
    }
  }
}

// Rows of any length: read twice, the second time from the caches.
template <bool FP16>
__global__ void __launch_bounds__(kRowThreads) int8_any_rows_kernel(const __grid_constant__ RowsParams p) {
  grid_dependency_release();
  grid_dependency_wait();
  __shared__ float red[2][kRowThreads / 32];
  const Team<kRowThreads> team{red};
  int turn = 0;
  for (long long b = blockIdx.y; b < p.batches; b += gridDim.y)
    for (long long r = blockIdx.x; r < p.rows_per_batch; r += gridDim.x, turn ^= 1) {
      const uint16_t* xr = p.x + b * p.x_batch_stride + r * p.x_row_stride;
      const long long row = b * p.rows_per_batch + r;
      int8_t* const qr = p.q + row * p.q_row_stride;
      uint32_t top = 0;
      for (int c = threadIdx.x; c < p.dim; c += kRowThreads) top = max(top, xr[c] & 0x7FFFu);
      const Int8Scale s = int8_scale(__float_as_uint(int8_unpack2<FP16>(team.max(top, turn)).x));
      const float inv17 = 17.f * s.inv;
      for (int c = threadIdx.x * 4; c < p.dim; c += kRowThreads * 4) {
        float2 t[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const float2 v = make_float2(c + 2 * i < p.dim ? int8_unpack2<FP16>(xr[c + 2 * i]).x : 0.f,
                                       c + 2 * i + 1 < p.dim ? int8_unpack2<FP16>(xr[c + 2 * i + 1]).x : 0.f);
          t[i] = add2(int8_steps_of_16bit(v, s.inv, inv17), both(kInt8Round));
        }
        const uint32_t v = s.inv == 0.f ? 0u : int8_bytes(t[0], t[1]);
        if (c + 4 <= p.dim) {
          *reinterpret_cast<uint32_t*>(qr + c) = v;
        } else {
          for (int i = 0; c + i < p.dim; ++i) qr[c + i] = static_cast<int8_t>((v >> (8 * i)) & 0xFFu);
        }
      }
      if (threadIdx.x == 0) p.q_scale[row] = int8_step(s);
    }
}

// CTAs for `ctas` beside one another on every SM over all batch entries, no more than there are rows for.
dim3 rows_grid(const RowsParams& p, long long teams, long long ctas) {
  const long long y = p.batches < 65535 ? p.batches : 65535;
  long long x = (148 * ctas + y - 1) / y;
  const long long most = (p.rows_per_batch + teams - 1) / teams;
  return dim3(static_cast<unsigned>(x < most ? x : most), static_cast<unsigned>(y));
}

template <bool FP16, int TEAM, int NCH, bool LN, bool VEC>
cudaError_t launch_rows(const RowsParams& p, cudaStream_t st) {
  constexpr auto kernel = int8_rows_kernel<FP16, TEAM, NCH, LN, VEC>;
  const size_t smem = LN ? static_cast<size_t>(p.dim) * 2 * sizeof(float) : 0;
  if (smem > 47 * 1024) {
    const cudaError_t e = allow_shared_memory<kernel, kMaxNormDim * 2 * static_cast<int>(sizeof(float))>();
    if (e != cudaSuccess) return e;
  }
  return launch_overlapped(kernel, rows_grid(p, kRowThreads / TEAM, rows_ctas(NCH, LN, VEC)), dim3(kRowThreads), smem, st, 1, p);
}

template <bool FP16, bool VEC>
cudaError_t launch_plain(const RowsParams& p, cudaStream_t st) {
  const int chunks = (p.dim + 7) / 8;
  if (chunks <= 32) return launch_rows<FP16, 32, 1, false, VEC>(p, st);
  if (chunks <= 64) return launch_rows<FP16, 32, 2, false, VEC>(p, st);
  if (chunks <= 96) return launch_rows<FP16, 32, 3, false, VEC>(p, st);
  if (chunks <= 128) return launch_rows<FP16, 32, 4, false, VEC>(p, st);
  if (chunks <= 192) return launch_rows<FP16, 64, 3, false, VEC>(p, st);
  if (chunks <= 256) return launch_rows<FP16, 64, 4, false, VEC>(p, st);
  if (chunks <= 384) return launch_rows<FP16, 128, 3, false, VEC>(p, st);
  if (chunks <= 512) return launch_rows<FP16, 128, 4, false, VEC>(p, st);
  if (chunks <= 768) return launch_rows<FP16, 256, 3, false, VEC>(p, st);
  if (chunks <= 1024) return launch_rows<FP16, 256, 4, false, VEC>(p, st);
  if (chunks <= 2048) return launch_rows<FP16, 256, 8, false, VEC>(p, st);
  return launch_overlapped(int8_any_rows_kernel<FP16>, rows_grid(p, 1, 8), dim3(kRowThreads), 0, st, 1, p);
}

// Unaligned rows: the teams, and so the sums, of aligned ones.
template <bool FP16, bool VEC>
cudaError_t launch_ln(const RowsParams& p, cudaStream_t st) {
  const int chunks = p.dim / 8;
  if (VEC && chunks <= 32) return launch_rows<FP16, 32, 1, true, true>(p, st);
  if (VEC && chunks <= 64) return launch_rows<FP16, 32, 2, true, true>(p, st);
  if (VEC && chunks <= 128) return launch_rows<FP16, 32, 4, true, true>(p, st);
  if (VEC && chunks <= 192) return launch_rows<FP16, 32, 6, true, true>(p, st);
  if (chunks <= 256) return launch_rows<FP16, 32, 8, true, VEC>(p, st);
  if (VEC && chunks <= 384) return launch_rows<FP16, 64, 6, true, true>(p, st);
  if (chunks <= 512) return launch_rows<FP16, 64, 8, true, VEC>(p, st);
  if (VEC && chunks <= 768) return launch_rows<FP16, 128, 6, true, true>(p, st);
  return launch_rows<FP16, 128, 8, true, VEC>(p, st);
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
  const bool flat = rows <= rows_per_batch || x_batch_stride == rows_per_batch * x_row_stride;  // one stride for all rows
  if (!flat && rows % rows_per_batch != 0) return set_error(HDIT_ERR_SHAPE, "rows must be a multiple of rows_per_batch");
  const long long batches = flat ? 1 : rows / rows_per_batch, per = flat ? rows : rows_per_batch;
  const uint16_t* const x_end = static_cast<const uint16_t*>(x) + (batches - 1) * x_batch_stride + (per - 1) * x_row_stride + dim;
  RowsParams p{static_cast<const uint16_t*>(x), x_end, nullptr, nullptr, static_cast<int8_t*>(q), scale, batches, per,
               x_batch_stride, x_row_stride, q_row_stride, 0, static_cast<int>(dim), 0.f, false};
  const bool vec = dim % 8 == 0 && !misaligned(x, x_row_stride) && (flat || x_batch_stride % 8 == 0);
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  HDIT_CUDA_OK((dtype == HDIT_FP16 ? (vec ? launch_plain<true, true>(p, st) : launch_plain<true, false>(p, st))
                                   : (vec ? launch_plain<false, true>(p, st) : launch_plain<false, false>(p, st))));
  return HDIT_OK;
}

extern "C" int hdit_ln_modulate_int8(int32_t dtype, const void* x, const void* shift, const void* scale, void* q, float* q_scale,
                                     int64_t rows, int64_t dim, int64_t rows_per_batch, int64_t x_batch_stride,
                                     int64_t x_row_stride, int64_t q_row_stride, int64_t mod_batch_stride, float eps, void* stream) {
  using namespace hdit;
  const int rc = check_rows(dtype, x, q, q_scale, rows, dim, rows_per_batch, q_row_stride);
  if (rc != HDIT_OK) return rc;
  if (dim % 8 != 0 || dim > kMaxNormDim) return set_error(HDIT_ERR_SHAPE, "row length must be a multiple of 8 and at most %d", kMaxNormDim);
  if (rows == 0) return HDIT_OK;
  if (shift == nullptr || scale == nullptr) return set_error(HDIT_ERR_BAD_ARG, "null shift / scale");
  if (((reinterpret_cast<uintptr_t>(shift) | reinterpret_cast<uintptr_t>(scale)) & 1) != 0)
    return set_error(HDIT_ERR_SHAPE, "shift / scale not aligned to their elements");
  if (rows > rows_per_batch && rows % rows_per_batch != 0) return set_error(HDIT_ERR_SHAPE, "rows must be a multiple of rows_per_batch");
  const bool one = rows <= rows_per_batch;
  RowsParams p{static_cast<const uint16_t*>(x), nullptr, static_cast<const uint16_t*>(shift), static_cast<const uint16_t*>(scale),
               static_cast<int8_t*>(q), q_scale, one ? 1 : rows / rows_per_batch, one ? rows : rows_per_batch, x_batch_stride, x_row_stride,
               q_row_stride, mod_batch_stride, static_cast<int>(dim), eps, !misaligned(shift, mod_batch_stride) && !misaligned(scale, mod_batch_stride)};
  const bool vec = !misaligned(x, x_row_stride) && (one || x_batch_stride % 8 == 0);
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  HDIT_CUDA_OK((dtype == HDIT_FP16 ? (vec ? launch_ln<true, true>(p, st) : launch_ln<true, false>(p, st))
                                   : (vec ? launch_ln<false, true>(p, st) : launch_ln<false, false>(p, st))));
  return HDIT_OK;
}
