// GroupNorm over channels-last images, with an activation, or with its rows (all channels of a pixel) as 8-bit integers
// (int8_rows.cuh) for a linear layer that follows:
//   y[b, r, c] = (x[b, r, c] - mean[b, g]) / sqrt(var[b, g] + eps) * weight[c] + bias[c],   g = c / (channels / groups)
// over rows r (pixels) and the channels of a group; biased variance.
//
// Two launches. The first one reads x once: a CTA takes a strip of rows of one image, each thread eight fixed channels, and
// leaves {mean, sum of squared distances from it} per group and strip. Sums are taken relative to the strip's first row, so
// that a mean far from zero costs no digits. The second one joins the strips (Chan's formula) and reads x again, each strip
// from its end to its start: what the first launch read last is still in L2.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include "host_common.h"
#include "int8_rows.cuh"

namespace hdit {
namespace {

constexpr int kMaxChannels = 4096;
constexpr int kGnThreads = 256;  // 512 for more than 2048 channels: a thread has eight of them

struct GnParams {
  const uint16_t* x;
  const uint16_t* weight;  // or null: 1
  const uint16_t* bias;    // or null: 0
  uint16_t* out;
  int8_t* q;
  float* q_scale;
  float2* partial;  // (batch, strips, groups): mean, sum of squared distances from it
  long long rows, x_batch_stride, x_row_stride, out_batch_stride, out_row_stride;  // q: out_row_stride only, rows of all images
  long long strip_rows;
  int strips, channels, groups, act;
  float eps;
  bool vec;
};

// Calls f(group, sub, n_sub) in groups of n_sub consecutive threads of a warp, the same number of times in all threads.
template <typename F>
__device__ __forceinline__ void for_groups(int groups, F f) {
  int n_sub = 32;
  while (n_sub > 1 && groups * n_sub > static_cast<int>(blockDim.x)) n_sub >>= 1;
  const int at_once = static_cast<int>(blockDim.x) / n_sub;
  for (int g0 = 0; g0 < groups; g0 += at_once) f(g0 + static_cast<int>(threadIdx.x) / n_sub, static_cast<int>(threadIdx.x) % n_sub, n_sub);
}
__device__ __forceinline__ float sub_sum(float v, int n_sub) {
  for (int o = n_sub >> 1; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

template <bool FP16>
__global__ void __launch_bounds__(512) group_norm_stats_kernel(const __grid_constant__ GnParams p) {
  grid_dependency_release();
  grid_dependency_wait();
  extern __shared__ float smem[];  // [lanes][channels] sums, then the same of squares
  const int chunks = p.channels / 8;
  const int lanes = static_cast<int>(blockDim.x) / chunks;  // rows at a time
  const int chunk = threadIdx.x % chunks, lane = threadIdx.x / chunks;
  const long long r0 = static_cast<long long>(blockIdx.x) * p.strip_rows;
  const long long r1 = r0 + p.strip_rows < p.rows ? r0 + p.strip_rows : p.rows;
  const uint16_t* xb = p.x + blockIdx.y * p.x_batch_stride;
  const int c = chunk * 8;
  float s[8], ss[8], pivot[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) s[i] = ss[i] = 0.f;
  if (lane < lanes) {
    const uint4 first = int8_load8(xb + r0 * p.x_row_stride, c, p.channels, p.vec);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 v = int8_unpack2<FP16>(reinterpret_cast<const uint32_t*>(&first)[i]);
      pivot[2 * i] = v.x;
      pivot[2 * i + 1] = v.y;
    }
    constexpr int kAhead = 4;  // rows in flight
    for (long long r = r0 + lane; r < r1; r += static_cast<long long>(kAhead) * lanes) {
      uint4 raw[kAhead];
#pragma unroll
      for (int k = 0; k < kAhead; ++k)
        raw[k] = r + static_cast<long long>(k) * lanes < r1 ? int8_load8(xb + (r + static_cast<long long>(k) * lanes) * p.x_row_stride, c, p.channels, p.vec) : first;
#pragma unroll
      for (int k = 0; k < kAhead; ++k) {
        const uint32_t* u = reinterpret_cast<const uint32_t*>(&raw[k]);
        if (r + static_cast<long long>(k) * lanes < r1) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float2 v = int8_unpack2<FP16>(u[i]);
            const float d0 = v.x - pivot[2 * i], d1 = v.y - pivot[2 * i + 1];
            s[2 * i] += d0;
            ss[2 * i] = fmaf(d0, d0, ss[2 * i]);
            s[2 * i + 1] += d1;
            ss[2 * i + 1] = fmaf(d1, d1, ss[2 * i + 1]);
          }
        }
      }
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      smem[lane * p.channels + c + i] = s[i];
      smem[(lanes + lane) * p.channels + c + i] = ss[i];
    }
  }
  __syncthreads();
  // per channel: mean and sum of squared distances from it, in the first lane's places
  const float n = static_cast<float>(r1 - r0);
  for (int ch = threadIdx.x; ch < p.channels; ch += blockDim.x) {
    float a = 0.f, q = 0.f;
    for (int l = 0; l < lanes; ++l) {
      a += smem[l * p.channels + ch];
      q += smem[(lanes + l) * p.channels + ch];
    }
    uint16_t first = xb[r0 * p.x_row_stride + ch];
    smem[ch] = int8_unpack2<FP16>(first).x + a / n;
    smem[lanes * p.channels + ch] = fmaxf(q - a * a / n, 0.f) + (q - q);  // keeps NaN
  }
  __syncthreads();
  const int per = p.channels / p.groups;
  float2* out = p.partial + (static_cast<long long>(blockIdx.y) * p.strips + blockIdx.x) * p.groups;
  for_groups(p.groups, [&](int g, int sub, int n_sub) {
    const bool live = g < p.groups;
    float mean = 0.f, m2 = 0.f;
    for (int k = sub; live && k < per; k += n_sub) mean += smem[g * per + k];
    mean = sub_sum(mean, n_sub) / static_cast<float>(per);
    for (int k = sub; live && k < per; k += n_sub) {
      const float d = smem[g * per + k] - mean;
      m2 += smem[lanes * p.channels + g * per + k] + n * d * d;
    }
    m2 = sub_sum(m2, n_sub);
    if (live && sub == 0) out[g] = make_float2(mean, m2);
  });
}

// {mean, 1 / deviation} of every group of image b into stat[groups].
__device__ __forceinline__ void group_norm_join(const GnParams& p, int b, float2* stat) {
  const float2* in = p.partial + static_cast<long long>(b) * p.strips * p.groups;
  const float per = static_cast<float>(p.channels / p.groups);
  const float n_full = static_cast<float>(p.strip_rows) * per;
  const float n_last = static_cast<float>(p.rows - p.strip_rows * (p.strips - 1)) * per;
  const float total = static_cast<float>(p.rows) * per;
  for_groups(p.groups, [&](int g, int sub, int n_sub) {
    const bool live = g < p.groups;
    const float base = live ? in[g].x : 0.f;
    float a = 0.f, q = 0.f;
    for (int k = sub; live && k < p.strips; k += n_sub) {
      const float2 v = in[static_cast<long long>(k) * p.groups + g];
      const float d = v.x - base, n = k == p.strips - 1 ? n_last : n_full;
      a = fmaf(n, d, a);
      q += fmaf(n * d, d, v.y);
    }
    a = sub_sum(a, n_sub);
    q = sub_sum(q, n_sub);
    const float far = a / total;  // of the mean from the first strip's
    const float var = q / total - far * far;
    if (live && sub == 0) stat[g] = make_float2(base + far, rsqrtf((var > 0.f ? var : var - var) + p.eps));
  });
}

// y = x * a + b with a = weight / deviation and b = bias - mean * a. Against (x - mean) * a + bias that costs half a unit of
// 2^-24 of mean * a: a 16-bit x resolves the deviation only while |mean| is below some 2^11 deviations, where this is
// under 2^-13 of the result's deviation.
template <bool FP16>
__device__ __forceinline__ float2 group_norm_factors(const GnParams& p, const float2* stat, int c) {
  const float2 st = stat[c / (p.channels / p.groups)];
  const uint32_t w = p.weight != nullptr ? p.weight[c] : (FP16 ? 0x3C00u : 0x3F80u), bi = p.bias != nullptr ? p.bias[c] : 0u;
  const float a = st.y * int8_unpack2<FP16>(w).x;
  return make_float2(a, fmaf(-st.x, a, int8_unpack2<FP16>(bi).x));
}

__device__ __forceinline__ float silu(float y) { return __fdividef(y, 1.f + __expf(-y)); }

template <bool FP16>
__device__ __forceinline__ uint32_t gn_pack(float lo, float hi) {
  if constexpr (FP16) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
  } else {
    const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
}

template <bool FP16, bool SILU>
__global__ void __launch_bounds__(512) group_norm_apply_kernel(const __grid_constant__ GnParams p) {
  grid_dependency_release();
  grid_dependency_wait();
  extern __shared__ float smem[];
  float2* stat = reinterpret_cast<float2*>(smem);
  group_norm_join(p, blockIdx.y, stat);
  __syncthreads();
  const int chunks = p.channels / 8;
  const int lanes = static_cast<int>(blockDim.x) / chunks;
  const int chunk = threadIdx.x % chunks, lane = threadIdx.x / chunks;
  if (lane >= lanes) return;
  const int c = chunk * 8;
  float a[8], b[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float2 f = group_norm_factors<FP16>(p, stat, c + i);
    a[i] = f.x;
    b[i] = f.y;
  }
  const long long r0 = static_cast<long long>(blockIdx.x) * p.strip_rows;
  const long long r1 = r0 + p.strip_rows < p.rows ? r0 + p.strip_rows : p.rows;
  const uint16_t* xb = p.x + blockIdx.y * p.x_batch_stride;
  uint16_t* ob = p.out + blockIdx.y * p.out_batch_stride;
  constexpr int kAhead = 4;
  for (long long r = r1 - 1 - lane; r >= r0; r -= static_cast<long long>(kAhead) * lanes) {
    uint4 raw[kAhead];
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      const long long rk = r - static_cast<long long>(k) * lanes;
      raw[k] = rk >= r0 ? int8_load8(xb + rk * p.x_row_stride, c, p.channels, p.vec) : make_uint4(0, 0, 0, 0);
    }
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      const long long rk = r - static_cast<long long>(k) * lanes;
      if (rk < r0) break;
      uint32_t* u = reinterpret_cast<uint32_t*>(&raw[k]);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 v = int8_unpack2<FP16>(u[i]);
        float y0 = fmaf(v.x, a[2 * i], b[2 * i]), y1 = fmaf(v.y, a[2 * i + 1], b[2 * i + 1]);
        if constexpr (SILU) y0 = silu(y0), y1 = silu(y1);
        u[i] = gn_pack<FP16>(y0, y1);
      }
      uint16_t* dst = ob + rk * p.out_row_stride + c;
      if (p.vec) {
        *reinterpret_cast<uint4*>(dst) = raw[k];
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) dst[i] = static_cast<uint16_t>(u[i / 2] >> (16 * (i & 1)));
      }
    }
  }
}

// The rows in 8 bits: TEAM threads hold a row of at most TEAM * NCH * 8 channels; factors of all channels in shared memory.
template <bool FP16, bool SILU, int TEAM, int NCH>
__global__ void __launch_bounds__(kRowThreads) group_norm_int8_kernel(const __grid_constant__ GnParams p) {
  grid_dependency_release();
  grid_dependency_wait();
  extern __shared__ float smem[];  // a[channels], b[channels], then {mean, 1 / deviation}[groups]
  __shared__ float red[2][kRowThreads / 32];
  float* fa = smem;
  float* fb = smem + p.channels;
  float2* stat = reinterpret_cast<float2*>(smem + 2 * p.channels);
  group_norm_join(p, blockIdx.y, stat);
  __syncthreads();
  for (int c = threadIdx.x; c < p.channels; c += kRowThreads) {
    const float2 f = group_norm_factors<FP16>(p, stat, c);
    fa[c] = f.x;
    fb[c] = f.y;
  }
  __syncthreads();
  const Team<TEAM> team{red};
  constexpr int kTeams = kRowThreads / TEAM;
  const int lane = threadIdx.x % TEAM;
  const long long r0 = static_cast<long long>(blockIdx.x) * p.strip_rows;
  const long long r1 = r0 + p.strip_rows < p.rows ? r0 + p.strip_rows : p.rows;
  const uint16_t* xb = p.x + blockIdx.y * p.x_batch_stride;
  int turn = 0;
  for (long long rt = r1 - kTeams; rt > r0 - kTeams; rt -= kTeams, turn ^= 1) {
    const long long r = rt + threadIdx.x / TEAM;
    const bool live = r >= r0;
    float y[NCH][8];
    float top = 0.f;
#pragma unroll
    for (int k = 0; k < NCH; ++k) {
      const int c = (k * TEAM + lane) * 8;
      if (live && c < p.channels) {
        const uint4 raw = int8_load8(xb + r * p.x_row_stride, c, p.channels, p.vec);
        const uint32_t* u = reinterpret_cast<const uint32_t*>(&raw);
        const float4* a4 = reinterpret_cast<const float4*>(fa + c);
        const float4* b4 = reinterpret_cast<const float4*>(fb + c);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const float4 av = a4[h], bv = b4[h];
          const float2 v0 = int8_unpack2<FP16>(u[2 * h]), v1 = int8_unpack2<FP16>(u[2 * h + 1]);
          y[k][4 * h] = fmaf(v0.x, av.x, bv.x);
          y[k][4 * h + 1] = fmaf(v0.y, av.y, bv.y);
          y[k][4 * h + 2] = fmaf(v1.x, av.z, bv.z);
          y[k][4 * h + 3] = fmaf(v1.y, av.w, bv.w);
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          if constexpr (SILU) y[k][i] = silu(y[k][i]);
          top = max_magnitude(top, y[k][i]);
        }
      }
    }
    const Int8Scale s = int8_scale(team.max(__float_as_uint(top) & 0x7FFFFFFFu, turn));
    if (live) {
      const long long row = blockIdx.y * p.rows + r;
#pragma unroll
      for (int k = 0; k < NCH; ++k) {
        const int c = (k * TEAM + lane) * 8;
        if (c < p.channels) {
          int8_put8_of(p.q + row * p.out_row_stride, c, s, y[k]);
        }
      }
      if (lane == 0) p.q_scale[row] = int8_step(s);
    }
  }
}

int gn_threads(int channels) { return channels > 2048 ? 512 : kGnThreads; }

// Strips per image: four CTAs per SM over all images, at least sixteen rows of every thread's channels each.
int strips_of(long long batch, long long rows, int channels) {
  const long long lanes = gn_threads(channels) / (channels / 8);
  long long n = (148 * 4 + batch - 1) / batch;
  const long long most = (rows + lanes * 16 - 1) / (lanes * 16);
  if (n > most) n = most;
  return static_cast<int>(n < 1 ? 1 : n);
}

int check_gn(int dtype, const void* x, const void* out, const void* partial, int64_t batch, int64_t rows, int64_t channels, int64_t groups,
             int act) {
  if (dtype != HDIT_BF16 && dtype != HDIT_FP16) return set_error(HDIT_ERR_BAD_ARG, "dtype must be bf16 or fp16");
  if (batch < 0 || rows < 0 || channels <= 0 || groups <= 0) return set_error(HDIT_ERR_BAD_ARG, "bad sizes");
  if (act != HDIT_ACT_NONE && act != HDIT_ACT_SILU) return set_error(HDIT_ERR_BAD_ARG, "unknown activation %d", act);
  if (channels % 8 != 0 || channels > kMaxChannels || channels % groups != 0)
    return set_error(HDIT_ERR_SHAPE, "channels must be a multiple of 8 and of groups, at most %d", kMaxChannels);
  if (batch > 65535 || rows > 0x7fffffffLL) return set_error(HDIT_ERR_TOO_LARGE, "at most 65535 images of 2^31 - 1 rows");
  if (batch == 0 || rows == 0) return HDIT_OK;
  if (x == nullptr || out == nullptr || partial == nullptr) return set_error(HDIT_ERR_BAD_ARG, "null x / out / scratch");
  if ((reinterpret_cast<uintptr_t>(partial) & 7) != 0) return set_error(HDIT_ERR_SHAPE, "scratch not 8-byte aligned");
  return HDIT_OK;
}

bool off16(const void* p, int64_t a, int64_t b) { return (reinterpret_cast<uintptr_t>(p) & 15) != 0 || a % 8 != 0 || b % 8 != 0; }

cudaError_t launch_stats(const GnParams& p, bool fp16, long long batch, cudaStream_t st) {
  const int threads = gn_threads(p.channels);
  const size_t smem = static_cast<size_t>(threads / (p.channels / 8)) * p.channels * 2 * sizeof(float);
  return launch_overlapped(fp16 ? group_norm_stats_kernel<true> : group_norm_stats_kernel<false>,
                           dim3(static_cast<unsigned>(p.strips), static_cast<unsigned>(batch)), dim3(static_cast<unsigned>(threads)), smem, st, 1, p);
}

template <bool FP16, bool SILU>
cudaError_t launch_int8(const GnParams& p, long long batch, cudaStream_t st) {
  const size_t smem = static_cast<size_t>(p.channels) * 2 * sizeof(float) + static_cast<size_t>(p.groups) * sizeof(float2);
  auto kernel = p.channels <= 256    ? group_norm_int8_kernel<FP16, SILU, 32, 1>
                : p.channels <= 512  ? group_norm_int8_kernel<FP16, SILU, 32, 2>
                : p.channels <= 1024 ? group_norm_int8_kernel<FP16, SILU, 32, 4>
                : p.channels <= 2048 ? group_norm_int8_kernel<FP16, SILU, 128, 2>
                                     : group_norm_int8_kernel<FP16, SILU, 128, 4>;
  // above 47 KB only where almost every channel is a group of its own
  const cudaError_t e = smem > 47 * 1024 ? cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem)) : cudaSuccess;
  if (e != cudaSuccess) return e;
  return launch_overlapped(kernel, dim3(static_cast<unsigned>(p.strips), static_cast<unsigned>(batch)), dim3(kRowThreads), smem, st, 1, p);
}

}  // namespace
}  // namespace hdit

extern "C" int64_t hdit_group_norm_scratch(int64_t batch, int64_t rows, int64_t channels, int64_t groups) {
  using namespace hdit;
  if (batch <= 0 || rows <= 0 || channels <= 0 || groups <= 0 || channels % 8 != 0 || channels > kMaxChannels) return 0;
  return batch * strips_of(batch, rows, static_cast<int>(channels)) * groups * static_cast<int64_t>(sizeof(float2));
}

extern "C" int hdit_group_norm(int32_t dtype, const void* x, const void* weight, const void* bias, void* out, void* scratch, int64_t batch,
                               int64_t rows, int64_t channels, int64_t groups, int64_t x_batch_stride, int64_t x_row_stride,
                               int64_t out_batch_stride, int64_t out_row_stride, float eps, int32_t act, void* stream) {
  using namespace hdit;
  const int rc = check_gn(dtype, x, out, scratch, batch, rows, channels, groups, act);
  if (rc != HDIT_OK || batch == 0 || rows == 0) return rc;
  GnParams p{static_cast<const uint16_t*>(x), static_cast<const uint16_t*>(weight), static_cast<const uint16_t*>(bias), static_cast<uint16_t*>(out),
             nullptr, nullptr, static_cast<float2*>(scratch), rows, x_batch_stride, x_row_stride, out_batch_stride, out_row_stride, 0, 0,
             static_cast<int>(channels), static_cast<int>(groups), act, eps,
             !off16(x, x_batch_stride, x_row_stride) && !off16(out, out_batch_stride, out_row_stride)};
  p.strips = strips_of(batch, rows, p.channels);
  p.strip_rows = (rows + p.strips - 1) / p.strips;
  p.strips = static_cast<int>((rows + p.strip_rows - 1) / p.strip_rows);
  const bool fp16 = dtype == HDIT_FP16;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  HDIT_CUDA_OK(launch_stats(p, fp16, batch, st));
  auto kernel = act == HDIT_ACT_SILU ? (fp16 ? group_norm_apply_kernel<true, true> : group_norm_apply_kernel<false, true>)
                                     : (fp16 ? group_norm_apply_kernel<true, false> : group_norm_apply_kernel<false, false>);
  HDIT_CUDA_OK(launch_overlapped(kernel, dim3(static_cast<unsigned>(p.strips), static_cast<unsigned>(batch)),
                                 dim3(static_cast<unsigned>(gn_threads(p.channels))), static_cast<size_t>(p.groups) * sizeof(float2), st, 1, p));
  return HDIT_OK;
}

extern "C" int hdit_group_norm_int8(int32_t dtype, const void* x, const void* weight, const void* bias, void* q, float* q_scale, void* scratch,
                                    int64_t batch, int64_t rows, int64_t channels, int64_t groups, int64_t x_batch_stride, int64_t x_row_stride,
                                    int64_t q_row_stride, float eps, int32_t act, void* stream) {
  using namespace hdit;
  const int rc = check_gn(dtype, x, q, scratch, batch, rows, channels, groups, act);
  if (rc != HDIT_OK) return rc;
  if ((reinterpret_cast<uintptr_t>(q) & 15) != 0 || q_row_stride % 16 != 0 || q_row_stride < channels)
    return set_error(HDIT_ERR_SHAPE, "8-bit rows need a 16-byte aligned pointer and a row stride that is a multiple of 16 and covers a row");
  if (batch == 0 || rows == 0) return HDIT_OK;
  if (q_scale == nullptr) return set_error(HDIT_ERR_BAD_ARG, "null scale");
  GnParams p{static_cast<const uint16_t*>(x), static_cast<const uint16_t*>(weight), static_cast<const uint16_t*>(bias), nullptr,
             static_cast<int8_t*>(q), q_scale, static_cast<float2*>(scratch), rows, x_batch_stride, x_row_stride, 0, q_row_stride, 0, 0,
             static_cast<int>(channels), static_cast<int>(groups), act, eps, !off16(x, x_batch_stride, x_row_stride)};
  p.strips = strips_of(batch, rows, p.channels);
  p.strip_rows = (rows + p.strips - 1) / p.strips;
  p.strips = static_cast<int>((rows + p.strip_rows - 1) / p.strip_rows);
  const bool fp16 = dtype == HDIT_FP16;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  HDIT_CUDA_OK(launch_stats(p, fp16, batch, st));
  const bool sl = act == HDIT_ACT_SILU;
  HDIT_CUDA_OK((fp16 ? (sl ? launch_int8<true, true>(p, batch, st) : launch_int8<true, false>(p, batch, st))
                     : (sl ? launch_int8<false, true>(p, batch, st) : launch_int8<false, false>(p, batch, st))));
  return HDIT_OK;
}
