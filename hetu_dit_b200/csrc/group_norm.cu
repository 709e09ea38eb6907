// GroupNorm over channels-last images, with an activation, or with its rows (all channels of a pixel) as 8-bit integers
// (int8_rows.cuh) for a linear layer that follows:
//   y[b, r, c] = (x[b, r, c] - mean[b, g]) / sqrt(var[b, g] + eps) * weight[c] + bias[c],   g = c / (channels / groups)
// over rows r (pixels) and the channels of a group; biased variance.
//
// Two launches of one CTA per SM. The first one reads x once: a CTA takes a strip of rows of one image, each thread eight fixed
// channels, and leaves {mean, sum of squared distances from it} per group and strip. Sums are taken relative to a value of the
// strip's first row, so that a mean far from zero costs no digits. The second one joins the strips (Chan's formula) and reads x
// again, each strip from its end to its start: what the first launch read last is still in L2. Every CTA joins the strips of
// its image by itself; with four strips per SM, read eight at a time by a thread, that alone took 3 us.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include "host_common.h"
#include "int8_rows.cuh"
#include "ptx_sm100.cuh"

namespace hdit {
namespace {

constexpr int kMaxChannels = 4096;
constexpr int kGnThreads = 512;  // what a CTA does beside its rows costs every warp some hundred instructions
constexpr int kAhead = 6;        // rows of a thread in flight

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

// Walks `count` rows of a thread, `step` elements apart: use(values of the row's eight channels, index). Groups of kAhead rows
// are on their way while the group before is used.
template <bool VEC, typename F>
__device__ __forceinline__ void walk_rows(const uint16_t* x, int c, int channels, int count, long long step, F use) {
  uint4 next[kAhead];
  const int full = count / kAhead;
  auto fetch = [&](int n) {
#pragma unroll
    for (int k = 0; k < kAhead; ++k)
      if (k < n) next[k] = int8_load8(x + k * step, c, channels, VEC);
    x += kAhead * step;
  };
  fetch(full > 0 ? kAhead : count);
  int at = 0;
  for (int f = 0; f < full; ++f) {
    uint4 raw[kAhead];
#pragma unroll
    for (int k = 0; k < kAhead; ++k) raw[k] = next[k];
    if (f + 1 < full) fetch(kAhead);
    else fetch(count - full * kAhead);
#pragma unroll
    for (int k = 0; k < kAhead; ++k) use(raw[k], at + k);
    at += kAhead;
  }
#pragma unroll
  for (int k = 0; k < kAhead; ++k)
    if (at + k < count) use(next[k], at + k);
}

template <bool FP16, bool VEC>
__global__ void __launch_bounds__(kGnThreads, 1) group_norm_stats_kernel(const __grid_constant__ GnParams p) {
  grid_dependency_release();
  grid_dependency_wait();
  extern __shared__ float smem[];  // [lanes][channels] sums, then the same of squares
  const int chunks = p.channels / 8;
  const int lanes = kGnThreads / chunks;  // rows at a time
  const int lane = threadIdx.x / chunks, c = (threadIdx.x - lane * chunks) * 8;
  const long long r0 = static_cast<long long>(blockIdx.x) * p.strip_rows;
  const int rows = static_cast<int>(r0 + p.strip_rows < p.rows ? p.strip_rows : p.rows - r0);
  const uint16_t* xs = p.x + blockIdx.y * p.x_batch_stride + r0 * p.x_row_stride;
  if (lane < lanes) {
    float s[8], ss[8], pivot[8];
    const uint4 first = int8_load8(xs, c, p.channels, VEC);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 v = int8_unpack2<FP16>(reinterpret_cast<const uint32_t*>(&first)[i]);
      pivot[2 * i] = v.x;
      pivot[2 * i + 1] = v.y;
      s[2 * i] = s[2 * i + 1] = ss[2 * i] = ss[2 * i + 1] = 0.f;
    }
    const int count = rows > lane ? (rows - lane + lanes - 1) / lanes : 0;
    walk_rows<VEC>(xs + lane * p.x_row_stride, c, p.channels, count, lanes * p.x_row_stride, [&](const uint4& raw, int) {
      const uint32_t* u = reinterpret_cast<const uint32_t*>(&raw);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 v = int8_unpack2<FP16>(u[i]);
        const float d0 = v.x - pivot[2 * i], d1 = v.y - pivot[2 * i + 1];
        s[2 * i] += d0;
        ss[2 * i] = fmaf(d0, d0, ss[2 * i]);
        s[2 * i + 1] += d1;
        ss[2 * i + 1] = fmaf(d1, d1, ss[2 * i + 1]);
      }
    });
    float4* to = reinterpret_cast<float4*>(smem + lane * p.channels + c);
    to[0] = make_float4(s[0], s[1], s[2], s[3]);
    to[1] = make_float4(s[4], s[5], s[6], s[7]);
    to = reinterpret_cast<float4*>(smem + (lanes + lane) * p.channels + c);
    to[0] = make_float4(ss[0], ss[1], ss[2], ss[3]);
    to[1] = make_float4(ss[4], ss[5], ss[6], ss[7]);
  }
  __syncthreads();
  // Over the lanes: `parts` neighbouring lanes of a warp to a channel. Then per channel, in the first lane's places: the mean,
  // and the sum of squared distances from it.
  int parts = 1;
  while (parts < 32 && parts < lanes && parts * 2 * p.channels <= kGnThreads) parts *= 2;
  const float inv_rows = 1.f / static_cast<float>(rows);
  for (int ch0 = 0; ch0 < p.channels; ch0 += kGnThreads / parts) {
    const int ch = ch0 + static_cast<int>(threadIdx.x) / parts, part = static_cast<int>(threadIdx.x) % parts;
    float a = 0.f, q = 0.f;
    if (ch < p.channels)
      for (int l = part; l < lanes; l += parts) {
        a += smem[l * p.channels + ch];
        q += smem[(lanes + l) * p.channels + ch];
      }
    a = sub_sum(a, parts);
    q = sub_sum(q, parts);
    if (ch < p.channels && part == 0) {  // no other thread reads this channel's first lane
      const float m2 = q - a * a * inv_rows;
      smem[ch] = int8_unpack2<FP16>(xs[ch]).x + a * inv_rows;
      smem[lanes * p.channels + ch] = m2 > 0.f ? m2 : m2 - m2;  // keeps NaN
    }
  }
  __syncthreads();
  const int per = p.channels / p.groups;
  const float n = static_cast<float>(rows), inv_per = 1.f / static_cast<float>(per);
  float2* out = p.partial + (static_cast<long long>(blockIdx.y) * p.strips + blockIdx.x) * p.groups;
  for_groups(p.groups, [&](int g, int sub, int n_sub) {
    const bool live = g < p.groups;
    float mean = 0.f, m2 = 0.f;
    for (int k = sub; live && k < per; k += n_sub) mean += smem[g * per + k];
    mean = sub_sum(mean, n_sub) * inv_per;
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
#pragma unroll 4
    for (int k = sub; k < (live ? p.strips : 0); k += n_sub) {
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

// y = x * a + b with a = weight / deviation and b = bias - mean * a, for all channels of image blockIdx.y into shared memory:
// `factors` holds a, then b, each first for the lower four channels of every chunk of eight, then for the upper four, so that
// threads' 16 bytes lie side by side; behind them stand the groups' statistics.
// Against (x - mean) * a + bias this form costs half a unit of 2^-24 of mean * a: a 16-bit x resolves the deviation only while
// |mean| is below some 2^11 deviations, where that is under 2^-13 of the result's deviation.
template <bool FP16>
__device__ __forceinline__ void group_norm_factors(const GnParams& p, float4* factors) {
  const int chunks = p.channels / 8, per = p.channels / p.groups;
  float2* stat = reinterpret_cast<float2*>(factors + 4 * chunks);
  group_norm_join(p, blockIdx.y, stat);
  __syncthreads();
  for (int c = threadIdx.x; c < p.channels; c += blockDim.x) {
    const float2 st = stat[c / per];
    const float a = st.y * (p.weight != nullptr ? int8_unpack2<FP16>(p.weight[c]).x : 1.f);
    float* to = reinterpret_cast<float*>(factors) + (c >> 3) * 4 + ((c >> 2) & 1) * chunks * 4 + (c & 3);
    to[0] = a;
    to[8 * chunks] = fmaf(-st.x, a, p.bias != nullptr ? int8_unpack2<FP16>(p.bias[c]).x : 0.f);
  }
  __syncthreads();
}

// y / (1 + exp(-y)): two operations of the special-function unit, each within 2^-22 of its result
__device__ __forceinline__ float silu(float y) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.f + ex2_approx(-1.4426950408889634f * y)));
  return y * r;
}

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

template <bool FP16, bool SILU, bool VEC>
__global__ void __launch_bounds__(kGnThreads, 1) group_norm_apply_kernel(const __grid_constant__ GnParams p) {
  grid_dependency_release();
  grid_dependency_wait();
  extern __shared__ float4 factors[];
  const int chunks = p.channels / 8;
  const int lanes = kGnThreads / chunks;
  const int lane = threadIdx.x / chunks, chunk = threadIdx.x - lane * chunks, c = chunk * 8;
  const long long r0 = static_cast<long long>(blockIdx.x) * p.strip_rows;
  const int rows = static_cast<int>(r0 + p.strip_rows < p.rows ? p.strip_rows : p.rows - r0);
  group_norm_factors<FP16>(p, factors);
  if (lane >= lanes) return;
  float a[8], b[8];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    *reinterpret_cast<float4*>(a + 4 * h) = factors[h * chunks + chunk];
    *reinterpret_cast<float4*>(b + 4 * h) = factors[(2 + h) * chunks + chunk];
  }
  // from the strip's end to its start
  const int count = rows > lane ? (rows - lane + lanes - 1) / lanes : 0;
  const long long out_step = lanes * p.out_row_stride;
  uint16_t* out = p.out + blockIdx.y * p.out_batch_stride + (r0 + rows - 1 - lane) * p.out_row_stride + c;
  walk_rows<VEC>(p.x + blockIdx.y * p.x_batch_stride + (r0 + rows - 1 - lane) * p.x_row_stride, c, p.channels, count, -lanes * p.x_row_stride,
                 [&](const uint4& raw, int i) {
                   uint4 y = raw;
                   uint32_t* u = reinterpret_cast<uint32_t*>(&y);
#pragma unroll
                   for (int k = 0; k < 4; ++k) {
                     const float2 v = int8_unpack2<FP16>(u[k]);
                     float y0 = fmaf(v.x, a[2 * k], b[2 * k]), y1 = fmaf(v.y, a[2 * k + 1], b[2 * k + 1]);
                     if constexpr (SILU) y0 = silu(y0), y1 = silu(y1);
                     u[k] = gn_pack<FP16>(y0, y1);
                   }
                   uint16_t* dst = out - i * out_step;
                   if constexpr (VEC) {
                     *reinterpret_cast<uint4*>(dst) = y;
                   } else {
#pragma unroll
                     for (int k = 0; k < 8; ++k) dst[k] = static_cast<uint16_t>(u[k / 2] >> (16 * (k & 1)));
                   }
                 });
}

// The rows in 8 bits: TEAM threads hold a row of at most TEAM * NCH * 8 channels and have the next one on its way; factors of
// all channels in shared memory.
template <bool FP16, bool SILU, int TEAM, int NCH, bool VEC>
__global__ void __launch_bounds__(kGnThreads, 1) group_norm_int8_kernel(const __grid_constant__ GnParams p) {
  grid_dependency_release();
  grid_dependency_wait();
  extern __shared__ float4 factors[];
  __shared__ float red[2][kGnThreads / 32];
  const int chunks = p.channels / 8;
  const Team<TEAM, kGnThreads> team{red};
  constexpr int kTeams = kGnThreads / TEAM;
  const int c0 = static_cast<int>(threadIdx.x % TEAM) * 8, first = static_cast<int>(threadIdx.x) / TEAM;
  const long long s0 = static_cast<long long>(blockIdx.x) * p.strip_rows;
  const int rows = static_cast<int>(s0 + p.strip_rows < p.rows ? p.strip_rows : p.rows - s0);
  const uint16_t* x = p.x + blockIdx.y * p.x_batch_stride + (s0 + rows - 1 - first) * p.x_row_stride;  // from the strip's end to its start
  uint4 next[NCH];
  auto fetch = [&] {
#pragma unroll
    for (int k = 0; k < NCH; ++k) {
      next[k] = make_uint4(0, 0, 0, 0);
      if (c0 + k * TEAM * 8 < p.channels) next[k] = int8_load8(x, c0 + k * TEAM * 8, p.channels, VEC);
    }
  };
  if (first < rows) fetch();
  group_norm_factors<FP16>(p, factors);
  int turn = 0;
  for (int r = first; r < rows; r += kTeams, turn ^= 1) {
    uint4 raw[NCH];
#pragma unroll
    for (int k = 0; k < NCH; ++k) raw[k] = next[k];
    x -= kTeams * p.x_row_stride;
    if (r + kTeams < rows) fetch();
    float y[NCH][8];
    float top = 0.f;
#pragma unroll
    for (int k = 0; k < NCH; ++k) {
      const int c = c0 + k * TEAM * 8;
      if (c >= p.channels) continue;
      const uint32_t* u = reinterpret_cast<const uint32_t*>(&raw[k]);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const float4 av = factors[h * chunks + (c >> 3)], bv = factors[(2 + h) * chunks + (c >> 3)];
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
    const Int8Scale s = int8_scale(team.max(__float_as_uint(top) & 0x7FFFFFFFu, turn));
    const long long row = blockIdx.y * p.rows + s0 + rows - 1 - r;
#pragma unroll
    for (int k = 0; k < NCH; ++k)
      if (c0 + k * TEAM * 8 < p.channels) int8_put8_of(p.q + row * p.out_row_stride, c0 + k * TEAM * 8, s, y[k]);
    if (c0 == 0) p.q_scale[row] = int8_step(s);
  }
}

// Strips per image: one CTA per SM over all images, at least two rows of every thread's channels each.
int strips_of(long long batch, long long rows, int channels) {
  const long long lanes = kGnThreads / (channels / 8);
  long long n = 148 / batch;
  const long long most = (rows + lanes * 2 - 1) / (lanes * 2);
  if (n > most) n = most;
  return static_cast<int>(n < 1 ? 1 : n);
}

void set_strips(GnParams& p, long long batch) {
  p.strips = strips_of(batch, p.rows, p.channels);
  p.strip_rows = (p.rows + p.strips - 1) / p.strips;
  p.strips = static_cast<int>((p.rows + p.strip_rows - 1) / p.strip_rows);
}

int check_gn(const hdit_group_norm_args* a) {
  if (a == nullptr) return set_error(HDIT_ERR_BAD_ARG, "null args");
  if (a->dtype != HDIT_BF16 && a->dtype != HDIT_FP16) return set_error(HDIT_ERR_BAD_ARG, "dtype must be bf16 or fp16");
  if (a->batch < 0 || a->rows < 0 || a->channels <= 0 || a->groups <= 0) return set_error(HDIT_ERR_BAD_ARG, "bad sizes");
  if (a->act != HDIT_ACT_NONE && a->act != HDIT_ACT_SILU) return set_error(HDIT_ERR_BAD_ARG, "unknown activation %d", a->act);
  if (a->channels % 8 != 0 || a->channels > kMaxChannels || a->channels % a->groups != 0)
    return set_error(HDIT_ERR_SHAPE, "channels must be a multiple of 8 and of groups, at most %d", kMaxChannels);
  if (a->batch > 65535 || a->rows > 0x7fffffffLL) return set_error(HDIT_ERR_TOO_LARGE, "at most 65535 images of 2^31 - 1 rows");
  if (a->batch == 0 || a->rows == 0) return HDIT_OK;
  if (a->x == nullptr || a->out == nullptr || a->scratch == nullptr) return set_error(HDIT_ERR_BAD_ARG, "null x / out / scratch");
  if ((reinterpret_cast<uintptr_t>(a->scratch) & 7) != 0) return set_error(HDIT_ERR_SHAPE, "scratch not 8-byte aligned");
  return HDIT_OK;
}

bool off16(const void* p, int64_t a, int64_t b) { return (reinterpret_cast<uintptr_t>(p) & 15) != 0 || a % 8 != 0 || b % 8 != 0; }

template <typename K>
cudaError_t launch_strips(K kernel, const GnParams& p, long long batch, size_t smem, cudaStream_t st) {
  // static shared memory counts, too
  const cudaError_t e = smem > 47 * 1024 ? cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem)) : cudaSuccess;
  if (e != cudaSuccess) return e;
  return launch_overlapped(kernel, dim3(static_cast<unsigned>(p.strips), static_cast<unsigned>(batch)), dim3(kGnThreads), smem, st, 1, p);
}

GnParams params_of(const hdit_group_norm_args* a, bool out_vec) {
  GnParams p{};
  p.x = static_cast<const uint16_t*>(a->x);
  p.weight = static_cast<const uint16_t*>(a->weight);
  p.bias = static_cast<const uint16_t*>(a->bias);
  p.out = static_cast<uint16_t*>(a->out);
  p.q = static_cast<int8_t*>(a->out);
  p.q_scale = a->out_scale;
  p.partial = static_cast<float2*>(a->scratch);
  p.rows = a->rows;
  p.x_batch_stride = a->x_batch_stride;
  p.x_row_stride = a->x_row_stride;
  p.out_batch_stride = a->out_batch_stride;
  p.out_row_stride = a->out_row_stride;
  p.channels = static_cast<int>(a->channels);
  p.groups = static_cast<int>(a->groups);
  p.act = a->act;
  p.eps = a->eps;
  p.vec = out_vec && !off16(a->x, a->x_batch_stride, a->x_row_stride);
  set_strips(p, a->batch);
  return p;
}

size_t factor_bytes(const GnParams& p) { return static_cast<size_t>(p.channels) * 2 * sizeof(float) + static_cast<size_t>(p.groups) * sizeof(float2); }

template <bool FP16, bool VEC>
cudaError_t launch_stats(const GnParams& p, long long batch, cudaStream_t st) {
  const size_t smem = static_cast<size_t>(kGnThreads / (p.channels / 8)) * p.channels * 2 * sizeof(float);
  return launch_strips(group_norm_stats_kernel<FP16, VEC>, p, batch, smem, st);
}

template <bool FP16, bool VEC>
cudaError_t launch_apply(const GnParams& p, long long batch, cudaStream_t st) {
  return p.act == HDIT_ACT_SILU ? launch_strips(group_norm_apply_kernel<FP16, true, VEC>, p, batch, factor_bytes(p), st)
                                : launch_strips(group_norm_apply_kernel<FP16, false, VEC>, p, batch, factor_bytes(p), st);
}

template <bool FP16, bool SILU, bool VEC>
cudaError_t launch_int8_act(const GnParams& p, long long batch, cudaStream_t st) {
  auto kernel = p.channels <= 256    ? group_norm_int8_kernel<FP16, SILU, 32, 1, VEC>
                : p.channels <= 512  ? group_norm_int8_kernel<FP16, SILU, 32, 2, VEC>
                : p.channels <= 1024 ? group_norm_int8_kernel<FP16, SILU, 32, 4, VEC>
                                     : group_norm_int8_kernel<FP16, SILU, 128, 4, VEC>;
  return launch_strips(kernel, p, batch, factor_bytes(p), st);
}

template <bool FP16, bool VEC>
cudaError_t launch_int8(const GnParams& p, long long batch, cudaStream_t st) {
  return p.act == HDIT_ACT_SILU ? launch_int8_act<FP16, true, VEC>(p, batch, st) : launch_int8_act<FP16, false, VEC>(p, batch, st);
}

#define HDIT_GN_OF(f, fp16, vec) ((fp16) ? ((vec) ? f<true, true> : f<true, false>) : ((vec) ? f<false, true> : f<false, false>))

}  // namespace
}  // namespace hdit

extern "C" int64_t hdit_group_norm_scratch(int64_t batch, int64_t rows, int64_t channels, int64_t groups) {
  using namespace hdit;
  if (batch <= 0 || rows <= 0 || channels <= 0 || groups <= 0 || channels % 8 != 0 || channels > kMaxChannels) return 0;
  return batch * strips_of(batch, rows, static_cast<int>(channels)) * groups * static_cast<int64_t>(sizeof(float2));
}

extern "C" int hdit_group_norm(const hdit_group_norm_args* a) {
  using namespace hdit;
  const int rc = check_gn(a);
  if (rc != HDIT_OK || a->batch == 0 || a->rows == 0) return rc;
  const GnParams p = params_of(a, !off16(a->out, a->out_batch_stride, a->out_row_stride));
  const bool fp16 = a->dtype == HDIT_FP16;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(a->stream);
  HDIT_CUDA_OK((HDIT_GN_OF(launch_stats, fp16, p.vec)(p, a->batch, st)));
  HDIT_CUDA_OK((HDIT_GN_OF(launch_apply, fp16, p.vec)(p, a->batch, st)));
  return HDIT_OK;
}

extern "C" int hdit_group_norm_int8(const hdit_group_norm_args* a) {
  using namespace hdit;
  const int rc = check_gn(a);
  if (rc != HDIT_OK) return rc;
  if ((reinterpret_cast<uintptr_t>(a->out) & 15) != 0 || a->out_row_stride % 16 != 0 || a->out_row_stride < a->channels)
    return set_error(HDIT_ERR_SHAPE, "8-bit rows need a 16-byte aligned pointer and a row stride that is a multiple of 16 and covers a row");
  if (a->batch == 0 || a->rows == 0) return HDIT_OK;
  if (a->out_scale == nullptr) return set_error(HDIT_ERR_BAD_ARG, "null scale");
  const GnParams p = params_of(a, true);
  const bool fp16 = a->dtype == HDIT_FP16;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(a->stream);
  HDIT_CUDA_OK((HDIT_GN_OF(launch_stats, fp16, p.vec)(p, a->batch, st)));
  HDIT_CUDA_OK((HDIT_GN_OF(launch_int8, fp16, p.vec)(p, a->batch, st)));
  return HDIT_OK;
}
