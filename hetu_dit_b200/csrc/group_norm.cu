// GroupNorm over channels-last images, with an activation, or with its rows (all channels of a pixel) as 8-bit integers
// (int8_rows.cuh) for a linear layer that follows:
//   y[b, r, c] = (x[b, r, c] - mean[b, g]) / sqrt(var[b, g] + eps) * weight[c] + bias[c],   g = c / (channels / groups)
// over rows r (pixels) and the channels of a group; biased variance.
//
// Two launches of one CTA per SM. The first one reads x once: a strip (a CTA) takes every strips-th tile of rows of an image,
// each thread eight fixed channels, and leaves {mean, sum of squared distances from it} per group and strip. Sums are taken
// relative to a value of the strip's first row, means relative to the group's pivot, its first value in the image, so that a
// mean far from zero costs no digits. The second one joins the strips
// (Chan's formula) and reads x again from its end to its start: what the first launch read last is still in L2. Every CTA joins
// the strips of its image by itself; with four strips per SM, read eight at a time by a thread, that alone took 3 us.
// All CTAs work on neighbouring tiles at a time: with one stretch of rows each, 1024 x 1024 x 128 took 148 us (4.8 TB/s of
// traffic in both launches), 143 like this.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include "gemm_common.cuh"
#include "host_common.h"
#include "int8_rows.cuh"
#include "ptx_sm100.cuh"

namespace hdit {
namespace {

constexpr int kMaxChannels = 4096;
constexpr int kAhead = 6;         // rows of a thread in flight
constexpr int cluster_threads(bool int8) { return int8 ? 512 : 256; }  // two CTAs to an SM, or few CTAs at all
constexpr int kGnThreads = 512;  // what a CTA does beside its rows costs every warp some hundred instructions

// How the rows of an image lie in tiles of `lanes` rows and the tiles in strips: strip k has tiles k, k + strips, ...; the last
// tile of all is `missing` rows short. Worked out on the host: a thread's 64-bit divisions cost more than its sums.
struct Strips {
  int strips, lanes;
  int tiles, longer;  // of a strip; the first `longer` strips have one more
  int last, missing;  // the strip with the last tile
  __host__ __device__ int tiles_of(int k) const { return tiles + (k < longer ? 1 : 0); }
  __host__ __device__ int rows_of(int k) const { return tiles_of(k) * lanes - (k == last ? missing : 0); }
  // rows of a lane of strip k
  __device__ __forceinline__ int rows_of_lane(int k, int lane) const { return tiles_of(k) - (k == last && lane >= lanes - missing ? 1 : 0); }
  __device__ __forceinline__ long long first(int k, int lane) const { return static_cast<long long>(k) * lanes + lane; }
  __device__ __forceinline__ long long step() const { return static_cast<long long>(strips) * lanes; }
};

struct GnParams {
  const uint16_t* x;
  const uint16_t* weight;  // or null: 1
  const uint16_t* bias;    // or null: 0
  uint16_t* out;
  int8_t* q;
  float* q_scale;
  float2* partial;  // (batch, strips, groups): mean from the pivot, sum of squared distances from the mean
  uint16_t* pivots;  // (batch, groups)
  long long rows, x_batch_stride, x_row_stride, out_batch_stride, out_row_stride;  // q: out_row_stride only, rows of all images
  Strips strips;
  int channels, groups, act, slab;
  float eps, inv_per;  // 1 / channels of a group
  bool vec;
};

// Group of a channel (below 4096: the product is off by less than the half that is added). Integer divisions one after the other
// between two barriers cost more than the sums there.
__device__ __forceinline__ int group_of(int channel, float inv_per) { return static_cast<int>((static_cast<float>(channel) + 0.5f) * inv_per); }

// Calls f(group, sub, n_sub) in groups of n_sub consecutive threads of a warp, the same number of times in all threads.
template <int THREADS, typename F>
__device__ __forceinline__ void for_groups(int groups, F f) {
  int shift = 5;
  while (shift > 0 && groups << shift > THREADS) --shift;
  const int sub = static_cast<int>(threadIdx.x) & ((1 << shift) - 1);
  for (int g0 = 0; g0 < groups; g0 += THREADS >> shift) f(g0 + (static_cast<int>(threadIdx.x) >> shift), sub, 1 << shift);
}
__device__ __forceinline__ float sub_sum(float v, int n_sub) {
  for (int o = n_sub >> 1; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// Walks `count` rows of a thread, `step` elements apart: use(values of the row's eight channels, index). Groups of kAhead rows
// are on their way while the group before is used; meanwhile() is called when the first ones are.
template <bool VEC, typename M, typename F>
__device__ __forceinline__ void walk_rows(const uint16_t* x, int c, int channels, int count, long long step, M meanwhile, F use) {
  uint4 next[kAhead];
  const int full = count / kAhead;
  auto fetch = [&](int n) {
#pragma unroll
    for (int k = 0; k < kAhead; ++k)
      if (k < n) next[k] = int8_load8(x + k * step, c, channels, VEC);
    x += kAhead * step;
  };
  fetch(full > 0 ? kAhead : count);
  meanwhile();
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

// Floats from one lane's sums to the next one's: lanes that are summed side by side are in banks of their own (two launches over 64 x 16 8.0 -> 6.5 us; the cluster over 4096 x 512 8.8 -> 7.9)
__host__ __device__ constexpr int stats_pitch(int channels) { return channels + 4; }
// of the cluster's sums; the factors take their place
__host__ __device__ constexpr int sums_bytes(int lanes, int channels) {
  return lanes * stats_pitch(channels) * 8 > channels * 12 ? lanes * stats_pitch(channels) * 8 : channels * 12;
}

// Statistics of strip k of an image of `rows` rows of `channels` channels at `x`. A thread passes its eight channels of every lanes-th
// row to keep(raw, index). smem: [lanes][stats_pitch(channels)] sums, then the same of squares. row0: the image's first row, which has
// the groups' pivots, is left there. put(group, {mean from the pivot, sum of squared distances from the mean}).
template <int THREADS, bool FP16, bool VEC, typename K, typename P>
__device__ __forceinline__ void strip_stats(const uint16_t* x, long long row_stride, const Strips& strips, int strip, int channels, int per, float inv_per, float* smem,
                                            uint16_t* row0, K keep, P put) {
  const int chunks = channels / 8;
  const int lanes = strips.lanes, pitch = stats_pitch(channels);  // rows at a time
  const int lane = threadIdx.x / chunks, c = (threadIdx.x - lane * chunks) * 8;
  const uint16_t* xs = x + static_cast<long long>(strip) * lanes * row_stride;  // the strip's first row
  if (lane < lanes) {
    float s[8], ss[8], first_row[8];
    uint4 image_row;
    const uint4 first = int8_load8(xs, c, channels, VEC);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 v = int8_unpack2<FP16>(reinterpret_cast<const uint32_t*>(&first)[i]);
      first_row[2 * i] = v.x;
      first_row[2 * i + 1] = v.y;
      s[2 * i] = s[2 * i + 1] = ss[2 * i] = ss[2 * i + 1] = 0.f;
    }
    walk_rows<VEC>(x + strips.first(strip, lane) * row_stride, c, channels, strips.rows_of_lane(strip, lane), strips.step() * row_stride, [&] {
      if (lane == 0) image_row = int8_load8(x, c, channels, VEC);
    }, [&](const uint4& raw, int at) {
      keep(raw, at);
      const uint32_t* u = reinterpret_cast<const uint32_t*>(&raw);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 v = int8_unpack2<FP16>(u[i]);
        const float d0 = v.x - first_row[2 * i], d1 = v.y - first_row[2 * i + 1];
        s[2 * i] += d0;
        ss[2 * i] = fmaf(d0, d0, ss[2 * i]);
        s[2 * i + 1] += d1;
        ss[2 * i + 1] = fmaf(d1, d1, ss[2 * i + 1]);
      }
    });
    if (lane == 0) *reinterpret_cast<uint4*>(row0 + c) = image_row;
    float4* to = reinterpret_cast<float4*>(smem + lane * pitch + c);
    to[0] = make_float4(s[0], s[1], s[2], s[3]);
    to[1] = make_float4(s[4], s[5], s[6], s[7]);
    to = reinterpret_cast<float4*>(smem + (lanes + lane) * pitch + c);
    to[0] = make_float4(ss[0], ss[1], ss[2], ss[3]);
    to[1] = make_float4(ss[4], ss[5], ss[6], ss[7]);
  }
  __syncthreads();
  // Over the lanes: `parts` neighbouring lanes of a warp to a channel. Then per channel, in the first lane's places: the mean from the
  // group's pivot, and the sum of squared distances from the mean.
  int shift = 0;
  while (shift < 5 && 1 << shift < lanes && 2 * channels << shift <= THREADS) ++shift;
  const int parts = 1 << shift, part = static_cast<int>(threadIdx.x) & (parts - 1);
  const float n = static_cast<float>(strips.rows_of(strip)), inv_rows = 1.f / n;
  for (int ch0 = 0; ch0 < channels; ch0 += THREADS >> shift) {
    const int ch = ch0 + (static_cast<int>(threadIdx.x) >> shift);
    float a = 0.f, q = 0.f;
    if (ch < channels)
      for (int l = part; l < lanes; l += parts) {
        a += smem[l * pitch + ch];
        q += smem[(lanes + l) * pitch + ch];
      }
    a = sub_sum(a, parts);
    q = sub_sum(q, parts);
    if (ch < channels && part == 0) {  // no other thread reads this channel's first lane
      const float m2 = q - a * a * inv_rows;
      smem[ch] = (int8_unpack2<FP16>(xs[ch]).x - int8_unpack2<FP16>(row0[group_of(ch, inv_per) * per]).x) + a * inv_rows;
      smem[lanes * pitch + ch] = m2 > 0.f ? m2 : m2 - m2;  // keeps NaN
    }
  }
  __syncthreads();
  for_groups<THREADS>(channels / per, [&](int g, int sub, int n_sub) {
    const bool live = g * per < channels;
    float mean = 0.f, m2 = 0.f;
    for (int k = sub; live && k < per; k += n_sub) mean += smem[g * per + k];
    mean = sub_sum(mean, n_sub) * inv_per;
    for (int k = sub; live && k < per; k += n_sub) {
      const float d = smem[g * per + k] - mean;
      m2 += smem[lanes * pitch + g * per + k] + n * d * d;
    }
    m2 = sub_sum(m2, n_sub);
    if (live && sub == 0) put(g, make_float2(mean, m2));
  });
}

template <bool FP16, bool VEC>
__global__ void __launch_bounds__(kGnThreads, 1) group_norm_stats_kernel(const __grid_constant__ GnParams p) {
  grid_dependency_release();
  grid_dependency_wait();
  extern __shared__ __align__(16) float smem[];
  const int per = p.channels / p.groups;
  uint16_t* row0 = reinterpret_cast<uint16_t*>(smem + p.strips.lanes * stats_pitch(p.channels) * 2);
  float2* out = p.partial + (static_cast<long long>(blockIdx.y) * p.strips.strips + blockIdx.x) * p.groups;
  strip_stats<kGnThreads, FP16, VEC>(p.x + blockIdx.y * p.x_batch_stride, p.x_row_stride, p.strips, static_cast<int>(blockIdx.x), p.channels, per, p.inv_per, smem,
                                     row0, [](const uint4&, int) {}, [&](int g, float2 v) {
                                       out[g] = v;
                                       if (blockIdx.x == 0) p.pivots[static_cast<long long>(blockIdx.y) * p.groups + g] = row0[g * per];
                                     });
}

// {mean from the pivot, 1 / deviation} of `groups` groups from `strips` strips of an image, `per` channels to a group, into
// stat[groups]. in(strip, group): the strip's {mean from the pivot, sum of squared distances from the mean}.
template <int THREADS, typename F>
__device__ __forceinline__ void join_strips(int groups, const Strips& strips, long long rows, int per, float eps, float2* stat, F in) {
  const float inv_total = 1.f / (static_cast<float>(rows) * static_cast<float>(per));
  for_groups<THREADS>(groups, [&](int g, int sub, int n_sub) {
    const bool live = g < groups;
    const float base = live ? in(0, g).x : 0.f;
    float a = 0.f, q = 0.f;
#pragma unroll 10
    for (int k = sub; k < (live ? strips.strips : 0); k += n_sub) {
      const float2 v = in(k, g);
      const float d = v.x - base, n = static_cast<float>(strips.rows_of(k)) * static_cast<float>(per);
      a = fmaf(n, d, a);
      q += fmaf(n * d, d, v.y);
    }
    a = sub_sum(a, n_sub);
    q = sub_sum(q, n_sub);
    const float far = a * inv_total;  // of the mean from the first strip's
    const float var = q * inv_total - far * far;
    if (live && sub == 0) stat[g] = make_float2(base + far, rsqrtf((var > 0.f ? var : var - var) + eps));
  });
}

// y = (x * a + b) + rest with a = weight / deviation and b + rest = bias - mean * a, for each channel in shared memory: `factors` holds
// a, b, rest, each first for the lower four channels of every chunk of eight, then for the upper four, so that threads' 16 bytes
// lie side by side. b alone would be off by half a unit of 2^-24 of mean * a, which at a constant image of 500 with an eps of 1e-6 is
// 0.03; `rest` is what its roundings lose (of the product by an FMA, of the sum by Knuth's two-sum). stat: {mean - pivot, 1 / deviation}.
__device__ __forceinline__ void put_factor(int c, int chunks, float2 stat, float weight, float bias, float pivot, float4* factors) {
  const float a = stat.y * weight;
  const float near = fmaf(-stat.x, a, bias), far = __fmul_rn(pivot, a);
  const float b = __fsub_rn(near, far), taken = __fsub_rn(b, near);
  const float rest = __fsub_rn(__fsub_rn(__fsub_rn(near, __fsub_rn(b, taken)), __fadd_rn(far, taken)), fmaf(pivot, a, -far));
  float* to = reinterpret_cast<float*>(factors) + (c >> 3) * 4 + ((c >> 2) & 1) * chunks * 4 + (c & 3);
  to[0] = a;
  to[8 * chunks] = b;
  to[16 * chunks] = isinf(b) ? 0.f : rest;  // a bias without a number: the difference of two of it would be none
}
__host__ __device__ constexpr int factor_bytes(int channels) { return channels * 12; }
template <bool FP16>
__device__ __forceinline__ float gn_weight(const GnParams& p, int c) { return p.weight != nullptr ? int8_unpack2<FP16>(p.weight[c]).x : 1.f; }
template <bool FP16>
__device__ __forceinline__ float gn_bias(const GnParams& p, int c) { return p.bias != nullptr ? int8_unpack2<FP16>(p.bias[c]).x : 0.f; }

// All channels' factors of image blockIdx.y; the groups' statistics stand behind them.
template <bool FP16>
__device__ __forceinline__ void group_norm_factors(const GnParams& p, float4* factors) {
  const int per = p.channels / p.groups;
  float2* stat = reinterpret_cast<float2*>(factors + factor_bytes(p.channels) / 16);
  const uint16_t* pivots = p.pivots + static_cast<long long>(blockIdx.y) * p.groups;
  const float2* in = p.partial + static_cast<long long>(blockIdx.y) * p.strips.strips * p.groups;
  float weight = 1.f, bias = 0.f;  // on their way while the strips are joined
  float pivot = 0.f;
  const int own = group_of(threadIdx.x, p.inv_per);
  if (threadIdx.x < p.channels) {
    weight = gn_weight<FP16>(p, threadIdx.x);
    bias = gn_bias<FP16>(p, threadIdx.x);
    pivot = int8_unpack2<FP16>(pivots[own]).x;
  }
  join_strips<kGnThreads>(p.groups, p.strips, p.rows, per, p.eps, stat, [&](int k, int g) { return in[static_cast<long long>(k) * p.groups + g]; });
  __syncthreads();
  if (threadIdx.x < p.channels) put_factor(threadIdx.x, p.channels / 8, stat[own], weight, bias, pivot, factors);
  for (int c = threadIdx.x + kGnThreads; c < p.channels; c += kGnThreads) {
    const int g = group_of(c, p.inv_per);
    put_factor(c, p.channels / 8, stat[g], gn_weight<FP16>(p, c), gn_bias<FP16>(p, c), int8_unpack2<FP16>(pivots[g]).x, factors);
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

// Eight channels of a row, normalised, to dst.
template <bool FP16, bool SILU, bool VEC>
__device__ __forceinline__ void apply8(const uint4& raw, const float (&a)[8], const float (&b)[8], const float (&rest)[8], uint16_t* dst) {
  uint4 y = raw;
  uint32_t* u = reinterpret_cast<uint32_t*>(&y);
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const float2 v = int8_unpack2<FP16>(u[k]);
    float y0 = fmaf(v.x, a[2 * k], b[2 * k]) + rest[2 * k], y1 = fmaf(v.y, a[2 * k + 1], b[2 * k + 1]) + rest[2 * k + 1];
    if constexpr (SILU) y0 = silu(y0), y1 = silu(y1);
    u[k] = gn_pack<FP16>(y0, y1);
  }
  if constexpr (VEC) {
    *reinterpret_cast<uint4*>(dst) = y;
  } else {
#pragma unroll
    for (int k = 0; k < 8; ++k) dst[k] = static_cast<uint16_t>(u[k / 2] >> (16 * (k & 1)));
  }
}
__device__ __forceinline__ void read_factors(const float4* factors, int chunks, int chunk, float (&a)[8], float (&b)[8], float (&rest)[8]) {
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    *reinterpret_cast<float4*>(a + 4 * h) = factors[h * chunks + chunk];
    *reinterpret_cast<float4*>(b + 4 * h) = factors[(2 + h) * chunks + chunk];
    *reinterpret_cast<float4*>(rest + 4 * h) = factors[(4 + h) * chunks + chunk];
  }
}

template <bool FP16, bool SILU, bool VEC>
__global__ void __launch_bounds__(kGnThreads, 1) group_norm_apply_kernel(const __grid_constant__ GnParams p) {
  grid_dependency_release();
  grid_dependency_wait();
  extern __shared__ float4 factors[];
  const int chunks = p.channels / 8;
  const int lanes = p.strips.lanes;
  const int lane = threadIdx.x / chunks, chunk = threadIdx.x - lane * chunks, c = chunk * 8;
  group_norm_factors<FP16>(p, factors);
  if (lane >= lanes) return;
  float a[8], b[8], rest[8];
  read_factors(factors, chunks, chunk, a, b, rest);
  // the strip's rows from the last to the first
  const int strip = static_cast<int>(blockIdx.x), count = p.strips.rows_of_lane(strip, lane);
  const long long step = p.strips.step(), last = p.strips.first(strip, lane) + (count - 1) * step, out_step = step * p.out_row_stride;
  uint16_t* out = p.out + blockIdx.y * p.out_batch_stride + last * p.out_row_stride + c;
  walk_rows<VEC>(p.x + blockIdx.y * p.x_batch_stride + last * p.x_row_stride, c, p.channels, count, -step * p.x_row_stride, [] {},
                 [&](const uint4& raw, int i) { apply8<FP16, SILU, VEC>(raw, a, b, rest, out - i * out_step); });
}

// A row in 8 bits, held by a team as NCH chunks of eight channels a thread.
template <bool FP16, bool SILU, int TEAM, int NCH, int THREADS>
__device__ __forceinline__ void row_to_int8(const GnParams& p, const Team<TEAM, THREADS>& team, int turn, const uint4 (&raw)[NCH], const float4* factors,
                                            int c0, long long row, bool live) {
  const int chunks = p.channels / 8;
  float2 y[NCH][4];
  float top = 0.f;
#pragma unroll
  for (int k = 0; k < NCH; ++k) {
    const int c = c0 + k * TEAM * 8;
    if (c >= p.channels) continue;
    const uint32_t* u = reinterpret_cast<const uint32_t*>(&raw[k]);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int at = (i >> 1) * chunks + (c >> 3);
      const float4 av = factors[at], bv = factors[2 * chunks + at], rv = factors[4 * chunks + at];
      const float2 v = fma2(int8_unpack2<FP16>(u[i]), i & 1 ? make_float2(av.z, av.w) : make_float2(av.x, av.y), i & 1 ? make_float2(bv.z, bv.w) : make_float2(bv.x, bv.y));
      y[k][i] = add2(v, i & 1 ? make_float2(rv.z, rv.w) : make_float2(rv.x, rv.y));
      if constexpr (SILU) y[k][i] = make_float2(silu(y[k][i].x), silu(y[k][i].y));
      top = max_magnitude(max_magnitude(top, y[k][i].x), y[k][i].y);
    }
  }
  const Int8Scale s = int8_scale(team.max(__float_as_uint(top) & 0x7FFFFFFFu, turn));
#pragma unroll
  for (int k = 0; k < NCH; ++k)
    if (live && c0 + k * TEAM * 8 < p.channels) int8_put8_of(p.q + row * p.out_row_stride, c0 + k * TEAM * 8, s, y[k]);
  if (live && c0 == 0) p.q_scale[row] = int8_step(s);
}

// The rows in 8 bits: TEAM threads hold a row of at most TEAM * NCH * 8 channels, ROWS of them at a time, and have the next ones
// on their way.
template <bool FP16, bool SILU, int TEAM, int NCH, int ROWS, bool VEC>
__global__ void __launch_bounds__(kGnThreads, 1) group_norm_int8_kernel(const __grid_constant__ GnParams p) {
  grid_dependency_release();
  grid_dependency_wait();
  extern __shared__ float4 factors[];
  __shared__ float red[2][kGnThreads / 32];
  const Team<TEAM, kGnThreads> team{red};
  constexpr int kTeams = kGnThreads / TEAM;
  const int c0 = static_cast<int>(threadIdx.x % TEAM) * 8;
  // every gridDim.x-th tile of kTeams * ROWS rows, from the last row to the first; a team has every kTeams-th row of a tile
  const long long step = static_cast<long long>(gridDim.x) * kTeams * ROWS, x_step = static_cast<long long>(kTeams) * p.x_row_stride;
  long long row = p.rows - 1 - (static_cast<long long>(blockIdx.x) * kTeams * ROWS + threadIdx.x / TEAM);
  long long end = p.rows - 1 - static_cast<long long>(blockIdx.x) * kTeams * ROWS;  // the tile's last row: the same in all teams
  const uint16_t* x = p.x + blockIdx.y * p.x_batch_stride + row * p.x_row_stride;
  uint4 next[ROWS][NCH];
  auto fetch = [&](long long at) {
#pragma unroll
    for (int i = 0; i < ROWS; ++i)
#pragma unroll
      for (int k = 0; k < NCH; ++k) {
        next[i][k] = make_uint4(0, 0, 0, 0);
        if (at >= i * kTeams && c0 + k * TEAM * 8 < p.channels) next[i][k] = int8_load8(x - i * x_step, c0 + k * TEAM * 8, p.channels, VEC);
      }
  };
  fetch(row);
  group_norm_factors<FP16>(p, factors);
  for (int turn = 0; end >= 0; row -= step, end -= step) {
    uint4 raw[ROWS][NCH];
#pragma unroll
    for (int i = 0; i < ROWS; ++i)
#pragma unroll
      for (int k = 0; k < NCH; ++k) raw[i][k] = next[i][k];
    x -= step * p.x_row_stride;
    if (end >= step) fetch(row - step);
#pragma unroll
    for (int i = 0; i < ROWS; ++i, turn ^= 1)
      row_to_int8<FP16, SILU, TEAM, NCH, kGnThreads>(p, team, turn, raw[i], factors, c0, blockIdx.y * p.rows + row - i * kTeams, row >= i * kTeams);
  }
}

// One launch for what fits the shared memory of a few SMs: a cluster of CTAs takes a slab of channels (whole groups) of an
// image, each CTA a strip of its rows, which stay in its shared memory between the two passes; the CTAs read each other's
// statistics there. p.strips: a strip is a CTA; p.slab: channels of a slab. Shared memory: the rows, the sums (then the
// factors), the strip's statistics, the groups' statistics. The image's first row, with the pivots, stays in between: `out` may be
// x, so nothing of x is read when the cluster has met.
template <bool FP16, bool SILU, bool VEC, bool INT8>
__global__ void __launch_bounds__(cluster_threads(INT8), INT8 ? 1 : 2) group_norm_cluster_kernel(const __grid_constant__ GnParams p) {
  grid_dependency_release();
  grid_dependency_wait();
  constexpr int kThreads = cluster_threads(INT8);
  extern __shared__ float4 smem4[];
  __shared__ float red[2][kThreads / 32];
  const int chunks = p.slab / 8, per = p.channels / p.groups, groups = p.slab / per;
  const int lanes = p.strips.lanes;
  const int lane = threadIdx.x / chunks, chunk = threadIdx.x - lane * chunks;
  const int slab0 = static_cast<int>(blockIdx.y) * p.slab;
  const int rank = static_cast<int>(blockIdx.x);
  uint4* held = reinterpret_cast<uint4*>(smem4);  // [tiles * lanes][chunks]
  float4* factors = smem4 + p.strips.tiles_of(0) * lanes * chunks;
  uint16_t* row0 = reinterpret_cast<uint16_t*>(factors + sums_bytes(lanes, p.slab) / 16);
  float2* strip = reinterpret_cast<float2*>(row0 + p.slab);
  float2* stat = strip + groups;
  float weight = 1.f, bias = 0.f;  // on their way while the statistics are made
  if (threadIdx.x < p.slab) {
    weight = gn_weight<FP16>(p, slab0 + threadIdx.x);
    bias = gn_bias<FP16>(p, slab0 + threadIdx.x);
  }
  strip_stats<kThreads, FP16, VEC>(
      p.x + blockIdx.z * p.x_batch_stride + slab0, p.x_row_stride, p.strips, rank, p.slab, per, p.inv_per, reinterpret_cast<float*>(factors), row0,
      [&](const uint4& raw, int at) { held[(at * lanes + lane) * chunks + chunk] = raw; },
      [&](int g, float2 v) { strip[g] = v; });
  __syncthreads();
  cluster_sync_all();
  join_strips<kThreads>(groups, p.strips, p.rows, per, p.eps, stat, [&](int k, int g) {
    float2 v;
    asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(map_to_cta(strip + g, static_cast<uint32_t>(k))) : "memory");
    return v;
  });
  __syncthreads();
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");  // this CTA has read the others' statistics
  auto put = [&](int c, float w, float b) {
    const int g = group_of(c, p.inv_per);
    put_factor(c, chunks, stat[g], w, b, int8_unpack2<FP16>(row0[g * per]).x, factors);
  };
  if (threadIdx.x < p.slab) put(threadIdx.x, weight, bias);
  for (int c = threadIdx.x + kThreads; c < p.slab; c += kThreads) put(c, gn_weight<FP16>(p, slab0 + c), gn_bias<FP16>(p, slab0 + c));
  __syncthreads();
  if constexpr (INT8) {
    const Team<32, kThreads> team{red};
    const int c0 = static_cast<int>(threadIdx.x & 31) * 8;
    const int mine = p.strips.rows_of(rank);
    for (int r = static_cast<int>(threadIdx.x) >> 5; r < mine; r += kThreads / 32) {
      uint4 raw[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) raw[k] = c0 + k * 256 < p.slab ? held[r * chunks + (c0 >> 3) + k * 32] : make_uint4(0, 0, 0, 0);
      const long long row = p.strips.first(rank, r % lanes) + r / lanes * p.strips.step();
      row_to_int8<FP16, SILU, 32, 4, kThreads>(p, team, 0, raw, factors, c0, blockIdx.z * p.rows + row, true);
    }
  } else if (lane < lanes) {
    float a[8], b[8], rest[8];
    read_factors(factors, chunks, chunk, a, b, rest);
    const int count = p.strips.rows_of_lane(rank, lane);
    uint16_t* out = p.out + blockIdx.z * p.out_batch_stride + p.strips.first(rank, lane) * p.out_row_stride + slab0 + chunk * 8;
    const long long out_step = p.strips.step() * p.out_row_stride;
    for (int at = 0; at < count; ++at) apply8<FP16, SILU, VEC>(held[(at * lanes + lane) * chunks + chunk], a, b, rest, out + at * out_step);
  }
  __syncwarp();
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");  // the others have read this CTA's
}

// Strips per image: one CTA per SM over all images, at least two tiles each.
int strips_of(long long batch, long long rows, int channels) {
  const long long lanes = kGnThreads / (channels / 8);
  long long n = 148 / batch;
  const long long most = (rows + lanes * 2 - 1) / (lanes * 2);
  if (n > most) n = most;
  return static_cast<int>(n < 1 ? 1 : n);
}

Strips make_strips(long long rows, int strips, int lanes) {
  const long long tiles = (rows + lanes - 1) / lanes;
  return {strips, lanes, static_cast<int>(tiles / strips), static_cast<int>(tiles % strips), static_cast<int>((tiles - 1) % strips),
          static_cast<int>(tiles * lanes - rows)};
}

// The one-launch form: whether the call fits it, and its slab, strips and shared memory.
constexpr int kClusterCtas = 8;
struct GnCluster {
  int slab;
  size_t smem;
};
bool cluster_of(long long batch, long long rows, int channels, int groups, bool int8, GnCluster* to) {
  const int per = channels / groups;
  int unit = per;  // whole groups and whole chunks
  while (unit % 8 != 0) unit += per;
  if ((int8 && (channels > 1024 || rows > 384)) || batch > 33 || rows > 33LL * 8 * 100 * 1024 / 2 / (batch * channels)) return false;
  for (int slab = int8 ? channels : unit; slab <= channels && slab / 8 <= cluster_threads(int8); slab += unit) {
    if (channels % slab != 0 || (slab < 32 && slab < channels)) continue;  // 64 bytes of a row at least
    const long long clusters = batch * (channels / slab), lanes = cluster_threads(int8) / (slab / 8);
    const long long tiles = ((rows + lanes - 1) / lanes + kClusterCtas - 1) / kClusterCtas;
    if (rows <= lanes * (kClusterCtas - 1)) continue;  // each CTA has rows
    const long long held = tiles * lanes * slab * 2, smem = held + sums_bytes(static_cast<int>(lanes), slab) + slab * 2 + slab / per * 16;
    // So many clusters of this size are on the GPU at a time; a second wave costs more than a second launch. 8-bit rows need all
    // channels of a pixel in one CTA, which leaves few CTAs: with 82 KB each, two images of 32 x 32 x 640 took 15 us, in two
    // launches 9.9; and a warp has a row, so many rows take long however short they are: 384 x 256 7.3 us against 7.6 in two
    // launches, 512 x 256 7.9 against 7.5, 6560 x 16 41 against 10.
    if (clusters <= (smem <= 100 * 1024 && !int8 ? 33 : 15) && smem <= 200 * 1024 && (!int8 || held <= 32 * 1024)) {
      *to = {slab, static_cast<size_t>(smem)};
      return true;
    }
  }
  return false;
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
  if (a->x == nullptr || a->out == nullptr) return set_error(HDIT_ERR_BAD_ARG, "null x / out");
  return HDIT_OK;
}

bool off16(const void* p, int64_t a, int64_t b) { return (reinterpret_cast<uintptr_t>(p) & 15) != 0 || a % 8 != 0 || b % 8 != 0; }

// of the two launches' kernels: the factors of 4096 channels and the statistics of as many groups
constexpr int kGnMaxBytes = factor_bytes(kMaxChannels) + kMaxChannels * static_cast<int>(sizeof(float2));

template <auto kKernel>
cudaError_t launch_strips(const GnParams& p, long long batch, size_t smem, cudaStream_t st) {
  // static shared memory counts, too
  const cudaError_t e = smem > 47 * 1024 ? allow_shared_memory<kKernel, kGnMaxBytes>() : cudaSuccess;
  if (e != cudaSuccess) return e;
  return launch_overlapped(kKernel, dim3(static_cast<unsigned>(p.strips.strips), static_cast<unsigned>(batch)), dim3(kGnThreads), smem, st, 1, p);
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
  p.inv_per = static_cast<float>(a->groups) / static_cast<float>(a->channels);
  p.vec = out_vec && !off16(a->x, a->x_batch_stride, a->x_row_stride);
  return p;
}

size_t apply_bytes(const GnParams& p) { return factor_bytes(p.channels) + static_cast<size_t>(p.groups) * sizeof(float2); }

template <bool FP16, bool VEC>
cudaError_t launch_stats(const GnParams& p, long long batch, cudaStream_t st) {
  const size_t smem = static_cast<size_t>(kGnThreads / (p.channels / 8)) * stats_pitch(p.channels) * 2 * sizeof(float) + p.channels * sizeof(uint16_t);
  return launch_strips<group_norm_stats_kernel<FP16, VEC>>(p, batch, smem, st);
}

template <bool FP16, bool VEC>
cudaError_t launch_apply(const GnParams& p, long long batch, cudaStream_t st) {
  return p.act == HDIT_ACT_SILU ? launch_strips<group_norm_apply_kernel<FP16, true, VEC>>(p, batch, apply_bytes(p), st)
                                : launch_strips<group_norm_apply_kernel<FP16, false, VEC>>(p, batch, apply_bytes(p), st);
}

template <bool FP16, bool SILU, bool VEC>
cudaError_t launch_int8_act(const GnParams& p, long long batch, cudaStream_t st) {
  const size_t smem = apply_bytes(p);
  if (p.channels <= 64) return launch_strips<group_norm_int8_kernel<FP16, SILU, 8, 1, 4, VEC>>(p, batch, smem, st);
  if (p.channels <= 128) return launch_strips<group_norm_int8_kernel<FP16, SILU, 16, 1, 4, VEC>>(p, batch, smem, st);
  if (p.channels <= 256) return launch_strips<group_norm_int8_kernel<FP16, SILU, 32, 1, 4, VEC>>(p, batch, smem, st);
  if (p.channels <= 512) return launch_strips<group_norm_int8_kernel<FP16, SILU, 32, 2, 2, VEC>>(p, batch, smem, st);
  if (p.channels <= 1024) return launch_strips<group_norm_int8_kernel<FP16, SILU, 32, 4, 1, VEC>>(p, batch, smem, st);
  return launch_strips<group_norm_int8_kernel<FP16, SILU, 128, 4, 1, VEC>>(p, batch, smem, st);
}

template <bool FP16, bool VEC>
cudaError_t launch_int8(const GnParams& p, long long batch, cudaStream_t st) {
  return p.act == HDIT_ACT_SILU ? launch_int8_act<FP16, true, VEC>(p, batch, st) : launch_int8_act<FP16, false, VEC>(p, batch, st);
}

template <bool FP16, bool SILU, bool VEC>
cudaError_t launch_cluster_act(const GnParams& p, const GnCluster& c, bool int8, long long batch, cudaStream_t st) {
  auto kernel = int8 ? group_norm_cluster_kernel<FP16, SILU, VEC, true> : group_norm_cluster_kernel<FP16, SILU, VEC, false>;
  const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 200 * 1024);
  if (e != cudaSuccess) return e;
  return launch_overlapped(kernel, dim3(kClusterCtas, static_cast<unsigned>(p.channels / c.slab), static_cast<unsigned>(batch)),
                           dim3(cluster_threads(int8)), c.smem, st, kClusterCtas, p);
}

template <bool FP16, bool VEC>
cudaError_t launch_cluster(const GnParams& p, const GnCluster& c, bool int8, long long batch, cudaStream_t st) {
  return p.act == HDIT_ACT_SILU ? launch_cluster_act<FP16, true, VEC>(p, c, int8, batch, st) : launch_cluster_act<FP16, false, VEC>(p, c, int8, batch, st);
}

#define HDIT_GN_OF(f, fp16, vec) ((fp16) ? ((vec) ? f<true, true> : f<true, false>) : ((vec) ? f<false, true> : f<false, false>))

int run_group_norm(const hdit_group_norm_args* a, bool int8) {
  GnParams p = params_of(a, int8 || !off16(a->out, a->out_batch_stride, a->out_row_stride));
  const bool fp16 = a->dtype == HDIT_FP16;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(a->stream);
  GnCluster c;
  if (cluster_of(a->batch, a->rows, p.channels, p.groups, int8, &c)) {
    p.slab = c.slab;
    p.strips = make_strips(a->rows, kClusterCtas, cluster_threads(int8) / (c.slab / 8));
    HDIT_CUDA_OK((HDIT_GN_OF(launch_cluster, fp16, p.vec)(p, c, int8, a->batch, st)));
    return HDIT_OK;
  }
  if (a->scratch == nullptr || (reinterpret_cast<uintptr_t>(a->scratch) & 7) != 0) return set_error(HDIT_ERR_BAD_ARG, "scratch is null or not 8-byte aligned");
  p.strips = make_strips(a->rows, strips_of(a->batch, a->rows, p.channels), kGnThreads / (p.channels / 8));
  p.pivots = reinterpret_cast<uint16_t*>(p.partial + a->batch * p.strips.strips * a->groups);
  HDIT_CUDA_OK((HDIT_GN_OF(launch_stats, fp16, p.vec)(p, a->batch, st)));
  if (int8) HDIT_CUDA_OK((HDIT_GN_OF(launch_int8, fp16, p.vec)(p, a->batch, st)));
  else HDIT_CUDA_OK((HDIT_GN_OF(launch_apply, fp16, p.vec)(p, a->batch, st)));
  return HDIT_OK;
}

}  // namespace
}  // namespace hdit

extern "C" int64_t hdit_group_norm_scratch(int64_t batch, int64_t rows, int64_t channels, int64_t groups, int32_t int8_rows) {
  using namespace hdit;
  GnCluster c;
  if (batch <= 0 || rows <= 0 || rows > 0x7fffffffLL || channels <= 0 || groups <= 0 || channels % 8 != 0 || channels > kMaxChannels || channels % groups != 0)
    return 0;
  if (cluster_of(batch, rows, static_cast<int>(channels), static_cast<int>(groups), int8_rows != 0, &c)) return 0;
  return batch * groups * (strips_of(batch, rows, static_cast<int>(channels)) * static_cast<int64_t>(sizeof(float2)) + 2);
}

extern "C" int hdit_group_norm(const hdit_group_norm_args* a) {
  using namespace hdit;
  const int rc = check_gn(a);
  if (rc != HDIT_OK || a->batch == 0 || a->rows == 0) return rc;
  // rows one after the other, and images one after the other or their rows in turn
  const int64_t row = a->out_row_stride, image = a->out_batch_stride;
  const bool rows_apart = a->rows == 1 || row >= a->channels;
  const bool images_apart = a->batch == 1 || image >= (a->rows - 1) * row + a->channels || (image >= a->channels && row >= (a->batch - 1) * image + a->channels);
  if (!rows_apart || !images_apart) return set_error(HDIT_ERR_SHAPE, "rows of out overlap");
  return run_group_norm(a, false);
}

extern "C" int hdit_group_norm_int8(const hdit_group_norm_args* a) {
  using namespace hdit;
  const int rc = check_gn(a);
  if (rc != HDIT_OK) return rc;
  if ((reinterpret_cast<uintptr_t>(a->out) & 15) != 0 || a->out_row_stride % 16 != 0 || a->out_row_stride < a->channels)
    return set_error(HDIT_ERR_SHAPE, "8-bit rows need a 16-byte aligned pointer and a row stride that is a multiple of 16 and covers a row");
  if (a->batch == 0 || a->rows == 0) return HDIT_OK;
  if (a->out_scale == nullptr) return set_error(HDIT_ERR_BAD_ARG, "null scale");
  return run_group_norm(a, true);
}
