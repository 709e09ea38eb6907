// The linear layer over 8-bit integers (int8_linear_sm100.cu) for a few rows, such as the adaLN vectors of an image or two: the
// weight is read once, nothing else counts, and a 128-row tensor-core tile would be nearly empty. The weight streams through
// registers into the warp-wide integer MMA (mma.sync m16n8k32: a contraction at the memory's rate leaves the tensor pipe
// idle, and tensor memory and TMA stages only lengthen the way of each byte):
//
//   sixteen output channels are the MMA's rows, the rows of x its columns. A CTA's eight warps take every
//   eighth 64-byte chunk of K each and add their exact integer sums in shared memory. In a chunk, lane t of a quad reads 16
//   bytes (16 t ..) of a row with one load and feeds them to two MMAs; which elements of K an MMA multiplies together does not
//   matter as long as both operands agree, so the rows of x lie in shared memory as they are.
//
// us, this kernel | 128 x 128 tiles, 8-bit rows: 9216 x 1536, 1 row 4.4 | 7.8, 8 rows 6.2 | 7.6, 16 rows 9.1 | 7.6 (as two column
// tiles); 18432 x 3072, 1 row 12.4 | 16.2, 8 rows 16.1 | 16.0: taken for up to eight rows. 16-bit rows are brought into 8 bits by every
// CTA for itself where there are one or two, or where the first pass over a row is one turn of its warps and no SM has two CTAs
// that do it: a launch less, 3 us on the host. us in a graph, so | after quantize_rows: 9216 x 1536, 2 rows 5.4 | 5.6; 2048 x 2048, 4
// rows 5.5 | 6.3; 1024 x 1024, 8 rows 4.4 | 5.3; 2368 x 512, 8 rows 3.6 | 4.5; 256 x 768, 8 rows 4.5 | 4.6. Not: 9216 x 1536, 4 rows
// 6.7 | 6.3; 9216 x 768, 8 rows 6.9 | 5.7; 6144 x 256, 8 rows 4.8 | 4.2 (many CTAs); 512 x 1536, 5 rows 5.3 | 4.9 (two turns).
#include "gemm_common.cuh"
#include "host_common.h"
#include "int8_linear.h"
#include "int8_rows.cuh"

namespace hdit {
namespace {

constexpr int kFewThreads = 256;
constexpr int kFewWarps = kFewThreads / 32;
constexpr int kChunksAhead = 4;
constexpr int kFewCtas = 4;  // to an SM
constexpr int kFewMaxBytes = 160 * 1024;  // of rows in shared memory

struct FewParams {
  const uint16_t* x;  // or null: a, a_scale hold the rows
  long long x_rows_per_batch, x_batch_stride, x_row_stride;
  const int8_t* a;
  long long lda;
  const float* a_scale;
  const int8_t* w;
  long long ldw;
  const float* w_scale;
  const uint16_t* bias;
  uint16_t* out;
  long long ldo;
  const uint16_t* residual;
  long long ldr;
  const uint16_t* gate;
  long long gate_batch_stride, rows_per_batch;
  int M, N, K, pitch, epilogue;
  bool vec;  // 16-bit rows are whole 16-byte chunks on 16-byte boundaries
};

__device__ __forceinline__ void mma_s8(int (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

template <bool FP16>
__global__ void __launch_bounds__(kFewThreads, kFewCtas) int8_linear_few_kernel(const __grid_constant__ FewParams p) {
  grid_dependency_release();
  grid_dependency_wait();
  extern __shared__ __align__(16) uint8_t rows8[];  // M rows of x, `pitch` bytes apart, zeros behind K
  __shared__ int sums[kFewWarps][16][kInt8FewRows + 1];
  __shared__ float row_scale[kInt8FewRows];
  __shared__ uint32_t tops[kFewWarps];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, t = lane & 3;
  const int n_chunks = (p.K + 63) / 64, groups = (p.N + 15) / 16;

  // the first weights are on their way while the rows are prepared
  uint4 lo[kChunksAhead], hi[kChunksAhead];  // of channels g and g + 8
  const int8_t *w_lo = nullptr, *w_hi = nullptr;
  auto channels = [&](int group) {
    const int n0 = min(group * 16 + g, p.N - 1), n1 = min(group * 16 + g + 8, p.N - 1);
    w_lo = p.w + n0 * p.ldw + t * 16;
    w_hi = p.w + n1 * p.ldw + t * 16;
  };
  auto fetch = [&](int chunk) {
#pragma unroll
    for (int i = 0; i < kChunksAhead; ++i) {
      const int at = (chunk + i * kFewWarps) * 64;
      lo[i] = hi[i] = make_uint4(0, 0, 0, 0);
      if (at + t * 16 < p.K) {  // the 16 bytes may reach into the row's padding: there the rows of x are zeros
        lo[i] = *reinterpret_cast<const uint4*>(w_lo + at);
        hi[i] = *reinterpret_cast<const uint4*>(w_hi + at);
      }
    }
  };
  channels(blockIdx.x);
  fetch(warp);

  if (p.x != nullptr) {
    // all rows at a time, a power of two of the warps to each
    const int per = kFewWarps >> (p.M > 4 ? 3 : p.M > 2 ? 2 : p.M - 1), m = warp / per;
    const int c0 = (static_cast<int>(threadIdx.x) - m * per * 32) * 8, step = per * 256;
    const uint16_t* xr = p.x;
    if (m < p.M) {
      xr += m / p.x_rows_per_batch * p.x_batch_stride + m % p.x_rows_per_batch * p.x_row_stride;
      uint32_t top2 = 0;
#pragma unroll 4
      for (int c = c0; c < p.K; c += step) {
        const uint4 raw = int8_load8(xr, c, p.K, p.vec);
        top2 = __vmaxu2(__vmaxu2(top2, __vmaxu2(raw.x & 0x7FFF7FFFu, raw.y & 0x7FFF7FFFu)), __vmaxu2(raw.z & 0x7FFF7FFFu, raw.w & 0x7FFF7FFFu));
      }
      const uint32_t v = __reduce_max_sync(0xffffffffu, (top2 & 0xFFFFu) > (top2 >> 16) ? top2 & 0xFFFFu : top2 >> 16);
      if (lane == 0) tops[warp] = v;
    }
    __syncthreads();
    if (m < p.M) {
      uint32_t top = 0;
      for (int w = 0; w < per; ++w) top = max(top, tops[m * per + w]);
      const Int8Scale s = int8_scale(__float_as_uint(int8_unpack2<FP16>(top).x));
      const float inv17 = 17.f * s.inv;
#pragma unroll 4
      for (int c = c0; c < p.pitch; c += step) {
        const uint4 raw = c < p.K ? int8_load8(xr, c, p.K, p.vec) : make_uint4(0, 0, 0, 0);
        int8_put8<FP16, false>(reinterpret_cast<int8_t*>(rows8) + m * p.pitch, c, p.pitch, s, inv17, raw);
      }
      if (c0 == 0) row_scale[m] = int8_step(s);
    }
  } else {
    const int chunks16 = p.pitch / 16;
    for (int i = threadIdx.x; i < p.M * chunks16; i += kFewThreads) {
      const int m = i / chunks16, c = (i - m * chunks16) * 16;
      uint4 v = make_uint4(0, 0, 0, 0);
      const int8_t* src = p.a + m * p.lda + c;
      if (c + 16 <= p.K) {
        v = *reinterpret_cast<const uint4*>(src);
      } else {
        uint32_t* e = reinterpret_cast<uint32_t*>(&v);
        for (int k = 0; c + k < p.K; ++k) e[k >> 2] |= static_cast<uint32_t>(static_cast<uint8_t>(src[k])) << (8 * (k & 3));
      }
      *reinterpret_cast<uint4*>(rows8 + m * p.pitch + c) = v;
    }
    if (threadIdx.x < p.M) row_scale[threadIdx.x] = p.a_scale[threadIdx.x];
  }
  __syncthreads();

  for (int group = blockIdx.x; group < groups; group += gridDim.x) {
    int acc[4] = {0, 0, 0, 0};
    for (int chunk = warp; chunk < n_chunks; chunk += kChunksAhead * kFewWarps) {
#pragma unroll
      for (int i = 0; i < kChunksAhead; ++i) {
        const int at = chunk + i * kFewWarps;
        if (at >= n_chunks) break;
        uint4 b = make_uint4(0, 0, 0, 0);
        if (g < p.M) b = *reinterpret_cast<const uint4*>(rows8 + g * p.pitch + at * 64 + t * 16);
        mma_s8(acc, lo[i].x, hi[i].x, lo[i].y, hi[i].y, b.x, b.y);
        mma_s8(acc, lo[i].z, hi[i].z, lo[i].w, hi[i].w, b.z, b.w);
      }
      if (chunk + kChunksAhead * kFewWarps < n_chunks) fetch(chunk + kChunksAhead * kFewWarps);
    }
    if (group + gridDim.x < groups) {
      channels(group + gridDim.x);
      fetch(warp);
    }
    // channels g (0, 1) and g + 8 (2, 3), rows 2 t and 2 t + 1
    sums[warp][g][2 * t] = acc[0];
    sums[warp][g][2 * t + 1] = acc[1];
    sums[warp][g + 8][2 * t] = acc[2];
    sums[warp][g + 8][2 * t + 1] = acc[3];
    __syncthreads();
    for (int i = threadIdx.x; i < p.M * 16; i += kFewThreads) {
      const int m = i >> 4, ch = i & 15, n = group * 16 + ch;
      int sum = 0;
#pragma unroll
      for (int w = 0; w < kFewWarps; ++w) sum += sums[w][ch][m];
      if (n < p.N) {
        const float bias = p.bias != nullptr ? to_f<FP16>(p.bias[n]) : 0.f;
        float v = int8_value2(sum, sum, row_scale[m], make_float2(p.w_scale[n], p.w_scale[n]), make_float2(bias, bias)).x;
        if (p.epilogue == HDIT_GEMM_BIAS_GELU_TANH) v = int8_gelu2(make_float2(v, v)).x;
        else if (p.epilogue == HDIT_GEMM_BIAS_GATE_RESIDUAL)
          v = fmaf(to_f<FP16>(p.gate[m / p.rows_per_batch * p.gate_batch_stride + n]), v, to_f<FP16>(p.residual[m * p.ldr + n]));
        p.out[m * p.ldo + n] = from_f<FP16>(v);
      }
    }
    __syncthreads();
  }
}

int few_pitch(long long k) {
  const long long p = (k + 63) / 64 * 64;
  return static_cast<int>(p % 128 == 0 ? p + 64 : p);  // eight rows' 64 bytes then lie in different banks two by two
}

template <bool FP16>
int launch_few(const FewParams& p, cudaStream_t st) {
  constexpr auto kernel = int8_linear_few_kernel<FP16>;
  const int smem = p.M * p.pitch;
  if (smem > 32 * 1024) HDIT_CUDA_OK((allow_shared_memory<kernel, kFewMaxBytes>()));
  const int groups = (p.N + 15) / 16, most = sm_count() * kFewCtas;
  HDIT_CUDA_OK(launch_overlapped(kernel, dim3(static_cast<unsigned>(groups < most ? groups : most)), dim3(kFewThreads), static_cast<size_t>(smem), st, 1, p));
  return HDIT_OK;
}

}  // namespace

bool int8_linear_few_takes(const hdit_int8_linear_args* a) {
  return a->m <= kInt8FewRows && a->m * few_pitch(a->k) <= kFewMaxBytes;
}
// Rows that take more than 44 KB leave the weights' stream too little of an SM's first-level cache, or room for one CTA only. us, here |
// in tiles: 3 rows of 8192 -> 3072 12.9 | 16.5, 5 rows (40 KB) 15.4 | 16.4, 6 rows (48 KB) 21.5 | 16.4; 12288 -> 12288, 3 rows (36 KB)
// 38 | 45, 4 rows (48 KB) 64 | 45. One or two rows always come here: they need no scratch.
bool int8_linear_few_pays(const hdit_int8_linear_args* a) { return a->m <= 2 || a->m * few_pitch(a->k) <= 44 * 1024; }
// Not where the result may take x's place (x = residual = out): a CTA would write what another one has yet to read.
bool int8_linear_few_quantizes(const hdit_int8_linear_args* a) {
  if (a->m > 2 && (a->k > (a->m > 4 ? 1024 : 2048) || a->n > 16 * 148)) return false;  // 1024 elements: four loads of a warp's lanes
  const int64_t per = a->x_rows_per_batch < a->m ? a->x_rows_per_batch : a->m, entries = (a->m + per - 1) / per;
  const uintptr_t x0 = reinterpret_cast<uintptr_t>(a->x), x1 = x0 + 2 * ((entries - 1) * a->x_batch_stride + (per - 1) * a->x_row_stride + a->k);
  const uintptr_t o0 = reinterpret_cast<uintptr_t>(a->out), o1 = o0 + 2 * ((a->m - 1) * a->ldo + a->n);
  return x1 <= o0 || o1 <= x0;
}

int int8_linear_few(const hdit_int8_linear_args* a) {
  FewParams p{};
  if (a->x != nullptr && int8_linear_few_quantizes(a)) {
    p.x = static_cast<const uint16_t*>(a->x);
    p.x_rows_per_batch = a->x_rows_per_batch;
    p.x_batch_stride = a->x_batch_stride;
    p.x_row_stride = a->x_row_stride;
    p.vec = a->k % 8 == 0 && (reinterpret_cast<uintptr_t>(a->x) & 15) == 0 && a->x_batch_stride % 8 == 0 && a->x_row_stride % 8 == 0;
  }
  p.a = static_cast<const int8_t*>(a->a);
  p.lda = a->lda;
  p.a_scale = a->a_scale;
  p.w = static_cast<const int8_t*>(a->w);
  p.ldw = a->ldw;
  p.w_scale = a->w_scale;
  p.bias = static_cast<const uint16_t*>(a->bias);
  p.out = static_cast<uint16_t*>(a->out);
  p.ldo = a->ldo;
  p.residual = static_cast<const uint16_t*>(a->residual);
  p.ldr = a->ldr;
  p.gate = static_cast<const uint16_t*>(a->gate);
  p.gate_batch_stride = a->gate_batch_stride;
  p.rows_per_batch = a->rows_per_batch > 0 ? a->rows_per_batch : a->m;
  p.M = static_cast<int>(a->m);
  p.N = static_cast<int>(a->n);
  p.K = static_cast<int>(a->k);
  p.pitch = few_pitch(a->k);
  p.epilogue = a->epilogue;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(a->stream);
  const bool fp16 = a->dtype == HDIT_FP16;
  return fp16 ? launch_few<true>(p, st) : launch_few<false>(p, st);
}

}  // namespace hdit
