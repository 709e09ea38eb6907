// Linear layer over 8-bit integers for sm_100a:  out = tail(s_x[m] s_w[n] sum_k q_x[m, k] q_w[n, k] + bias[n]).
//
// q_x is (M, K) and q_w (N, K), both K-contiguous signed bytes with one fp32 scale per row. The integer sums are exact (32-bit
// accumulators in tensor memory, tcgen05.mma kind::i8); everything after them runs in fp32 and is rounded to the 16-bit
// result once. The kernel has the frame of the 16-bit linear layer (gemm_sm100.cu): persistent CTAs, a TMA producer warp, an
// MMA warp, epilogue warps, two accumulators, optionally CTA pairs. A stage is 128 bytes of K as there -- 128 elements, four
// MMAs of 32 -- so operand bytes per clock are the same and the main loop of a tile takes half the time for the same K; the
// epilogue has half the time to hide behind it.
//
//   epilogue     per 32 x 64 piece of a warp: scales and bias of the warp's columns wait in shared memory since before
//                the accumulator was ready (a lane would else wait for the same 64 values from global memory one after
//                the other); the residual's piece is brought in by full 128-byte lines through the staging buffer and the
//                result leaves through it the same way, in place.
//
// All waits are bounded, see gemm_sm100.cu.
#include <math.h>

#include "gemm_common.cuh"
#include "host_common.h"

namespace hdit {
namespace {

constexpr int kTileKBytes = 128;  // one swizzle row

enum Int8Wait : int {
  Q_PROD_EMPTY = 211,
  Q_MMA_FULL = 212,
  Q_MMA_ACC_EMPTY = 213,
  Q_EPI_ACC_FULL = 214,
};

// Instruction descriptor for kind::i8: signed operands, both K-major, 32-bit integer accumulators, no saturation.
constexpr uint32_t make_idesc_i8(uint32_t m, uint32_t n) {
  return (2u << 4) | (1u << 7) | (1u << 10) | ((n >> 3) << 17) | ((m >> 4) << 24);
}

__device__ __forceinline__ void umma_i8(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t"
      ".reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n\t"
      "}"
      :
      : "r"(d_tmem), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void umma_i8_pair(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t"
      ".reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n\t"
      "}"
      :
      : "r"(d_tmem), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}

struct Int8Params {
  CUtensorMap a_map;
  CUtensorMap w_map;
  int M, N, k_blocks;
  int m_tiles, n_tiles, group_m;
  const float* a_scale;
  const float* w_scale;
  const uint16_t* bias;
  uint16_t* out;
  long long ldo;
  const uint16_t* residual;
  long long ldr;
  const uint16_t* gate;
  long long gate_batch_stride;
  int rows_per_batch;
  bool vec;  // rows of out and residual are whole 16-byte chunks
  int32_t* status;
};

template <int BN, bool PAIR>
struct Int8Cfg {
  // Four warps reach the 128 lanes of an accumulator; a second team takes the other half of the columns
  static constexpr int kPieces = BN / 64;
  static constexpr int kColTeams = BN >= 128 ? 2 : 1;
  static constexpr int kTeamPieces = (kPieces + kColTeams - 1) / kColTeams;  // the last team may have fewer
  static constexpr int kEpiWarps = 4 * kColTeams;
  static constexpr int kThreads = 64 + 32 * kEpiWarps;
  static constexpr int kTileRows = PAIR ? 256 : 128;
  static constexpr int kBRows = PAIR ? BN / 2 : BN;
  static constexpr int kABytes = 128 * kTileKBytes;
  static constexpr int kBBytes = kBRows * kTileKBytes;
  static constexpr int kStageBytes = kABytes + kBBytes;
  static constexpr int kStagingBytes = kEpiWarps * 4096;  // 32 rows x 64 columns of 16 bits per epilogue warp
  static constexpr int kColBytes = kEpiWarps * kTeamPieces * 64 * 12;  // scale, bias, gate of a warp's columns, fp32
  static constexpr int kBarBytes = 256;
  static constexpr int kStagesFit = (kMaxSmem - 1024 - kBarBytes - kStagingBytes - kColBytes) / kStageBytes;
  static constexpr int kStages = kStagesFit > 8 ? 8 : kStagesFit;
  static constexpr int kAccCols = BN == 192 ? 256 : BN;
  static constexpr int kTmemCols = 2 * kAccCols;
  static constexpr int kSmemBytes = 1024 + kStages * kStageBytes + kStagingBytes + kColBytes + kBarBytes;
  static_assert(kStages >= 3, "ring too short");
  static_assert(kTmemCols == 128 || kTmemCols == 256 || kTmemCols == 512, "TMEM allocation must be a power of two");
};

// Tile index -> (tile row, tile column): bands of group_m tile rows, column-major inside a band, as in gemm_sm100.cu
__device__ __forceinline__ void int8_tile_coords(const Int8Params& p, int tile, int& m_t, int& n_t) {
  const int per_band = p.group_m * p.n_tiles;
  const int band = tile / per_band, r = tile - band * per_band;
  const int m0 = band * p.group_m;
  const int rows = min(p.group_m, p.m_tiles - m0);
  n_t = r / rows;
  m_t = m0 + (r - n_t * rows);
}

template <int BN, bool PAIR, bool FP16, int EPI>
__global__ void __launch_bounds__(Int8Cfg<BN, PAIR>::kThreads, 1) int8_linear_kernel(const __grid_constant__ Int8Params p) {
  using C = Int8Cfg<BN, PAIR>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* stage_base = smem;
  uint8_t* staging_base = smem + C::kStages * C::kStageBytes;
  float* col_base = reinterpret_cast<float*>(staging_base + C::kStagingBytes);
  uint64_t* full = reinterpret_cast<uint64_t*>(staging_base + C::kStagingBytes + C::kColBytes);
  uint64_t* empty = full + 8;
  uint64_t* acc_full = empty + 8;
  uint64_t* acc_empty = acc_full + 2;
  uint64_t* drain_bar = acc_empty + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain_bar + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const uint32_t rank = PAIR ? cluster_ctarank() : 0u;
  const bool leader = rank == 0;
  const int unit = PAIR ? static_cast<int>(blockIdx.x >> 1) : static_cast<int>(blockIdx.x);
  const int n_units = PAIR ? static_cast<int>(gridDim.x >> 1) : static_cast<int>(gridDim.x);
  const int total_tiles = p.m_tiles * p.n_tiles;

  if (threadIdx.x == 0) {
    tma_prefetch_desc(&p.a_map);
    tma_prefetch_desc(&p.w_map);
    for (int s = 0; s < C::kStages; ++s) {
      mbar_init(&full[s], 1);  // pair: only the even CTA's is used; both CTAs' copies complete on it
      mbar_init(&empty[s], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&acc_full[i], 1);
      mbar_init(&acc_empty[i], PAIR ? 2 * C::kEpiWarps : C::kEpiWarps);
    }
    mbar_init(drain_bar, 1);
    *abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == 1) {
    if constexpr (PAIR) {
      tmem_alloc_pair(tmem_slot, C::kTmemCols);
      tmem_relinquish_pair();
    } else {
      tmem_alloc(tmem_slot, C::kTmemCols);
      tmem_relinquish();
    }
  }
  tc_fence_before();
  __syncthreads();
  if constexpr (PAIR) cluster_sync_all();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  grid_dependency_release();
  grid_dependency_wait();

  if (warp == 0) {
    // ------------------------------------------------------------------ TMA producer
    if (elect_one()) {
      uint32_t it = 0;
      bool ok = true;
      for (int tile = unit; tile < total_tiles && ok; tile += n_units) {
        int m_t, n_t;
        int8_tile_coords(p, tile, m_t, n_t);
        const int a_row = m_t * C::kTileRows + static_cast<int>(rank) * 128;
        const int w_row = n_t * BN + static_cast<int>(rank) * C::kBRows;
        for (int kb = 0; kb < p.k_blocks; ++kb, ++it) {
          const uint32_t s = it % C::kStages, round = it / C::kStages;
          if (round > 0 && !mbar_wait_bounded(&empty[s], (round - 1) & 1, abort_flag, kSpinLimit)) {
            report_failure(p.status, abort_flag, HDIT_ERR_PEER_TIMEOUT, Q_PROD_EMPTY, static_cast<int>(it));
            ok = false;
            break;
          }
          uint8_t* a_dst = stage_base + s * C::kStageBytes;
          if constexpr (PAIR) {
            // the even CTA announces both CTAs' bytes, see gemm_sm100.cu
            if (leader) mbar_expect_tx(&full[s], 2 * C::kStageBytes);
            const uint32_t bar = map_to_cta(&full[s], 0);
            tma_load_2d_pair(a_dst, &p.a_map, bar, kb * kTileKBytes, a_row);
            tma_load_2d_pair(a_dst + C::kABytes, &p.w_map, bar, kb * kTileKBytes, w_row);
          } else {
            mbar_expect_tx(&full[s], C::kStageBytes);
            tma_load_2d(a_dst, &p.a_map, &full[s], kb * kTileKBytes, a_row);
            tma_load_2d(a_dst + C::kABytes, &p.w_map, &full[s], kb * kTileKBytes, w_row);
          }
        }
      }
      if (PAIR && !leader) {
        // copies of this CTA complete on the partner's barrier: after a failure give them time to land
        if (*abort_flag != 0)
          for (int i = 0; i < 64; ++i) __nanosleep(1000);
      } else if (*abort_flag != 0) {
        volatile int never = 0;
        for (uint32_t s = 0; s < static_cast<uint32_t>(C::kStages) && s < it; ++s) {
          const uint32_t last = ((it - 1 - s) / C::kStages) * C::kStages + s;  // last issue that used stage s
          if (last < it) mbar_wait_bounded(&full[s], (last / C::kStages) & 1, &never, kSpinLimit);
        }
      }
    }
  } else if (warp == 1) {
    if (elect_one() && (!PAIR || leader)) {
      // ------------------------------------------------------------------ MMA issuer
      constexpr uint32_t idesc = make_idesc_i8(PAIR ? 256 : 128, BN);
      uint32_t it = 0;
      uint32_t local = 0;
      bool ok = true;
      for (int tile = unit; tile < total_tiles && ok; tile += n_units, ++local) {
        const uint32_t acc = local & 1, use = local >> 1;
        if (use > 0 && !mbar_wait_bounded(&acc_empty[acc], (use - 1) & 1, abort_flag, kSpinLimit)) {
          report_failure(p.status, abort_flag, HDIT_ERR_PEER_TIMEOUT, Q_MMA_ACC_EMPTY, static_cast<int>(local));
          ok = false;
          break;
        }
        tc_fence_after();
        const uint32_t d_tmem = tmem_base + acc * C::kAccCols;
        for (int kb = 0; kb < p.k_blocks; ++kb, ++it) {
          const uint32_t s = it % C::kStages, round = it / C::kStages;
          if (!mbar_wait_bounded(&full[s], round & 1, abort_flag, kSpinLimit)) {
            report_failure(p.status, abort_flag, HDIT_ERR_PEER_TIMEOUT, Q_MMA_FULL, static_cast<int>(it));
            ok = false;
            break;
          }
          tc_fence_after();
          const uint32_t a_addr = smem_u32(stage_base + s * C::kStageBytes);
          const uint64_t a_desc = make_smem_desc_sw128(a_addr, 16, 1024);
          const uint64_t b_desc = make_smem_desc_sw128(a_addr + C::kABytes, 16, 1024);
#pragma unroll
          for (int kk = 0; kk < kTileKBytes / 32; ++kk) {
            const uint64_t off = static_cast<uint64_t>((kk * 32) >> 4);
            if constexpr (PAIR) umma_i8_pair(d_tmem, a_desc + off, b_desc + off, idesc, (kb | kk) != 0 ? 1u : 0u);
            else umma_i8(d_tmem, a_desc + off, b_desc + off, idesc, (kb | kk) != 0 ? 1u : 0u);
          }
          if constexpr (PAIR) tc_commit_pair(&empty[s]);
          else tc_commit(&empty[s]);
        }
        if (ok) {
          if constexpr (PAIR) tc_commit_pair(&acc_full[acc]);
          else tc_commit(&acc_full[acc]);
        }
      }
      if (*abort_flag != 0) {
        volatile int never = 0;
        if constexpr (PAIR) tc_commit_pair(drain_bar);
        else tc_commit(drain_bar);
        mbar_wait_bounded(drain_bar, 0, &never, kSpinLimit);
      }
    }
  } else {
    // ------------------------------------------------------------------ epilogue
    const int quarter = warp & 3;  // the TMEM lanes this warp may read: [32 * quarter, 32 * quarter + 32)
    const int team = (warp - 2) >> 2;
    const int c0 = team * C::kTeamPieces, c1 = min(C::kPieces, c0 + C::kTeamPieces);
    uint8_t* staging = staging_base + (warp - 2) * 4096;
    float* col_scale = col_base + (warp - 2) * (C::kTeamPieces * 64 * 3);
    float* col_bias = col_scale + C::kTeamPieces * 64;
    float* col_gate = col_bias + C::kTeamPieces * 64;
    const int sub_row = lane >> 3, chunk = lane & 7;  // full lines: 4 rows per instruction, 8 lanes per row
    uint32_t local = 0;
    for (int tile = unit; tile < total_tiles; tile += n_units, ++local) {
      int m_t, n_t;
      int8_tile_coords(p, tile, m_t, n_t);
      const uint32_t acc = local & 1, use = local >> 1;
      const long long row0 = static_cast<long long>(m_t) * C::kTileRows + static_cast<long long>(rank) * 128 + quarter * 32;
      const long long my_row = row0 + lane;
      const int tile_col = n_t * BN + c0 * 64;  // first column of this warp
      // one batch entry for all rows of the warp: its gate waits beside the scales; else each row reads its own
      long long batch = 0;
      bool one_batch = true;
      if constexpr (EPI == HDIT_GEMM_BIAS_GATE_RESIDUAL) {
        const unsigned first = static_cast<unsigned>(row0 < p.M ? row0 : 0), last = static_cast<unsigned>(row0 + 31 < p.M ? row0 + 31 : p.M - 1);
        const unsigned b_first = first / static_cast<unsigned>(p.rows_per_batch);
        one_batch = first > last || b_first == last / static_cast<unsigned>(p.rows_per_batch);
        batch = one_batch ? b_first : (my_row < p.M ? static_cast<unsigned>(my_row) / static_cast<unsigned>(p.rows_per_batch) : b_first);
      }
      const float row_scale = my_row < p.M ? p.a_scale[my_row] : 0.f;
      __syncwarp();  // everyone is done with the previous tile's columns
      for (int i = lane; i < C::kTeamPieces * 64; i += 32) {
        const int col = tile_col + i;
        const bool in = col < p.N;
        col_scale[i] = in ? p.w_scale[col] : 0.f;
        col_bias[i] = in && p.bias != nullptr ? to_f<FP16>(p.bias[col]) : 0.f;
        if constexpr (EPI == HDIT_GEMM_BIAS_GATE_RESIDUAL)
          if (one_batch) col_gate[i] = in ? to_f<FP16>(p.gate[batch * p.gate_batch_stride + col]) : 0.f;
      }
      __syncwarp();
      bool waited = false;
      bool ok = true;
#pragma unroll 1
      for (int c = c0; c < c1; ++c) {
        const int col0 = n_t * BN + c * 64;
        const int col = col0 + chunk * 8;
        const int at = (c - c0) * 64;
        if constexpr (EPI == HDIT_GEMM_BIAS_GATE_RESIDUAL) {
          // the residual's 32 x 64 values to the staging buffer (16-byte chunk j of row r sits at chunk j ^ (r & 7))
          uint4 xv[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const long long row = row0 + i * 4 + sub_row;
            xv[i] = make_uint4(0, 0, 0, 0);
            if (row < p.M && col < p.N) {
              const uint16_t* src = p.residual + row * p.ldr + col;
              if (p.vec) {
                xv[i] = *reinterpret_cast<const uint4*>(src);
              } else {
                uint16_t* e = reinterpret_cast<uint16_t*>(&xv[i]);
#pragma unroll
                for (int k = 0; k < 8; ++k) e[k] = col + k < p.N ? src[k] : uint16_t(0);
              }
            }
          }
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const int rl = i * 4 + sub_row;
            *reinterpret_cast<uint4*>(staging + rl * 128 + ((chunk ^ (rl & 7)) << 4)) = xv[i];
          }
          __syncwarp();
        }
        if (!waited) {
          waited = true;
          if (!__all_sync(0xffffffffu, mbar_wait_bounded(&acc_full[acc], use & 1, abort_flag, kSpinLimit))) {
            if (lane == 0) report_failure(p.status, abort_flag, HDIT_ERR_PEER_TIMEOUT, Q_EPI_ACC_FULL, static_cast<int>(local));
            ok = false;
            break;
          }
          tc_fence_after();
        }
        const uint32_t taddr = tmem_base + (static_cast<uint32_t>(quarter * 32) << 16) + acc * C::kAccCols + c * 64;
        uint32_t r[64];
        tmem_ld32(taddr, *reinterpret_cast<uint32_t(*)[32]>(&r[0]));
        tmem_ld32(taddr + 32, *reinterpret_cast<uint32_t(*)[32]>(&r[32]));
        tc_wait_ld();
        if (c == c1 - 1) {
          // the accumulator is in registers: hand it back to the MMA warp
          tc_fence_before();
          __syncwarp();
          if (lane == 0) {
            if constexpr (PAIR) mbar_arrive_remote(map_to_cta(&acc_empty[acc], 0));
            else mbar_arrive(&acc_empty[acc]);
          }
        }
        // row `lane`: scale, bias, tail, one rounding
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          float v[8];
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const float4 s4 = *reinterpret_cast<const float4*>(col_scale + at + j * 8 + h * 4);
            const float4 b4 = *reinterpret_cast<const float4*>(col_bias + at + j * 8 + h * 4);
            const uint32_t* a4 = &r[j * 8 + h * 4];
            v[h * 4 + 0] = fmaf(static_cast<float>(static_cast<int>(a4[0])) * row_scale, s4.x, b4.x);
            v[h * 4 + 1] = fmaf(static_cast<float>(static_cast<int>(a4[1])) * row_scale, s4.y, b4.y);
            v[h * 4 + 2] = fmaf(static_cast<float>(static_cast<int>(a4[2])) * row_scale, s4.z, b4.z);
            v[h * 4 + 3] = fmaf(static_cast<float>(static_cast<int>(a4[3])) * row_scale, s4.w, b4.w);
          }
          uint4* place = reinterpret_cast<uint4*>(staging + lane * 128 + ((j ^ (lane & 7)) << 4));
          if constexpr (EPI == HDIT_GEMM_BIAS_GELU_TANH) {
#pragma unroll
            for (int k = 0; k < 8; ++k) v[k] = gelu_tanh_f(v[k]);
          } else if constexpr (EPI == HDIT_GEMM_BIAS_GATE_RESIDUAL) {
            const uint4 x4 = *place;
            const uint16_t* xe = reinterpret_cast<const uint16_t*>(&x4);
            if (one_batch) {
#pragma unroll
              for (int k = 0; k < 8; ++k) v[k] = fmaf(col_gate[at + j * 8 + k], v[k], to_f<FP16>(xe[k]));
            } else {
#pragma unroll
              for (int k = 0; k < 8; ++k) {
                const int gc = col0 + j * 8 + k;
                const float g = gc < p.N ? to_f<FP16>(p.gate[batch * p.gate_batch_stride + gc]) : 0.f;
                v[k] = fmaf(g, v[k], to_f<FP16>(xe[k]));
              }
            }
          }
          *place = make_uint4(pack2<FP16>(v[0], v[1]), pack2<FP16>(v[2], v[3]), pack2<FP16>(v[4], v[5]), pack2<FP16>(v[6], v[7]));
        }
        __syncwarp();
        if (col < p.N) {
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const int rl = i * 4 + sub_row;
            const long long row = row0 + rl;
            if (row >= p.M) continue;
            const uint4 v = *reinterpret_cast<const uint4*>(staging + rl * 128 + ((chunk ^ (rl & 7)) << 4));
            uint16_t* dst = p.out + row * p.ldo + col;
            if (p.vec) {
              *reinterpret_cast<uint4*>(dst) = v;
            } else {
              const uint16_t* e = reinterpret_cast<const uint16_t*>(&v);
#pragma unroll
              for (int k = 0; k < 8; ++k)
                if (col + k < p.N) dst[k] = e[k];
            }
          }
        }
        __syncwarp();  // the staging buffer is overwritten by the next piece
      }
      if (!ok) break;
    }
  }

  tc_fence_before();
  __syncthreads();
  if constexpr (PAIR) cluster_sync_all();
  if (warp == 1) {
    tc_fence_after();
    if constexpr (PAIR) tmem_dealloc_pair(tmem_base, C::kTmemCols);
    else tmem_dealloc(tmem_base, C::kTmemCols);
  }
}

// ------------------------------------------------------------------ host side
// Map of a (rows, K) matrix of bytes with K contiguous; box = 128 bytes x box_rows rows. What lies outside reads as 0.
int encode_bytes(CUtensorMap* map, const void* ptr, long long rows, long long k, long long ld, int box_rows) {
  EncodeTiledFn enc = encode_fn();
  if (enc == nullptr) return set_error(HDIT_ERR_CUDA, "cuTensorMapEncodeTiled entry point unavailable");
  cuuint64_t dims[2] = {static_cast<cuuint64_t>(k), static_cast<cuuint64_t>(rows)};
  cuuint64_t strides[1] = {static_cast<cuuint64_t>(ld)};
  cuuint32_t box[2] = {static_cast<cuuint32_t>(kTileKBytes), static_cast<cuuint32_t>(box_rows)};
  cuuint32_t estr[2] = {1, 1};
  const CUresult r = enc(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(ptr), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                         CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS)
    return set_error(HDIT_ERR_CUDA, "cuTensorMapEncodeTiled failed with CUresult %d (rows=%lld k=%lld ld=%lld)", static_cast<int>(r), rows, k, ld);
  return HDIT_OK;
}

template <int BN, bool PAIR, bool FP16, int EPI>
int launch_int8(Int8Params& p, const hdit_int8_linear_args* a) {
  using C = Int8Cfg<BN, PAIR>;
  auto kernel = int8_linear_kernel<BN, PAIR, FP16, EPI>;
  static thread_local int last_dev = -1;  // the attribute is per device
  int dev = 0;
  HDIT_CUDA_OK(cudaGetDevice(&dev));
  if (dev != last_dev) {
    HDIT_CUDA_OK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmemBytes));
    last_dev = dev;
  }
  int rc = encode_bytes(&p.a_map, a->a, a->m, a->k, a->lda, 128);
  if (rc != HDIT_OK) return rc;
  rc = encode_bytes(&p.w_map, a->w, a->n, a->k, a->ldw, C::kBRows);
  if (rc != HDIT_OK) return rc;
  const long long ctas = a->max_ctas > 0 ? a->max_ctas : sm_count();
  const long long m_tiles = (a->m + C::kTileRows - 1) / C::kTileRows, n_tiles = (a->n + BN - 1) / BN;
  if (m_tiles * n_tiles > 0x7fffffffLL) return set_error(HDIT_ERR_TOO_LARGE, "more than 2^31 output tiles");
  p.m_tiles = static_cast<int>(m_tiles);
  p.n_tiles = static_cast<int>(n_tiles);
  long long units = PAIR ? (ctas / 2 > 0 ? ctas / 2 : 1) : ctas;
  // band height: a wave of `units` tiles should read about as many bytes of q_x as of q_w
  int g = static_cast<int>(sqrt(static_cast<double>(units) * BN / C::kTileRows) + 0.5);
  if (g < 1) g = 1;
  if (g > p.m_tiles) g = p.m_tiles;
  p.group_m = g;
  if (units > m_tiles * n_tiles) units = m_tiles * n_tiles;
  HDIT_CUDA_OK(launch_overlapped(kernel, dim3(static_cast<unsigned>(PAIR ? 2 * units : units)), dim3(C::kThreads), C::kSmemBytes,
                                 reinterpret_cast<cudaStream_t>(a->stream), PAIR ? 2 : 1, p));
  return HDIT_OK;
}

template <int BN, bool PAIR>
int launch_int8_of(Int8Params& p, const hdit_int8_linear_args* a) {
  const bool fp16 = a->dtype == HDIT_FP16;
  switch (a->epilogue) {
    case HDIT_GEMM_BIAS: return fp16 ? launch_int8<BN, PAIR, true, 0>(p, a) : launch_int8<BN, PAIR, false, 0>(p, a);
    case HDIT_GEMM_BIAS_GELU_TANH: return fp16 ? launch_int8<BN, PAIR, true, 1>(p, a) : launch_int8<BN, PAIR, false, 1>(p, a);
    default: return fp16 ? launch_int8<BN, PAIR, true, 2>(p, a) : launch_int8<BN, PAIR, false, 2>(p, a);
  }
}

}  // namespace
}  // namespace hdit

extern "C" int hdit_int8_linear(const hdit_int8_linear_args* a) {
  using namespace hdit;
  if (a == nullptr) return set_error(HDIT_ERR_BAD_ARG, "null args");
  if (a->dtype != HDIT_BF16 && a->dtype != HDIT_FP16) return set_error(HDIT_ERR_BAD_ARG, "dtype must be bf16 or fp16");
  if (a->epilogue < HDIT_GEMM_BIAS || a->epilogue > HDIT_GEMM_BIAS_GATE_RESIDUAL) return set_error(HDIT_ERR_BAD_ARG, "unknown epilogue %d", a->epilogue);
  if (a->m < 0 || a->n <= 0 || a->k <= 0) return set_error(HDIT_ERR_BAD_ARG, "bad m / n / k");
  if (a->m > 0x7fffff00LL || a->n > 0x7fffff00LL) return set_error(HDIT_ERR_TOO_LARGE, "m and n must fit 31 bits");
  if (a->k > HDIT_INT8_MAX_K) return set_error(HDIT_ERR_TOO_LARGE, "k above %d could overflow the 32-bit sums", HDIT_INT8_MAX_K);
  if (a->m == 0) return HDIT_OK;
  if (a->a == nullptr || a->a_scale == nullptr || a->w == nullptr || a->w_scale == nullptr || a->out == nullptr)
    return set_error(HDIT_ERR_BAD_ARG, "null a / w / scale / out");
  auto bad_rows = [&](const void* ptr, long long ld) { return (reinterpret_cast<uintptr_t>(ptr) & 15) != 0 || ld % 16 != 0 || ld < a->k; };
  if (bad_rows(a->a, a->lda) || bad_rows(a->w, a->ldw))
    return set_error(HDIT_ERR_SHAPE, "8-bit rows need a 16-byte aligned pointer and a row stride that is a multiple of 16 and covers a row");
  if (((reinterpret_cast<uintptr_t>(a->a_scale) | reinterpret_cast<uintptr_t>(a->w_scale)) & 3) != 0 ||
      ((reinterpret_cast<uintptr_t>(a->out) | reinterpret_cast<uintptr_t>(a->bias) | reinterpret_cast<uintptr_t>(a->residual) |
        reinterpret_cast<uintptr_t>(a->gate)) & 1) != 0)
    return set_error(HDIT_ERR_SHAPE, "a pointer is not aligned to its elements");
  if (a->ldo < a->n) return set_error(HDIT_ERR_SHAPE, "rows of out overlap");
  const bool gated = a->epilogue == HDIT_GEMM_BIAS_GATE_RESIDUAL;
  if (gated && (a->residual == nullptr || a->gate == nullptr || a->rows_per_batch <= 0))
    return set_error(HDIT_ERR_BAD_ARG, "the gated-residual epilogue needs residual, gate and rows_per_batch > 0");
  if (gated && a->ldr < a->n) return set_error(HDIT_ERR_SHAPE, "rows of residual overlap");
  Int8Params p;
  memset(&p, 0, sizeof(p));
  p.M = static_cast<int>(a->m);
  p.N = static_cast<int>(a->n);
  p.k_blocks = static_cast<int>((a->k + kTileKBytes - 1) / kTileKBytes);
  p.a_scale = a->a_scale;
  p.w_scale = a->w_scale;
  p.bias = static_cast<const uint16_t*>(a->bias);
  p.out = static_cast<uint16_t*>(a->out);
  p.ldo = a->ldo;
  p.residual = static_cast<const uint16_t*>(a->residual);
  p.ldr = a->ldr;
  p.gate = static_cast<const uint16_t*>(a->gate);
  p.gate_batch_stride = a->gate_batch_stride;
  p.rows_per_batch = static_cast<int>(a->rows_per_batch > 0 && a->rows_per_batch < a->m ? a->rows_per_batch : a->m);
  auto whole = [&](const void* ptr, long long ld) { return (reinterpret_cast<uintptr_t>(ptr) & 15) == 0 && ld % 8 == 0; };
  p.vec = a->n % 8 == 0 && whole(a->out, a->ldo) && (!gated || whole(a->residual, a->ldr));
  p.status = device_status_ptr();
  if (p.status == nullptr) return HDIT_ERR_CUDA;
  if (a->x != nullptr) {
    // 16-bit rows: into 8 bits first, in the caller's a / a_scale
    const int rc = hdit_quantize_rows(a->dtype, a->x, const_cast<void*>(a->a), const_cast<float*>(a->a_scale), a->m, a->k, a->x_rows_per_batch,
                                      a->x_batch_stride, a->x_row_stride, a->lda, a->stream);
    if (rc != HDIT_OK) return rc;
  }
  if (a->tile < 0 || a->tile > 4) return set_error(HDIT_ERR_BAD_ARG, "tile must be 0 (choose) to 4");
  int tile = a->tile;
  if (tile == 0) {
    // Fewest waves, each weighted by a tile's time relative to 128 x 128 of output per SM
    const long long sms = a->max_ctas > 0 ? a->max_ctas : sm_count();
    struct Cand { int tile, rows, cols, units_div; double per_tile; };
    const Cand cand[4] = {{1, 128, 128, 1, 1.25}, {2, 256, 128, 2, 1.2}, {3, 256, 192, 2, 1.725}, {4, 256, 256, 2, 2.1}};
    double best = -1.0;
    for (const Cand& c : cand) {
      const long long units = sms / c.units_div > 0 ? sms / c.units_div : 1;
      const long long tiles = ((a->m + c.rows - 1) / c.rows) * ((a->n + c.cols - 1) / c.cols);
      const double cost = static_cast<double>((tiles + units - 1) / units) * c.per_tile;
      if (best < 0 || cost < best) best = cost, tile = c.tile;
    }
  }
  switch (tile) {
    case 1: return launch_int8_of<128, false>(p, a);
    case 2: return launch_int8_of<128, true>(p, a);
    case 3: return launch_int8_of<192, true>(p, a);
    default: return launch_int8_of<256, true>(p, a);
  }
}
