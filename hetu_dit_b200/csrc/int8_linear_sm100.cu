// Linear layer over 8-bit integers for sm_100a:  out = tail(s_x[m] s_w[n] sum_k q_x[m, k] q_w[n, k] + bias[n]).
//
// q_x is (M, K) and q_w (N, K), both K-contiguous signed bytes with one fp32 scale per row. The integer sums are exact (32-bit
// accumulators in tensor memory, tcgen05.mma kind::i8); everything after them runs in fp32 and is rounded to the 16-bit
// result once. The kernel has the frame of the 16-bit linear layer (gemm_sm100.cu): persistent CTAs, a TMA producer warp, an
// MMA warp, epilogue warps, two accumulators, optionally CTA pairs. A stage is 128 bytes of K as there -- 128 elements, four
// MMAs of 32 -- so operand bytes per clock are the same and the main loop of a tile takes half the time for the same K; the
// epilogue has half the time to hide behind it.
//
//   epilogue     per 32 x 32 piece of a warp, a lane to a row: scales, bias and gate of the warp's columns wait in shared
//                memory (they are fetched while the tile before is worked on), the residual's piece comes into the staging
//                buffer by TMA one piece ahead, the result takes its place there and leaves by TMA. Sixteen warps for 256 columns:
//                with eight over pieces of 64 columns a scheduler had two to hide the chain TMEM - scales - staging behind, 3.5 k
//                cycles a tile instead of 2.9 k (16384 x 512 -> 1536 19.9 us, now 18.0).
//
// All waits are bounded, see gemm_sm100.cu.
#include <limits.h>
#include <math.h>

#include "gemm_common.cuh"
#include "host_common.h"
#include "int8_linear.h"

namespace hdit {
namespace {

constexpr int kTileKBytes = 128;  // one swizzle row
constexpr int kPieceBytes = 2048;  // 32 rows x 32 columns of 16 bits, 64-byte swizzle: chunk j of row r sits at chunk j ^ (r / 2 % 4)

enum Int8Wait : int {
  Q_PROD_EMPTY = 211,
  Q_MMA_FULL = 212,
  Q_MMA_ACC_EMPTY = 213,
  Q_EPI_ACC_FULL = 214,
  Q_EPI_RESIDUAL = 215,
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

// ---- results leave shared memory by TMA
__device__ __forceinline__ void tma_store_2d(const void* tmap, const void* smem_src, int c0, int c1) {
  asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%2, %3}], [%1];"
               :
               : "l"(reinterpret_cast<uint64_t>(tmap)), "r"(smem_u32(smem_src)), "r"(c0), "r"(c1)
               : "memory");
}
__device__ __forceinline__ void tma_store_commit() { asm volatile("cp.async.bulk.commit_group;" ::: "memory"); }
// All but the last N stores of this thread have read their shared memory.
template <int N>
__device__ __forceinline__ void tma_store_wait_read() {
  asm volatile("cp.async.bulk.wait_group.read %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ void tma_store_wait_all() { asm volatile("cp.async.bulk.wait_group 0;" ::: "memory"); }

// Column k of row i of a staged piece.
__device__ __forceinline__ uint16_t* staged(uint8_t* stage, int i, int k) {
  return reinterpret_cast<uint16_t*>(stage + i * 64 + (((k >> 3) ^ ((i >> 1) & 3)) << 4) + (k & 7) * 2);
}

// Pieces of matrices whose rows start on no 16-byte boundary, which TMA cannot move: 32-bit words where they lie on one, half a
// warp to a row, and what a row has before its first and behind its last whole word by a lane to a row. A row that starts inside
// of a word is staged one element to the left in between, so that words go from and to shared memory as they are. g: the piece's
// first element, `rows` x `cols` of it exist. All of a warp's loads are on their way before the first is needed: one row after the
// other, 1813 x 3122 -> 6387 with a gated residual took 100 us.
struct RaggedPiece {
  uint32_t word[16];
  uint16_t first, last;
};
__device__ __forceinline__ int starts_inside(const uint16_t* row) { return static_cast<int>(reinterpret_cast<uintptr_t>(row) >> 1) & 1; }
// Word `lane & 15` of row `lane >> 4` + 2 i; (row >> 1) & 3 is i & 3.
__device__ __forceinline__ uint32_t* staged_word(uint8_t* stage, int i, int lane) {
  return reinterpret_cast<uint32_t*>(stage + ((lane >> 4) + 2 * i) * 64 + ((((lane >> 2) & 3) ^ (i & 3)) << 4) + (lane & 3) * 4);
}
__device__ __forceinline__ void ragged_load(RaggedPiece& v, const uint16_t* g, long long ld, int rows, int cols, int lane) {
  const uint16_t* at = g + (lane >> 4) * ld;
  const int col = 2 * (lane & 15) + starts_inside(at), live = col + 1 < cols ? rows - (lane >> 4) : 0;
  at += col;
#pragma unroll
  for (int i = 0; i < 16; ++i, at += 2 * ld) v.word[i] = 2 * i < live ? *reinterpret_cast<const uint32_t*>(at) : 0u;
  const uint16_t* own = g + lane * ld;
  v.first = lane < rows && starts_inside(own) ? own[0] : uint16_t(0);
  v.last = lane < rows && ((cols - starts_inside(own)) & 1) ? own[cols - 1] : uint16_t(0);
}
__device__ __forceinline__ void ragged_stage(const RaggedPiece& v, uint8_t* stage, const uint16_t* g, long long ld, int rows, int cols, int lane) {
#pragma unroll
  for (int i = 0; i < 16; ++i) *staged_word(stage, i, lane) = v.word[i];
  __syncwarp();
  const int inside = starts_inside(g + lane * ld);
  uint32_t before = static_cast<uint32_t>(v.first) << 16;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    uint4* const chunk = reinterpret_cast<uint4*>(staged(stage, lane, j * 8));
    const uint4 w = *chunk;
    *chunk = make_uint4(__funnelshift_l(before, w.x, inside * 16), __funnelshift_l(w.x, w.y, inside * 16), __funnelshift_l(w.y, w.z, inside * 16),
                        __funnelshift_l(w.z, w.w, inside * 16));
    before = w.w;
  }
  if ((cols - inside) & 1) *staged(stage, lane, cols - 1) = v.last;
}
__device__ __forceinline__ void ragged_store(uint16_t* g, long long ld, int rows, int cols, uint8_t* stage, int lane) {
  uint16_t* const own = g + lane * ld;
  const int inside = starts_inside(own);
  if (lane < rows) {
    if (inside) own[0] = *staged(stage, lane, 0);
    if ((cols - inside) & 1) own[cols - 1] = *staged(stage, lane, cols - 1);
  }
  uint4 w[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) w[j] = *reinterpret_cast<const uint4*>(staged(stage, lane, j * 8));
#pragma unroll
  for (int j = 0; j < 4; ++j)
    *reinterpret_cast<uint4*>(staged(stage, lane, j * 8)) =
        make_uint4(__funnelshift_r(w[j].x, w[j].y, inside * 16), __funnelshift_r(w[j].y, w[j].z, inside * 16), __funnelshift_r(w[j].z, w[j].w, inside * 16),
                   __funnelshift_r(w[j].w, j < 3 ? w[j + 1 < 4 ? j + 1 : 3].x : 0u, inside * 16));
  __syncwarp();
  uint16_t* at = g + (lane >> 4) * ld;
  const int col = 2 * (lane & 15) + starts_inside(at), live = col + 1 < cols ? rows - (lane >> 4) : 0;
  at += col;
#pragma unroll
  for (int i = 0; i < 16; ++i, at += 2 * ld)
    if (2 * i < live) *reinterpret_cast<uint32_t*>(at) = *staged_word(stage, i, lane);
}

struct alignas(64) Int8Params {
  CUtensorMap a_map;
  CUtensorMap w_map;
  CUtensorMap out_map;  // boxes of 32 columns x 32 rows, where tma_out / tma_residual say so
  CUtensorMap residual_map;
  int M, N, k_blocks;
  int m_tiles, n_tiles, group_m;
  uint32_t a_bytes;  // of a stage: the rows of a CTA's tile that any tile has; what the others' places hold is summed and dropped
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
  bool tma_out, tma_residual;  // rows start on 16-byte boundaries
  int tma_cols;                // results' pieces up to this column leave by TMA
  int32_t* status;
};

template <int BN, bool PAIR, int EPI>
struct Int8Cfg {
  // Four warps, a team, reach the 128 lanes of an accumulator; each team has 64 of its columns in two pieces of 32
  static constexpr int kTeamCols = 64, kTeamPieces = 2;
  static constexpr int kColTeams = BN / kTeamCols;
  static constexpr int kEpiWarps = 4 * kColTeams;
  static constexpr int kThreads = 64 + 32 * kEpiWarps;
  static constexpr int kTileRows = PAIR ? 256 : 128;
  static constexpr int kBRows = PAIR ? BN / 2 : BN;
  static constexpr int kABytes = 128 * kTileKBytes;
  static constexpr int kBBytes = kBRows * kTileKBytes;
  static constexpr int kStageBytes = kABytes + kBBytes;
  // pieces of 32 rows x 32 columns of 16 bits per epilogue warp: two where a residual comes in beside the result that leaves.
  // A second buffer costs a stage or two of the ring, which 256 columns miss more: 4608 x 12288 x 3072 + GELU took 137 us with 4
  // stages and two buffers (of 64 columns), 124 with 6 and one.
  static constexpr int kBufs = EPI == HDIT_GEMM_BIAS_GATE_RESIDUAL ? 2 : 1;
  static constexpr int kStagingBytes = kEpiWarps * kBufs * kPieceBytes;
  // barriers and the columns' scales, bias and gate: what is left of 227 KB beside six stages of 32 KB and one piece per warp
  static constexpr int kSmallBytes = 3072;
  static constexpr int kStagesFit = (kMaxSmem - kSmallBytes - kStagingBytes) / kStageBytes;
  static constexpr int kStages = kStagesFit > 8 ? 8 : kStagesFit;
  static constexpr int kAccCols = BN == 192 ? 256 : BN;
  static constexpr int kTmemCols = 2 * kAccCols;
  static constexpr int kSmemBytes = kSmallBytes + kStages * kStageBytes + kStagingBytes;
  static_assert(512 + kColTeams * kTeamCols * 10 <= kSmallBytes, "no room for the columns");
  static_assert(kStageBytes % 1024 == 0, "TMA tiles start at multiples of the swizzle's 1024 bytes");
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

// PLAIN_RESIDUAL: no bulk copy can move the residual. A kernel of its own: its pieces in registers cost the other one, at 256 columns
// with 96 registers a thread, 76 bytes of spills.
template <int BN, bool PAIR, bool FP16, int EPI, bool PLAIN_RESIDUAL>
__global__ void __launch_bounds__(Int8Cfg<BN, PAIR, EPI>::kThreads, 1) int8_linear_kernel(const __grid_constant__ Int8Params p) {
  using C = Int8Cfg<BN, PAIR, EPI>;
  extern __shared__ __align__(1024) uint8_t smem[];
  uint64_t* full = reinterpret_cast<uint64_t*>(smem);
  uint64_t* empty = full + 8;
  uint64_t* acc_full = empty + 8;
  uint64_t* acc_empty = acc_full + 2;
  uint64_t* drain_bar = acc_empty + 2;
  uint64_t* res_bars = drain_bar + 1;  // two for each epilogue warp
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(res_bars + 2 * C::kEpiWarps);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  static_assert((8 + 8 + 2 + 2 + 1 + 2 * C::kEpiWarps + 1) * 8 <= 512, "barriers");
  uint8_t* col_base = smem + 512;
  uint8_t* stage_base = smem + C::kSmallBytes;
  uint8_t* staging_base = stage_base + C::kStages * C::kStageBytes;

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
    for (int i = 0; i < 2 * C::kEpiWarps; ++i) mbar_init(&res_bars[i], 1);
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
      const uint32_t stage_bytes = (C::kBBytes + p.a_bytes) * (PAIR ? 2 : 1);
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
            if (leader) mbar_expect_tx(&full[s], stage_bytes);
            const uint32_t bar = map_to_cta(&full[s], 0);
            tma_load_2d_pair(a_dst, &p.a_map, bar, kb * kTileKBytes, a_row);
            tma_load_2d_pair(a_dst + C::kABytes, &p.w_map, bar, kb * kTileKBytes, w_row);
          } else {
            mbar_expect_tx(&full[s], stage_bytes);
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
    constexpr bool kGated = EPI == HDIT_GEMM_BIAS_GATE_RESIDUAL;
    constexpr bool kTmaResidual = kGated && !PLAIN_RESIDUAL;
    const int quarter = warp & 3;  // the TMEM lanes this warp may read: [32 * quarter, 32 * quarter + 32)
    const int team = (warp - 2) >> 2;
    uint8_t* const staging = staging_base + (warp - 2) * (C::kBufs * kPieceBytes);
    uint64_t* const res_full = res_bars + (warp - 2) * 2;
    const int t_col = (threadIdx.x - 64) & 127;  // the column of its team that this thread fetches
    float* const col_scale = reinterpret_cast<float*>(col_base + team * (C::kTeamCols * 10));
    float* const col_bias = col_scale + C::kTeamCols;
    uint16_t* const col_gate = reinterpret_cast<uint16_t*>(col_bias + C::kTeamCols);
    auto team_sync = [&] { asm volatile("bar.sync %0, 128;" ::"r"(1 + team) : "memory"); };

    // what the tile needs beside its sums; fetched one tile ahead
    int row0 = 0;           // first row of the warp
    int tile_col = 0;       // first column of the team
    bool one_batch = true;  // all rows of the team have one batch entry: its gate waits in shared memory, else each row reads its own
    float row_scale = 0.f, f_scale = 0.f;
    uint16_t f_bias = 0, f_gate = 0;
    auto fetch = [&](int tile) {
      int m_t, n_t;
      int8_tile_coords(p, tile, m_t, n_t);
      const int team_row0 = m_t * C::kTileRows + static_cast<int>(rank) * 128;
      row0 = team_row0 + quarter * 32;
      tile_col = n_t * BN + team * C::kTeamCols;
      unsigned batch = 0;
      if constexpr (kGated) {
        const unsigned first = static_cast<unsigned>(team_row0 < p.M ? team_row0 : 0);
        const unsigned last = static_cast<unsigned>(team_row0 + 127 < p.M ? team_row0 + 127 : p.M - 1);
        const unsigned per = static_cast<unsigned>(p.rows_per_batch);
        batch = first / per;
        one_batch = first > last || batch == last / per;
      }
      row_scale = row0 + lane < p.M ? p.a_scale[row0 + lane] : 0.f;
      const int col = tile_col + t_col;
      if (t_col < C::kTeamCols) {
        const bool in = col < p.N;
        f_scale = in ? p.w_scale[col] : 0.f;
        f_bias = in && p.bias != nullptr ? p.bias[col] : uint16_t(0);
        if constexpr (kGated) f_gate = in && one_batch ? p.gate[static_cast<long long>(batch) * p.gate_batch_stride + col] : uint16_t(0);
      }
    };
    // pieces are numbered through all tiles; piece i has staging buffer i % kBufs
    uint32_t piece = 0, res_phase = 0, res_pending = 0;
    auto issue_residual = [&](int row, int col, uint32_t buf) {
      if (lane == 0 && row < p.M && col < p.N) {
        mbar_expect_tx(&res_full[buf], kPieceBytes);
        tma_load_2d(staging + buf * kPieceBytes, &p.residual_map, &res_full[buf], col, row);
      }
      if (row < p.M && col < p.N) res_pending |= 1u << buf;
    };
    uint32_t local = 0;
    bool ok = true;
    if (unit < total_tiles) {
      fetch(unit);
      if constexpr (kTmaResidual) issue_residual(row0, tile_col, 0);
    }
    for (int tile = unit; tile < total_tiles; tile += n_units, ++local) {
      const uint32_t acc = local & 1, use = local >> 1;
      const int my_row0 = row0;
      const int my_col = tile_col;
      const bool my_one_batch = one_batch;
      const float my_scale = row_scale;
      team_sync();  // everyone is done with the previous tile's columns
      if (t_col < C::kTeamCols) {
        col_scale[t_col] = f_scale;
        col_bias[t_col] = to_f<FP16>(f_bias);
        if constexpr (kGated) col_gate[t_col] = f_gate;
      }
      team_sync();
      if (!ok) continue;  // after a failure: the team's other warps still meet the barriers
      if (tile + n_units < total_tiles) fetch(tile + n_units);
      if constexpr (PLAIN_RESIDUAL) {
        // both pieces, into buffers that the tile before has left, while its sums are on their way
        static_assert(C::kTeamPieces == 2 && C::kBufs == 2, "a buffer for each piece of a tile");
        RaggedPiece v[2];
        auto piece_at = [&](int c, auto f) {
          if (my_row0 < p.M && my_col + c * 32 < p.N)
            f(p.residual + my_row0 * p.ldr + my_col + c * 32, min(32, p.M - my_row0), min(32, p.N - my_col - c * 32));
        };
#pragma unroll
        for (int c = 0; c < 2; ++c) piece_at(c, [&](const uint16_t* g, int rows, int cols) { ragged_load(v[c], g, p.ldr, rows, cols, lane); });
        if (lane == 0) tma_store_wait_read<0>();
        __syncwarp();
#pragma unroll
        for (int c = 0; c < 2; ++c)
          piece_at(c, [&](const uint16_t* g, int rows, int cols) { ragged_stage(v[c], staging + c * kPieceBytes, g, p.ldr, rows, cols, lane); });
        __syncwarp();
      }
      if (!__all_sync(0xffffffffu, mbar_wait_bounded(&acc_full[acc], use & 1, abort_flag, kSpinLimit))) {
        if (lane == 0) report_failure(p.status, abort_flag, HDIT_ERR_PEER_TIMEOUT, Q_EPI_ACC_FULL, static_cast<int>(local));
        ok = false;
        continue;
      }
      tc_fence_after();
#pragma unroll 1
      for (int c = 0; c < C::kTeamPieces; ++c, ++piece) {
        const uint32_t buf = C::kBufs == 1 ? 0 : piece & 1;
        uint8_t* const stage = staging + buf * kPieceBytes;
        const int at = c * 32, col0 = my_col + at;
        const bool in = my_row0 < p.M && col0 < p.N;
        const uint32_t taddr = tmem_base + (static_cast<uint32_t>(quarter * 32) << 16) + acc * C::kAccCols + team * C::kTeamCols + at;
        uint32_t r[32];
        tmem_ld32(taddr, r);
        if constexpr (kTmaResidual) {
          // the next piece's residual, into the buffer that the previous piece's result has left
          fence_proxy_async_smem();  // where it left by plain loads
          if (lane == 0) tma_store_wait_read<0>();
          __syncwarp();
          if (c + 1 < C::kTeamPieces) issue_residual(my_row0, col0 + 32, buf ^ 1);
          else if (tile + n_units < total_tiles) issue_residual(row0, tile_col, buf ^ 1);
          if (in) {
            if (!__all_sync(0xffffffffu, mbar_wait_bounded(&res_full[buf], (res_phase >> buf) & 1, abort_flag, kSpinLimit))) {
              if (lane == 0) report_failure(p.status, abort_flag, HDIT_ERR_PEER_TIMEOUT, Q_EPI_RESIDUAL, static_cast<int>(piece));
              ok = false;
              break;
            }
            res_phase ^= 1u << buf;
            res_pending &= ~(1u << buf);
          }
        } else if constexpr (!kGated) {
          if (lane == 0) tma_store_wait_read<C::kBufs - 1>();  // the buffer's last result has left
          __syncwarp();
        }
        tc_wait_ld();
        if (c == C::kTeamPieces - 1) {
          // the accumulator is in registers: hand it back to the MMA warp
          tc_fence_before();
          __syncwarp();
          if (lane == 0) {
            if constexpr (PAIR) mbar_arrive_remote(map_to_cta(&acc_empty[acc], 0));
            else mbar_arrive(&acc_empty[acc]);
          }
        }
        // Row `lane`: scale, bias, tail, one rounding. What eight columns need is read before the eight ones before are
        // written: the compiler cannot tell that the two do not overlap, and two warps per scheduler hide little of a chain of
        // reads and writes.
        uint8_t* const own = stage + lane * 64;
        const int swizzle = (lane >> 1) & 3;
        float4 s4[2], b4[2];
        uint4 x4, g8;
        auto read = [&](int j) {
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            s4[h] = *reinterpret_cast<const float4*>(col_scale + at + j * 8 + h * 4);
            b4[h] = *reinterpret_cast<const float4*>(col_bias + at + j * 8 + h * 4);
          }
          if constexpr (kGated) {
            g8 = *reinterpret_cast<const uint4*>(col_gate + at + j * 8);
            x4 = *reinterpret_cast<const uint4*>(own + ((j ^ swizzle) << 4));
          }
        };
        read(0);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          float2 v[4];
#pragma unroll
          for (int h = 0; h < 4; ++h) {
            const float4 s = s4[h >> 1], b = b4[h >> 1];
            v[h] = int8_value2(static_cast<int>(r[j * 8 + h * 2]), static_cast<int>(r[j * 8 + h * 2 + 1]), my_scale,
                               h & 1 ? make_float2(s.z, s.w) : make_float2(s.x, s.y), h & 1 ? make_float2(b.z, b.w) : make_float2(b.x, b.y));
          }
          if constexpr (EPI == HDIT_GEMM_BIAS_GELU_TANH) {
#pragma unroll
            for (int h = 0; h < 4; ++h) v[h] = int8_gelu2(v[h]);
          } else if constexpr (kGated) {
            const uint16_t* xe = reinterpret_cast<const uint16_t*>(&x4);
            const uint16_t* ge = reinterpret_cast<const uint16_t*>(&g8);
            float g[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) g[k] = to_f<FP16>(ge[k]);
            if (!my_one_batch) {
              const long long row = my_row0 + lane;
              const uint16_t* gr = p.gate + (row < p.M ? static_cast<unsigned>(row) / static_cast<unsigned>(p.rows_per_batch) : 0u) * p.gate_batch_stride;
#pragma unroll
              for (int k = 0; k < 8; ++k) {
                const int gc = col0 + j * 8 + k;
                g[k] = gc < p.N ? to_f<FP16>(gr[gc]) : 0.f;
              }
            }
#pragma unroll
            for (int h = 0; h < 4; ++h)
              v[h] = fma2(make_float2(g[2 * h], g[2 * h + 1]), v[h], make_float2(to_f<FP16>(xe[2 * h]), to_f<FP16>(xe[2 * h + 1])));
          }
          if (j < 3) read(j + 1);
          *reinterpret_cast<uint4*>(own + ((j ^ swizzle) << 4)) =
              make_uint4(pack2<FP16>(v[0].x, v[0].y), pack2<FP16>(v[1].x, v[1].y), pack2<FP16>(v[2].x, v[2].y), pack2<FP16>(v[3].x, v[3].y));
        }
        if (p.tma_out && col0 + 32 <= p.tma_cols) {
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) {
            if (in) tma_store_2d(&p.out_map, stage, col0, my_row0);
            tma_store_commit();
          }
        } else {
          __syncwarp();
          if (in) ragged_store(p.out + my_row0 * p.ldo + col0, p.ldo, min(32, p.M - my_row0), min(32, p.N - col0), stage, lane);
          __syncwarp();
        }
      }
    }
    // copies in flight must have left or landed before the CTA's shared memory is given back
    if (lane == 0) tma_store_wait_all();
    if constexpr (kTmaResidual) {
      volatile int never = 0;
      for (uint32_t buf = 0; buf < 2; ++buf)
        if ((res_pending >> buf) & 1) mbar_wait_bounded(&res_full[buf], (res_phase >> buf) & 1, &never, kSpinLimit);
    }
    __syncwarp();
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

// Map of a (rows, n) matrix of 16-bit values for the epilogue's pieces.
int encode_pieces(CUtensorMap* map, const void* ptr, long long rows, long long n, long long ld, int dtype) {
  EncodeTiledFn enc = encode_fn();
  if (enc == nullptr) return set_error(HDIT_ERR_CUDA, "cuTensorMapEncodeTiled entry point unavailable");
  cuuint64_t dims[2] = {static_cast<cuuint64_t>(n), static_cast<cuuint64_t>(rows)};
  cuuint64_t strides[1] = {static_cast<cuuint64_t>(ld) * 2};
  cuuint32_t box[2] = {32, 32};
  cuuint32_t estr[2] = {1, 1};
  const CUtensorMapDataType dt = dtype == HDIT_FP16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
  const CUresult r = enc(map, dt, 2, const_cast<void*>(ptr), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_64B,
                         CU_TENSOR_MAP_L2_PROMOTION_NONE, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS)
    return set_error(HDIT_ERR_CUDA, "cuTensorMapEncodeTiled failed with CUresult %d (rows=%lld n=%lld ld=%lld)", static_cast<int>(r), rows, n, ld);
  return HDIT_OK;
}

template <int BN, bool PAIR, bool FP16, int EPI, bool PLAIN_RESIDUAL = false>
int launch_int8(Int8Params& p, const hdit_int8_linear_args* a) {
  using C = Int8Cfg<BN, PAIR, EPI>;
  constexpr auto kernel = int8_linear_kernel<BN, PAIR, FP16, EPI, PLAIN_RESIDUAL>;
  HDIT_CUDA_OK((allow_shared_memory<kernel, C::kSmemBytes>()));
  // Boxes of rows that lie outside cost more than rows: 16 x 6144 -> 9216 took 22.9 us with boxes of 128 rows, 15.0 with 16; 128 rows take 15.8.
  const int a_rows = a->m < 128 ? static_cast<int>((a->m + 7) / 8 * 8) : 128;
  p.a_bytes = static_cast<uint32_t>(a_rows * kTileKBytes);
  int rc = encode_bytes(&p.a_map, a->a, a->m, a->k, a->lda, a_rows);
  if (rc != HDIT_OK) return rc;
  rc = encode_bytes(&p.w_map, a->w, a->n, a->k, a->ldw, C::kBRows);
  if (rc != HDIT_OK) return rc;
  if (p.tma_out && (rc = encode_pieces(&p.out_map, a->out, a->m, a->n, a->ldo, a->dtype)) != HDIT_OK) return rc;
  if (p.tma_residual && (rc = encode_pieces(&p.residual_map, a->residual, a->m, a->n, a->ldr, a->dtype)) != HDIT_OK) return rc;
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
    default:
      if (!p.tma_residual) return fp16 ? launch_int8<BN, PAIR, true, 2, true>(p, a) : launch_int8<BN, PAIR, false, 2, true>(p, a);
      return fp16 ? launch_int8<BN, PAIR, true, 2>(p, a) : launch_int8<BN, PAIR, false, 2>(p, a);
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
  if (a->w == nullptr || a->w_scale == nullptr || a->out == nullptr) return set_error(HDIT_ERR_BAD_ARG, "null w / scale / out");
  if (a->x != nullptr && (a->x_rows_per_batch <= 0 || (reinterpret_cast<uintptr_t>(a->x) & 1) != 0))
    return set_error(HDIT_ERR_BAD_ARG, "x needs x_rows_per_batch > 0 and the alignment of its elements");
  if (a->tile < 0 || a->tile > 5) return set_error(HDIT_ERR_BAD_ARG, "tile must be 0 (choose) to 5");
  if (a->tile == 5 && !int8_linear_few_takes(a)) return set_error(HDIT_ERR_SHAPE, "too many rows, or too long ones, for the kernel for a few rows");
  const bool few = a->tile == 5 || (a->tile == 0 && int8_linear_few_takes(a) && int8_linear_few_pays(a));
  const bool own_rows = few && a->x != nullptr && int8_linear_few_quantizes(a);  // a and a_scale are not used
  if (!(own_rows && a->m <= 2) && (a->a == nullptr || a->a_scale == nullptr)) return set_error(HDIT_ERR_BAD_ARG, "null a / a_scale");
  auto bad_rows = [&](const void* ptr, long long ld) { return (reinterpret_cast<uintptr_t>(ptr) & 15) != 0 || ld % 16 != 0 || ld < a->k; };
  if ((!own_rows && bad_rows(a->a, a->lda)) || bad_rows(a->w, a->ldw))
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
  p.tma_out = whole(a->out, a->ldo);
  // A copy writes whole 16 bytes of a row: where N ends inside of them, the last piece would overwrite what lies behind the row.
  p.tma_cols = p.N % 8 == 0 ? INT_MAX : p.N;
  p.tma_residual = gated && whole(a->residual, a->ldr);
  p.status = device_status_ptr();
  if (p.status == nullptr) return HDIT_ERR_CUDA;
  if (a->x != nullptr && !own_rows) {
    // 16-bit rows: into 8 bits first, in the caller's a / a_scale
    const int rc = hdit_quantize_rows(a->dtype, a->x, const_cast<void*>(a->a), const_cast<float*>(a->a_scale), a->m, a->k, a->x_rows_per_batch,
                                      a->x_batch_stride, a->x_row_stride, a->lda, a->stream);
    if (rc != HDIT_OK) return rc;
  }
  if (few) return int8_linear_few(a);
  int tile = a->tile;
  if (tile == 0) {
    // Fewest waves, each weighted by a tile's time relative to 128 x 128 of output per SM (0.145 us per 128 of K), as for the 16-bit
    // layers, whose operands take as many bytes per clock; a pair starts 0.3 us later. us with 128 x 128, 256 x 128, 256 x 192, 256 x 256:
    // 154 x 1536 -> 1536 5.7, 5.9, 7.1, 8.4; 512 x 12288 -> 3072 25.5, 22.5, 28.3, 34.2; 2192 x 3072 -> 3072 19.3, 18.3, 16.9, 19.8; 8192 x
    // 1536 -> 4608 54, 50, 45, 43; 16384 x 512 -> 512 10.7, 10.7, 10.2, 9.5. Over 24 shapes the choice is 2 % from the best.
    const long long sms = a->max_ctas > 0 ? a->max_ctas : sm_count();
    struct Cand { int tile, rows, cols, units_div; double per_tile; };
    const Cand cand[4] = {{1, 128, 128, 1, 1.25}, {2, 256, 128, 2, 1.2}, {3, 256, 192, 2, 1.725}, {4, 256, 256, 2, 2.1}};
    const double pair_start = 2.0 / p.k_blocks;
    double best = -1.0;
    for (const Cand& c : cand) {
      const long long units = sms / c.units_div > 0 ? sms / c.units_div : 1;
      const long long tiles = ((a->m + c.rows - 1) / c.rows) * ((a->n + c.cols - 1) / c.cols);
      const double cost = static_cast<double>((tiles + units - 1) / units) * c.per_tile + (c.units_div == 2 ? pair_start : 0.0);
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
