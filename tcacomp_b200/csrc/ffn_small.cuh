// ffn_small.cuh -- the contractions of ffn_gemm.cuh for few rows, or few output tiles: a tile per CTA, the contracted
// axis of a tile cut over the CTAs of a cluster, two CTAs per SM.
//
// The operands change places: the tensor core's 128 rows are 128 output COLUMNS (the weights, or the gradient of Dw), its
// N dimension is TM output rows (16, 32, 64 or 128), so that one token costs the tensor core a sixteenth of what a padded
// 128-row tile would, and the weights stream through shared memory once whatever the number of rows:
//
//   form    128-row operand (per K block of 64)         TM-row operand
//   Fwd     b [K, N], N-major: 128 columns              a [M, K], K-major
//   Gated   64 columns of the gate, 64 of up            a [M, K], K-major
//   Dx      b [N, K], K-major: 128 rows                 a [M, K], K-major; both pairs one after the other
//   Dw      b [K, N], N-major: 128 columns              a [K, M], M-major
//
// Bound: HBM, reading the weights once (one token, 4096 x 4096: 33.5 MB, 5.1 us). What matters is bytes in flight -- a
// CTA's ring takes what shared memory there is, half of it where two CTAs share an SM -- and the path behind the last
// block, measured with clock stamps: a cluster barrier costs about 1,300 cycles and a row of outputs read back through
// distributed shared memory another 400, so the ranges meet in one step instead. The 128 columns of a tile are dealt out
// to the CTAs of its cluster; each CTA writes its fp32 partial sums into the owners' receive buffers (st.shared::cluster)
// and arrives on their barriers, and an owner adds what it received in ascending order of the ranges, then bias,
// activation, product, residual. The sums have a fixed order; nothing is atomic. Cluster barriers remain only for
// lifetimes, arrived at early and waited for late.
//
// Measured in graphs of launches: one token 4096 x 4096 7.7-9.8 us (8 ranges), 16 tokens through two weights of 4096 x 11008
// 33.4 us (5.4 TB/s of weights, 82 % of the copy rate), 64 rows 9.2, 128 rows 11.0 us.
//
// The CTAs of a cluster wait for one another while each holds TMEM, so an SM's 512 columns must suffice for all CTAs that
// fit on it: at most 1.3 columns per KB of shared memory of any kernel here beside this one (128 of 97 KB, 256 of 193 KB
// in gemm_bias_act.cu), 300 in all; kernels that take all 512 columns leave no room for a second CTA.
#pragma once

#include "activation.cuh"
#include "ffn_gemm.h"
#include "sm100_ptx.cuh"

namespace tcab {

constexpr int kSmallThreads = 256;
constexpr int kSmallMaxStages = 12;

struct FfnSmallArgs {
  CUtensorMap wide[2], rows[2];  // the 128-row operand, the TM-row operand
  __nv_bfloat16* c[2];
  __nv_bfloat16* z[2];
  const float* bias[2];
  const __nv_bfloat16* residual;
  uint32_t M, N, K, pairs;
  uint32_t ks, blocks_per_range;  // CTAs per tile (1, 2, 4, 8), K blocks of each
  uint32_t stages;
  int act;
  int beside;  // FfnProblem::beside
};

struct FfnSmallKernel {
  const void* fn;
  uint32_t stage_bytes, receive_bytes;
  cudaError_t (*status)(int*);
};

template <int TM>
struct FfnSmall {
  static constexpr int WIDE_BYTES = 128 * 128, ROWS_BYTES = TM * 128, STAGE = WIDE_BYTES + ROWS_BYTES;
  static constexpr int RECEIVE_BYTES = TM * 128 * 4;  // [range][row][128 / ks columns] fp32
  static constexpr int TMEM_COLS = TM < 32 ? 32 : TM;
};

namespace {

__device__ int g_small_status = 0;

// activations of eight values by a run-time choice: a tile has few of them per thread
__device__ __forceinline__ void act_values_any(int act, float (&v)[8]) {
  switch (act) {
    case TCAB_ACT_RELU: act_values<TCAB_ACT_RELU>(v); break;
    case TCAB_ACT_SILU: act_values<TCAB_ACT_SILU>(v); break;
    case TCAB_ACT_GELU: act_values<TCAB_ACT_GELU>(v); break;
    case TCAB_ACT_GELU_TANH: act_values<TCAB_ACT_GELU_TANH>(v); break;
    case TCAB_ACT_SIGMOID: act_values<TCAB_ACT_SIGMOID>(v); break;
    default: break;
  }
}
__device__ __forceinline__ uint4 pack8(const float (&v)[8]) {
  uint32_t w[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(v[2 * j], v[2 * j + 1]);
    w[j] = *reinterpret_cast<const uint32_t*>(&h);
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}
template <int FORM, int TM>
__global__ void __launch_bounds__(kSmallThreads, 2)
ffn_small_kernel(const __grid_constant__ FfnSmallArgs args) {
  using C = FfnSmall<TM>;
  constexpr bool GATED = FORM == kFfnGated, WIDE_MN = FORM != kFfnDx, ROWS_MN = FORM == kFfnDw;
  constexpr uint32_t TN = GATED ? 64 : 128;  // output columns per tile
  extern __shared__ uint8_t smem_raw[];
  __shared__ __align__(8) uint64_t bar_full[kSmallMaxStages];
  __shared__ __align__(8) uint64_t bar_empty[kSmallMaxStages];
  __shared__ __align__(8) uint64_t bar_acc;
  __shared__ __align__(8) uint64_t bar_received;  // one arrival per range
  __shared__ uint32_t tmem_slot;
  __shared__ int abort_flag;

  const uint32_t ring = (ptx::smem_u32(smem_raw) + 1023u) & ~1023u;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  volatile int* abort_p = &abort_flag;
  const uint32_t M = args.M, N = args.N, ks = args.ks, stages = args.stages;
  const uint32_t receive = ring + stages * C::STAGE, first_blocks = min(stages, 3u);
  const uint32_t rank = ks > 1 ? ptx::cluster_ctarank() : 0u;  // the range; clusters are ks x 1 x 1 over a 1-D grid
  const uint32_t tiles_m = (M + TM - 1) / TM, tiles_n = (N + TN - 1) / TN, tiles_one = tiles_m * tiles_n;
  uint32_t tile = blockIdx.x / ks;
  const uint32_t which = FORM == kFfnDw && tile >= tiles_one ? 1u : 0u;
  tile -= which * tiles_one;
  // neighbouring tiles share the 128-row operand: it leaves HBM once
  const uint32_t m0 = (tile % tiles_m) * TM, n0 = (tile / tiles_m) * TN;
  const uint32_t seg_kb = (args.K + 63) / 64, all_kb = FORM == kFfnDx ? seg_kb * args.pairs : seg_kb;
  const uint32_t kb0 = min(rank * args.blocks_per_range, all_kb), num_kb = min(args.blocks_per_range, all_kb - kb0);

  auto issue = [&](uint32_t i, uint32_t stage) {  // K block kb0 + i into a stage
    const uint32_t kb = kb0 + i, seg = FORM == kFfnDx && kb >= seg_kb ? 1u : 0u;
    const int32_t k = static_cast<int32_t>((kb - seg * seg_kb) * 64);
    const uint32_t bar = ptx::smem_u32(&bar_full[stage]), wide = ring + stage * C::STAGE, rows = wide + C::WIDE_BYTES;
    ptx::mbar_expect_tx(bar, C::STAGE);
    if (GATED) {
      ptx::tma_load_2d(wide, &args.wide[0], bar, static_cast<int32_t>(n0), k);
      ptx::tma_load_2d(wide + 8192, &args.wide[1], bar, static_cast<int32_t>(n0), k);
    } else if (WIDE_MN) {
      ptx::tma_load_2d(wide, &args.wide[which], bar, static_cast<int32_t>(n0), k);
      ptx::tma_load_2d(wide + 8192, &args.wide[which], bar, static_cast<int32_t>(n0 + 64), k);
    } else {
      ptx::tma_load_2d(wide, &args.wide[seg], bar, k, static_cast<int32_t>(n0));
    }
    if (ROWS_MN) {
#pragma unroll
      for (int j = 0; j < TM / 64; ++j)
        ptx::tma_load_2d(rows + j * 8192, &args.rows[0], bar, static_cast<int32_t>(m0 + j * 64), k);
    } else {
      ptx::tma_load_2d(rows, &args.rows[seg], bar, k, static_cast<int32_t>(m0));
    }
  };

  if (threadIdx.x == 0) {
    abort_flag = 0;
    for (uint32_t s = 0; s < stages; ++s) {
      ptx::mbar_init(ptx::smem_u32(&bar_full[s]), 1);
      ptx::mbar_init(ptx::smem_u32(&bar_empty[s]), 1);
    }
    ptx::mbar_init(ptx::smem_u32(&bar_acc), 1);
    ptx::mbar_init(ptx::smem_u32(&bar_received), ks);
    ptx::fence_barrier_init();
    ptx::fence_proxy_async();
    if (!args.beside) ptx::pdl_wait();
    // the first blocks are under way before the TMEM allocation and the barrier below; the others follow it: a full ring
    // of copies from one thread takes 1,500 cycles
    for (uint32_t i = 0; i < num_kb && i < first_blocks; ++i) issue(i, i);
  }
  __syncwarp();
  if (ks > 1) ptx::cluster_arrive();  // this CTA's barriers are initialised
  if (warp == 1) {
    ptx::tmem_alloc(ptx::smem_u32(&tmem_slot), C::TMEM_COLS);
    ptx::tmem_relinquish();
  }
  ptx::tc_fence_before();
  __syncthreads();
  ptx::tc_fence_after();
  ptx::pdl_launch();
  const uint32_t tmem = tmem_slot;

  if (warp == 0) {
    if (lane == 0) {
      for (uint32_t i = first_blocks; i < stages && i < num_kb; ++i) issue(i, i);
      uint32_t stage = 0, phase = 0;
      for (uint32_t i = stages; i < num_kb; ++i) {
        if (!ptx::mbar_wait(ptx::smem_u32(&bar_empty[stage]), phase, abort_p)) break;
        issue(i, stage);
        if (++stage == stages) { stage = 0; phase ^= 1u; }
      }
    }
  } else if (warp == 1) {
    if (lane == 0 && num_kb > 0) {
      constexpr uint32_t idesc = ptx::idesc_bf16_f32(128, TM, WIDE_MN ? 1 : 0, ROWS_MN ? 1 : 0);
      uint32_t stage = 0, phase = 0;
      bool ok = true;
      for (uint32_t i = 0; i < num_kb; ++i) {
        if (!ptx::mbar_wait(ptx::smem_u32(&bar_full[stage]), phase, abort_p)) { ok = false; break; }
        ptx::tc_fence_after();
        const uint32_t wide = ring + stage * C::STAGE, rows = wide + C::WIDE_BYTES;
#pragma unroll
        for (int k = 0; k < 4; ++k) {  // descriptors as in ffn_gemm.cuh
          const uint64_t adesc = WIDE_MN ? ptx::smem_desc_sw128(wide + k * 2048, 8192, 1024) : ptx::smem_desc_sw128(wide + k * 32, 16, 1024);
          const uint64_t bdesc = ROWS_MN ? ptx::smem_desc_sw128(rows + k * 2048, 8192, 1024) : ptx::smem_desc_sw128(rows + k * 32, 16, 1024);
          ptx::mma_bf16(tmem, adesc, bdesc, idesc, (i | static_cast<uint32_t>(k)) != 0u);
        }
        ptx::mma_commit(ptx::smem_u32(&bar_empty[stage]));
        if (++stage == stages) { stage = 0; phase ^= 1u; }
      }
      if (ok) ptx::mma_commit(ptx::smem_u32(&bar_acc));
    }
  }
  __syncwarp();
  if (!args.beside) ptx::pdl_wait();  // every thread: what follows reads and writes global memory
  const uint32_t live_rows = min(static_cast<uint32_t>(TM), M - m0);
  // A lane of TMEM is a column of the tile. Its owner is the CTA that stores it; there it is column `mine` of the range.
  const uint32_t col = (static_cast<uint32_t>(warp) & 3u) * 32 + lane, per = TN / ks;  // columns per owner (of each projection)
  const uint32_t owner = (GATED ? col % 64 : col) / per, in_owner = (GATED ? col % 64 : col) % per;
  const uint32_t width = GATED ? 2 * per : per;  // Gated: gate's columns, then up's
  const uint32_t mine = in_owner + (GATED && col >= 64 ? per : 0u);
  const uint32_t local = receive + (rank * live_rows * width + mine) * 4;
  const uint32_t dest = ks > 1 ? ptx::mapa(local, owner) : local;
  if (ks > 1) ptx::cluster_wait();  // the peers' barriers are initialised (arrived at before the K loop)
  constexpr int HALF = C::TMEM_COLS >= 64 ? C::TMEM_COLS / 2 : 32;  // rows per warp: two warps share a quarter of the lanes
  const uint32_t row_base = (static_cast<uint32_t>(warp) >> 2) * HALF;
  bool ok = true;
  if (num_kb > 0) {
    ok = ptx::mbar_wait(ptx::smem_u32(&bar_acc), 0, abort_p);
    ptx::tc_fence_after();
  }
  if (row_base < live_rows && row_base < TM) {
#pragma unroll
    for (int q = 0; q < HALF / 32; ++q) {
      uint32_t r[32];
      if (num_kb > 0 && ok) {
        ptx::tmem_ld_32x32(tmem + (((static_cast<uint32_t>(warp) & 3u) * 32u) << 16) + row_base + q * 32, r);
        ptx::tmem_ld_wait_for(r);
      } else {  // an empty range
#pragma unroll
        for (int j = 0; j < 32; ++j) r[j] = 0u;
      }
#pragma unroll
      for (int j = 0; j < 32; ++j) {
        const uint32_t row = row_base + q * 32 + j;
        if (row < live_rows) ptx::st_cluster_f32(dest + row * width * 4, __uint_as_float(r[j]));
      }
    }
  }
  ptx::tc_fence_before();
  __syncthreads();
  // one arrival per range and owner, ordered after every thread's stores by the barrier above and the release
  if (threadIdx.x < ks) ptx::mbar_arrive_cluster(ks > 1 ? ptx::mapa(ptx::smem_u32(&bar_received), threadIdx.x) : ptx::smem_u32(&bar_received));
  if (warp == 1) {
    ptx::tc_fence_after();
    ptx::tmem_dealloc(tmem, C::TMEM_COLS);
  }
  if (!ptx::mbar_wait_cluster(ptx::smem_u32(&bar_received), 0, abort_p)) ok = false;
  __syncwarp();
  if (ks > 1) ptx::cluster_arrive_relaxed();  // nothing of this CTA is outstanding on a peer

  // This CTA's columns in groups of eight (ks <= 8: a CTA owns at least eight).
  const float* got = reinterpret_cast<const float*>(smem_raw + (receive - ptx::smem_u32(smem_raw)));
  const uint32_t groups = per / 8;
  for (uint32_t i = threadIdx.x; i < live_rows * groups; i += kSmallThreads) {
    const uint32_t row = i / groups, g = i % groups, m = m0 + row, n = n0 + rank * per + g * 8;
    if (n >= N || !ok) continue;  // N % 8 == 0: the eight columns are inside together
    const size_t at = static_cast<size_t>(m) * N + n;
    uint4 res = make_uint4(0u, 0u, 0u, 0u);
    if (FORM == kFfnFwd && args.residual != nullptr) res = *reinterpret_cast<const uint4*>(args.residual + at);
    float v[2][8];
#pragma unroll
    for (int s = 0; s < (GATED ? 2 : 1); ++s) {
      const float* from = got + row * width + s * per + g * 8;
#pragma unroll
      for (int j = 0; j < 8; ++j) v[s][j] = 0.0f;
      for (uint32_t r = 0; r < ks; ++r) {  // ascending ranges: ascending k
        const float4 a = *reinterpret_cast<const float4*>(from + r * live_rows * width), b = *reinterpret_cast<const float4*>(from + r * live_rows * width + 4);
        v[s][0] += a.x; v[s][1] += a.y; v[s][2] += a.z; v[s][3] += a.w;
        v[s][4] += b.x; v[s][5] += b.y; v[s][6] += b.z; v[s][7] += b.w;
      }
      if ((FORM == kFfnFwd || GATED) && args.bias[s] != nullptr) {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[s][j] += __ldg(args.bias[s] + n + j);
      }
      if ((FORM == kFfnFwd || GATED) && args.z[s] != nullptr) *reinterpret_cast<uint4*>(args.z[s] + at) = pack8(v[s]);
    }
    if (FORM == kFfnFwd || GATED) act_values_any(args.act, v[0]);
    if (GATED) {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[0][j] *= v[1][j];
    } else if (FORM == kFfnFwd && args.residual != nullptr) {
      const uint32_t w[4] = {res.x, res.y, res.z, res.w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        v[0][2 * j] += __uint_as_float(w[j] << 16);
        v[0][2 * j + 1] += __uint_as_float(w[j] & 0xffff0000u);
      }
    }
    *reinterpret_cast<uint4*>(args.c[which] + at) = pack8(v[0]);
  }
  if (threadIdx.x == 0 && abort_flag != 0) g_small_status = 1;
  if (args.beside) ptx::pdl_wait();
  if (ks > 1) {
    __syncwarp();
    ptx::cluster_wait();  // no CTA leaves while a peer may still signal it
  }
}

cudaError_t read_small_status(int* out) { return cudaMemcpyFromSymbol(out, g_small_status, sizeof(int)); }

template <int FORM, int TM>
FfnSmallKernel ffn_small_of() {
  return {reinterpret_cast<const void*>(ffn_small_kernel<FORM, TM>), FfnSmall<TM>::STAGE, FfnSmall<TM>::RECEIVE_BYTES, read_small_status};
}

}  // namespace

}  // namespace tcab
