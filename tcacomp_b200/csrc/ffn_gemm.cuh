// ffn_gemm.cuh -- one persistent tcgen05 kernel for the contractions of a feed-forward layer: forward with bias,
// activation and residual in the epilogue, the two projections of a gated layer with activation and product, and the
// two contractions of a backward pass. bf16 operands, fp32 accumulators in TMEM, bf16 results rounded once.
//
// Operands are taken as they lie in memory; no form copies or transposes anything:
//   form    a                      b                                       tile of b in shared memory
//   Fwd     [M, K], K-major        [K, N], N-major                         BN columns
//   Gated   [M, K], K-major        [K, N] twice, N-major                   BN / 2 columns of each
//   Dx      [M, K] (twice)         [N, K] (twice), K-major                 BN rows; the K loop runs over both pairs
//   Dw      [K, M], M-major        [K, N] (twice), N-major                 BN columns; tiles of the second output follow
//
// Roles: warp 0 (one lane) is the TMA producer, warp 1 (one lane) issues the MMAs, warps 2-9 are the epilogue. A K block
// is 64 wide; a tile of BM x BN takes BM / 128 accumulators of 128 x BN, and TMEM holds 512 / BN of them in a ring, so
// that with BM = 128 the epilogue of a tile runs under the K loop of the next. With BM = BN = 256 the two accumulators
// of a tile fill TMEM: a warp pulls its whole share of the first into registers, hands it back, and refills each
// register block from the second as soon as it has been consumed (what costs time there is how long the next tile's
// first MMAs wait for an accumulator, see gemm_bias_act.cu).
//
// Results leave through 32 x 32 boxes in two alternating staging buffers per warp and TMA stores, which clip ragged
// edges. Loads past an edge read zeros. Every wait is bounded (sm100_ptx.cuh); a wait that gives up ends the kernel
// with a status word.
#pragma once

#include "activation.cuh"
#include "ffn_gemm.h"
#include "sm100_ptx.cuh"

namespace tcab {

constexpr int kFfnBK = 64, kFfnEpiWarps = 8, kFfnThreads = 64 + 32 * kFfnEpiWarps;
constexpr int kFfnAtom = kFfnBK * 128;  // a box of 64 x 64 bf16
constexpr int kFfnStageBox = 32 * 64;   // a box of 32 x 32 bf16 results

struct FfnArgs {
  CUtensorMap a[2], b[2], c[2], z[2];
  const float* bias[2];
  const __nv_bfloat16* residual;
  uint32_t M, N, K;
  uint32_t pairs;  // Dx: contracted pairs (1, 2); Dw: outputs (1, 2)
  int save;        // Fwd, Gated: also store the projections
};

// What a translation unit of this kernel family gives: an instance, its dynamic shared memory and its status word
// (1: an instance gave up on a wait).
struct FfnKernel {
  const void* fn;
  size_t smem;
  cudaError_t (*status)(int*);
};

template <int BM, int BN>
struct FfnTile {
  static constexpr int NACC = BM / 128, SLOTS = 512 / BN;
  static constexpr int A_BYTES = BM * 128, B_BYTES = BN * 128, STAGE = A_BYTES + B_BYTES;
  static constexpr int STAGES = (BM + BN >= 512) ? 3 : (BM + BN >= 384) ? 4 : 6;
  static constexpr size_t SMEM = static_cast<size_t>(STAGES) * STAGE + kFfnEpiWarps * 2 * kFfnStageBox + 1024;
};

struct FfnCoord {
  uint32_t m, n;
};
// Bands of 8 tile rows, so that the CTAs running at the same time share slabs of a and b in L2.
__device__ __forceinline__ FfnCoord ffn_coord(uint32_t t, uint32_t tiles_m, uint32_t tiles_n) {
  const uint32_t band = 8 * tiles_n, first_m = (t / band) * 8, rows = min(8u, tiles_m - first_m), r = t % band;
  return {first_m + r % rows, r / rows};
}

namespace {  // one translation unit per form and activation: each has a status word of its own

__device__ int g_ffn_status = 0;

cudaError_t read_status(int* out) { return cudaMemcpyFromSymbol(out, g_ffn_status, sizeof(int)); }

template <int FORM, int ACT, int BM, int BN>
__global__ void __launch_bounds__(kFfnThreads, 1)
ffn_gemm_kernel(const __grid_constant__ FfnArgs args) {
  using C = FfnTile<BM, BN>;
  constexpr bool A_MN = FORM == kFfnDw, B_NK = FORM == kFfnDx, GATED = FORM == kFfnGated;
  constexpr bool EPILOGUE = FORM == kFfnFwd || FORM == kFfnGated;
  constexpr int TN = GATED ? BN / 2 : BN;  // output columns per tile
  extern __shared__ uint8_t smem_raw[];
  __shared__ __align__(8) uint64_t bar_full[C::STAGES];
  __shared__ __align__(8) uint64_t bar_empty[C::STAGES];
  __shared__ __align__(8) uint64_t bar_acc_full[C::SLOTS];
  __shared__ __align__(8) uint64_t bar_acc_empty[C::SLOTS];
  __shared__ __align__(16) float bias_s[EPILOGUE ? BN : 4];  // the current tile's (zeros past N)
  __shared__ uint32_t tmem_base_slot;
  __shared__ int abort_flag;

  const uint32_t smem_base = (ptx::smem_u32(smem_raw) + 1023u) & ~1023u;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  volatile int* abort_p = &abort_flag;

  const uint32_t M = args.M, N = args.N;
  const uint32_t tiles_m = (M + BM - 1) / BM, tiles_n1 = (N + TN - 1) / TN;
  const uint32_t tiles_one = tiles_m * tiles_n1;  // tiles of one output
  const uint32_t num_tiles = FORM == kFfnDw ? tiles_one * args.pairs : tiles_one;
  const uint32_t seg_kb = (args.K + kFfnBK - 1) / kFfnBK;
  const uint32_t num_kb = FORM == kFfnDx ? seg_kb * args.pairs : seg_kb;

  if (threadIdx.x == 0) {
    abort_flag = 0;
    for (int s = 0; s < C::STAGES; ++s) {
      ptx::mbar_init(ptx::smem_u32(&bar_full[s]), 1);
      ptx::mbar_init(ptx::smem_u32(&bar_empty[s]), 1);
    }
    for (int s = 0; s < C::SLOTS; ++s) {
      ptx::mbar_init(ptx::smem_u32(&bar_acc_full[s]), 1);
      ptx::mbar_init(ptx::smem_u32(&bar_acc_empty[s]), kFfnEpiWarps);
    }
    ptx::fence_barrier_init();
    ptx::fence_proxy_async();
  }
  if (warp == 1) {
    ptx::tmem_alloc(ptx::smem_u32(&tmem_base_slot), 512);
    ptx::tmem_relinquish();
  }
  ptx::tc_fence_before();
  __syncthreads();
  ptx::tc_fence_after();
  const uint32_t tmem_base = tmem_base_slot;

  if (warp == 0) {
    // ---------------- TMA producer ----------------
    if (lane == 0) {
      uint32_t stage = 0, phase = 0;
      bool ok = true;
      for (uint32_t t = blockIdx.x; ok && t < num_tiles; t += gridDim.x) {
        const uint32_t which = FORM == kFfnDw && t >= tiles_one ? 1u : 0u;
        const FfnCoord tc = ffn_coord(t - which * tiles_one, tiles_m, tiles_n1);
        const int32_t m0 = static_cast<int32_t>(tc.m * BM), n0 = static_cast<int32_t>(tc.n * TN);
        for (uint32_t kb = 0; kb < num_kb; ++kb) {
          if (!ptx::mbar_wait(ptx::smem_u32(&bar_empty[stage]), phase ^ 1u, abort_p)) { ok = false; break; }
          const uint32_t full = ptx::smem_u32(&bar_full[stage]);
          const uint32_t a_dst = smem_base + stage * C::STAGE, b_dst = a_dst + C::A_BYTES;
          const uint32_t seg = FORM == kFfnDx && kb >= seg_kb ? 1u : 0u;
          const int32_t k0 = static_cast<int32_t>((kb - seg * seg_kb) * kFfnBK);
          ptx::mbar_expect_tx(full, C::STAGE);
          if (A_MN) {
#pragma unroll
            for (int j = 0; j < BM / 64; ++j) ptx::tma_load_2d(a_dst + j * kFfnAtom, &args.a[0], full, m0 + j * 64, k0);
          } else {
            ptx::tma_load_2d(a_dst, &args.a[seg], full, k0, m0);
          }
          if (B_NK) {
            ptx::tma_load_2d(b_dst, &args.b[seg], full, k0, n0);
          } else if (GATED) {
#pragma unroll
            for (int j = 0; j < BN / 64; ++j)
              ptx::tma_load_2d(b_dst + j * kFfnAtom, &args.b[j / (BN / 128)], full, n0 + (j % (BN / 128)) * 64, k0);
          } else {
#pragma unroll
            for (int j = 0; j < BN / 64; ++j) ptx::tma_load_2d(b_dst + j * kFfnAtom, &args.b[which], full, n0 + j * 64, k0);
          }
          if (++stage == C::STAGES) { stage = 0; phase ^= 1u; }
        }
      }
    }
  } else if (warp == 1) {
    // ---------------- MMA issuer ----------------
    if (lane == 0) {
      constexpr uint32_t idesc = ptx::idesc_bf16_f32(128, BN, A_MN ? 1 : 0, B_NK ? 0 : 1);
      uint32_t stage = 0, phase = 0, unit = 0;
      bool ok = true;
      for (uint32_t t = blockIdx.x; ok && t < num_tiles; t += gridDim.x, unit += C::NACC) {
        for (uint32_t kb = 0; ok && kb < num_kb; ++kb) {
          if (!ptx::mbar_wait(ptx::smem_u32(&bar_full[stage]), phase, abort_p)) { ok = false; break; }
          ptx::tc_fence_after();
          const uint32_t a_src = smem_base + stage * C::STAGE, b_src = a_src + C::A_BYTES;
#pragma unroll
          for (int a = 0; a < C::NACC; ++a) {
            const uint32_t slot = (unit + a) % C::SLOTS;
            if (kb == 0) {  // the epilogue must have drained this accumulator
              if (!ptx::mbar_wait(ptx::smem_u32(&bar_acc_empty[slot]), (((unit + a) / C::SLOTS) & 1u) ^ 1u, abort_p)) { ok = false; break; }
              ptx::tc_fence_after();
            }
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              // K-major: rows of 128 bytes in groups of eight 1024 B apart, a step of 16 k is 32 B inside the row.
              // MN-major: atoms of 64 x 64 kFfnAtom apart, groups of eight k rows 1024 B apart, a step is 16 k rows.
              const uint64_t adesc = A_MN ? ptx::smem_desc_sw128(a_src + a * 2 * kFfnAtom + k * 2048, kFfnAtom, 1024)
                                          : ptx::smem_desc_sw128(a_src + a * (128 * 128) + k * 32, 16, 1024);
              const uint64_t bdesc = B_NK ? ptx::smem_desc_sw128(b_src + k * 32, 16, 1024)
                                          : ptx::smem_desc_sw128(b_src + k * 2048, kFfnAtom, 1024);
              ptx::mma_bf16(tmem_base + slot * BN, adesc, bdesc, idesc, (kb | static_cast<uint32_t>(k)) != 0u);
            }
            if (kb + 1 == num_kb) ptx::mma_commit(ptx::smem_u32(&bar_acc_full[slot]));  // this accumulator is complete
          }
          if (!ok) break;
          ptx::mma_commit(ptx::smem_u32(&bar_empty[stage]));
          if (++stage == C::STAGES) { stage = 0; phase ^= 1u; }
        }
      }
    }
  } else {
    // ---------------- epilogue ----------------
    const int e = warp - 2;
    const uint32_t quad = static_cast<uint32_t>(warp) & 3u;  // the TMEM lanes a warp may read: 32 * (warp % 4)
    const uint32_t half = static_cast<uint32_t>(e) >> 2;
    constexpr int NB = BN / 64;              // register blocks of 32 columns per warp and accumulator
    constexpr int OB = GATED ? NB / 2 : NB;  // result boxes per accumulator (Gated: blocks q and OB + q are gate and up)
    const uint32_t stage_box = smem_base + C::STAGES * C::STAGE + e * 2 * kFfnStageBox;
    const uint32_t sw = (static_cast<uint32_t>(lane) >> 1) & 3u;
    uint32_t unit = 0, nstore = 0;
    bool ok = true;

    // Column (inside the accumulator) of register block q of this warp.
    auto block_col = [&](int q) -> uint32_t {
      if (GATED) return (q < OB ? 0u : BN / 2u) + half * (BN / 4) + (q < OB ? q : q - OB) * 32u;
      return half * (BN / 2) + q * 32u;
    };
    // 32 rows x 32 columns, packed bf16 pairs, to global memory through the staging buffer whose turn it is.
    auto put_box = [&](const uint32_t (&w)[16], const CUtensorMap* map, uint32_t row0, uint32_t col0) {
      const uint32_t buf = stage_box + (nstore & 1u) * kFfnStageBox;
      ++nstore;
      if (lane == 0) ptx::tma_store_wait_read_1();  // the store before the last one has left this buffer
      __syncwarp();
      const uint32_t my_row = buf + static_cast<uint32_t>(lane) * 64u;
#pragma unroll
      for (uint32_t v = 0; v < 4; ++v) ptx::st_shared_v4(my_row + ((v ^ sw) * 16u), w[v * 4], w[v * 4 + 1], w[v * 4 + 2], w[v * 4 + 3]);
      ptx::fence_proxy_async();
      __syncwarp();
      if (lane == 0) {
        // a box outside the result commits an empty group: the wait above counts groups
        if (row0 < M && col0 < N) ptx::tma_store_2d(map, buf, static_cast<int32_t>(col0), static_cast<int32_t>(row0));
        ptx::tma_store_commit();
      }
    };
    auto pack = [](float lo, float hi) -> uint32_t {
      const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
      return *reinterpret_cast<const uint32_t*>(&h);
    };
    // The residual of one box: this lane's row, 32 columns.
    auto load_residual = [&](uint4 (&q)[4], uint32_t row, uint32_t col0) {
#pragma unroll
      for (int v = 0; v < 4; ++v) {
        q[v] = make_uint4(0u, 0u, 0u, 0u);
        if (row < M && col0 + v * 8 < N)
          q[v] = __ldcs(reinterpret_cast<const uint4*>(args.residual + static_cast<size_t>(row) * N + col0 + v * 8));
      }
    };

    for (uint32_t t = blockIdx.x; t < num_tiles; t += gridDim.x, unit += C::NACC) {
      const uint32_t which = FORM == kFfnDw && t >= tiles_one ? 1u : 0u;
      const FfnCoord tc = ffn_coord(t - which * tiles_one, tiles_m, tiles_n1);
      if (EPILOGUE && args.bias[0] != nullptr) {
        // The tile's bias to shared memory while the K loop runs. No warp leaves this loop early, also after a wait has
        // given up: the barriers need all of them.
        ptx::named_bar_sync(1, kFfnEpiWarps * 32);  // every warp has finished with the previous tile's values
        const uint32_t et = threadIdx.x - 64u;
        if (et < BN) {
          const uint32_t side = GATED && et >= TN ? 1u : 0u, col = tc.n * TN + et - side * TN;
          bias_s[et] = col < N ? __ldg(args.bias[side] + col) : 0.0f;
        }
        ptx::named_bar_sync(1, kFfnEpiWarps * 32);
      }
      const bool have_bias = EPILOGUE && args.bias[0] != nullptr;
      const bool have_res = FORM == kFfnFwd && args.residual != nullptr;
      const uint32_t row_a = tc.m * BM + quad * 32, out_col = tc.n * TN + half * (TN / 2);
      uint4 res[4], res_next[4];
      if (have_res && ok) load_residual(res_next, row_a + lane, out_col);

      uint32_t r[NB][32];
      auto acc_addr = [&](uint32_t a) { return tmem_base + ((quad * 32u) << 16) + ((unit + a) % C::SLOTS) * BN; };
      auto wait_acc = [&](uint32_t a) {
        if (ok && !ptx::mbar_wait(ptx::smem_u32(&bar_acc_full[(unit + a) % C::SLOTS]), ((unit + a) / C::SLOTS) & 1u, abort_p)) ok = false;
        ptx::tc_fence_after();
      };
      auto release_acc = [&](uint32_t a) {
        ptx::tc_fence_before();
        if (lane == 0) ptx::mbar_arrive(ptx::smem_u32(&bar_acc_empty[(unit + a) % C::SLOTS]));
      };
      if (num_kb > 0) {
        wait_acc(0);
        if (!ok) continue;
#pragma unroll
        for (int q = 0; q < NB; ++q) ptx::tmem_ld_32x32(acc_addr(0) + block_col(q), r[q]);
#pragma unroll
        for (int q = 0; q < NB; ++q) ptx::tmem_ld_wait_for(r[q]);
        release_acc(0);
      } else {  // an empty contraction: the accumulators' initial value
#pragma unroll
        for (int q = 0; q < NB; ++q)
#pragma unroll
          for (int j = 0; j < 32; ++j) r[q][j] = 0u;
      }
#pragma unroll
      for (int a = 0; a < C::NACC; ++a) {
        const uint32_t row0 = row_a + a * 128;
        if (a > 0 && num_kb > 0) {
#pragma unroll
          for (int q = 0; q < NB; ++q) ptx::tmem_ld_wait_for(r[q]);
          release_acc(a);
        }
#pragma unroll
        for (int q = 0; q < OB; ++q) {
          const uint32_t col0 = out_col + q * 32;
          uint32_t w[16];
          if (!EPILOGUE) {
#pragma unroll
            for (int j = 0; j < 16; ++j) w[j] = pack(__uint_as_float(r[q][2 * j]), __uint_as_float(r[q][2 * j + 1]));
          } else {
            if (have_res) {
#pragma unroll
              for (int v = 0; v < 4; ++v) res[v] = res_next[v];
              // the next box's residual is under way while this one is computed
              if (q + 1 < OB) load_residual(res_next, row0 + lane, col0 + 32);
              else if (a + 1 < C::NACC) load_residual(res_next, row0 + 128 + lane, out_col);
            }
            if (have_bias) {
#pragma unroll
              for (int j = 0; j < 32; j += 4) {
                const float4 b0 = *reinterpret_cast<const float4*>(bias_s + block_col(q) + j);
                r[q][j] = __float_as_uint(__uint_as_float(r[q][j]) + b0.x);
                r[q][j + 1] = __float_as_uint(__uint_as_float(r[q][j + 1]) + b0.y);
                r[q][j + 2] = __float_as_uint(__uint_as_float(r[q][j + 2]) + b0.z);
                r[q][j + 3] = __float_as_uint(__uint_as_float(r[q][j + 3]) + b0.w);
                if (GATED) {
                  constexpr int up = GATED ? OB : 0;
                  const float4 b1 = *reinterpret_cast<const float4*>(bias_s + block_col(up + q) + j);
                  r[up + q][j] = __float_as_uint(__uint_as_float(r[up + q][j]) + b1.x);
                  r[up + q][j + 1] = __float_as_uint(__uint_as_float(r[up + q][j + 1]) + b1.y);
                  r[up + q][j + 2] = __float_as_uint(__uint_as_float(r[up + q][j + 2]) + b1.z);
                  r[up + q][j + 3] = __float_as_uint(__uint_as_float(r[up + q][j + 3]) + b1.w);
                }
              }
            }
            if (args.save) {
#pragma unroll
              for (int j = 0; j < 16; ++j) w[j] = pack(__uint_as_float(r[q][2 * j]), __uint_as_float(r[q][2 * j + 1]));
              put_box(w, &args.z[0], row0, col0);
              if (GATED) {
                constexpr int up = GATED ? OB : 0;
#pragma unroll
                for (int j = 0; j < 16; ++j) w[j] = pack(__uint_as_float(r[up + q][2 * j]), __uint_as_float(r[up + q][2 * j + 1]));
                put_box(w, &args.z[1], row0, col0);
              }
            }
#pragma unroll
            for (int j = 0; j < 16; ++j) {
              float f0 = act_value<ACT>(__uint_as_float(r[q][2 * j])), f1 = act_value<ACT>(__uint_as_float(r[q][2 * j + 1]));
              if (GATED) {
                constexpr int up = GATED ? OB : 0;
                f0 *= __uint_as_float(r[up + q][2 * j]);
                f1 *= __uint_as_float(r[up + q][2 * j + 1]);
              } else if (have_res) {
                const uint32_t p = j % 4 == 0 ? res[j / 4].x : j % 4 == 1 ? res[j / 4].y : j % 4 == 2 ? res[j / 4].z : res[j / 4].w;
                f0 += __uint_as_float(p << 16);
                f1 += __uint_as_float(p & 0xffff0000u);
              }
              w[j] = pack(f0, f1);
            }
          }
          if (a + 1 < C::NACC && num_kb > 0) {  // this block's registers are free: refill them from the next accumulator
            if (q == 0) wait_acc(a + 1);
            if (ok) {
              ptx::tmem_ld_32x32(acc_addr(a + 1) + block_col(q), r[q]);
              if (GATED) ptx::tmem_ld_32x32(acc_addr(a + 1) + block_col(OB + q), r[GATED ? OB + q : q]);
            }
          }
          put_box(w, &args.c[which], row0, col0);
        }
        if (!ok) break;
      }
    }
    if (lane == 0) ptx::tma_store_wait_all();  // every box has reached global memory before the CTA exits
  }

  ptx::tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    ptx::tc_fence_after();
    ptx::tmem_dealloc(tmem_base, 512);
  }
  if (threadIdx.x == 0 && abort_flag != 0) g_ffn_status = 1;
}

// The kernel of a form, an activation and a tile shape (0: 256 x 256, 1: 128 x 256, 2: 128 x 128).
template <int FORM, int ACT>
FfnKernel ffn_kernel_of(int shape) {
  switch (shape) {
    case 0: return {reinterpret_cast<const void*>(ffn_gemm_kernel<FORM, ACT, 256, 256>), FfnTile<256, 256>::SMEM, read_status};
    case 1: return {reinterpret_cast<const void*>(ffn_gemm_kernel<FORM, ACT, 128, 256>), FfnTile<128, 256>::SMEM, read_status};
    default: return {reinterpret_cast<const void*>(ffn_gemm_kernel<FORM, ACT, 128, 128>), FfnTile<128, 128>::SMEM, read_status};
  }
}

}  // namespace
}  // namespace tcab
