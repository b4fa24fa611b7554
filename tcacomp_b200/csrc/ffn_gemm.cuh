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
// A tile is 512 x 256 or 256 x 256 on a pair of CTAs (cta_group::2: each loads its rows of a and half of b's columns, the
// leader issues the MMAs), or 128 x 128 on one CTA. Roles: warp 0 (one lane) is the TMA producer, warp 1 (one lane) issues
// the MMAs, warps 4-11 are the epilogue and take most of the registers. A K block is 64 wide; an accumulator is 128 rows x
// BN columns per CTA, and TMEM holds 512 / BN of them. With 256 x 256 and 128 x 128 they form a ring, so that the epilogue
// of a tile -- activations, products, residuals, up to three stored matrices -- runs under the K loop of the next. With
// 512 x 256 a tile takes both accumulators: the first is read into registers and handed back before anything is computed,
// the second follows block by block.
//
// Bound: the tensor pipe up to where the power limit lowers the clock; from some thousand rows on, energy per product.
// 8192^3 without an activation: 512 x 256 1,395 TFLOP/s (tensor pipe 85 % busy at 1,342 MHz), 256 x 256 1,305 (92 % at
// 1,170: it moves half as many bytes again). Two K blocks share a ring stage where there is room: a stage's wait, signal
// and commit cost 15 % of the K loop with one block each (256 x 256 .80 -> .91 busy; 128 x 128 tiles, 512 x 4096 x 4096:
// 25.7 -> 20.1 us, from there on L2: 16 TB/s of operand tiles). 256 x 128 tiles on pairs were no faster than 128 x 128
// (20.2 us there, 14.2 against 11.1 for 256 x 256 at 1003 x 1000 x 2728) and are not built.
//
// Results leave as 32 x 32 boxes: a lane holds a row of 32 columns, the box turns in a 2 KB buffer of the warp, and four
// 16-byte stores per lane write 64-byte row segments. (TMA stores from two such buffers were measured first: about 1,000
// cycles per box, most of them waiting for a buffer to be read, against 250; where a CTA has one tile, nothing hides
// that.) A residual takes the same way in. Loads past an edge read zeros. Every wait is bounded (sm100_ptx.cuh); a wait
// that gives up ends the kernel with a status word.
#pragma once

#include "activation.cuh"
#include "ffn_gemm.h"
#include "sm100_ptx.cuh"

namespace tcab {

constexpr int kFfnBK = 64, kFfnEpiWarps = 8, kFfnThreads = 128 + 32 * kFfnEpiWarps;
constexpr int kFfnAtom = kFfnBK * 128;  // a box of 64 x 64 bf16
constexpr int kFfnStageBox = 32 * 64;   // a box of 32 x 32 bf16 results

struct FfnArgs {
  CUtensorMap a[2], b[2];
  __nv_bfloat16* c[2];
  __nv_bfloat16* z[2];
  const float* bias[2];
  const __nv_bfloat16* residual;
  uint32_t M, N, K;
  uint32_t pairs;  // Dx: contracted pairs (1, 2); Dw: outputs (1, 2)
  int save;        // Fwd, Gated: also store the projections
  int beside;      // FfnProblem::beside
};

// What a translation unit of this kernel family gives: an instance, its dynamic shared memory and its status word
// (1: an instance gave up on a wait).
struct FfnKernel {
  const void* fn;
  size_t smem;
  cudaError_t (*status)(int*);
};

// A tile of (128 NACC CTAS) x BN on CTAS SMs. A CTA holds NACC accumulators of 128 rows x BN columns of it and loads, per
// K block, the 128 NACC rows of a that belong to them and BN / CTAS columns of b. KPS K blocks share a ring stage.
template <int CTAS, int NACC_, int BN, int KPS_>
struct FfnTile {
  static constexpr int NACC = NACC_, KPS = KPS_, BM = 128 * NACC * CTAS, B_COLS = BN / CTAS, SLOTS = 512 / BN;
  static constexpr int A_BYTES = NACC * 128 * 128, B_BYTES = B_COLS * 128, BLOCK = A_BYTES + B_BYTES, STAGE = KPS * BLOCK;
  static constexpr int STAGES = 192 * 1024 / STAGE;
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

template <int FORM, int ACT, int CTAS, int NACC, int BN, int KPS>
__global__ void __launch_bounds__(kFfnThreads, 1)
ffn_gemm_kernel(const __grid_constant__ FfnArgs args) {
  using C = FfnTile<CTAS, NACC, BN, KPS>;
  constexpr bool PAIR = CTAS == 2;
  constexpr bool A_MN = FORM == kFfnDw, B_NK = FORM == kFfnDx, GATED = FORM == kFfnGated;
  constexpr bool EPILOGUE = FORM == kFfnFwd || FORM == kFfnGated;
  constexpr int TN = GATED ? BN / 2 : BN;  // output columns per tile
  extern __shared__ uint8_t smem_raw[];
  __shared__ __align__(8) uint64_t bar_full[C::STAGES];       // PAIR: used in the leader, bytes of both CTAs land here
  __shared__ __align__(8) uint64_t bar_empty[C::STAGES];      // in each CTA
  __shared__ __align__(8) uint64_t bar_acc_full[C::SLOTS];    // in each CTA
  __shared__ __align__(8) uint64_t bar_acc_empty[C::SLOTS];   // PAIR: used in the leader, both CTAs' epilogue warps arrive
  __shared__ __align__(16) float bias_s[EPILOGUE ? BN : 4];  // the current tile's (zeros past N)
  __shared__ uint32_t tmem_base_slot;
  __shared__ int abort_flag;

  const uint32_t smem_base = (ptx::smem_u32(smem_raw) + 1023u) & ~1023u;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = PAIR ? ptx::cluster_ctarank() : 0u;
  const bool leader = rank == 0;
  volatile int* abort_p = &abort_flag;

  const uint32_t M = args.M, N = args.N;
  const uint32_t tiles_m = (M + C::BM - 1) / C::BM, tiles_n1 = (N + TN - 1) / TN;
  const uint32_t tiles_one = tiles_m * tiles_n1;  // tiles of one output
  const uint32_t num_tiles = FORM == kFfnDw ? tiles_one * args.pairs : tiles_one;
  const uint32_t seg_st = (args.K + kFfnBK * KPS - 1) / (kFfnBK * KPS);  // ring stages per contracted pair
  const uint32_t num_st = FORM == kFfnDx ? seg_st * args.pairs : seg_st;
  const uint32_t first = blockIdx.x / CTAS, step = gridDim.x / CTAS;

  if (threadIdx.x == 0) {
    abort_flag = 0;
    for (int s = 0; s < C::STAGES; ++s) {
      ptx::mbar_init(ptx::smem_u32(&bar_full[s]), 1);
      ptx::mbar_init(ptx::smem_u32(&bar_empty[s]), 1);
    }
    for (int s = 0; s < C::SLOTS; ++s) {
      ptx::mbar_init(ptx::smem_u32(&bar_acc_full[s]), 1);
      ptx::mbar_init(ptx::smem_u32(&bar_acc_empty[s]), CTAS * kFfnEpiWarps);
    }
    ptx::fence_barrier_init();
    ptx::fence_proxy_async();
    ptx::prefetch_tensormap(&args.a[0]);
    ptx::prefetch_tensormap(&args.b[0]);
    if (GATED || (FORM >= kFfnDx && args.pairs == 2)) ptx::prefetch_tensormap(&args.b[1]);
  }
  __syncwarp();
  if (PAIR) ptx::cluster_arrive();  // this CTA's barriers are initialised
  if (warp == 1) {
    if (PAIR) {
      ptx::tmem_alloc_pair(ptx::smem_u32(&tmem_base_slot), 512);
      ptx::tmem_relinquish_pair();
    } else {
      ptx::tmem_alloc(ptx::smem_u32(&tmem_base_slot), 512);
      ptx::tmem_relinquish();
    }
  }
  ptx::tc_fence_before();
  __syncthreads();
  if (PAIR) ptx::cluster_wait();  // the peer's barriers must be initialised before anything of this CTA can signal them
  ptx::tc_fence_after();
  const uint32_t tmem_base = tmem_base_slot;
  if (!args.beside) ptx::pdl_wait();
  ptx::pdl_launch();

  // Register split: 384 threads x 168 at launch = 64,512; 128 x 40 + 256 x 224 = 62,464 afterwards.
  if (warp < 4) {
    ptx::setmaxnreg_dec<40>();
    if (warp == 0) {
      // ---------------- TMA producer (every CTA) ----------------
      if (lane == 0) {
        auto load = [&](uint32_t dst, const CUtensorMap* map, uint32_t bar, int32_t x, int32_t y) {
          if (PAIR) ptx::tma_load_2d_pair(dst, map, bar, x, y);
          else ptx::tma_load_2d(dst, map, bar, x, y);
        };
        uint32_t stage = 0, phase = 0;
        bool ok = true;
        for (uint32_t t = first; ok && t < num_tiles; t += step) {
          const uint32_t which = FORM == kFfnDw && t >= tiles_one ? 1u : 0u;
          const FfnCoord tc = ffn_coord(t - which * tiles_one, tiles_m, tiles_n1);
          const int32_t m0 = static_cast<int32_t>(tc.m * C::BM + rank * 128);  // accumulator a: + a * 128 CTAS
          // Gated: a pair's first CTA loads the gate's columns, its second the same columns of up
          const int32_t n0 = static_cast<int32_t>(tc.n * TN + (GATED ? 0u : rank * C::B_COLS));
          for (uint32_t st = 0; st < num_st; ++st) {
            if (!ptx::mbar_wait_parked(ptx::smem_u32(&bar_empty[stage]), phase ^ 1u, abort_p)) { ok = false; break; }
            const uint32_t full = PAIR ? ptx::mapa(ptx::smem_u32(&bar_full[stage]), 0) : ptx::smem_u32(&bar_full[stage]);
            const uint32_t seg = FORM == kFfnDx && st >= seg_st ? 1u : 0u;
            if (leader) ptx::mbar_expect_tx(ptx::smem_u32(&bar_full[stage]), CTAS * C::STAGE);
#pragma unroll
            for (int kk = 0; kk < KPS; ++kk) {
              const uint32_t a_dst = smem_base + stage * C::STAGE + kk * C::BLOCK, b_dst = a_dst + C::A_BYTES;
              const int32_t k0 = static_cast<int32_t>(((st - seg * seg_st) * KPS + kk) * kFfnBK);
#pragma unroll
              for (int a = 0; a < NACC; ++a) {
                const int32_t row = m0 + a * 128 * CTAS;
                if (A_MN) {
                  load(a_dst + a * 2 * kFfnAtom, &args.a[0], full, row, k0);
                  load(a_dst + a * 2 * kFfnAtom + kFfnAtom, &args.a[0], full, row + 64, k0);
                } else {
                  load(a_dst + a * 2 * kFfnAtom, &args.a[seg], full, k0, row);
                }
              }
              if (B_NK) {
                load(b_dst, &args.b[seg], full, k0, n0);
              } else {
#pragma unroll
                for (int j = 0; j < C::B_COLS / 64; ++j) {
                  constexpr int per = GATED && !PAIR ? BN / 128 : 64;  // Gated on one CTA: boxes of gate, then of up
                  const uint32_t side = GATED ? (PAIR ? rank : static_cast<uint32_t>(j / per)) : which;
                  load(b_dst + j * kFfnAtom, &args.b[side], full, n0 + (j % per) * 64, k0);
                }
              }
            }
            if (++stage == C::STAGES) { stage = 0; phase ^= 1u; }
          }
        }
      }
    } else if (warp == 1) {
      // ---------------- MMA issuer (the leader CTA) ----------------
      if (leader && lane == 0) {
        constexpr uint32_t idesc = ptx::idesc_bf16_f32(128 * CTAS, BN, A_MN ? 1 : 0, B_NK ? 0 : 1);
        auto multiply = [&](uint32_t stage, uint32_t a, uint32_t slot, bool fresh) {
#pragma unroll
          for (int kk = 0; kk < KPS; ++kk) {
            const uint32_t a_src = smem_base + stage * C::STAGE + kk * C::BLOCK + a * 2 * kFfnAtom;
            const uint32_t b_src = smem_base + stage * C::STAGE + kk * C::BLOCK + C::A_BYTES;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              // K-major: rows of 128 bytes in groups of eight 1024 B apart, a step of 16 k is 32 B inside the row.
              // MN-major: atoms of 64 x 64 kFfnAtom apart, groups of eight k rows 1024 B apart, a step is 16 k rows.
              const uint64_t adesc = A_MN ? ptx::smem_desc_sw128(a_src + k * 2048, kFfnAtom, 1024)
                                          : ptx::smem_desc_sw128(a_src + k * 32, 16, 1024);
              const uint64_t bdesc = B_NK ? ptx::smem_desc_sw128(b_src + k * 32, 16, 1024)
                                          : ptx::smem_desc_sw128(b_src + k * 2048, kFfnAtom, 1024);
              const uint32_t more = fresh && kk == 0 && k == 0 ? 0u : 1u;
              if (PAIR) ptx::mma_bf16_pair(tmem_base + slot * BN, adesc, bdesc, idesc, more);
              else ptx::mma_bf16(tmem_base + slot * BN, adesc, bdesc, idesc, more);
            }
          }
        };
        auto commit = [&](uint64_t* bar) {
          if (PAIR) ptx::mma_commit_pair(ptx::smem_u32(bar), 3);  // on both CTAs' barriers
          else ptx::mma_commit(ptx::smem_u32(bar));
        };
        uint32_t stage = 0, phase = 0, unit = 0;
        bool ok = true;
        for (uint32_t t = first; ok && num_st > 0 && t < num_tiles; t += step, unit += NACC) {
          // The first accumulator's products of the tile's first stages go out before the second accumulator is waited
          // for: the epilogue hands that one back a few thousand cycles later.
          const uint32_t ahead = NACC > 1 ? (num_st < C::STAGES ? num_st : C::STAGES) : 0u;
#pragma unroll
          for (int a = 0; a < NACC; ++a) {
            const uint32_t slot = (unit + a) % C::SLOTS;
            uint32_t s2 = stage, p2 = phase;
            // the epilogue must have drained this accumulator
            ok = ok && ptx::mbar_wait_parked(ptx::smem_u32(&bar_acc_empty[slot]), (((unit + a) / C::SLOTS) & 1u) ^ 1u, abort_p);
            if (!ok) break;
            ptx::tc_fence_after();
            for (uint32_t st = 0; st < ahead; ++st) {
              if (a == 0) {
                if (!ptx::mbar_wait_parked(ptx::smem_u32(&bar_full[s2]), p2, abort_p)) { ok = false; break; }
                ptx::tc_fence_after();
              }
              multiply(s2, a, slot, st == 0);
              if (a == NACC - 1) commit(&bar_empty[s2]);
              if (++s2 == C::STAGES) { s2 = 0; p2 ^= 1u; }
            }
            if (!ok) break;
            if (ahead > 0 && ahead == num_st) commit(&bar_acc_full[slot]);
            if (a == NACC - 1) {
              stage = s2;
              phase = p2;
            }
          }
          for (uint32_t st = ahead; ok && st < num_st; ++st) {
            if (!ptx::mbar_wait_parked(ptx::smem_u32(&bar_full[stage]), phase, abort_p)) { ok = false; break; }
            ptx::tc_fence_after();
#pragma unroll
            for (int a = 0; a < NACC; ++a) {
              const uint32_t slot = (unit + a) % C::SLOTS;
              multiply(stage, a, slot, NACC == 1 && st == 0);
              if (NACC > 1 && st + 1 == num_st) commit(&bar_acc_full[slot]);  // this accumulator is complete
            }
            commit(&bar_empty[stage]);
            if (NACC == 1 && st + 1 == num_st) commit(&bar_acc_full[unit % C::SLOTS]);
            if (++stage == C::STAGES) { stage = 0; phase ^= 1u; }
          }
        }
      }
    }
  } else {
    ptx::setmaxnreg_inc<224>();
    // ---------------- epilogue (every CTA drains its own rows) ----------------
    const int e = warp - 4;
    const uint32_t quad = static_cast<uint32_t>(warp) & 3u;  // the TMEM lanes a warp may read: 32 * (warp % 4)
    const uint32_t half = static_cast<uint32_t>(e) >> 2;
    constexpr int NB = BN / 64;              // register blocks of 32 columns per warp and accumulator
    constexpr int OB = GATED ? NB / 2 : NB;  // result boxes per accumulator (Gated: blocks q and OB + q are gate and up)
    const uint32_t stage_box = smem_base + C::STAGES * C::STAGE + e * 2 * kFfnStageBox;
    const uint32_t sw = (static_cast<uint32_t>(lane) >> 1) & 3u;
    uint32_t unit = 0;
    bool ok = true;

    // This lane's place in a turned box: rows lane / 4 + 8 i, the 16-byte chunk lane % 4 of their 64 bytes.
    const uint32_t trow = static_cast<uint32_t>(lane) >> 2, tchunk = static_cast<uint32_t>(lane) & 3u;
    const uint32_t my_row = stage_box + static_cast<uint32_t>(lane) * 64u;
    auto turned = [&](uint32_t i) { return (trow + 8 * i) * 64u + ((tchunk ^ (((trow + 8 * i) >> 1) & 3u)) * 16u); };
    // 32 rows x 32 columns, packed bf16 pairs, to global memory.
    auto put_box = [&](const uint32_t (&w)[16], __nv_bfloat16* to, uint32_t row0, uint32_t col0) {
      __syncwarp();  // every lane has read the previous box
#pragma unroll
      for (uint32_t v = 0; v < 4; ++v) ptx::st_shared_v4(my_row + ((v ^ sw) * 16u), w[v * 4], w[v * 4 + 1], w[v * 4 + 2], w[v * 4 + 3]);
      __syncwarp();
      const uint32_t col = col0 + tchunk * 8;
      uint4* at = reinterpret_cast<uint4*>(to + static_cast<size_t>(row0 + trow) * N + col);
#pragma unroll
      for (uint32_t i = 0; i < 4; ++i)  // N % 8 == 0: a chunk is inside or outside as a whole
        if (row0 + trow + 8 * i < M && col < N) at[static_cast<size_t>(i) * N] = ptx::ld_shared_u4(stage_box + turned(i));
    };
    auto pack = [](uint32_t lo, uint32_t hi) -> uint32_t {
      const __nv_bfloat162 h = __floats2bfloat162_rn(__uint_as_float(lo), __uint_as_float(hi));
      return *reinterpret_cast<const uint32_t*>(&h);
    };
    auto add_bias = [&](uint32_t (&r)[32], const float* b) {
#pragma unroll
      for (int j = 0; j < 32; j += 4) {
        const float4 q = *reinterpret_cast<const float4*>(b + j);
        r[j] = __float_as_uint(__uint_as_float(r[j]) + q.x);
        r[j + 1] = __float_as_uint(__uint_as_float(r[j + 1]) + q.y);
        r[j + 2] = __float_as_uint(__uint_as_float(r[j + 2]) + q.z);
        r[j + 3] = __float_as_uint(__uint_as_float(r[j + 3]) + q.w);
      }
    };
    // The residual of one box, turned like a result: whole 64-byte row segments from global memory, ...
    auto load_residual = [&](uint4 (&q)[4], uint32_t row0, uint32_t col0) {
      const uint32_t col = col0 + tchunk * 8;
      const uint4* at = reinterpret_cast<const uint4*>(args.residual + static_cast<size_t>(row0 + trow) * N + col);
#pragma unroll
      for (uint32_t i = 0; i < 4; ++i) {
        q[i] = make_uint4(0u, 0u, 0u, 0u);
        if (row0 + trow + 8 * i < M && col < N) q[i] = at[static_cast<size_t>(i) * N];
      }
    };
    // ... and through the warp's second buffer to this lane's row of 32 columns.
    auto turn_residual = [&](uint4 (&q)[4]) {
      const uint32_t buf = kFfnStageBox;
      __syncwarp();
#pragma unroll
      for (uint32_t i = 0; i < 4; ++i) ptx::st_shared_v4(stage_box + buf + turned(i), q[i].x, q[i].y, q[i].z, q[i].w);
      __syncwarp();
#pragma unroll
      for (uint32_t v = 0; v < 4; ++v) q[v] = ptx::ld_shared_u4(my_row + buf + ((v ^ sw) * 16u));
    };

    for (uint32_t t = first; t < num_tiles; t += step, unit += NACC) {
      const uint32_t which = FORM == kFfnDw && t >= tiles_one ? 1u : 0u;
      const FfnCoord tc = ffn_coord(t - which * tiles_one, tiles_m, tiles_n1);
      const bool have_bias = EPILOGUE && args.bias[0] != nullptr;
      const bool have_res = FORM == kFfnFwd && args.residual != nullptr;
      if (have_bias) {
        // The tile's bias to shared memory while the K loop runs. No warp leaves this loop early, also after a wait has
        // given up: the barriers need all of them.
        ptx::named_bar_sync(1, kFfnEpiWarps * 32);  // every warp has finished with the previous tile's values
        const uint32_t et = threadIdx.x - 128u;
        if (et < BN) {
          const uint32_t side = GATED && et >= TN ? 1u : 0u, col = tc.n * TN + et - side * TN;
          bias_s[et] = col < N ? __ldg(args.bias[side] + col) : 0.0f;
        }
        ptx::named_bar_sync(1, kFfnEpiWarps * 32);
      }
      const uint32_t row_t = tc.m * C::BM + rank * 128 + quad * 32, out_col = tc.n * TN + half * (TN / 2);
      // Block q of this warp: result columns out_col + 32 q; its accumulator columns (Gated: of gate, of up).
      auto acc_addr = [&](int a, int q) {
        const uint32_t col = GATED ? (q < OB ? 0u : static_cast<uint32_t>(TN)) + half * (TN / 2) + (q < OB ? q : q - OB) * 32u
                                   : half * (TN / 2) + q * 32u;
        return tmem_base + ((quad * 32u) << 16) + ((unit + a) % C::SLOTS) * BN + col;
      };
      auto wait_acc = [&](int a) {
        if (ok && !ptx::mbar_wait_parked(ptx::smem_u32(&bar_acc_full[(unit + a) % C::SLOTS]), ((unit + a) / C::SLOTS) & 1u, abort_p)) ok = false;
        ptx::tc_fence_after();
      };
      auto release_acc = [&](int a) {
        ptx::tc_fence_before();
        // A signal that no later tile waits for is not sent: nothing of this CTA may be under way to a peer that has left.
        if (lane == 0 && t + step * (C::SLOTS / NACC) < num_tiles) {
          const uint32_t bar = ptx::smem_u32(&bar_acc_empty[(unit + a) % C::SLOTS]);
          if (PAIR) ptx::mbar_arrive_cluster(ptx::mapa(bar, 0));
          else ptx::mbar_arrive(bar);
        }
      };
      uint4 res[4];
      if (have_res) {
        // this warp's share of the tile's residual on its way to L2 while the K loop runs
#pragma unroll
        for (int a = 0; a < NACC; ++a) {
          const uint32_t row = row_t + a * 128 * CTAS + lane;
          if (row < M && out_col < N)
            ptx::prefetch_l2(args.residual + static_cast<size_t>(row) * N + out_col, min(static_cast<uint32_t>(TN / 2), N - out_col) * 2u);
        }
        load_residual(res, row_t, out_col);
      }
      // From accumulators to packed results: bias, the stored projections, activation, product or residual. `up` is r
      // itself where there is no second projection. The next box's residual is under way afterwards.
      auto finish = [&](uint32_t (&r)[32], uint32_t (&up)[32], uint32_t (&w)[16], int a, int q) {
        const uint32_t row0 = row_t + a * 128 * CTAS, col0 = out_col + q * 32;
        if constexpr (EPILOGUE) {
          if (have_bias) {
            add_bias(r, bias_s + half * (TN / 2) + q * 32);
            if constexpr (GATED) add_bias(up, bias_s + TN + half * (TN / 2) + q * 32);
          }
          if (args.save) {
#pragma unroll
            for (int j = 0; j < 16; ++j) w[j] = pack(r[2 * j], r[2 * j + 1]);
            put_box(w, args.z[0], row0, col0);
            if constexpr (GATED) {
#pragma unroll
              for (int j = 0; j < 16; ++j) w[j] = pack(up[2 * j], up[2 * j + 1]);
              put_box(w, args.z[1], row0, col0);
            }
          }
#pragma unroll
          for (int j0 = 0; j0 < 32; j0 += 8) {
            float f[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) f[j] = __uint_as_float(r[j0 + j]);
            act_values<ACT>(f);
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              if constexpr (GATED) f[j] *= __uint_as_float(up[j0 + j]);
              r[j0 + j] = __float_as_uint(f[j]);
            }
          }
          if (have_res) {
            turn_residual(res);
#pragma unroll
            for (int v = 0; v < 4; ++v) {
              const uint32_t p[4] = {res[v].x, res[v].y, res[v].z, res[v].w};
#pragma unroll
              for (int j = 0; j < 4; ++j) {
                r[v * 8 + 2 * j] = __float_as_uint(__uint_as_float(r[v * 8 + 2 * j]) + __uint_as_float(p[j] << 16));
                r[v * 8 + 2 * j + 1] = __float_as_uint(__uint_as_float(r[v * 8 + 2 * j + 1]) + __uint_as_float(p[j] & 0xffff0000u));
              }
            }
            if (q + 1 < OB) load_residual(res, row0, col0 + 32);
            else if (a + 1 < NACC) load_residual(res, row0 + 128 * CTAS, out_col);
          }
        }
#pragma unroll
        for (int j = 0; j < 16; ++j) w[j] = pack(r[2 * j], r[2 * j + 1]);
      };
      if (num_st > 0) {
        wait_acc(0);
        if (!ok) continue;
      }
      if constexpr (NACC == 1) {
        // One accumulator per tile and more in TMEM: there is no hurry to hand it back. The boxes go through one copy of
        // the code: where a CTA has a single tile, fetching the instructions of four unrolled boxes for the first time
        // took longer than running them (about 1,000 cycles each).
#pragma unroll 1
        for (int q = 0; q < OB; ++q) {
          uint32_t r[32], up[GATED ? 32 : 1], w[16];
          if (num_st > 0) {
            ptx::tmem_ld_32x32(acc_addr(0, q), r);
            if constexpr (GATED) {
              ptx::tmem_ld_32x32(acc_addr(0, OB + q), up);
              ptx::tmem_ld_wait_for(up);
            }
            ptx::tmem_ld_wait_for(r);
            if (q + 1 == OB) release_acc(0);
          } else {  // an empty contraction: the accumulators' initial value
#pragma unroll
            for (int j = 0; j < 32; ++j) {
              r[j] = 0u;
              if constexpr (GATED) up[j] = 0u;
            }
          }
          if constexpr (GATED) finish(r, up, w, 0, q);
          else finish(r, r, w, 0, q);
          put_box(w, args.c[which], row_t, out_col + q * 32);
        }
      } else {
        uint32_t r[NB][32];
        if (num_st > 0) {
          // the whole share of the first accumulator into registers: it is handed back before anything is computed
#pragma unroll
          for (int q = 0; q < NB; ++q) ptx::tmem_ld_32x32(acc_addr(0, q), r[q]);
#pragma unroll
          for (int q = 0; q < NB; ++q) ptx::tmem_ld_wait_for(r[q]);
          release_acc(0);
        } else {
#pragma unroll
          for (int q = 0; q < NB; ++q)
#pragma unroll
            for (int j = 0; j < 32; ++j) r[q][j] = 0u;
        }
#pragma unroll
        for (int a = 0; a < NACC; ++a) {
          if (a > 0 && num_st > 0) {
#pragma unroll
            for (int q = 0; q < NB; ++q) ptx::tmem_ld_wait_for(r[q]);
            release_acc(a);
          }
#pragma unroll
          for (int q = 0; q < OB; ++q) {
            constexpr int up = GATED ? OB : 0;
            uint32_t w[16];
            finish(r[q], r[up + q], w, a, q);
            if (a + 1 < NACC && num_st > 0) {  // this block's registers are free: refill them from the next accumulator
              if (q == 0) wait_acc(a + 1);
              if (ok) {
                ptx::tmem_ld_32x32(acc_addr(a + 1, q), r[q]);
                if constexpr (GATED) ptx::tmem_ld_32x32(acc_addr(a + 1, up + q), r[up + q]);
              }
            }
            put_box(w, args.c[which], row_t + a * 128 * CTAS, out_col + q * 32);
          }
          if (!ok) break;
        }
      }
    }
  }

  ptx::tc_fence_before();
  __syncthreads();
  if (PAIR) {  // neither CTA may exit or free TMEM while the other can still signal it or read its shared memory
    ptx::cluster_arrive_relaxed();
    ptx::cluster_wait();
  }
  if (warp == 1) {
    ptx::tc_fence_after();
    if (PAIR) ptx::tmem_dealloc_pair(tmem_base, 512);
    else ptx::tmem_dealloc(tmem_base, 512);
  }
  if (threadIdx.x == 0 && abort_flag != 0) g_ffn_status = 1;
  if (args.beside) ptx::pdl_wait();
}

// The kernel of a form, an activation and a tile shape.
template <int FORM, int ACT, int CTAS, int NACC, int BN, int KPS>
FfnKernel ffn_kernel_shape() {
  return {reinterpret_cast<const void*>(ffn_gemm_kernel<FORM, ACT, CTAS, NACC, BN, KPS>), FfnTile<CTAS, NACC, BN, KPS>::SMEM, read_status};
}
template <int FORM, int ACT>
FfnKernel ffn_kernel_of(int shape) {
  switch (shape) {
    case 0: return ffn_kernel_shape<FORM, ACT, 2, 2, 256, 1>();
    case 1: return ffn_kernel_shape<FORM, ACT, 2, 1, 256, 2>();
    default: return ffn_kernel_shape<FORM, ACT, 1, 1, 128, 2>();
  }
}

}  // namespace
}  // namespace tcab
