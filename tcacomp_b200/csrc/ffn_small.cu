// ffn_small.cu -- the instances of ffn_small.cuh and their launch.
#include "ffn_small.cuh"

namespace tcab {
namespace {

FfnSmallKernel small_kernel(int form, int tm) {
#define TCAB_CASE(F, R) if (form == F && tm == R) return ffn_small_of<F, R>();
  TCAB_CASE(kFfnFwd, 16) TCAB_CASE(kFfnFwd, 32) TCAB_CASE(kFfnFwd, 64) TCAB_CASE(kFfnFwd, 128)
  TCAB_CASE(kFfnGated, 16) TCAB_CASE(kFfnGated, 32) TCAB_CASE(kFfnGated, 64) TCAB_CASE(kFfnGated, 128)
  TCAB_CASE(kFfnDx, 16) TCAB_CASE(kFfnDx, 32) TCAB_CASE(kFfnDx, 64) TCAB_CASE(kFfnDx, 128)
  TCAB_CASE(kFfnDw, 64) TCAB_CASE(kFfnDw, 128)
#undef TCAB_CASE
  return {nullptr, 0, 0, nullptr};
}

}  // namespace

int ffn_small_status(int* out) {
  if (read_small_status(out) != cudaSuccess) {
    cudaGetLastError();
    return fail(TCAB_ERR_CUDA, "device_status: cannot read a status word");
  }
  return TCAB_OK;
}

// Rows of the tile and CTAs per tile, by an estimate in microseconds that follows what was measured on B200 with graphs of
// launches (contractions over 64 to 4096, outputs of 4096 columns):
//   before the first and behind the last block: 3.2 (16 or 32 rows), 4.3 (64), 5.8 (128); + 0.1, 0.2, 1.1 (6 from 64 rows on)
//   for 2, 4, 8 ranges
//   a block of 64: 0.33, or the time HBM takes for the blocks of all ranges (6.3 TB/s from two CTAs per SM, 4.6 from one)
// 1 x 4096 x 4096: 22.3, 14.6, 11.7, 9.5 us for 1, 2, 4, 8 ranges; 128 rows: 27.6, 17.1, 12.8, 26.6.
FfnSmallPlan ffn_small_plan(int form, uint32_t m, uint32_t n, uint32_t k, uint32_t pairs, int sms, int forced_ks) {
  FfnSmallPlan p;
  p.tm = m <= 16 && form != kFfnDw ? 16 : m <= 32 && form != kFfnDw ? 32 : m <= 64 ? 64 : 128;
  const uint64_t tn = form == kFfnGated ? 64 : 128;
  const uint64_t wide = (n + tn - 1) / tn * (form == kFfnDw ? pairs : 1);
  p.tiles = (static_cast<uint64_t>(m) + p.tm - 1) / p.tm * wide;
  const uint64_t blocks = (static_cast<uint64_t>(k) + 63) / 64 * (form == kFfnDx ? pairs : 1);
  p.us = 1e300;
  for (uint32_t ks = 1; ks <= 8; ks *= 2) {
    if (forced_ks > 0 && ks != (forced_ks >= 8 ? 8u : forced_ks >= 4 ? 4u : forced_ks >= 2 ? 2u : 1u)) continue;
    if (forced_ks <= 0 && ks > 1 && blocks < 2ull * ks) break;
    const uint64_t ctas = p.tiles * ks, per = (blocks + ks - 1) / ks;
    const int per_sm = p.tm < 128 && ctas > static_cast<uint64_t>(sms) ? 2 : 1;
    const uint64_t slots = static_cast<uint64_t>(sms) * per_sm, rounds = (ctas + slots - 1) / slots;
    const double resident = static_cast<double>(ctas < slots ? ctas : slots) / static_cast<double>(p.tiles);
    double block = static_cast<double>(wide) * resident * 16384.0 / (per_sm == 2 ? 6.3e6 : 4.6e6);
    if (block < 0.33) block = 0.33;
    const double ranges = ks == 1 ? 0.0 : ks == 2 ? 0.1 : ks == 4 ? 0.2 : p.tm <= 32 ? 1.1 : 6.0;
    const double us = (p.tm <= 32 ? 3.2 : p.tm == 64 ? 4.3 : 5.8) * (0.5 + 0.5 * static_cast<double>(rounds)) + ranges +
                      static_cast<double>(rounds * per) * block;
    if (us < p.us) {
      p.us = us;
      p.ks = ks;
      p.blocks_per_range = static_cast<uint32_t>(per);
      p.per_sm = per_sm;
    }
  }
  return p;
}

int launch_ffn_small(const char* op, int form, const FfnProblem& p, int sms, cudaStream_t s) {
  const uint32_t pairs = p.b[1] != nullptr ? 2 : 1;
  const FfnSmallPlan plan = ffn_small_plan(form, p.M, p.N, p.K, pairs, sms, tune(kFfn).p3);
  const FfnSmallKernel k = small_kernel(form, plan.tm);
  const uint32_t room = (plan.per_sm == 2 ? 112u : 225u) * 1024 - 1024 - k.receive_bytes;
  uint32_t stages = room / k.stage_bytes;
  if (stages > kSmallMaxStages) stages = kSmallMaxStages;
  if (stages > plan.blocks_per_range && plan.blocks_per_range > 0) stages = plan.blocks_per_range;
  const size_t smem = static_cast<size_t>(stages) * k.stage_bytes + k.receive_bytes + 1024;
  FfnSmallArgs args = {};
  args.M = p.M;
  args.N = p.N;
  args.K = p.K;
  args.pairs = pairs;
  args.ks = plan.ks;
  args.blocks_per_range = plan.blocks_per_range;
  args.stages = stages;
  args.act = p.act;
  args.beside = p.beside ? 1 : 0;
  args.residual = p.residual;
  for (int i = 0; i < 2; ++i) {
    args.c[i] = p.c[i];
    args.z[i] = p.z[i];
    args.bias[i] = p.bias[i];
  }
  if (p.K > 0) {
    for (uint32_t i = 0; i < pairs; ++i) {
      if (form == kFfnDx) TCAB_TRY_RC(make_tensor_map(op, &args.wide[i], p.b[i], p.N, p.K, 128, 64));
      else TCAB_TRY_RC(make_tensor_map(op, &args.wide[i], p.b[i], p.K, p.N, 64, 64));
      if (form == kFfnDw) {
        if (i == 0) TCAB_TRY_RC(make_tensor_map(op, &args.rows[0], p.a[0], p.K, p.M, 64, 64));
      } else if (i == 0 || form == kFfnDx) {
        TCAB_TRY_RC(make_tensor_map(op, &args.rows[i], p.a[i], p.M, p.K, static_cast<uint32_t>(plan.tm), 64));
      }
    }
  }
  TCAB_TRY_RC(reserve_smem(op, k.fn, smem));
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(plan.tiles * plan.ks));
  cfg.blockDim = dim3(kSmallThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = plan.ks;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.numAttrs = 2;
  void* params[] = {&args};
  const cudaError_t le = cudaLaunchKernelExC(&cfg, k.fn, params);
  count_launch();
  if (le != cudaSuccess) {
    cudaGetLastError();
    return fail(TCAB_ERR_CUDA, "%s: launch failed: %s", op, cudaGetErrorString(le));
  }
  return TCAB_OK;
}

}  // namespace tcab
