// ffn_gemm.cu -- host side of ffn_gemm.cuh: which tile shape a problem takes, its tensor maps and the launch.
#include "ffn_gemm.cuh"

namespace tcab {

FfnKernel ffn_kernel_dx(int shape);
FfnKernel ffn_kernel_dw(int shape);
FfnKernel ffn_kernel_fwd_none(int shape);
FfnKernel ffn_kernel_fwd_relu(int shape);
FfnKernel ffn_kernel_fwd_silu(int shape);
FfnKernel ffn_kernel_fwd_gelu(int shape);
FfnKernel ffn_kernel_fwd_gelu_tanh(int shape);
FfnKernel ffn_kernel_gated_relu(int shape);
FfnKernel ffn_kernel_gated_silu(int shape);
FfnKernel ffn_kernel_gated_gelu(int shape);
FfnKernel ffn_kernel_gated_gelu_tanh(int shape);
FfnKernel ffn_kernel_gated_sigmoid(int shape);

namespace {

FfnKernel kernel_of(int form, int act, int shape) {
  if (form == kFfnDx) return ffn_kernel_dx(shape);
  if (form == kFfnDw) return ffn_kernel_dw(shape);
  if (form == kFfnFwd) {
    switch (act) {
      case TCAB_ACT_NONE: return ffn_kernel_fwd_none(shape);
      case TCAB_ACT_RELU: return ffn_kernel_fwd_relu(shape);
      case TCAB_ACT_SILU: return ffn_kernel_fwd_silu(shape);
      case TCAB_ACT_GELU: return ffn_kernel_fwd_gelu(shape);
      case TCAB_ACT_GELU_TANH: return ffn_kernel_fwd_gelu_tanh(shape);
      default: return {nullptr, 0, nullptr};
    }
  }
  switch (act) {
    case TCAB_ACT_RELU: return ffn_kernel_gated_relu(shape);
    case TCAB_ACT_SILU: return ffn_kernel_gated_silu(shape);
    case TCAB_ACT_GELU: return ffn_kernel_gated_gelu(shape);
    case TCAB_ACT_GELU_TANH: return ffn_kernel_gated_gelu_tanh(shape);
    case TCAB_ACT_SIGMOID: return ffn_kernel_gated_sigmoid(shape);
    default: return {nullptr, 0, nullptr};
  }
}

// The tile shapes of ffn_kernel_of.
constexpr int kShapes = 3, kCtas[kShapes] = {2, 2, 1}, kRows[kShapes] = {512, 256, 128}, kBN[kShapes] = {256, 256, 128};

// The kernel: a tile shape of the persistent one, or kShapes for ffn_small.cuh. An estimate in microseconds per shape --
// what a launch costs before its first and behind its last block, rounds over the SMs (pairs of SMs), blocks of 64 per
// round -- fitted to outputs of 1003 x 2728, 1024 x 2816 and 512 x 4096 over 64 ... 2048 (graphs of launches):
//   512 x 256 on pairs 8.3 + 0.49 per block, 256 x 256 on pairs 5.8 + 0.30, 128 x 128 3.6 + 0.25.
// Both sides of it, us for 512 x 256, 256 x 256, 128 x 128, the small kernel (the choice first): 512 x 4096 x 4096 20.1 for
// 128 x 128, against 42.5, 22.5, 26.5; 1003 x 1000 x 2728 11.2 for 256 x 256, against 17.3, 16.7, 24.9; 2048 x 4096 x 4096
// 46.5 for 512 x 256, against 47.8, 77.4, 103; 256 x 4096 x 4096 16.1 for the small one, against 41.8, 22.3, 19.0.
// Over many rounds the 512 x 256 tile wins (8192^3: 1,395 TFLOP/s against 1,305 for 256 x 256): it moves the fewest bytes.
struct Choice {
  int shape;
  double us;
  uint32_t ctas;  // at once at most
};
Choice choose(int form, uint32_t m, uint32_t n, uint32_t k, uint32_t pairs, int sm, bool shared_l2 = false) {
  static const double kFixed[kShapes] = {8.3, 5.8, 3.6}, kBlock[kShapes] = {0.49, 0.30, 0.25}, kEpilogue[kShapes] = {4.0, 2.2, 1.0};
  const uint64_t sms = static_cast<uint64_t>(sm);
  const uint64_t outs = form == kFfnDw ? pairs : 1, blocks = (static_cast<uint64_t>(k) + 63) / 64 * (form == kFfnDx ? pairs : 1);
  const FfnSmallPlan small = ffn_small_plan(form, m, n, k, pairs, sm, 0);
  int best = kShapes;
  double best_us = small.us;
  uint64_t best_ctas = small.tiles * small.ks;
  for (int s = 0; s < kShapes; ++s) {
    const uint64_t bm = kRows[s], tn = static_cast<uint64_t>(form == kFfnGated ? kBN[s] / 2 : kBN[s]);
    const uint64_t tiles = (m + bm - 1) / bm * ((n + tn - 1) / tn) * outs, at_once = sms / kCtas[s];
    if (at_once == 0) continue;
    const uint64_t rounds = (tiles + at_once - 1) / at_once;
    // a round's end is hidden where two accumulators alternate; the 512 x 256 tile pays part of it every time
    double round = static_cast<double>(blocks) * (s == 2 && shared_l2 ? 0.40 : kBlock[s]) + (s == 0 ? 3.0 : 0.8);
    if (round < kEpilogue[s]) round = kEpilogue[s];  // few blocks: the time of storing a tile
    const double us = kFixed[s] + static_cast<double>(rounds) * round;
    if (us < best_us - 1e-9) {
      best_us = us;
      best = s;
      best_ctas = (tiles < at_once ? tiles : at_once) * kCtas[s];
    }
  }
  return {best, best_us, static_cast<uint32_t>(best_ctas < sms ? best_ctas : sms)};
}

}  // namespace

// Rows and columns of a tile of the kernel that a contraction takes, the CTAs that share a tile's contracted axis and the
// K blocks of 64 that each of them takes (ffn_small.cuh: columns are 128, of a gated pair 64 each).
void ffn_plan(int form, uint32_t m, uint32_t n, uint32_t k, uint32_t pairs, int sms, uint32_t* rows, uint32_t* cols, uint32_t* ranges,
              uint32_t* blocks) {
  const int shape = choose(form, m, n, k, pairs, sms).shape;
  if (shape == kShapes) {
    const FfnSmallPlan p = ffn_small_plan(form, m, n, k, pairs, sms, 0);
    *rows = static_cast<uint32_t>(p.tm);
    *cols = form == kFfnGated ? 64 : 128;
    *ranges = p.ks;
    *blocks = p.blocks_per_range;
    return;
  }
  *rows = static_cast<uint32_t>(kRows[shape]);
  *cols = static_cast<uint32_t>(form == kFfnGated ? kBN[shape] / 2 : kBN[shape]);
  *ranges = 1;
  *blocks = static_cast<uint32_t>((static_cast<uint64_t>(k) + 63) / 64 * (form == kFfnDx ? pairs : 1));
}

int ffn_device_status(int* out) {
  *out = 0;
  TCAB_TRY_RC(ffn_small_status(out));
  for (int form = kFfnFwd; form <= kFfnDw; ++form)
    for (int act = TCAB_ACT_NONE; act <= TCAB_ACT_SIGMOID; ++act) {
      if (form >= kFfnDx && act != TCAB_ACT_NONE) continue;
      const FfnKernel k = kernel_of(form, act, 0);
      int one = 0;
      if (k.fn == nullptr) continue;
      if (k.status(&one) != cudaSuccess) {
        cudaGetLastError();
        return fail(TCAB_ERR_CUDA, "device_status: cannot read a status word");
      }
      if (one != 0) *out = one;
    }
  return TCAB_OK;
}

int launch_ffn_gemm(const char* op, int form, const FfnProblem& p, cudaStream_t s, FfnTaken* taken) {
  if (p.M == 0 || p.N == 0) return TCAB_OK;
  const Tune& tn = tune(kFfn);
  const uint32_t pairs = p.b[1] != nullptr ? 2 : 1;
  int sms = sm_count();
  Choice choice = choose(form, p.M, p.N, p.K, pairs, sms);
  if (p.beside && p.taken > 0 && p.taken < static_cast<uint32_t>(sms)) {
    // After the launch beside it with all SMs (some 2 us of its start are hidden), or with it on those that it leaves.
    // Backward passes, us: 800 x 768 x 2048 19.6 after, 15.7 with it; 200 x 1024 x 4096 17.0, 13.5; 515 x 1032 x 2056 20.8,
    // 19.9 with 256 x 256 tiles and 21.9 with 128 x 128, whose operand tiles both kernels then draw from L2.
    const int rest = sms - static_cast<int>(p.taken);
    const Choice alone = choose(form, p.M, p.N, p.K, pairs, rest, true);
    if ((alone.us > p.taken_us ? alone.us : p.taken_us) < p.taken_us + choice.us - 2.0) {
      choice = alone;
      sms = rest;
    }
  }
  if (taken != nullptr) *taken = {choice.ctas, choice.us};
  const int shape = tn.p1 > 0 && tn.p1 <= kShapes + 1 ? tn.p1 - 1 : choice.shape;
  if (shape == kShapes) return launch_ffn_small(op, form, p, sms, s);
  const uint32_t ctas = kCtas[shape], bm = kRows[shape], bn = kBN[shape], tile_n = form == kFfnGated ? bn / 2 : bn;
  FfnArgs args = {};
  args.M = p.M;
  args.N = p.N;
  args.K = p.K;
  args.pairs = pairs;
  args.bias[0] = p.bias[0];
  args.bias[1] = p.bias[1];
  args.residual = p.residual;
  args.save = p.z[0] != nullptr ? 1 : 0;
  args.beside = p.beside ? 1 : 0;
  const int nb = static_cast<int>(pairs);
  if (p.K > 0) {
    if (form == kFfnDw) {
      TCAB_TRY_RC(make_tensor_map(op, &args.a[0], p.a[0], p.K, p.M, 64, 64));
    } else {
      TCAB_TRY_RC(make_tensor_map(op, &args.a[0], p.a[0], p.M, p.K, 128, 64));
      if (form == kFfnDx && nb == 2) TCAB_TRY_RC(make_tensor_map(op, &args.a[1], p.a[1], p.M, p.K, 128, 64));
    }
    for (int i = 0; i < nb; ++i) {
      if (form == kFfnDx) TCAB_TRY_RC(make_tensor_map(op, &args.b[i], p.b[i], p.N, p.K, bn / ctas, 64));
      else TCAB_TRY_RC(make_tensor_map(op, &args.b[i], p.b[i], p.K, p.N, 64, 64));
    }
  }
  for (int i = 0; i < 2; ++i) {
    args.c[i] = p.c[i];
    args.z[i] = p.z[i];
  }
  const FfnKernel k = kernel_of(form, p.act, shape);
  if (k.fn == nullptr) return fail(TCAB_ERR_UNSUPPORTED, "%s: no kernel for activation %d", op, p.act);
  TCAB_TRY_RC(reserve_smem(op, k.fn, k.smem));
  const uint64_t tiles = static_cast<uint64_t>((p.M + bm - 1) / bm) * ((p.N + tile_n - 1) / tile_n) * (form == kFfnDw ? nb : 1);
  uint64_t groups = (tn.p0 > 0 ? static_cast<uint64_t>(tn.p0) : static_cast<uint64_t>(sms)) / ctas;
  if (groups > tiles) groups = tiles;
  if (groups < 1) groups = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(groups * ctas));
  cfg.blockDim = dim3(kFfnThreads);
  cfg.dynamicSmemBytes = k.smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = ctas;
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
