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

// The tile shape: fewest rounds over the SMs (pairs of SMs), weighted by what a round of each shape costs.
int pick_shape(int form, const FfnProblem& p) {
  static const double kCost[kShapes] = {1.0, 0.55, 0.36};  // of a round of one tile per CTA or pair
  const uint64_t sms = static_cast<uint64_t>(sm_count()), outs = form == kFfnDw && p.b[1] != nullptr ? 2 : 1;
  int best = 0;
  double best_cost = 1e300;
  for (int s = 0; s < kShapes; ++s) {
    const uint64_t bm = kRows[s], tn = static_cast<uint64_t>(form == kFfnGated ? kBN[s] / 2 : kBN[s]);
    const uint64_t tiles = (p.M + bm - 1) / bm * ((p.N + tn - 1) / tn) * outs, at_once = sms / kCtas[s];
    if (at_once == 0) continue;
    const double cost = static_cast<double>((tiles + at_once - 1) / at_once) * kCost[s];
    if (cost < best_cost - 1e-9) {
      best_cost = cost;
      best = s;
    }
  }
  return best;
}

}  // namespace

int ffn_device_status(int* out) {
  *out = 0;
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

int launch_ffn_gemm(const char* op, int form, const FfnProblem& p, cudaStream_t s) {
  if (p.M == 0 || p.N == 0) return TCAB_OK;
  const Tune& tn = tune(kFfn);
  const int shape = tn.p1 > 0 && tn.p1 <= kShapes ? tn.p1 - 1 : pick_shape(form, p);
  const uint32_t ctas = kCtas[shape], bm = kRows[shape], bn = kBN[shape], tile_n = form == kFfnGated ? bn / 2 : bn;
  FfnArgs args = {};
  args.M = p.M;
  args.N = p.N;
  args.K = p.K;
  args.pairs = p.b[1] != nullptr ? 2 : 1;
  args.bias[0] = p.bias[0];
  args.bias[1] = p.bias[1];
  args.residual = p.residual;
  args.save = p.z[0] != nullptr ? 1 : 0;
  const int nb = p.b[1] != nullptr ? 2 : 1;
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
  const int nc = form == kFfnDw ? nb : 1;
  for (int i = 0; i < nc; ++i) TCAB_TRY_RC(make_tensor_map(op, &args.c[i], p.c[i], p.M, p.N, 32, 32));
  for (int i = 0; i < 2; ++i)
    if (p.z[i] != nullptr) TCAB_TRY_RC(make_tensor_map(op, &args.z[i], p.z[i], p.M, p.N, 32, 32));

  const FfnKernel k = kernel_of(form, p.act, shape);
  if (k.fn == nullptr) return fail(TCAB_ERR_UNSUPPORTED, "%s: no kernel for activation %d", op, p.act);
  const cudaError_t ae = cudaFuncSetAttribute(k.fn, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(k.smem));
  if (ae != cudaSuccess) {
    cudaGetLastError();
    return fail(TCAB_ERR_CUDA, "%s: cannot reserve %zu bytes of shared memory: %s", op, k.smem, cudaGetErrorString(ae));
  }
  const uint64_t tiles = static_cast<uint64_t>((p.M + bm - 1) / bm) * ((p.N + tile_n - 1) / tile_n) * (form == kFfnDw ? nb : 1);
  uint64_t groups = (tn.p0 > 0 ? static_cast<uint64_t>(tn.p0) : static_cast<uint64_t>(sm_count())) / ctas;
  if (groups > tiles) groups = tiles;
  if (groups < 1) groups = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(groups * ctas));
  cfg.blockDim = dim3(kFfnThreads);
  cfg.dynamicSmemBytes = k.smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = ctas;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
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
