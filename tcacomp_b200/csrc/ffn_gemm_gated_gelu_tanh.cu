// ffn_gemm_gated_gelu_tanh.cu -- ffn_gemm_kernel, form kFfnGated, activation gelu_tanh (one translation unit per instance: they
// compile side by side).
#include "ffn_gemm.cuh"

namespace tcab {
FfnKernel ffn_kernel_gated_gelu_tanh(int shape) { return ffn_kernel_of<kFfnGated, TCAB_ACT_GELU_TANH>(shape); }
}  // namespace tcab
