// ffn_gemm_gated_relu.cu -- ffn_gemm_kernel, form kFfnGated, activation relu (one translation unit per instance: they
// compile side by side).
#include "ffn_gemm.cuh"

namespace tcab {
FfnKernel ffn_kernel_gated_relu(int shape) { return ffn_kernel_of<kFfnGated, TCAB_ACT_RELU>(shape); }
}  // namespace tcab
