// ffn_gemm_fwd_relu.cu -- ffn_gemm_kernel, form kFfnFwd, activation relu (one translation unit per instance: they
// compile side by side).
#include "ffn_gemm.cuh"

namespace tcab {
FfnKernel ffn_kernel_fwd_relu(int shape) { return ffn_kernel_of<kFfnFwd, TCAB_ACT_RELU>(shape); }
}  // namespace tcab
