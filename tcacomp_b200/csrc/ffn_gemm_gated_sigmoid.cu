// ffn_gemm_gated_sigmoid.cu -- ffn_gemm_kernel, form kFfnGated, activation sigmoid (one translation unit per instance: they
// compile side by side).
#include "ffn_gemm.cuh"

namespace tcab {
FfnKernel ffn_kernel_gated_sigmoid(int shape) { return ffn_kernel_of<kFfnGated, TCAB_ACT_SIGMOID>(shape); }
}  // namespace tcab
