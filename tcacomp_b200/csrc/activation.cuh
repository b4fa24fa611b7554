// activation.cuh -- the activations of the contraction epilogues and their slopes, in fp32.
//
//   relu       max(z, 0)                               slope z > 0 (0 at z = 0)
//   silu       z s,  s = 1 / (1 + exp(-z))             s (1 + z (1 - s))
//   sigmoid    s                                       s (1 - s)
//   gelu       z Phi(z), Phi the normal distribution   Phi(z) + z phi(z)
//   gelu_tanh  z (1 + tanh v) / 2 = z / (1 + exp(-2 v)),  v = sqrt(2 / pi) (z + 0.044715 z^3)
//                                                      s + z s (1 - s) 2 v',  s = 1 / (1 + exp(-2 v))
//
// exp is the hardware's exp2 with the argument scaled in fp32 (relative error about 2^-22 + |z| 2^-24) and the quotient
// a reciprocal (2 ulp): every result is rounded to bf16's 8 bits afterwards or summed in fp32 over many rows. The
// logistic form of gelu_tanh is the same function as the tanh form and costs one exp2 and one reciprocal.
#pragma once

#include "common.cuh"

#ifdef __CUDACC__
namespace tcab {

__device__ __forceinline__ float logistic(float z) { return __fdividef(1.0f, 1.0f + __expf(-z)); }
__device__ __forceinline__ float normal_cdf(float z) { return 0.5f + 0.5f * erff(z * 0.70710678118654752f); }

template <int ACT>
__device__ __forceinline__ float act_value(float z) {
  if constexpr (ACT == TCAB_ACT_RELU) return z <= 0.0f ? 0.0f : z;  // a NaN stays a NaN
  if constexpr (ACT == TCAB_ACT_SILU) return z * logistic(z);
  if constexpr (ACT == TCAB_ACT_SIGMOID) return logistic(z);
  if constexpr (ACT == TCAB_ACT_GELU) return z * normal_cdf(z);
  if constexpr (ACT == TCAB_ACT_GELU_TANH) return z * logistic(1.5957691216057308f * (z + 0.044715f * z * z * z));
  return z;
}

// value and slope together: the gated backward pass needs both
template <int ACT>
__device__ __forceinline__ void act_value_slope(float z, float* value, float* slope) {
  if constexpr (ACT == TCAB_ACT_RELU) {
    *value = act_value<ACT>(z);
    *slope = z > 0.0f ? 1.0f : 0.0f;
  } else if constexpr (ACT == TCAB_ACT_SILU) {
    const float s = logistic(z);
    *value = z * s;
    *slope = s + z * s * (1.0f - s);
  } else if constexpr (ACT == TCAB_ACT_SIGMOID) {
    const float s = logistic(z);
    *value = s;
    *slope = s * (1.0f - s);
  } else if constexpr (ACT == TCAB_ACT_GELU) {
    const float p = normal_cdf(z);
    *value = z * p;
    *slope = p + z * 0.3989422804014327f * __expf(-0.5f * z * z);
  } else if constexpr (ACT == TCAB_ACT_GELU_TANH) {
    const float z2 = fminf(z * z, 1e6f);  // s is 0 or 1 long before: keeps 0 * inf out of the second term
    const float s = logistic(1.5957691216057308f * z * (1.0f + 0.044715f * z2));
    *value = z * s;
    *slope = s + z * s * (1.0f - s) * (1.5957691216057308f * (1.0f + 0.134145f * z2));
  } else {
    *value = z;
    *slope = 1.0f;
  }
}

}  // namespace tcab
#endif
