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
//
// Phi: the upper tail of the normal distribution is Q(x) = exp(-x^2 / 2) t (b1 + t (b2 + t (b3 + t (b4 + t b5)))) with
// t = 1 / (1 + 0.2316419 x), x >= 0 (Abramowitz and Stegun, Handbook of Mathematical Functions, 26.2.17, with
// 1 / sqrt(2 pi) taken into the coefficients): absolute error below 7.5e-8, about what an fp32 erf leaves of 1 + erf. The
// tail form keeps gelu(z) = max(z, 0) - |z| Q(|z|) free of cancellation on the negative side, and its exponential is the
// density that the slope needs.
//
// Everything works on eight values at a time, step by step over all eight, multiply-adds two at a time (FFMA2): an
// epilogue has two warps per scheduler, so one value's chain of a reciprocal, an exp2 and a dozen multiply-adds has to
// overlap with its neighbours'. An 8192^3 product with gelu (TFLOP/s): one value after the other with erff 1,090, with
// the tail form 1,250, eight at a time 1,360; without an activation 1,400-1,435.
#pragma once

#include "f32x2.cuh"

#ifdef __CUDACC__
namespace tcab {

// s = 1 / (1 + exp(-z))
__device__ __forceinline__ void logistic8(const float (&z)[8], float (&s)[8]) {
  float e[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) e[j] = exp2_hw(-1.4426950408889634f * z[j]);
#pragma unroll
  for (int j = 0; j < 8; ++j) s[j] = rcp_hw(1.0f + e[j]);
}

// e = exp(-z^2 / 2), q = Q(|z|)
__device__ __forceinline__ void normal_tail8(const float (&z)[8], float (&e)[8], float (&q)[8]) {
  float t[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) t[j] = rcp_hw(fmaf(0.2316419f, fabsf(z[j]), 1.0f));
#pragma unroll
  for (int j = 0; j < 4; ++j) {  // -z^2 / 2 in units of ln 2
    const f32x2 zp = pair_of(z[2 * j], z[2 * j + 1]);
    pair_to(mul_pair(mul_pair(zp, spread<f32x2>(-0.7213475204444817f)), zp), e[2 * j], e[2 * j + 1]);
  }
#pragma unroll
  for (int j = 0; j < 8; ++j) e[j] = exp2_hw(e[j]);
  f32x2 tp[4], p[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    tp[j] = pair_of(t[2 * j], t[2 * j + 1]);
    p[j] = fma_pair(tp[j], spread<f32x2>(0.5307027143f), spread<f32x2>(-0.7265760131f));
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) p[j] = fma_pair(tp[j], p[j], spread<f32x2>(0.7107068707f));
#pragma unroll
  for (int j = 0; j < 4; ++j) p[j] = fma_pair(tp[j], p[j], spread<f32x2>(-0.1422483683f));
#pragma unroll
  for (int j = 0; j < 4; ++j) p[j] = fma_pair(tp[j], p[j], spread<f32x2>(0.1274147959f));
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    p[j] = mul_pair(p[j], mul_pair(tp[j], pair_of(e[2 * j], e[2 * j + 1])));
    pair_to(p[j], q[2 * j], q[2 * j + 1]);
  }
}

// gelu from the tail; the cap keeps infinity * 0 out of it
__device__ __forceinline__ float gelu_of_tail(float z, float q) { return fmaxf(z, 0.0f) - fminf(fabsf(z), 1e30f) * q; }

// v = act(v)
template <int ACT>
__device__ __forceinline__ void act_values(float (&v)[8]) {
  float s[8];
  if constexpr (ACT == TCAB_ACT_RELU) {
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = v[j] <= 0.0f ? 0.0f : v[j];  // a NaN stays a NaN
  } else if constexpr (ACT == TCAB_ACT_SILU || ACT == TCAB_ACT_SIGMOID) {
    logistic8(v, s);
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = ACT == TCAB_ACT_SILU ? v[j] * s[j] : s[j];
  } else if constexpr (ACT == TCAB_ACT_GELU) {
    float e[8];
    normal_tail8(v, e, s);
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = gelu_of_tail(v[j], s[j]);
  } else if constexpr (ACT == TCAB_ACT_GELU_TANH) {
    float u[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) u[j] = 1.5957691216057308f * v[j] * fmaf(0.044715f * v[j], v[j], 1.0f);
    logistic8(u, s);
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] *= s[j];
  }
}

// act(z) and act'(z) together: the gated backward pass needs both
template <int ACT>
__device__ __forceinline__ void act_values_slopes(const float (&z)[8], float (&value)[8], float (&slope)[8]) {
  float s[8];
  if constexpr (ACT == TCAB_ACT_RELU) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      value[j] = z[j] <= 0.0f ? 0.0f : z[j];
      slope[j] = z[j] > 0.0f ? 1.0f : 0.0f;
    }
  } else if constexpr (ACT == TCAB_ACT_SILU || ACT == TCAB_ACT_SIGMOID) {
    logistic8(z, s);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      value[j] = ACT == TCAB_ACT_SILU ? z[j] * s[j] : s[j];
      slope[j] = ACT == TCAB_ACT_SILU ? fmaf(z[j] * s[j], 1.0f - s[j], s[j]) : s[j] * (1.0f - s[j]);
    }
  } else if constexpr (ACT == TCAB_ACT_GELU) {
    float e[8];
    normal_tail8(z, e, s);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      value[j] = gelu_of_tail(z[j], s[j]);
      slope[j] = fmaf(z[j] * 0.3989422804014327f, e[j], z[j] < 0.0f ? s[j] : 1.0f - s[j]);
    }
  } else if constexpr (ACT == TCAB_ACT_GELU_TANH) {
    float u[8], z2[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      z2[j] = fminf(z[j] * z[j], 1e6f);  // s is 0 or 1 long before: keeps 0 * infinity out of the slope's second term
      u[j] = 1.5957691216057308f * z[j] * fmaf(0.044715f, z2[j], 1.0f);
    }
    logistic8(u, s);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      value[j] = z[j] * s[j];
      slope[j] = fmaf(value[j] * (1.0f - s[j]), 1.5957691216057308f * fmaf(0.134145f, z2[j], 1.0f), s[j]);
    }
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      value[j] = z[j];
      slope[j] = 1.0f;
    }
  }
}

}  // namespace tcab
#endif
