// f32x2.cuh -- two fp32 values per register pair: sm_100 multiplies and adds them with one instruction (FFMA2), each half
// rounded like the scalar operation. For kernels whose limit is the issue rate rather than memory.
#pragma once

#include "common.cuh"

#ifdef __CUDACC__
namespace tcab {

using f32x2 = float2;

__device__ __forceinline__ f32x2 pair_of(float lo, float hi) { return make_float2(lo, hi); }
__device__ __forceinline__ void pair_to(f32x2 p, float& lo, float& hi) {
  lo = p.x;
  hi = p.y;
}
__device__ __forceinline__ float pair_sum(f32x2 p) { return p.x + p.y; }
__device__ __forceinline__ f32x2 fma_pair(f32x2 a, f32x2 b, f32x2 c) { return __ffma2_rn(a, b, c); }
__device__ __forceinline__ f32x2 mul_pair(f32x2 a, f32x2 b) { return __fmul2_rn(a, b); }
__device__ __forceinline__ f32x2 add_pair(f32x2 a, f32x2 b) { return __fadd2_rn(a, b); }

// the same operations on one value, for kernels that handle both
__device__ __forceinline__ float fma_pair(float a, float b, float c) { return fmaf(a, b, c); }
__device__ __forceinline__ float mul_pair(float a, float b) { return a * b; }
__device__ __forceinline__ float add_pair(float a, float b) { return a + b; }
__device__ __forceinline__ float pair_sum(float a) { return a; }
template <typename Num>
__device__ __forceinline__ Num spread(float v);
template <>
__device__ __forceinline__ float spread<float>(float v) { return v; }
template <>
__device__ __forceinline__ f32x2 spread<f32x2>(float v) { return pair_of(v, v); }
// two bf16 values in a word, widened / rounded to nearest even
__device__ __forceinline__ f32x2 pair_of_bf16(uint32_t w) { return pair_of(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u)); }
__device__ __forceinline__ uint32_t bf16_of_pair(f32x2 p) {
  float lo, hi;
  pair_to(p, lo, hi);
  const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// The special-function unit's exp2 and reciprocal (2 ulp); subnormal arguments and results are zero.
__device__ __forceinline__ float exp2_hw(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float rcp_hw(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

}  // namespace tcab
#endif
