// Activations of the linear operators' epilogues and their derivatives, in fp32.
//
//   relu       max(z, 0)
//   gelu       z * Phi(z),  Phi(z) = (1 + erf(z / sqrt(2))) / 2
//   gelu_tanh  z * (1 + tanh(a * (z + 0.044715 z^3))) / 2,  a = sqrt(2 / pi)
//   silu       z / (1 + exp(-z))
#pragma once

#include "common.cuh"
#include "swiglu.cuh"

namespace moe {

// tanh through one exponential of a non-positive argument (it cannot overflow); near 0 its
// absolute error is of the order of 2^-24, which is all that 1 + tanh needs.
__device__ __forceinline__ float tanh_exp(float u) {
  const float t = expf(-2.f * fabsf(u));
  return copysignf((1.f - t) / (1.f + t), u);
}

// The normal distribution function by Abramowitz and Stegun's formula 7.1.26 for erf (absolute
// error below 1.5e-7), with the hardware's exponential.
__device__ __forceinline__ float normal_cdf_fast(float z) {
  const float x = fabsf(z) * 0.70710678f;
  const float t = __fdividef(1.f, fmaf(0.3275911f, x, 1.f));
  float p = fmaf(1.061405429f, t, -1.453152027f);
  p = fmaf(p, t, 1.421413741f);
  p = fmaf(p, t, -0.284496736f);
  p = fmaf(p, t, 0.254829592f);
  const float tail = 0.5f * p * t * __expf(-0.5f * z * z);
  return z > 0.f ? 1.f - tail : tail;
}

// FAST: for values that are rounded to 16 bits next.  The hardware's exponential and division, whose
// errors (a few 2^-22 here) lie far below half a step of fp16 (2^-12): CUDA's erff, expf and IEEE
// division took 100 us of the 8192 x 4096 x 11008 product's epilogue.
template <int ACT, bool FAST>
__device__ __forceinline__ float act_fwd(float z) {
  if constexpr (ACT == MOE_ACT_RELU) return z > 0.f ? z : (z != z ? z : 0.f);
  if constexpr (FAST) {
    if constexpr (ACT == MOE_ACT_GELU) return z * normal_cdf_fast(z);
    // (1 + tanh(u)) / 2 = 1 / (1 + exp(-2u))
    if constexpr (ACT == MOE_ACT_GELU_TANH)
      return __fdividef(z, 1.f + __expf(-1.59576912f * (z + 0.044715f * z * z * z)));
    if constexpr (ACT == MOE_ACT_SILU) return __fdividef(z, 1.f + __expf(-z));
  } else {
    if constexpr (ACT == MOE_ACT_GELU) return 0.5f * z * (1.f + erff(z * 0.70710678f));
    if constexpr (ACT == MOE_ACT_GELU_TANH)
      return 0.5f * z * (1.f + tanh_exp(0.79788456f * (z + 0.044715f * z * z * z)));
    if constexpr (ACT == MOE_ACT_SILU) return z * sigmoid_f32(z);
  }
  return z;
}

template <int ACT, bool FAST>
__device__ __forceinline__ float act_bwd(float z) {
  if constexpr (ACT == MOE_ACT_RELU) return z > 0.f ? 1.f : (z != z ? z : 0.f);
  if constexpr (ACT == MOE_ACT_GELU) {
    if constexpr (FAST) return normal_cdf_fast(z) + z * (__expf(-0.5f * z * z) * 0.39894228f);
    return 0.5f * (1.f + erff(z * 0.70710678f)) + z * (expf(-0.5f * z * z) * 0.39894228f);
  }
  if constexpr (ACT == MOE_ACT_GELU_TANH) {
    const float u = 0.79788456f * (z + 0.044715f * z * z * z);
    const float half = FAST ? __fdividef(1.f, 1.f + __expf(-2.f * u)) : 0.5f * (1.f + tanh_exp(u));
    // beyond |z| = 8 the second term is below 2^-24 of the first and z^2 may overflow
    const float zc = fminf(fmaxf(z, -8.f), 8.f);
    return half + 2.f * zc * half * (1.f - half) * 0.79788456f * (1.f + 0.134145f * zc * zc);
  }
  if constexpr (ACT == MOE_ACT_SILU) {
    const float s = FAST ? __fdividef(1.f, 1.f + __expf(-z)) : sigmoid_f32(z);
    // s is 0 far below -100; the bound keeps 0 * inf out at z = -inf
    return s * (1.f + fmaxf(z, -100.f) * (1.f - s));
  }
  return 1.f;
}

// Runs the statements with the activation code as a compile-time constant ACT.
#define MOE_SWITCH_ACT(code, ACT, ...)                                        \
  switch (code) {                                                             \
    case MOE_ACT_RELU: { constexpr int ACT = MOE_ACT_RELU; __VA_ARGS__; break; }           \
    case MOE_ACT_GELU: { constexpr int ACT = MOE_ACT_GELU; __VA_ARGS__; break; }           \
    case MOE_ACT_GELU_TANH: { constexpr int ACT = MOE_ACT_GELU_TANH; __VA_ARGS__; break; } \
    case MOE_ACT_SILU: { constexpr int ACT = MOE_ACT_SILU; __VA_ARGS__; break; }           \
    default: { constexpr int ACT = MOE_ACT_NONE; __VA_ARGS__; break; }                     \
  }

template <bool FAST>
__device__ __forceinline__ float act_fwd_rt(int act, float z) {
  MOE_SWITCH_ACT(act, A, return (act_fwd<A, FAST>(z)));
  return z;
}

}  // namespace moe
