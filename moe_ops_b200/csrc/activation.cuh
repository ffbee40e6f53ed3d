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

// FAST: for values that are rounded to 16 bits next: the hardware's exponential, reciprocal and a
// fitted normal distribution, with a relative error below 2^-15 (most of it the rounding of the
// exponential's argument, up to 100), an eighth of half a step of fp16.  (CUDA's erff, expf and IEEE
// division took 100 us of the 8192 x 4096 x 11008 product's epilogue.)
template <bool FAST>
__device__ __forceinline__ float exp_of(float v) { return FAST ? __expf(v) : expf(v); }
// 1 / v for v >= 1.  FAST: within one unit in the last place, without __fdividef's scaling of other v.
template <bool FAST>
__device__ __forceinline__ float reciprocal(float v) {
  if constexpr (!FAST) return 1.f / v;
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}

// 1 / (1 + exp(-v)) and its derivative, through an exponential that cannot overflow and without a
// difference: both keep their relative accuracy where they are small.
struct Logistic {
  float s, ds;
};
template <bool FAST>
__device__ __forceinline__ Logistic logistic(float v) {
  const float e = exp_of<FAST>(-fabsf(v));
  const float r = reciprocal<FAST>(1.f + e);
  return {r * (v < 0.f ? e : 1.f), e * r * r};
}

// The normal distribution function Phi.  FAST: Phi(-a) = t P(t) exp(-a^2 / 2), t = 1 / (1 + 0.35 a),
// with P of degree 6 fitted here (iterated weighted least squares over 0 <= a <= 14.5) so that Phi is
// off by at most 2^-24 absolutely and 2^-17 relatively.
template <bool FAST>
__device__ __forceinline__ float normal_cdf(float z) {
  if constexpr (!FAST) return normcdff(z);
  const float t = reciprocal<true>(fmaf(0.35f, fabsf(z), 1.f));
  float p = fmaf(0.044112293f, t, -0.182377315f);
  p = fmaf(p, t, 0.207723782f);
  p = fmaf(p, t, 0.011725331f);
  p = fmaf(p, t, 0.141921700f);
  p = fmaf(p, t, 0.137139676f);
  p = fmaf(p, t, 0.139754564f);
  const float tail = p * t * __expf(-0.5f * z * z);
  return z > 0.f ? 1.f - tail : tail;
}

constexpr float kGeluTanh = 1.59576912f;  // 2 sqrt(2 / pi): (1 + tanh(u)) / 2 = 1 / (1 + exp(-2u))

template <int ACT, bool FAST>
__device__ __forceinline__ float act_fwd(float z) {
  if constexpr (ACT == MOE_ACT_RELU) return z > 0.f ? z : (z != z ? z : 0.f);
  if constexpr (ACT == MOE_ACT_GELU) return z * normal_cdf<FAST>(z);
  if constexpr (ACT == MOE_ACT_GELU_TANH || ACT == MOE_ACT_SILU)
    return z * logistic<FAST>(ACT == MOE_ACT_SILU ? z : kGeluTanh * (z + 0.044715f * z * z * z)).s;
  return z;
}

// At z = +-infinity the derivatives take their limits, 1 and 0: the factor z beside an exponential
// is bounded where that exponential is 0 (from |z| = 104 on, 14 for gelu).
template <int ACT, bool FAST>
__device__ __forceinline__ float act_bwd(float z) {
  const float zc = fminf(fmaxf(z, -128.f), 128.f);
  if constexpr (ACT == MOE_ACT_RELU) return z > 0.f ? 1.f : (z != z ? z : 0.f);
  if constexpr (ACT == MOE_ACT_GELU)
    return normal_cdf<FAST>(z) + zc * (exp_of<FAST>(-0.5f * z * z) * 0.39894228f);
  if constexpr (ACT == MOE_ACT_GELU_TANH) {
    const Logistic l = logistic<FAST>(kGeluTanh * (z + 0.044715f * z * z * z));
    return fmaf(l.ds, kGeluTanh * zc * (1.f + 0.134145f * zc * zc), l.s);
  }
  if constexpr (ACT == MOE_ACT_SILU) {
    const Logistic l = logistic<FAST>(z);
    return fmaf(l.ds, zc, l.s);
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
