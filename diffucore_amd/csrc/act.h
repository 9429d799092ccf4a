// Activations and their slopes in float32, shared by the passes that apply
// them.
#pragma once

#include "common.h"

namespace dc {

// Two forms of GELU, without the cancellation the textbook forms have in the
// negative tail, with the hardware exp2 / reciprocal (the passes that run them
// are VALU-bound, and the library erf / tanh cost about twice as much):
//   tanh form: 0.5 x (1 + tanh u) = x / (1 + 2^(-2 u log2 e)), u = sqrt(2 / pi)
//   (x + 0.044715 x^3);
//   erf form: 1 + erf(x / sqrt 2) = erfc(z) for x < 0, 2 - erfc(z) for x >= 0,
//   z = |x| / sqrt 2, erfc by the Chebyshev-fitted form of Press et al.,
//   Numerical Recipes (2nd ed., section 6.2, erfcc): t = 1 / (1 + z / 2),
//   erfc(z) = t exp(-z^2 - 1.26551223 + t P(t)) with P of degree 9, whose
//   relative error is below 1.2e-7 for every z >= 0.
// Both keep a small relative error over the whole line.
constexpr float LOG2E = 1.4426950408889634f;

// The constants of u, log2 e, the 1 / sqrt 2 of z and the 0.5 are folded into
// the coefficients: x * x is exact in float32 for a 16-bit x, so both forms
// round less often than with z and u written out. Largest relative error over
// all finite 16-bit |x| < 10 with exact exp2 / reciprocal, before -> now: tanh
// form 1.0e-5 -> 6.3e-6, erf form 7.5e-6 -> 3.3e-6 (both in the far negative
// tail; 1.7e-6 -> 1.4e-6 and 2.2e-6 -> 9e-7 for |x| < 5).
//
// -2 u log2 e = x (A + B x^2), A = -2 log2 e sqrt(2 / pi) and B = 0.044715 A each rounded once
constexpr float GELU_TANH_A = -2.302208198144325f, GELU_TANH_B = -0.1029432395800235f;

__device__ __forceinline__ float gelu_tanh_f32(float x) {
  return x * __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(x * __builtin_fmaf(x * x, GELU_TANH_B, GELU_TANH_A)));
}

// erfc(|x| / sqrt 2) / 2, the normal distribution's tail beyond |x|
__device__ __forceinline__ float normal_tail(float x) {
  // t 2^(log2 e (-z^2 - 1.26551223 + t P(t)) - 1), z^2 = x^2 / 2
  const float t = __builtin_amdgcn_rcpf(__builtin_fmaf(0.5f * 0.7071067811865476f, fabsf(x), 1.0f));
  float p = __builtin_fmaf(0.17087277f * LOG2E, t, -0.82215223f * LOG2E);
  p = __builtin_fmaf(p, t, 1.48851587f * LOG2E);
  p = __builtin_fmaf(p, t, -1.13520398f * LOG2E);
  p = __builtin_fmaf(p, t, 0.27886807f * LOG2E);
  p = __builtin_fmaf(p, t, -0.18628806f * LOG2E);
  p = __builtin_fmaf(p, t, 0.09678418f * LOG2E);
  p = __builtin_fmaf(p, t, 0.37409196f * LOG2E);
  p = __builtin_fmaf(p, t, 1.00002368f * LOG2E);
  p = __builtin_fmaf(p, t, -1.26551223f * LOG2E - 1.0f);
  return t * __builtin_amdgcn_exp2f(__builtin_fmaf(x * x, -0.5f * LOG2E, p));
}

__device__ __forceinline__ float gelu_erf_f32(float x) {
  const float h = normal_tail(x);
  // the float's sign, not the 16-bit input's: comparing that would keep the
  // packed inputs live to the end (fp16: 58 VGPRs, 8 waves per SIMD; 68 and 7)
  x = materialize(x);
  return x * (x < 0.0f ? h : 1.0f - h);
}

// s = 1 / (1 + 2^e), the gate of the sigmoid-shaped activations (x s), with e
// = x (A + B x^2) for the tanh form of GELU and e = -q log2(e) x else (q = 1
// SiLU, q = 1.702 the sigmoid approximation of GELU).
template <int ACT>
__device__ __forceinline__ float sigmoid_gate(float x) {
  float e;
  if constexpr (ACT == DC_ACT_GELU_TANH) e = x * __builtin_fmaf(x * x, GELU_TANH_B, GELU_TANH_A);
  else if constexpr (ACT == DC_ACT_QUICK_GELU) e = x * (-1.702f * LOG2E);
  else e = x * -LOG2E;
  return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(e));
}

// ACT(x).
template <int ACT>
__device__ __forceinline__ float act_value(float x) {
  if constexpr (ACT == DC_ACT_NONE) return x;
  else if constexpr (ACT == DC_ACT_GELU_ERF) return gelu_erf_f32(x);
  else return x * sigmoid_gate<ACT>(x);
}

// ACT(x) and its slope at x:
//   erf form     Phi(x) + x phi(x)
//   x s(x)       s + x s (1 - s) d,  d = -e'(x) ln 2
// At |x| = 128 phi and s (or 1 - s) have underflowed to 0, so every slope is 0
// or 1: x is held there, as x phi(x) and x s (1 - s) d turn into inf * 0 further
// out (NaN stays NaN).
template <int ACT>
__device__ __forceinline__ float act_slope(float x, float& value) {
  if constexpr (ACT == DC_ACT_NONE) {
    value = x;
    return 1.0f;
  } else {
    const float c = x > 128.0f ? 128.0f : x < -128.0f ? -128.0f : x;
    if constexpr (ACT == DC_ACT_GELU_ERF) {
      const float h = normal_tail(c), cdf = c < 0.0f ? h : 1.0f - h;
      value = (x > c ? x : c) * cdf;
      return __builtin_fmaf(c * 0.3989422804014327f, __builtin_amdgcn_exp2f(c * c * (-0.5f * LOG2E)), cdf);
    } else {
      const float s = sigmoid_gate<ACT>(c);
      constexpr float LN2 = 0.6931471805599453f;
      float d;
      if constexpr (ACT == DC_ACT_GELU_TANH) d = __builtin_fmaf(c * c, -3.0f * LN2 * GELU_TANH_B, -LN2 * GELU_TANH_A);
      else d = ACT == DC_ACT_QUICK_GELU ? 1.702f : 1.0f;
      value = (x > c ? x : c) * s;
      return __builtin_fmaf(c * s * (1.0f - s), d, s);
    }
  }
}

// f(std::integral_constant<int, ACT>{}) for a runtime activation: one uniform
// branch around code that is compiled for each.
template <class F>
__device__ __forceinline__ void with_act(int act, F&& f) {
  switch (act) {
    case DC_ACT_GELU_ERF: f(std::integral_constant<int, DC_ACT_GELU_ERF>{}); break;
    case DC_ACT_GELU_TANH: f(std::integral_constant<int, DC_ACT_GELU_TANH>{}); break;
    case DC_ACT_SILU: f(std::integral_constant<int, DC_ACT_SILU>{}); break;
    case DC_ACT_QUICK_GELU: f(std::integral_constant<int, DC_ACT_QUICK_GELU>{}); break;
    default: f(std::integral_constant<int, DC_ACT_NONE>{}); break;
  }
}

// ---------------------------------------------------------------- unaligned vectors

// N consecutive 16-bit or 32-bit values whose address need only be aligned to
// one element (rows of an odd width): the compiler still makes one wide access
// of it, which global memory takes at any address on gfx950.
struct __attribute__((packed, aligned(2))) U16x8 { uint32_t v[4]; };
struct __attribute__((packed, aligned(4))) U32x4 { uint32_t v[4]; };

__device__ __forceinline__ uint4 load16_any(const uint16_t* p) {
  const U16x8 u = *reinterpret_cast<const U16x8*>(p);
  return make_uint4(u.v[0], u.v[1], u.v[2], u.v[3]);
}
__device__ __forceinline__ void store16_any(uint16_t* p, uint4 v) {
  U16x8 u;
  u.v[0] = v.x, u.v[1] = v.y, u.v[2] = v.z, u.v[3] = v.w;
  *reinterpret_cast<U16x8*>(p) = u;
}

}  // namespace dc
