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

// Wide accesses whose address need only be aligned to one element (rows of an
// odd width): the compiler makes one access of each, which global memory takes
// at any address on gfx950.
template <class E, int N>
struct __attribute__((packed, aligned(sizeof(E)))) AnyWords { uint32_t v[N]; };

template <class E, int N>
__device__ __forceinline__ AnyWords<E, N> load_words(const E* p) {
  return *reinterpret_cast<const AnyWords<E, N>*>(p);
}
template <class E, int N>
__device__ __forceinline__ void store_words(E* p, AnyWords<E, N> w) {
  *reinterpret_cast<AnyWords<E, N>*>(p) = w;
}

// A 16-byte chunk of a row of which `n` elements are left: whole, or the row's
// tail (the rest read as 0) in at most one access of each power of two.
__device__ __forceinline__ uint4 load_chunk16(const uint16_t* p, int64_t n) {
  if (n >= 8) {
    const auto u = load_words<uint16_t, 4>(p);
    return make_uint4(u.v[0], u.v[1], u.v[2], u.v[3]);
  }
  const int k = n > 0 ? (int)n : 0;
  uint32_t a0 = 0u, a1 = 0u, b = 0u, c = 0u;
  if (k & 4) {
    const auto u = load_words<uint16_t, 2>(p);
    a0 = u.v[0], a1 = u.v[1];
  }
  if (k & 2) b = load_words<uint16_t, 1>(p + (k & 4)).v[0];
  if (k & 1) c = p[k & 6];
  const uint32_t bc = k & 2 ? b : c, cz = k & 2 ? c : 0u;   // the words after the four
  return k & 4 ? make_uint4(a0, a1, bc, cz) : make_uint4(bc, cz, 0u, 0u);
}
__device__ __forceinline__ void store_chunk16(uint16_t* p, int64_t n, uint4 v) {
  if (n >= 8) {
    store_words<uint16_t, 4>(p, {{v.x, v.y, v.z, v.w}});
    return;
  }
  const int k = n > 0 ? (int)n : 0;
  uint32_t bc = v.x, cz = v.y;
  if (k & 4) {
    store_words<uint16_t, 2>(p, {{v.x, v.y}});
    bc = v.z, cz = v.w;
  }
  if (k & 2) store_words<uint16_t, 1>(p + (k & 4), {{bc}});
  if (k & 1) p[k & 6] = (uint16_t)(k & 2 ? cz : bc);
}
// 8 bytes of a row of which `n` are left.
__device__ __forceinline__ uint2 load_chunk8(const uint8_t* p, int64_t n) {
  if (n >= 8) {
    const auto u = load_words<uint8_t, 2>(p);
    return make_uint2(u.v[0], u.v[1]);
  }
  const int k = n > 0 ? (int)n : 0;
  uint32_t a = 0u, t = 0u;   // the first four, and what follows them
  if (k & 4) a = load_words<uint8_t, 1>(p).v[0];
  const uint8_t* q = p + (k & 4);
  for (int e = 0; e < (k & 3); ++e) t |= (uint32_t)q[e] << (8 * e);
  return k & 4 ? make_uint2(a, t) : make_uint2(t, 0u);
}
__device__ __forceinline__ void store_chunk8(uint8_t* p, int64_t n, uint2 v) {
  if (n >= 8) {
    store_words<uint8_t, 2>(p, {{v.x, v.y}});
    return;
  }
  const int k = n > 0 ? (int)n : 0;
  uint32_t t = v.x;
  if (k & 4) {
    store_words<uint8_t, 1>(p, {{v.x}});
    t = v.y;
  }
  uint8_t* q = p + (k & 4);
  for (int e = 0; e < (k & 3); ++e) q[e] = (uint8_t)(t >> (8 * e));
}
__device__ __forceinline__ float4 load_chunk32(const float* p, int64_t n) {
  float4 f = make_float4(0.f, 0.f, 0.f, 0.f);
  if (n >= 4) {
    const auto u = load_words<float, 4>(p);
    return make_float4(__uint_as_float(u.v[0]), __uint_as_float(u.v[1]), __uint_as_float(u.v[2]),
                       __uint_as_float(u.v[3]));
  }
  if (n > 0) f.x = p[0];
  if (n > 1) f.y = p[1];
  if (n > 2) f.z = p[2];
  return f;
}
__device__ __forceinline__ void store_chunk32(float* p, int64_t n, float4 f) {
  if (n >= 4) {
    store_words<float, 4>(p, {{__float_as_uint(f.x), __float_as_uint(f.y), __float_as_uint(f.z),
                               __float_as_uint(f.w)}});
    return;
  }
  if (n > 0) p[0] = f.x;
  if (n > 1) p[1] = f.y;
  if (n > 2) p[2] = f.z;
}

}  // namespace dc
