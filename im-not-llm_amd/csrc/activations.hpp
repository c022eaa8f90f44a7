// Activations and their derivatives in f32, from v_exp_f32 and v_rcp_f32 (an
// ulp each).
#pragma once

#include "inl_common.hpp"
#include "../../include/inl_train.h"

namespace inl {

enum : int32_t {
  ACT_NONE = INL_ACT_NONE,
  ACT_RELU = INL_ACT_RELU,
  ACT_SILU = INL_ACT_SILU,
  ACT_GELU_TANH = INL_ACT_GELU_TANH,
  ACT_GELU_ERF = INL_ACT_GELU_ERF,
};

struct ActPair {
  float value, slope;
};

__device__ __forceinline__ float act_sigmoid(float v) {
  return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-1.44269504088896f * v));
}

// Phi(v), the normal distribution function, with q = e^(-v^2 / 2): for x = |v| /
// sqrt(2), erfc(x) = t (a1 + t (a2 + ... a5 t)) e^(-x^2), t = 1 / (1 + 0.3275911 x)
// (Hastings; Abramowitz and Stegun 7.1.26, absolute error 1.5e-7). The tail is
// erfc itself, so that large negative v keep their relative size.
__device__ __forceinline__ float act_phi(float v, float q) {
  const float x = fabsf(v) * 0.707106781186548f;
  const float t = __builtin_amdgcn_rcpf(__builtin_fmaf(0.3275911f, x, 1.0f));
  float s = __builtin_fmaf(t, 1.061405429f, -1.453152027f);
  s = __builtin_fmaf(t, s, 1.421413741f);
  s = __builtin_fmaf(t, s, -0.284496736f);
  s = __builtin_fmaf(t, s, 0.254829592f);
  const float half_tail = 0.5f * t * s * q;
  return v < 0.f ? half_tail : 1.0f - half_tail;
}

// gelu_tanh(v) = v sigmoid(2u), 2u = 2 sqrt(2 / pi) (v + 0.044715 v^3)
__device__ __forceinline__ float act_gelu_gate(float v) {
  return act_sigmoid(v * __builtin_fmaf(v * v, 0.0713548162f, 1.59576912f));
}

__device__ __forceinline__ float act_apply(int32_t act, float v) {
  switch (act) {
    case ACT_RELU: return v > 0.f ? v : (v != v ? v : 0.f);
    case ACT_SILU: return v * act_sigmoid(v);
    case ACT_GELU_TANH: return v * act_gelu_gate(v);
    case ACT_GELU_ERF: {
      // v Phi(v) = v / 2 + |v| / 2 (1 - erfc(|v| / sqrt(2))), erfc(x) = (1 + a1 x + ... + a6 x^6)^-16
      // (Hastings; Abramowitz and Stegun 7.1.28, absolute error 3e-7; a_i here times
      // 2^(-i/2)). One reciprocal and no exponential: of 128 outputs per lane and
      // tile the form of act_phi took 10 us of a 20,011 x 768 x 768 layer's 38.
      const float x = fabsf(v);
      float d = __builtin_fmaf(x, 5.3829750e-6f, 4.8890636e-5f);
      d = __builtin_fmaf(x, d, 3.8003575e-5f);
      d = __builtin_fmaf(x, d, 3.2776263e-3f);
      d = __builtin_fmaf(x, d, 2.1141006e-2f);
      d = __builtin_fmaf(x, d, 4.9867347e-2f);
      d = __builtin_fmaf(x, d, 1.0f);
      d *= d;
      d *= d;
      d *= d;
      d *= d;
      return __builtin_fmaf(0.5f * x, 1.0f - __builtin_amdgcn_rcpf(d), 0.5f * v);
    }
    default: return v;
  }
}

__device__ __forceinline__ f32x4 act_apply4(int32_t act, f32x4 v) {
  f32x4 r = v;
  switch (act) {   // uniform: one branch for the four values
#define INL_ACT4(A)                                              \
  case A:                                                        \
    _Pragma("unroll") for (int e = 0; e < 4; ++e) r[e] = act_apply(A, v[e]); \
    break;
    INL_ACT4(ACT_RELU)
    INL_ACT4(ACT_SILU)
    INL_ACT4(ACT_GELU_TANH)
    INL_ACT4(ACT_GELU_ERF)
#undef INL_ACT4
    default: break;
  }
  return r;
}

__device__ __forceinline__ ActPair act_pair(int32_t act, float v) {
  switch (act) {
    case ACT_RELU: return {act_apply(ACT_RELU, v), v > 0.f ? 1.f : (v != v ? v : 0.f)};
    case ACT_SILU: {
      const float s = act_sigmoid(v);
      return {v * s, s * __builtin_fmaf(v, 1.0f - s, 1.0f)};
    }
    case ACT_GELU_TANH: {
      const float s = act_gelu_gate(v);
      const float d = __builtin_fmaf(v * v, 0.214064449f, 1.59576912f);   // d(2u) / dv
      return {v * s, s * __builtin_fmaf(v * (1.0f - s), d, 1.0f)};
    }
    case ACT_GELU_ERF: {
      const float q = __builtin_amdgcn_exp2f(-0.721347520444482f * v * v);
      const float f = act_phi(v, q);
      return {v * f, __builtin_fmaf(v * 0.398942280401433f, q, f)};
    }
    default: return {v, 1.f};
  }
}

}  // namespace inl
