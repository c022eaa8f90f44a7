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

// Phi(-x), x >= 0, the normal distribution's tail, as 2^-Q(x): -log2 Phi(-x) goes as
// x^2 / 2 and log x, which a polynomial follows with one exponential and no
// reciprocal. The coefficients are a fit of our own, Q(0) = 1 exactly, that spends its
// error as 2.7e-4 of the tail or 2.7e-7 of 1, whichever is less; in f32 arithmetic 3e-4
// and 4e-7, up to x = 8. Past that it falls faster than the tail does (below 1e-15). NaN
// stays NaN, an infinite x gives 0. An erfc of absolute accuracy only, as
// v / 2 (1 + erf), left nothing of v = -5.5 (off by 0.57 of its value). Of 20,011 x 768 outputs
// this form takes 8 us beside the products, the power of a polynomial with its
// reciprocal before it 8.7.
__device__ __forceinline__ float act_tail(float x) {
  float q = __builtin_fmaf(x, 1.0045712e-7f, -1.1652755e-6f);
  q = __builtin_fmaf(x, q, -2.7316801e-5f);
  q = __builtin_fmaf(x, q, 7.3941034e-4f);
  q = __builtin_fmaf(x, q, -7.9598976e-3f);
  q = __builtin_fmaf(x, q, 5.3172562e-2f);
  q = __builtin_fmaf(x, q, 4.5898059e-1f);
  q = __builtin_fmaf(x, q, 1.1511295f);
  q = __builtin_fmaf(x, q, 1.0f);
  return __builtin_amdgcn_exp2f(-q);
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
      // v Phi(v), the tail by itself where v < 0: nothing cancels, and small results
      // keep their relative size
      const float t = act_tail(fabsf(v));
      return v * (v < 0.f ? t : 1.0f - t);
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
      // (past 16, where s is 0 or 1, the square would leave the range before v does; the
      // median drops NaN, which s carries)
      const float s = act_gelu_gate(v), w = __builtin_amdgcn_fmed3f(v, -16.0f, 16.0f);
      const float d = __builtin_fmaf(w * w, 0.214064449f, 1.59576912f);   // d(2u) / dv
      return {v * s, s * __builtin_fmaf(w * (1.0f - s), d, 1.0f)};
    }
    case ACT_GELU_ERF: {
      const float q = __builtin_amdgcn_exp2f(-0.721347520444482f * v * v);
      const float t = act_tail(fabsf(v)), f = v < 0.f ? t : 1.0f - t;
      return {v * f, __builtin_fmaf(v * 0.398942280401433f, q, f)};
    }
    default: return {v, 1.f};
  }
}

}  // namespace inl
