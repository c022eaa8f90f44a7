// Gradients of packed varlen attention (attn_bwd.hip): parameters of the kernels.
#pragma once

#include "attn_kernels.hpp"

namespace inl {

// A text of the batch, longest first: its first row, its length, and the first unit
// (block of own rows) of it among all units of a kernel.
struct BwdText {
  int32_t start, len, unit;
};

// Texts that fit into a kernel's arguments (3 KB of the 4 KB that a launch takes).
constexpr int BWD_INLINE = 256;

struct AttnBwdParams {
  const char* q;
  const char* k;
  const char* v;
  const char* o;
  const char* dout;
  char* dq;
  char* dk;
  char* dv;
  float* stat;             // [2][h_q][rows]: -log-sum-exp / c, then -delta
  const BwdText* texts;    // null: in `own`
  int64_t q_stride, k_stride, v_stride, o_stride, do_stride, dq_stride, dk_stride, dv_stride;  // bytes
  int64_t rows;
  int32_t n_texts, h_q, h_kv, group, head_dim, causal, window;
  float c, scale;          // scale * log2(e) (the exponent's), scale
  BwdText own[BWD_INLINE];
};

}  // namespace inl
