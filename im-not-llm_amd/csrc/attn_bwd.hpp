// Gradients of packed varlen attention (attn_bwd.hip): parameters of the kernels.
#pragma once

#include "attn_kernels.hpp"

namespace inl {

// A text of the batch: its first row, its length, and the first unit (block of own rows) of
// it among all units of its class.
struct BwdText {
  int32_t start, len, unit;
};

// Texts that fit into a kernel's arguments (3 KB of the 4 KB that a launch takes).
constexpr int BWD_INLINE = 256;
constexpr int BWD_CLASSES = 8;

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
  int32_t h_q, h_kv, group, head_dim, causal, window;
  float c, scale;          // scale * log2(e) (the exponent's), scale
  // Workgroup i works for key head (i % (h_kv classes)) % h_kv, on texts of class (i % (h_kv classes)) / h_kv.
  int32_t classes;
  int32_t first[BWD_CLASSES + 1];   // texts of class c: [first[c], first[c + 1])
  int32_t units[BWD_CLASSES];       // and their units
  BwdText own[BWD_INLINE];
};

}  // namespace inl
