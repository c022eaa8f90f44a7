/*
 * inl_train.h - C ABI of the layer and head ops with their gradients, on one
 * MI355X (gfx950): what fine-tuning the encoders of inl_encoder.h needs beside
 * its forward. Conventions are those of inl_hip.h: device pointers, int status
 * + inl_last_error(), work on the caller's stream, the caller owns every
 * buffer. Nothing is allocated and nothing synchronised, so every call can be
 * captured into a graph.
 *
 * Matrices are rows of bf16 (strides in elements between rows, 0 = packed),
 * 16-byte aligned, row lengths and strides multiples of 8 elements; products
 * accumulate in f32 on the matrix cores. Other shapes are refused
 * (INL_E_UNSUPPORTED).
 *
 * Workspaces: device memory of at least the size the *_workspace_size call
 * gives for the same desc, 16-byte aligned, untouched until the call has
 * completed on `stream`. Calls that may overlap (two streams, two graphs that
 * run at one time) need a workspace each. Results do not depend on what it
 * holds, and equal calls give equal bits.
 */
#ifndef INL_TRAIN_H
#define INL_TRAIN_H

#include <stddef.h>
#include <stdint.h>

#include "inl_hip.h"

#ifdef __cplusplus
extern "C" {
#endif

enum inl_act {
  INL_ACT_NONE = 0,
  INL_ACT_RELU = 1,
  INL_ACT_SILU = 2,       /* v / (1 + exp(-v)) */
  INL_ACT_GELU_TANH = 3,  /* v / 2 (1 + tanh(sqrt(2 / pi) (v + 0.044715 v^3))) */
  INL_ACT_GELU_ERF = 4    /* v Phi(v) */
};

/* ------------------------------------------------------------------------
 * Linear layer with bias, activation and residual in its epilogue:
 *   pre = x . w^T + bias;  y = act(pre) + residual
 * inl_gemm_bf16_fwd (inl_encoder.h) is the bias-free one. w is [n, k], the
 * checkpoint's [out, in].
 * --------------------------------------------------------------------- */
typedef struct inl_dense_desc {
  int64_t m;               /* rows of x, >= 0 */
  int64_t n, k;            /* outputs, inputs */
  int64_t x_stride;
  int64_t w_stride;
  int64_t y_stride;        /* y and dy */
  int64_t residual_stride;
  int64_t pre_stride;
  int64_t dx_stride;
  int64_t dw_stride;
  int32_t act;             /* enum inl_act */
  int32_t out_dtype;       /* of y: INL_F32 or INL_BF16 */
  int32_t residual_dtype;  /* of residual */
  int32_t dx_dtype;        /* of dx */
  int32_t dw_dtype;        /* of dw */
} inl_dense_desc;

int inl_dense_workspace_size(const inl_dense_desc* desc, int32_t backward, size_t* bytes);

/* bias: f32 [n] or NULL; residual: [m, n] or NULL (it may be y itself, of its type
 * and stride); pre: bf16 [m, n] or NULL, receives x . w^T + bias for the backward.
 * Everything up to y (and pre) stays in f32: one rounding each. y and pre otherwise
 * share no byte with another argument: x itself is refused, as x is read until the
 * last of y is written. */
int inl_dense_fwd(const inl_dense_desc* desc, const void* x, const void* w, const float* bias, const void* residual,
                  void* y, void* pre, void* workspace, size_t workspace_bytes, void* stream);

/* With dz = dy * act'(pre):
 *   dx = dz . w,  dw = dz^T . x,  dbias[c] = sum over rows of dz (f32 [n])
 * dy: bf16 [m, n]; pre: what the forward stored (NULL with INL_ACT_NONE). The
 * gradient of the residual is dy itself. dx, dw, dbias: NULL = not computed.
 * The products read dz rounded to bf16; dbias sums it unrounded. m = 0 gives
 * dw = 0 and dbias = 0. */
int inl_dense_bwd(const inl_dense_desc* desc, const void* dy, const void* x, const void* w, const void* pre, void* dx,
                  void* dw, float* dbias, void* workspace, size_t workspace_bytes, void* stream);

/* ------------------------------------------------------------------------
 * Gated feed-forward block:
 *   gate = x . w_gate^T, up = x . w_up^T;  h = act(gate) * up;
 *   y = h . w_down^T + residual
 * (crates/inl-text/src/qwen3/mod.rs:96-116 with INL_ACT_SILU, gemma2.rs:233-254
 * with INL_ACT_GELU_TANH, the gated MLP of crates/inl-sparse/src/modernbert.rs
 * with INL_ACT_GELU_ERF). w_gate_up: [2 inner, hidden], gate rows then up rows;
 * w_down: [hidden, inner]; both packed. gate, up and their product are one
 * launch, the down projection with its residual another.
 * --------------------------------------------------------------------- */
typedef struct inl_gated_ffn_desc {
  int64_t m;
  int64_t hidden, inner;
  int64_t x_stride;
  int64_t y_stride;        /* y and dy */
  int64_t residual_stride;
  int64_t dx_stride;
  int32_t act;             /* INL_ACT_SILU, INL_ACT_GELU_TANH, INL_ACT_GELU_ERF or INL_ACT_RELU */
  int32_t out_dtype;       /* of y */
  int32_t residual_dtype;
  int32_t dx_dtype;
  int32_t dw_dtype;        /* of dw_gate_up and dw_down */
} inl_gated_ffn_desc;

int inl_gated_ffn_workspace_size(const inl_gated_ffn_desc* desc, int32_t backward, size_t* bytes);

/* residual: [m, hidden] or NULL (it may be y itself, and either may be x). pre (bf16 [m, 2 inner]:
 * gate, then up) and h (bf16 [m, inner]), packed, are stored for the backward,
 * both or neither (NULL). h is rounded to bf16 before the down projection. */
int inl_gated_ffn_fwd(const inl_gated_ffn_desc* desc, const void* x, const void* w_gate_up, const void* w_down,
                      const void* residual, void* y, void* pre, void* h, void* workspace, size_t workspace_bytes,
                      void* stream);

/* With dh = dy . w_down (f32), d_gate = dh * up * act'(gate), d_up = dh *
 * act(gate), both rounded to bf16:
 *   dx = [d_gate d_up] . w_gate_up;  dw_gate_up = [d_gate d_up]^T . x;
 *   dw_down = dy^T . h
 * dx, dw_gate_up, dw_down: NULL = not computed. */
int inl_gated_ffn_bwd(const inl_gated_ffn_desc* desc, const void* dy, const void* x, const void* w_gate_up,
                      const void* w_down, const void* pre, const void* h, void* dx, void* dw_gate_up, void* dw_down,
                      void* workspace, size_t workspace_bytes, void* stream);

/* ------------------------------------------------------------------------
 * Softmax cross entropy of scores that are never stored:
 *   s[r, v] = scale * x[r] . w[v] + bias[v]
 *   lse[r] = log sum_v exp(s[r, v]);  loss[r] = lse[r] - s[r, targets[r]]
 * for a vocabulary (w: the decoder) or for the documents of a batch (w: their
 * embeddings, scale: 1 / temperature, targets: each query's document). Beside
 * inl_splade_decoder_max_fwd, which takes a maximum of such products. A row
 * whose target is ignore_index has loss 0 and a gradient of 0 whatever its scores
 * are (its lse is given; dw still multiplies its x by 0); another target outside
 * [0, vocab) gives a NaN loss and, in the backward, NaN in its row of dx and in all
 * of dw. A bias of -inf takes an entry out (with all of them out lse is -inf, loss
 * NaN). x: [m, hidden], w: [vocab, hidden]; any vocab >= 1.
 * --------------------------------------------------------------------- */
typedef struct inl_softmax_xent_desc {
  int64_t m;
  int64_t vocab, hidden;
  int64_t x_stride;
  int64_t w_stride;
  int64_t dx_stride;
  int64_t dw_stride;
  float scale;
  int32_t ignore_index;
  int32_t dx_dtype;
  int32_t dw_dtype;
} inl_softmax_xent_desc;

int inl_softmax_xent_workspace_size(const inl_softmax_xent_desc* desc, int32_t backward, size_t* bytes);

/* bias: f32 [vocab] or NULL; targets: int32 [m]; loss, lse: f32 [m] */
int inl_softmax_xent_fwd(const inl_softmax_xent_desc* desc, const void* x, const void* w, const float* bias,
                         const int32_t* targets, float* loss, float* lse, void* workspace, size_t workspace_bytes,
                         void* stream);

/* With g[r, v] = dloss[r] (exp(s[r, v] - lse[r]) - [v == targets[r]]):
 *   dx = scale g . w,  dw = scale g^T . x,  dbias = sum over rows of g
 * lse: the forward's; dloss: f32 [m]. The vocabulary is taken in pieces: g of
 * one piece (bf16, dloss rounded with it) is all of it that exists at a time; dx
 * adds up in f32.
 * dbias (f32 [vocab]) sums the bf16 values. dx, dw, dbias: NULL = not
 * computed. */
int inl_softmax_xent_bwd(const inl_softmax_xent_desc* desc, const float* dloss, const float* lse, const void* x,
                         const void* w, const float* bias, const int32_t* targets, void* dx, void* dw, float* dbias,
                         void* workspace, size_t workspace_bytes, void* stream);

/* ------------------------------------------------------------------------
 * Gradients of inl_norm_rope_qk_fwd (inl_hip.h): for y = R(x / rms(x) * weight)
 * per (token, head), with R the rotation of the head's rotary part,
 *   dn = R^T dy;  dweight = sum over tokens and heads of dn * x / rms(x);
 *   dx = (weight dn - xhat mean(weight dn xhat)) / rms(x),  xhat = x / rms(x)
 * in f32. x and dx are in desc->dtype, dy in desc->out_dtype with y_row_stride;
 * dx_row_stride: elements, 0 = heads * head_dim. 0 < q_heads <= desc->heads; with q_heads ==
 * heads there are no k heads (dk_weight NULL). dq_weight, dk_weight: f32
 * [head_dim], NULL = not computed. The roundings that the desc's round_norm
 * and round_tables ask for pass gradients through unchanged (tables rounded as
 * in the forward). A token whose table row is out of range gets NaN in dx and
 * in dweight. dx may be dy or x itself where types and strides are equal; it
 * overlaps them nowhere else.
 * --------------------------------------------------------------------- */
int inl_norm_rope_bwd_workspace_size(const inl_norm_rope_desc* desc, size_t* bytes);
int inl_norm_rope_qk_bwd(const inl_norm_rope_desc* desc, int32_t q_heads, const void* dy, const void* x, void* dx,
                         int64_t dx_row_stride, const void* q_weight, const void* k_weight, const int32_t* rows, const float* cos,
                         const float* sin, const float* cos2, const float* sin2, float* dq_weight, float* dk_weight,
                         void* workspace, size_t workspace_bytes, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* INL_TRAIN_H */
