// The gated feed-forward block and its gradients: five products, the element-wise
// parts in their epilogues.
//
//   forward   h = act(x . w_gate^T) * (x . w_up^T)     one launch (EPI_GATED), 4 m hidden inner flops
//             y = h . w_down^T + residual              2 m hidden inner
//   backward  dh = dy . w_down, d_gate and d_up from it and the stored gate and
//             up in the epilogue: dh never reaches memory  2 m hidden inner
//             dw_down = dy^T . h                       2
//             dx = [d_gate d_up] . w_gate_up           4
//             dw_gate_up = [d_gate d_up]^T . x         4
//
// 20,011 rows, 768 x 1,152, forward: 107 to 120 us by card (gate and up 71, down 43; 890 to 990
// TFLOP/s), 7 more where pre and h are stored. 16,384 rows, 1,024 x 4,096, backward: 764 to 786 us
// (1,050 to 1,080): the gate gradients' product stands beside the bytes of its epilogue (98 us of
// products, 537 MB, matrix cores 26 % busy), the others run at 2.0 to 2.1 GHz of 2.4 (58 to 65 %
// busy). One row of 1,024 x 2,816: 6.3 us.
//
// h, d_gate and d_up are rounded to bf16, the type of the products' operands. The outputs feel
// it: y is 1.9e-3 of its norm from 64 bits (1.7e-3 with its own rounding alone), dx and
// dw_gate_up 2.3e-3 (1.7e-3). gate, up, dh and the activation stay in f32 in between.
#include "train_ops.hpp"

namespace inl {

namespace {

int ffn_check(const inl_gated_ffn_desc* d) {
  if (!d) return fail(INL_E_INVALID, "gated_ffn: desc is NULL");
  if (d->m < 0 || d->hidden <= 0 || d->inner <= 0)
    return fail(INL_E_INVALID, "gated_ffn: m must be >= 0, hidden and inner > 0");
  if (d->hidden % 8 || d->inner % 8) return fail(INL_E_UNSUPPORTED, "gated_ffn: hidden and inner must be multiples of 8");
  if (d->m >= ((int64_t)1 << 31) - 256 || d->hidden > (1 << 20) || d->inner > (1 << 20))
    return fail(INL_E_UNSUPPORTED, "gated_ffn: m must stay below 2^31 - 256, hidden and inner at most 2^20");
  if (d->act <= INL_ACT_NONE || d->act > INL_ACT_GELU_ERF)
    return fail(INL_E_INVALID, "gated_ffn: act must be INL_ACT_RELU, SILU, GELU_TANH or GELU_ERF");
  return INL_OK;
}

constexpr int MAX_SPLITS = 32;

struct FfnPlan {
  TilePlan h{}, y{}, dh, dwd, dx, dwgu;   // h and y without tiles: splits 0
  int cus = 0;
};
int ffn_plan(const inl_gated_ffn_desc& d, bool backward, FfnPlan* p) {
  const bool few_h = few_rows(d.m, d.inner, d.hidden, true), few_y = few_rows(d.m, d.hidden, d.inner, false);
  if (!backward && few_h && few_y) return INL_OK;
  int rc = device_cus(&p->cus);
  if (rc) return rc;
  if (!backward) {
    if (!few_h) p->h = tile_plan(d.m, d.inner, d.hidden, 0, true, MAX_SPLITS, p->cus);
    if (!few_y) p->y = tile_plan(d.m, d.hidden, d.inner, 0, false, MAX_SPLITS, p->cus);
    return INL_OK;
  }
  p->dh = tile_plan(d.m, d.inner, d.hidden, 1, false, MAX_SPLITS, p->cus);
  p->dwd = tile_plan(d.hidden, d.inner, d.m, 2, false, MAX_SPLITS, p->cus);
  p->dx = tile_plan(d.m, d.hidden, 2 * d.inner, 1, false, MAX_SPLITS, p->cus);
  p->dwgu = tile_plan(2 * d.inner, d.hidden, d.m, 2, false, MAX_SPLITS, p->cus);
  return INL_OK;
}

// The workspace: h (forward) or [d_gate d_up] (backward), then split partials.
size_t rows_bytes(const inl_gated_ffn_desc& d, bool backward) {
  return (size_t)d.m * (size_t)d.inner * (backward ? 4 : 2);
}
size_t ffn_need(const inl_gated_ffn_desc& d, const FfnPlan& p, bool backward) {
  Carve c(nullptr);
  c.take(rows_bytes(d, backward));
  if (backward)
    c.take(std::max(std::max(tile_part_bytes(p.dh, d.m, d.inner), tile_part_bytes(p.dwd, d.hidden, d.inner)),
                    std::max(tile_part_bytes(p.dx, d.m, d.hidden), tile_part_bytes(p.dwgu, 2 * d.inner, d.hidden))));
  else
    c.take(std::max(tile_part_bytes(p.h, d.m, 2 * d.inner), tile_part_bytes(p.y, d.m, d.hidden)));
  return c.used;
}

}  // namespace

}  // namespace inl

extern "C" int inl_gated_ffn_workspace_size(const inl_gated_ffn_desc* d, int32_t backward, size_t* bytes) {
  using namespace inl;
  if (!bytes) return fail(INL_E_INVALID, "gated_ffn: bytes is NULL");
  int rc = ffn_check(d);
  if (rc) return rc;
  FfnPlan plan;
  if ((rc = ffn_plan(*d, backward != 0, &plan))) return rc;
  *bytes = ffn_need(*d, plan, backward != 0);
  return INL_OK;
}

extern "C" int inl_gated_ffn_fwd(const inl_gated_ffn_desc* d, const void* x, const void* w_gate_up, const void* w_down,
                                 const void* residual, void* y, void* pre, void* h, void* ws, size_t ws_bytes,
                                 void* stream) {
  using namespace inl;
  hipStream_t st = (hipStream_t)stream;
  int rc = ffn_check(d);
  if (rc) return rc;
  if ((pre == nullptr) != (h == nullptr)) return fail(INL_E_INVALID, "gated_ffn: pre and h are stored together");
  if (d->m == 0) return INL_OK;
  const int64_t xs = d->x_stride ? d->x_stride : d->hidden, ys = d->y_stride ? d->y_stride : d->hidden;
  const int64_t rs = d->residual_stride ? d->residual_stride : d->hidden;
  if ((rc = check_rows("gated_ffn: x", x, d->hidden, xs, INL_BF16))) return rc;
  if ((rc = check_rows("gated_ffn: w_gate_up", w_gate_up, d->hidden, d->hidden, INL_BF16))) return rc;
  if ((rc = check_rows("gated_ffn: w_down", w_down, d->inner, d->inner, INL_BF16))) return rc;
  if ((rc = check_rows("gated_ffn: y", y, d->hidden, ys, d->out_dtype))) return rc;
  if (residual && (rc = check_rows("gated_ffn: residual", residual, d->hidden, rs, d->residual_dtype))) return rc;
  if (pre && (rc = check_rows("gated_ffn: pre", pre, 2 * d->inner, 2 * d->inner, INL_BF16))) return rc;
  if (h && (rc = check_rows("gated_ffn: h", h, d->inner, d->inner, INL_BF16))) return rc;
  FfnPlan plan;
  if ((rc = ffn_plan(*d, false, &plan))) return rc;
  if ((rc = check_workspace("gated_ffn", ws, ws_bytes, ffn_need(*d, plan, false)))) return rc;
  Carve c(ws);
  char* hb = c.take(rows_bytes(*d, false));
  float* part = (float*)c.take(0);
  if (h) hb = (char*)h;
  TileParams p{};
  p.x = (const char*)x;
  p.xs_b = xs * 2;
  p.w = (const char*)w_gate_up;
  p.ws_b = d->hidden * 2;
  p.m = d->m;
  p.n = (int32_t)d->inner;
  p.k = (int32_t)d->hidden;
  p.y = hb;
  p.ys = d->inner;
  p.alpha = p.beta = 1.f;
  p.pre = (char*)pre;
  p.ps = 2 * d->inner;
  p.act = d->act;
  if ((rc = !plan.h.splits ? few_dense(p, true, true, st) : tile_nt_gated(p, plan.h, part, plan.cus, st))) return rc;
  p.x = hb;
  p.xs_b = d->inner * 2;
  p.w = (const char*)w_down;
  p.ws_b = d->inner * 2;
  p.n = (int32_t)d->hidden;
  p.k = (int32_t)d->inner;
  p.y = (char*)y;
  p.ys = ys;
  p.res = (const char*)residual;
  p.rs = rs;
  p.res_bf16 = d->residual_dtype == INL_BF16;
  p.pre = nullptr;
  p.act = ACT_NONE;
  const bool out16 = d->out_dtype == INL_BF16;
  return !plan.y.splits ? few_dense(p, false, out16, st) : tile_nt_linear(p, plan.y, out16, part, plan.cus, st);
}

extern "C" int inl_gated_ffn_bwd(const inl_gated_ffn_desc* d, const void* dy, const void* x, const void* w_gate_up,
                                 const void* w_down, const void* pre, const void* h, void* dx, void* dw_gate_up,
                                 void* dw_down, void* ws, size_t ws_bytes, void* stream) {
  using namespace inl;
  hipStream_t st = (hipStream_t)stream;
  int rc = ffn_check(d);
  if (rc) return rc;
  const int64_t xs = d->x_stride ? d->x_stride : d->hidden, ys = d->y_stride ? d->y_stride : d->hidden;
  const int64_t dxs = d->dx_stride ? d->dx_stride : d->hidden;
  if (dx && !dtype_ok(d->dx_dtype)) return fail(INL_E_INVALID, "gated_ffn: dx_dtype must be INL_F32 or INL_BF16");
  if (dw_gate_up && (rc = check_rows("gated_ffn: dw_gate_up", dw_gate_up, d->hidden, d->hidden, d->dw_dtype))) return rc;
  if (dw_down && (rc = check_rows("gated_ffn: dw_down", dw_down, d->inner, d->inner, d->dw_dtype))) return rc;
  if (d->m == 0) {
    if (dw_gate_up && (rc = fill_zero(dw_gate_up, 2 * d->inner, d->hidden, d->hidden, d->dw_dtype, st))) return rc;
    return dw_down ? fill_zero(dw_down, d->hidden, d->inner, d->inner, d->dw_dtype, st) : INL_OK;
  }
  if ((rc = check_rows("gated_ffn: dy", dy, d->hidden, ys, INL_BF16))) return rc;
  const bool inner_grads = dx || dw_gate_up;
  if (inner_grads) {
    if ((rc = check_rows("gated_ffn: w_down", w_down, d->inner, d->inner, INL_BF16))) return rc;
    if ((rc = check_rows("gated_ffn: pre", pre, 2 * d->inner, 2 * d->inner, INL_BF16))) return rc;
  }
  if (dx && (rc = check_rows("gated_ffn: dx", dx, d->hidden, dxs, d->dx_dtype))) return rc;
  if (dx && (rc = check_rows("gated_ffn: w_gate_up", w_gate_up, d->hidden, d->hidden, INL_BF16))) return rc;
  if (dw_gate_up && (rc = check_rows("gated_ffn: x", x, d->hidden, xs, INL_BF16))) return rc;
  if (dw_down && (rc = check_rows("gated_ffn: h", h, d->inner, d->inner, INL_BF16))) return rc;
  FfnPlan plan;
  if ((rc = ffn_plan(*d, true, &plan))) return rc;
  if ((rc = check_workspace("gated_ffn", ws, ws_bytes, ffn_need(*d, plan, true)))) return rc;
  Carve c(ws);
  char* dgu = c.take(rows_bytes(*d, true));
  float* part = (float*)c.take(0);
  TileParams p{};
  p.alpha = p.beta = 1.f;
  if (inner_grads) {
    p.x = (const char*)dy;
    p.xs_b = ys * 2;
    p.w = (const char*)w_down;
    p.ws_b = d->inner * 2;
    p.m = d->m;
    p.n = (int32_t)d->inner;
    p.k = (int32_t)d->hidden;
    p.y = dgu;
    p.ys = 2 * d->inner;
    p.pre = (char*)pre;
    p.ps = 2 * d->inner;
    p.act = d->act;
    if ((rc = tile_nn_dgated(p, plan.dh, part, plan.cus, st))) return rc;
  }
  p.pre = nullptr;
  p.act = ACT_NONE;
  if (dw_down) {
    p.x = (const char*)dy;
    p.xs_b = ys * 2;
    p.w = (const char*)h;
    p.ws_b = d->inner * 2;
    p.m = d->hidden;
    p.n = (int32_t)d->inner;
    p.k = (int32_t)d->m;
    p.y = (char*)dw_down;
    p.ys = d->inner;
    if ((rc = tile_tn_linear(p, plan.dwd, d->dw_dtype == INL_BF16, part, plan.cus, st))) return rc;
  }
  if (dx) {
    p.x = dgu;
    p.xs_b = d->inner * 4;
    p.w = (const char*)w_gate_up;
    p.ws_b = d->hidden * 2;
    p.m = d->m;
    p.n = (int32_t)d->hidden;
    p.k = (int32_t)(2 * d->inner);
    p.y = (char*)dx;
    p.ys = dxs;
    if ((rc = tile_nn_linear(p, plan.dx, d->dx_dtype == INL_BF16, part, plan.cus, st))) return rc;
  }
  if (dw_gate_up) {
    p.x = dgu;
    p.xs_b = d->inner * 4;
    p.w = (const char*)x;
    p.ws_b = xs * 2;
    p.m = 2 * d->inner;
    p.n = (int32_t)d->hidden;
    p.k = (int32_t)d->m;
    p.y = (char*)dw_gate_up;
    p.ys = d->hidden;
    if ((rc = tile_tn_linear(p, plan.dwgu, d->dw_dtype == INL_BF16, part, plan.cus, st))) return rc;
  }
  return INL_OK;
}
