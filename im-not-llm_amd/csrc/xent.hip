// Softmax cross entropy of scores that are never stored, and its gradients.
//
//   forward   s = scale x . w^T + bias; lse = log sum exp s; loss = lse - s_target
//     One pass of the tiled product; its epilogue (EPI_XENT) keeps of each row
//     and 128 (64, 32) columns the maximum and the sum of exponentials under
//     it, and the target's score where it passes by. A second kernel joins the
//     column blocks: 2 x 4 bytes per 128 scores instead of the scores.
//     2 m vocab hidden flops. 4,099 rows, 50,002 entries, hidden 768: 305 to 331 us by card
//     (some 1,000 TFLOP/s): the product under the power limit, 14 rounds of tiles for
//     13.0, and 4.5 us of exponentials per tile.
//   backward  g = dloss (exp(s - lse) - onehot), in pieces of the vocabulary: the
//     scores again (EPI_DXENT writes g in bf16), dw of the piece = scale g^T . x,
//     dx += scale g . w. 6 m vocab hidden flops. 2,048 rows, 151,669 entries, hidden
//     1,024: 1.72 to 1.80 ms (1,060 to 1,110 TFLOP/s); a piece's scores 139 us, dw 107, dx 103
//     and 14 for the join of its k splits. g is rounded to bf16, the type of the products'
//     operands: here dx and dw move by 2e-4 of their norm for it, under the rounding of a
//     bf16 output (1.7e-3); a dloss that is the same for every row moves them by its own
//     rounding, 3.9e-3 at most (1 / 255; 1 / 2,048 is exact). dbias sums those values, which the pieces read anyway, in f32.
#include "train_ops.hpp"

namespace inl {

namespace {

int xent_check(const inl_softmax_xent_desc* d) {
  if (!d) return fail(INL_E_INVALID, "softmax_xent: desc is NULL");
  if (d->m < 0 || d->vocab <= 0 || d->hidden <= 0)
    return fail(INL_E_INVALID, "softmax_xent: m must be >= 0, vocab and hidden > 0");
  if (d->hidden % 8) return fail(INL_E_UNSUPPORTED, "softmax_xent: hidden must be a multiple of 8");
  if (d->m >= ((int64_t)1 << 31) - 256 || d->vocab > (1 << 28) || d->hidden > (1 << 21))
    return fail(INL_E_UNSUPPORTED, "softmax_xent: m must stay below 2^31 - 256, vocab at most 2^28, hidden at most 2^21");
  return INL_OK;
}

// Columns per statistics block of a shape.
int stat_cols(int shape) { return shape == 0 ? 128 : shape == 1 ? 64 : 32; }
int tile_cols(int shape) { return shape == 0 ? TileShapeOf<0>::BN : shape == 1 ? TileShapeOf<1>::BN : TileShapeOf<2>::BN; }

// Statistics blocks along the vocabulary: whole tiles, those past the end hold
// (-inf, 0).
int64_t stat_blocks(int shape, int64_t vocab) {
  const int64_t tiles = (vocab + tile_cols(shape) - 1) / tile_cols(shape);
  return tiles * (tile_cols(shape) / stat_cols(shape));
}

// lse and loss from the blocks' statistics: the 16 waves of a workgroup take every
// 16th block for 64 rows, then meet in LDS. Bound by latency: 4,099 rows are 65
// workgroups for 256 CUs, and a wave folds some 25 of the 392 blocks (50,002 entries) one
// after another: 6.0 us for 12.9 MB, 2.1 TB/s. 1,024 rows x 128 blocks 3.9 us, mostly launch.
constexpr int JOIN_WAVES = 16;
__global__ __launch_bounds__(JOIN_WAVES * 64) void xent_join_kernel(const float2* part, int64_t blocks, int64_t m,
                                                                    const int32_t* target, const float* at,
                                                                    int32_t ignore, int64_t vocab, float* loss,
                                                                    float* lse) {
  __shared__ float2 red[JOIN_WAVES][64];
  constexpr float LOG2E = 1.44269504088896f;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t row = blockIdx.x * 64LL + lane;
  float top = -INFINITY, sum = 0.f;
  auto fold = [&](float2 q) {
    const float t = fmaxf(top, q.x);
    const float base = t == -INFINITY ? 0.f : t;
    sum = sum * __builtin_amdgcn_exp2f((top - base) * LOG2E) + q.y * __builtin_amdgcn_exp2f((q.x - base) * LOG2E);
    top = t;
  };
  if (row < m) {
#pragma unroll 4
    for (int64_t b = wave; b < blocks; b += JOIN_WAVES) fold(part[b * m + row]);
  }
  red[wave][lane] = make_float2(top, sum);
  __syncthreads();
  if (wave || row >= m) return;
#pragma unroll
  for (int w = 1; w < JOIN_WAVES; ++w) fold(red[w][lane]);
  const float logs = logf(sum);
  lse[row] = top + logs;
  const int32_t t = target[row];
  // (top - score) + log: a small loss beside large scores keeps its digits
  loss[row] = t == ignore ? 0.f : (t < 0 || t >= vocab) ? __builtin_nanf("") : (top - at[row]) + logs;
}

constexpr int MAX_SPLITS = 32;

// Vocabulary entries per piece: g of a piece is some 128 MiB, so that dw and dx
// read it from the 256 MB Infinity Cache, in whole 256-column tiles; at most 2^21, the
// longest row that the products' descriptors take.
int64_t piece_cols(int64_t m, int64_t vocab) {
  int64_t p = std::min<int64_t>(((int64_t)1 << 26) / std::max<int64_t>(m, 1), (int64_t)1 << 21);
  p = std::min(std::max<int64_t>(p, 4096), vocab);
  return (p + 255) / 256 * 256;
}

struct XentPlan {
  TilePlan s;              // forward
  int64_t piece;           // columns of g
  TilePlan g, dw, dx;      // of a whole piece
  int cus = 0;
};
int xent_plan(const inl_softmax_xent_desc& d, XentPlan* p) {
  int rc = device_cus(&p->cus);
  if (rc) return rc;
  p->s = tile_plan(d.m, d.vocab, d.hidden, 0, false, 1, p->cus);
  p->piece = piece_cols(d.m, d.vocab);
  p->g = tile_plan(d.m, p->piece, d.hidden, 0, false, 1, p->cus);
  p->dw = tile_plan(std::min(p->piece, d.vocab), d.hidden, d.m, 2, false, MAX_SPLITS, p->cus);
  p->dx = tile_plan(d.m, d.hidden, p->piece, 1, false, MAX_SPLITS, p->cus);
  return INL_OK;
}

size_t xent_need(const inl_softmax_xent_desc& d, const XentPlan& p, bool backward) {
  Carve c(nullptr);
  if (!backward) {
    c.take((size_t)stat_blocks(p.s.shape, d.vocab) * (size_t)d.m * 8);
    c.take((size_t)d.m * 4);
    return c.used;
  }
  c.take((size_t)d.m * (size_t)p.piece * 2);
  c.take((size_t)d.m * (size_t)d.hidden * 4);
  c.take(colsum_bytes(d.m, p.piece));
  c.take(std::max(tile_part_bytes(p.dw, std::min(p.piece, d.vocab), d.hidden), tile_part_bytes(p.dx, d.m, d.hidden)));
  return c.used;
}

}  // namespace

}  // namespace inl

extern "C" int inl_softmax_xent_workspace_size(const inl_softmax_xent_desc* d, int32_t backward, size_t* bytes) {
  using namespace inl;
  if (!bytes) return fail(INL_E_INVALID, "softmax_xent: bytes is NULL");
  int rc = xent_check(d);
  if (rc) return rc;
  XentPlan plan;
  if ((rc = xent_plan(*d, &plan))) return rc;
  *bytes = xent_need(*d, plan, backward != 0);
  return INL_OK;
}

extern "C" int inl_softmax_xent_fwd(const inl_softmax_xent_desc* d, const void* x, const void* w, const float* bias,
                                    const int32_t* targets, float* loss, float* lse, void* ws, size_t ws_bytes,
                                    void* stream) {
  using namespace inl;
  hipStream_t st = (hipStream_t)stream;
  int rc = xent_check(d);
  if (rc) return rc;
  if (d->m == 0) return INL_OK;
  const int64_t xs = d->x_stride ? d->x_stride : d->hidden, wst = d->w_stride ? d->w_stride : d->hidden;
  if ((rc = check_rows("softmax_xent: x", x, d->hidden, xs, INL_BF16))) return rc;
  if ((rc = check_rows("softmax_xent: w", w, d->hidden, wst, INL_BF16))) return rc;
  if ((uintptr_t)bias & 15) return fail(INL_E_INVALID, "softmax_xent: bias must be 16-byte aligned");
  if (!targets || !loss || !lse) return fail(INL_E_INVALID, "softmax_xent: targets, loss or lse is NULL");
  XentPlan plan;
  if ((rc = xent_plan(*d, &plan))) return rc;
  if ((rc = check_workspace("softmax_xent", ws, ws_bytes, xent_need(*d, plan, false)))) return rc;
  Carve c(ws);
  const int64_t blocks = stat_blocks(plan.s.shape, d->vocab);
  float2* part = (float2*)c.take((size_t)blocks * (size_t)d->m * 8);
  float* at = (float*)c.take((size_t)d->m * 4);
  TileParams p{};
  p.x = (const char*)x;
  p.w = (const char*)w;
  p.xs_b = xs * 2;
  p.ws_b = wst * 2;
  p.m = d->m;
  p.n = (int32_t)d->vocab;
  p.k = (int32_t)d->hidden;
  p.alpha = d->scale;
  p.bias = bias;
  p.target = targets;
  p.ignore = d->ignore_index;
  p.at = at;
  p.part = part;
  if ((rc = tile_nt_xent(p, plan.s, plan.cus, st))) return rc;
  hipLaunchKernelGGL(xent_join_kernel, dim3((unsigned)((d->m + 63) / 64)), dim3(JOIN_WAVES * 64), 0, st, part, blocks, d->m,
                     targets, at, d->ignore_index, d->vocab, loss, lse);
  INL_HIP_TRY(hipGetLastError());
  return INL_OK;
}

extern "C" int inl_softmax_xent_bwd(const inl_softmax_xent_desc* d, const float* dloss, const float* lse, const void* x,
                                    const void* w, const float* bias, const int32_t* targets, void* dx, void* dw,
                                    float* dbias, void* ws, size_t ws_bytes, void* stream) {
  using namespace inl;
  hipStream_t st = (hipStream_t)stream;
  int rc = xent_check(d);
  if (rc) return rc;
  const int64_t xs = d->x_stride ? d->x_stride : d->hidden, wst = d->w_stride ? d->w_stride : d->hidden;
  const int64_t dxs = d->dx_stride ? d->dx_stride : d->hidden, dws = d->dw_stride ? d->dw_stride : d->hidden;
  if (dx && !dtype_ok(d->dx_dtype)) return fail(INL_E_INVALID, "softmax_xent: dx_dtype must be INL_F32 or INL_BF16");
  if (dw && (rc = check_rows("softmax_xent: dw", dw, d->hidden, dws, d->dw_dtype))) return rc;
  if (d->m == 0) {
    if (dw && (rc = fill_zero(dw, d->vocab, d->hidden, dws, d->dw_dtype, st))) return rc;
    return dbias ? fill_zero(dbias, 1, d->vocab, d->vocab, INL_F32, st) : INL_OK;
  }
  if ((rc = check_rows("softmax_xent: x", x, d->hidden, xs, INL_BF16))) return rc;
  if ((rc = check_rows("softmax_xent: w", w, d->hidden, wst, INL_BF16))) return rc;
  if (dx && (rc = check_rows("softmax_xent: dx", dx, d->hidden, dxs, d->dx_dtype))) return rc;
  if ((uintptr_t)bias & 15) return fail(INL_E_INVALID, "softmax_xent: bias must be 16-byte aligned");
  if (!targets || !dloss || !lse) return fail(INL_E_INVALID, "softmax_xent: targets, dloss or lse is NULL");
  if (!dx && !dw && !dbias) return INL_OK;
  XentPlan plan;
  if ((rc = xent_plan(*d, &plan))) return rc;
  if ((rc = check_workspace("softmax_xent", ws, ws_bytes, xent_need(*d, plan, true)))) return rc;
  Carve c(ws);
  char* g = c.take((size_t)d->m * (size_t)plan.piece * 2);
  float* dxf = (float*)c.take((size_t)d->m * (size_t)d->hidden * 4);
  float* sums = (float*)c.take(colsum_bytes(d->m, plan.piece));
  float* part = (float*)c.take(0);
  for (int64_t v0 = 0; v0 < d->vocab; v0 += plan.piece) {
    const int64_t cols = std::min(plan.piece, d->vocab - v0), cols8 = (cols + 7) / 8 * 8;
    const bool last = v0 + cols == d->vocab;
    const char* wp = (const char*)w + v0 * wst * 2;
    TileParams p{};
    p.x = (const char*)x;
    p.w = wp;
    p.xs_b = xs * 2;
    p.ws_b = wst * 2;
    p.m = d->m;
    p.n = (int32_t)cols;
    p.k = (int32_t)d->hidden;
    p.alpha = d->scale;
    p.bias = bias ? bias + v0 : nullptr;
    p.target = targets;
    p.ignore = d->ignore_index;
    p.col0 = (int32_t)v0;
    p.lse = lse;
    p.dl = dloss;
    p.vocab = (int32_t)d->vocab;
    p.y = g;
    p.ys = plan.piece;
    p.n_store = (int32_t)cols8;
    if ((rc = tile_nt_dxent(p, plan.g, plan.cus, st))) return rc;
    if (dbias && (rc = act_bwd(d->m, cols, g, plan.piece, nullptr, 0, ACT_NONE, nullptr, dbias + v0, sums, st))) return rc;
    TileParams q{};
    q.alpha = d->scale;
    q.beta = 1.f;
    q.act = ACT_NONE;
    q.x = g;
    q.xs_b = plan.piece * 2;
    if (dw) {
      q.w = (const char*)x;
      q.ws_b = xs * 2;
      q.m = cols;
      q.n = (int32_t)d->hidden;
      q.k = (int32_t)d->m;
      q.y = (char*)dw + v0 * dws * dtype_size(d->dw_dtype);
      q.ys = dws;
      if ((rc = tile_tn_linear(q, plan.dw, d->dw_dtype == INL_BF16, part, plan.cus, st))) return rc;
    }
    if (dx) {
      // dx adds up in f32 over the pieces and is rounded with the last one
      q.w = wp;
      q.ws_b = wst * 2;
      q.m = d->m;
      q.n = (int32_t)d->hidden;
      q.k = (int32_t)cols;
      q.res = v0 ? (const char*)dxf : nullptr;
      q.rs = d->hidden;
      q.res_bf16 = 0;
      q.y = last ? (char*)dx : (char*)dxf;
      q.ys = last ? dxs : d->hidden;
      TilePlan t = plan.dx;
      if (cols != plan.piece) {   // the last piece: the same splits or fewer
        const int64_t kst = (cols + TG_BK - 1) / TG_BK;
        t.splits = (int)((kst + t.kper - 1) / t.kper);
      }
      if ((rc = tile_nn_linear(q, t, last && d->dx_dtype == INL_BF16, part, plan.cus, st))) return rc;
    }
  }
  return INL_OK;
}
