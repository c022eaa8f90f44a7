// Gradients of the q/k prologue y = R(x / rms(x) * weight), per (token, head):
//
//   dn   = R^T dy                     (the rotation by the negative angle)
//   xhat = x / rms(x)
//   dweight += dn * xhat
//   dx   = (weight dn - xhat mean(weight dn xhat)) / rms(x)
//
// Bound by memory: x and dy read once, dx written once (125 us for 32,003 tokens of
// 16 + 8 heads of 128 in bf16, 4.7 TB/s; a copy reaches 4.8; f32 5.2). The layout is
// the forward's (norm_rope.hip): G = head_dim / 8 lanes own a unit of four heads (f32:
// two) of a token, 8 values of every head each, so the two sums of a row are one
// cross-lane reduction each and a rotation partner is a lane away. Units, not whole
// tokens, so that a short batch fills the card too: 500 tokens took 28 us when a lane
// group walked all the heads of its token, and take 11.6. A lane keeps its 8 columns of
// dq_weight and dk_weight in f32 registers over all units of its workgroup; the groups
// of a workgroup meet in LDS, the workgroups in a second kernel, in a fixed order.
#include <type_traits>

#include "norm_rope.hpp"
#include "train_ops.hpp"

namespace inl {

namespace {

struct NormRopeBwdParams {
  const char* dy;
  const char* x;
  char* dx;
  const char* qw;
  const char* kw;
  const int32_t* rows;
  const float* cos;
  const float* sin;
  const float* cos2;
  const float* sin2;
  float* part;             // [workgroups][2 head_dim], or null
  int64_t n_tokens, x_stride, y_stride, d_stride;
  int32_t heads, q_heads, head_dim;
  int32_t norm, rotary_dim, sections, table_rows, round_tables;
  float eps;
};

// TX: x and dx, TY: dy. HB heads of a token are in flight at a time.
template <typename TX, typename TY, int G>
__global__ __launch_bounds__(256) void norm_rope_bwd_kernel(NormRopeBwdParams p) {
  constexpr int HB = sizeof(TX) == 2 ? 4 : 2;
  constexpr int GROUPS = 256 / G;
  __shared__ float red[256][17];
  const int lane = threadIdx.x & 63;
  const int j = lane & (G - 1);
  const int grp = threadIdx.x / G;
  const bool adjacent = p.sections == INL_ROPE_INTERLEAVED;
  const bool inner8 = p.rotary_dim == 8 && p.sections == INL_ROPE_HALF;

  // rotation geometry of this lane, as in the forward: 0 none, 1 pairs (e, e + 4),
  // 2 a partner lane, 3 pairs (2i, 2i + 1)
  int mode = 0, partner = lane, half = 0, tw = p.rotary_dim >> 1, tcol = 0;
  bool first = true, second_sec = false, xor_partner = false;
  if (p.rotary_dim > 0) {
    if (inner8) {
      mode = j == 0 ? 1 : 0;
    } else if (adjacent) {
      mode = 8 * j < p.rotary_dim ? 3 : 0;
      tcol = mode ? 4 * j : 0;
    } else {
      const int sec = p.sections == INL_ROPE_AXIAL ? G >> 1 : p.rotary_dim >> 3;
      second_sec = p.sections == INL_ROPE_AXIAL && j >= sec;
      const int jj = j - (second_sec ? sec : 0);
      half = sec >> 1;
      tw = half * 8;
      xor_partner = half > 0 && (half & (half - 1)) == 0;
      if (jj < sec) {
        mode = 2;
        first = jj < half;
        partner = lane + (first ? half : -half);
        tcol = 8 * (first ? jj : jj - half);
      }
    }
  }
  const float* ct = second_sec ? p.cos2 : p.cos;
  const float* st = second_sec ? p.sin2 : p.sin;

  float wq[8], wk[8], dq[8] = {}, dk[8] = {};
#pragma unroll
  for (int e = 0; e < 8; ++e) wq[e] = wk[e] = 1.f;
  if (p.norm && p.qw) load8<TX>(p.qw + 8 * j * (int)sizeof(TX), wq);
  if (p.norm && p.kw) load8<TX>(p.kw + 8 * j * (int)sizeof(TX), wk);

  // units: HB heads of a token, a lane group each; every lane of a wave runs the
  // same iterations (the reductions need all of them)
  const int chunks = (p.heads + HB - 1) / HB;
  const int64_t units = p.n_tokens * chunks, step = (int64_t)gridDim.x * GROUPS;
  const int64_t step_tok = step / chunks;
  const int step_chunk = (int)(step - step_tok * chunks);
  int64_t u = (int64_t)blockIdx.x * GROUPS + grp, tok = u / chunks;
  int chunk = (int)(u - tok * chunks);
  for (int64_t u0 = u - grp; u0 < units; u0 += step) {
    const bool valid = tok < p.n_tokens;
    const int64_t tc = valid ? tok : 0;
    const int h0 = chunk * HB;
    tok += step_tok;
    chunk += step_chunk;
    if (chunk >= chunks) {
      chunk -= chunks;
      ++tok;
    }
    const char* yt = p.dy + (tc * p.y_stride + 8 * j) * (int64_t)sizeof(TY);
    const char* xt = p.x + (tc * p.x_stride + 8 * j) * (int64_t)sizeof(TX);
    char* dt = p.dx + (tc * p.d_stride + 8 * j) * (int64_t)sizeof(TX);
    Raw8 ry[HB], rx[HB];
#pragma unroll
    for (int i = 0; i < HB; ++i) {
      const int64_t h = min(h0 + i, p.heads - 1) * (int64_t)p.head_dim;
      load_raw<TY>(yt + h * (int64_t)sizeof(TY), ry[i]);
      if (p.norm) load_raw<TX>(xt + h * (int64_t)sizeof(TX), rx[i]);
    }
    float c[8], sn[8];
    bool bad = false;
    if (p.rotary_dim > 0) {
      const int32_t pos = p.rows[tc];
      bad = mode != 0 && (pos < 0 || pos >= p.table_rows);
      const int64_t at = (int64_t)min(max(pos, 0), p.table_rows - 1) * tw + tcol;
      if (inner8 || adjacent) {
        const f32x4 c4 = *reinterpret_cast<const f32x4*>(ct + at), s4 = *reinterpret_cast<const f32x4*>(st + at);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          c[e] = adjacent ? c4[e >> 1] : c4[e & 3];
          sn[e] = adjacent ? s4[e >> 1] : s4[e & 3];
        }
      } else {
        load8<float>(reinterpret_cast<const char*>(ct + at), c);
        load8<float>(reinterpret_cast<const char*>(st + at), sn);
      }
      if (p.round_tables)
#pragma unroll
        for (int e = 0; e < 8; ++e) { c[e] = round_bf16(c[e]); sn[e] = round_bf16(sn[e]); }
    }
#pragma unroll
    for (int i = 0; i < HB; ++i) {
      const bool live = valid && h0 + i < p.heads;
      float d[8];
      unpack8<TY>(ry[i], d);
      if (mode == 1) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float a = d[e], b = d[e + 4];
          d[e] = a * c[e] + b * sn[e];
          d[e + 4] = b * c[e] - a * sn[e];
        }
      } else if (mode == 3) {
#pragma unroll
        for (int e = 0; e < 8; e += 2) {
          const float a = d[e], b = d[e + 1];
          d[e] = a * c[e] + b * sn[e];
          d[e + 1] = b * c[e] - a * sn[e];
        }
      }
      if (p.rotary_dim > 0 && !inner8 && !adjacent) {   // uniform
        float pv[8];
        if (xor_partner)
          xor_lanes8(d, pv, half, lane);
        else
#pragma unroll
          for (int e = 0; e < 8; ++e) pv[e] = __shfl(d[e], partner, 64);
        if (mode == 2)
#pragma unroll
          for (int e = 0; e < 8; ++e) d[e] = first ? d[e] * c[e] + pv[e] * sn[e] : d[e] * c[e] - pv[e] * sn[e];
      }
      if (bad)
#pragma unroll
        for (int e = 0; e < 8; ++e) d[e] = __builtin_nanf("");
      if (p.norm) {
        const bool is_q = h0 + i < p.q_heads;
        float v[8];
        unpack8<TX>(rx[i], v);
        float ss = 0.f;
#pragma unroll
        for (int e = 0; e < 8; ++e) ss += v[e] * v[e];
        ss = group_sum<G>(ss);
        const float inv = 1.0f / sqrtf(ss / (float)p.head_dim + p.eps);
        float dot = 0.f, wd[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          v[e] *= inv;
          const float dw = d[e] * v[e];
          if (live) {
            dq[e] += is_q ? dw : 0.f;
            dk[e] += is_q ? 0.f : dw;
          }
          wd[e] = d[e] * (is_q ? wq[e] : wk[e]);
          dot += wd[e] * v[e];
        }
        dot = group_sum<G>(dot) / (float)p.head_dim;
#pragma unroll
        for (int e = 0; e < 8; ++e) d[e] = inv * (wd[e] - v[e] * dot);
      }
      if (live) store8<TX>(dt + (h0 + i) * (int64_t)p.head_dim * (int64_t)sizeof(TX), d);
    }
  }
  if (!p.part) return;   // uniform
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    red[threadIdx.x][e] = dq[e];
    red[threadIdx.x][8 + e] = dk[e];
  }
  __syncthreads();
  for (int c = threadIdx.x; c < 2 * p.head_dim; c += 256) {
    const int k = c >= p.head_dim, col = c - k * p.head_dim;
    float s = 0.f;
#pragma unroll 8
    for (int g = 0; g < GROUPS; ++g) s += red[g * G + (col >> 3)][8 * k + (col & 7)];
    p.part[(int64_t)blockIdx.x * 2 * p.head_dim + c] = s;
  }
}

// Workgroups, at most four per CU: each adds a row of partial sums to join. Eight take
// 29 us for 4,000 tokens where four take 24, and no less for 32,003. (A unit has two
// heads or more.)
int64_t bwd_groups(int64_t n_tokens, int heads, int head_dim, int cus) {
  const int64_t per = 256 / (head_dim / 8), units = n_tokens * ((heads + 1) / 2);
  return std::max<int64_t>(1, std::min<int64_t>((units + per - 1) / per, (int64_t)cus * 4));
}

}  // namespace

}  // namespace inl

extern "C" int inl_norm_rope_bwd_workspace_size(const inl_norm_rope_desc* d, size_t* bytes) {
  using namespace inl;
  if (!d || !bytes) return fail(INL_E_INVALID, "norm_rope_bwd: desc or bytes is NULL");
  if (d->n_tokens < 0 || d->heads <= 0 || d->head_dim < 8 || d->head_dim > 512)
    return fail(INL_E_INVALID, "norm_rope_bwd: bad n_tokens/heads/head_dim");
  int cus = 0, rc = device_cus(&cus);
  if (rc) return rc;
  *bytes = d->norm ? (size_t)bwd_groups(d->n_tokens, d->heads, d->head_dim, cus) * 2 * d->head_dim * 4 : 0;
  return INL_OK;
}

extern "C" int inl_norm_rope_qk_bwd(const inl_norm_rope_desc* d, int32_t q_heads, const void* dy, const void* x,
                                    void* dx, int64_t dx_row_stride, const void* q_weight, const void* k_weight,
                                    const int32_t* rows, const float* cos, const float* sin, const float* cos2, const float* sin2,
                                    float* dq_weight, float* dk_weight, void* ws, size_t ws_bytes, void* stream) {
  using namespace inl;
  hipStream_t st = (hipStream_t)stream;
  const int32_t none = 0;   // no tokens, no rows
  int rc = norm_rope_check(d, d && d->n_tokens == 0 ? &none : rows, cos, sin, cos2, sin2);
  if (rc) return rc;
  if (q_heads <= 0 || q_heads > d->heads) return fail(INL_E_INVALID, "norm_rope_bwd: need 0 < q_heads <= heads");
  if (q_heads == d->heads && (k_weight || dk_weight))
    return fail(INL_E_INVALID, "norm_rope_bwd: no k heads for k_weight or dk_weight");
  if (!d->norm && (dq_weight || dk_weight)) return fail(INL_E_INVALID, "norm_rope_bwd: no norm, no weight gradients");
  const int hd = d->head_dim;
  if (d->n_tokens == 0) {
    if (dq_weight && (rc = fill_zero(dq_weight, 1, hd, hd, INL_F32, st))) return rc;
    return dk_weight ? fill_zero(dk_weight, 1, hd, hd, INL_F32, st) : INL_OK;
  }
  const int64_t row = (int64_t)d->heads * hd;
  const int64_t xs = d->x_row_stride ? d->x_row_stride : row, ys = d->y_row_stride ? d->y_row_stride : row;
  const int64_t ds = dx_row_stride ? dx_row_stride : row;
  if (xs < row || ys < row || ds < row || ((xs | ds) * dtype_size(d->dtype)) % 16 || (ys * dtype_size(d->out_dtype)) % 16)
    return fail(INL_E_INVALID, "norm_rope_bwd: row strides must cover all heads, in 16-byte multiples");
  if (!dy || !dx || (d->norm && !x) ||
      (((uintptr_t)dy | (uintptr_t)dx | (uintptr_t)x | (uintptr_t)q_weight | (uintptr_t)k_weight) & 15))
    return fail(INL_E_INVALID, "norm_rope_bwd: dy, x, dx and the weights must be non-null and 16-byte aligned");
  // a unit of heads is read before it is written: at its own place, or nowhere near
  auto apart = [&](const void* at, int64_t stride, int32_t dtype) {
    if (at == dx && dtype == d->dtype && (stride == ds || d->n_tokens == 1)) return true;
    const int64_t in = dtype_size(dtype), out = dtype_size(d->dtype);
    return !rows_meet({at, d->n_tokens, row * in, stride * in}, {dx, d->n_tokens, row * out, ds * out});
  };
  if (!apart(dy, ys, d->out_dtype) || (d->norm && !apart(x, xs, d->dtype)))
    return fail(INL_E_INVALID, "norm_rope_bwd: dx overlaps dy or x, of another type or stride");
  int cus = 0;
  if ((rc = device_cus(&cus))) return rc;
  const int64_t groups = bwd_groups(d->n_tokens, d->heads, hd, cus);
  const bool sums = dq_weight || dk_weight;
  if (sums && (rc = check_workspace("norm_rope_bwd", ws, ws_bytes, (size_t)groups * 2 * hd * 4))) return rc;
  NormRopeBwdParams p{};
  p.dy = (const char*)dy;
  p.x = (const char*)x;
  p.dx = (char*)dx;
  p.qw = (const char*)q_weight;
  p.kw = (const char*)k_weight;
  p.rows = rows;
  p.cos = cos;
  p.sin = sin;
  p.cos2 = cos2;
  p.sin2 = sin2;
  p.part = sums ? (float*)ws : nullptr;
  p.n_tokens = d->n_tokens;
  p.x_stride = xs;
  p.y_stride = ys;
  p.d_stride = ds;
  p.heads = d->heads;
  p.q_heads = q_heads;
  p.head_dim = hd;
  p.norm = d->norm;
  p.rotary_dim = d->rotary_dim;
  p.sections = d->sections;
  p.table_rows = d->table_rows;
  p.round_tables = d->round_tables;
  p.eps = d->eps;
  const dim3 grid((unsigned)groups), block(256);
  auto launch = [&](auto tx, auto ty) {
    using TX = decltype(tx);
    using TY = decltype(ty);
    switch (hd >> 3) {
      case 1: hipLaunchKernelGGL((norm_rope_bwd_kernel<TX, TY, 1>), grid, block, 0, st, p); break;
      case 2: hipLaunchKernelGGL((norm_rope_bwd_kernel<TX, TY, 2>), grid, block, 0, st, p); break;
      case 4: hipLaunchKernelGGL((norm_rope_bwd_kernel<TX, TY, 4>), grid, block, 0, st, p); break;
      case 8: hipLaunchKernelGGL((norm_rope_bwd_kernel<TX, TY, 8>), grid, block, 0, st, p); break;
      case 16: hipLaunchKernelGGL((norm_rope_bwd_kernel<TX, TY, 16>), grid, block, 0, st, p); break;
      case 32: hipLaunchKernelGGL((norm_rope_bwd_kernel<TX, TY, 32>), grid, block, 0, st, p); break;
      default: hipLaunchKernelGGL((norm_rope_bwd_kernel<TX, TY, 64>), grid, block, 0, st, p);
    }
  };
  if (d->dtype == INL_BF16 && d->out_dtype == INL_BF16) launch(bf16{}, bf16{});
  else if (d->dtype == INL_BF16) launch(bf16{}, float{});
  else if (d->out_dtype == INL_BF16) launch(float{}, bf16{});
  else launch(float{}, float{});
  INL_HIP_TRY(hipGetLastError());
  return sums ? colsum_join((const float*)ws, groups, 2 * hd, dq_weight, hd, dk_weight, st) : INL_OK;
}
