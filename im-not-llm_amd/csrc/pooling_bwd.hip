// Gradients of the mean and last-token pooling (pooling.hip). Bound by the rows they write:
// a workgroup takes PB_ROWS rows, finds the text of the first in cu (64 entries per step of
// the search), and writes them text by text.
//
// Mean: a lane owns 8 columns of the text's gradient, made once in registers, and writes
// them to every PASS-th row. Through the unit length y = m / s it needs |m|^2 and m . d, two sums
// over the row that each workgroup makes by itself (8 KB read per 64 KB written).
//
// Last token: y = z / |z|, z = x / rms(x) w. y does not change with the size of x but for the
// epsilons: with size^2 = |z|^2 + e, e = 1e-12, the mean that the norm's gradient subtracts is
// mean(dn x / rms) = (x w . d) e / (rms size^3 n), no difference of near values. So one pass of
// three sums (x^2, (x w)^2, x w . d) gives the gradient.
//
// Mean of 26,923 x 768 rows in bf16: 10.8 us (3.9 TB/s; 17.1 with a search for the text in rounds of
// dependent loads). Last token of 14,716 x 1,024: 8.2 (3.7 TB/s; 9.1 with a text's columns loaded in turn) and
// 3.6 for the join of dweight. 16 rows per workgroup instead of 32: the same; 64: 9.3.
#include <algorithm>

#include "norm_rope.hpp"
#include "train_ops.hpp"

#include "inl_train.h"

namespace inl {

namespace {

constexpr int PB_ROWS = 32;
constexpr int PB_KEPT = 4;
constexpr float PB_UNIT_EPS = 1e-12f;

// Number of entries of cu[0 .. n] that are <= r: one more than the text of row r (if any). The
// whole wave takes part: up to 255 texts in one round of loads, more in a search of 64 ways.
__device__ __forceinline__ int cu_upto(const int32_t* cu, int n, int64_t r) {
  const int lane = threadIdx.x & 63;
  if (n < 256) {
    int count = 0;
    int32_t e[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) e[i] = cu[min(lane + 64 * i, n)];
#pragma unroll
    for (int i = 0; i < 4; ++i)
      count += __builtin_popcountll(__builtin_amdgcn_ballot_w64(lane + 64 * i <= n && (int64_t)e[i] <= r));
    return count;
  }
  int lo = 0, hi = n + 1;   // the answer is in [lo, hi]
  while (hi > lo) {
    const int step = (hi - lo + 63) / 64;
    const int at = lo + (lane + 1) * step - 1;   // the last entry of each of 64 pieces
    const bool in = at < hi && (int64_t)cu[at] <= r;
    const int pieces = __builtin_popcountll(__builtin_amdgcn_ballot_w64(in));
    lo += pieces * step;
    hi = min(hi, lo + step - 1);
  }
  return lo;
}

// Sums of N values over the workgroup, in all lanes.
template <int N>
__device__ __forceinline__ void wg_sums(float (&v)[N], float (*red)[4]) {
  __syncthreads();
#pragma unroll
  for (int i = 0; i < N; ++i) {
    v[i] = wave_sum(v[i]);
    if ((threadIdx.x & 63) == 0) red[i][threadIdx.x >> 6] = v[i];
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = (red[i][0] + red[i][1]) + (red[i][2] + red[i][3]);
}

template <typename T>
__device__ __forceinline__ float ld1(const char* p, int64_t i) {
  if constexpr (sizeof(T) == 2) return (float)reinterpret_cast<const bf16*>(p)[i];
  else return reinterpret_cast<const float*>(p)[i];
}
template <typename T>
__device__ __forceinline__ void st1(char* p, int64_t i, float v) {
  if constexpr (sizeof(T) == 2) reinterpret_cast<bf16*>(p)[i] = (bf16)v;
  else reinterpret_cast<float*>(p)[i] = v;
}

template <int V>
__device__ __forceinline__ void load_cols(const float* p, float (&v)[V]) {
#pragma unroll
  for (int e = 0; e < V; ++e) v[e] = p[e];
}

// V columns per lane: 8 (16-byte aligned rows of multiples of 8 columns) or 1.
template <typename T, int V>
__global__ __launch_bounds__(256) void pool_mean_bwd_kernel(const int32_t* cu, int n_texts, int dim, int64_t rows,
                                                            const float* dp, const float* mean, char* out, int64_t stride) {
  __shared__ float red[2][4];
  const int64_t first = (int64_t)blockIdx.x * PB_ROWS, last = min(first + PB_ROWS, rows);
  const int lanes = dim / V;                         // lanes of a row
  const int pass = max(1, 256 / lanes);              // rows written side by side
  const int sub = lanes <= 256 ? threadIdx.x / lanes : 0;
  const int l0 = lanes <= 256 ? threadIdx.x - sub * lanes : threadIdx.x;
  int b = n_texts ? cu_upto(cu, n_texts, first) - 1 : 0;
  for (int64_t r = first; r < last; ++b) {           // text b (none before the first or behind the last one)
    const bool some = b >= 0 && b < n_texts;
    const int64_t end = b < n_texts ? min(last, max(r, (int64_t)cu[b + 1])) : last;
    if (end == r) continue;                          // (b only grows, to n_texts at most)
    float by_d = 0.f, by_m = 0.f;                    // the gradient is by_d d - by_m mean
    const int64_t row = some ? (int64_t)b * dim : 0;
    // a lane's columns of the first round stay in registers from the sums to the gradient
    float d0[V] = {}, m0[V] = {};
    if (some && l0 < lanes) {
      load_cols<V>(dp + row + (int64_t)l0 * V, d0);
      if (mean) load_cols<V>(mean + row + (int64_t)l0 * V, m0);
    }
    if (some) {
      by_d = 1.f / (float)((int64_t)cu[b + 1] - cu[b]);
      if (mean) {
        float s[2] = {0.f, 0.f};                     // |mean|^2, mean . d
        if (sub == 0)
          for (int l = l0; l < lanes; l += 256) {
            float d[V], m[V];
#pragma unroll
            for (int e = 0; e < V; ++e) {
              d[e] = d0[e];
              m[e] = m0[e];
            }
            if (l != l0) {
              load_cols<V>(dp + row + (int64_t)l * V, d);
              load_cols<V>(mean + row + (int64_t)l * V, m);
            }
#pragma unroll
            for (int e = 0; e < V; ++e) {
              s[0] += m[e] * m[e];
              s[1] += m[e] * d[e];
            }
          }
        wg_sums<2>(s, red);
        const float s2 = s[0] + PB_UNIT_EPS;
        by_d /= sqrtf(s2);
        by_m = by_d * s[1] / s2;
      }
    }
    for (int l = l0; l < lanes && sub < pass; l += 256) {
      float g[V];
      if (l != l0 && some) {
        load_cols<V>(dp + row + (int64_t)l * V, d0);
        if (mean) load_cols<V>(mean + row + (int64_t)l * V, m0);
      }
#pragma unroll
      for (int e = 0; e < V; ++e) g[e] = some ? by_d * d0[e] - (mean ? by_m * m0[e] : 0.f) : 0.f;
      for (int64_t i = r + sub; i < end; i += pass) {
        if constexpr (V == 8) store8<T>(out + (i * stride + (int64_t)l * 8) * (int64_t)sizeof(T), g);
        else st1<T>(out, i * stride + l, g[0]);
      }
    }
    r = end;
  }
}

// Workgroups [0, n_texts): the last row of a text; the others: zeros in every other row.
template <typename T, typename TO, int V>
__global__ __launch_bounds__(256) void pool_last_bwd_kernel(const int32_t* cu, int n_texts, int dim, int64_t rows,
                                                            const char* hidden, int64_t stride, const char* weight,
                                                            float eps, const float* dp, char* out, int64_t os,
                                                            float* part) {
  if ((int)blockIdx.x < n_texts) {
    __shared__ float red[3][4];
    const int b = blockIdx.x;
    const int64_t row = (int64_t)cu[b + 1] - 1;
    const float* d = dp + (int64_t)b * dim;
    float* dw = part ? part + (int64_t)b * dim : nullptr;
    if (cu[b + 1] <= cu[b] || row < 0 || row >= rows) {   // no row, no gradient
      if (dw)
        for (int c = threadIdx.x; c < dim; c += 256) dw[c] = 0.f;
      return;
    }
    const char* x = hidden + row * stride * (int64_t)sizeof(T);
    // the first PB_KEPT columns of a lane stay in registers: their loads are under way together
    float kx[PB_KEPT], kw[PB_KEPT], kd[PB_KEPT];
    float s[3] = {0.f, 0.f, 0.f};
#pragma unroll
    for (int k = 0; k < PB_KEPT; ++k) {
      const int c = min((int)threadIdx.x + 256 * k, dim - 1);
      kx[k] = ld1<T>(x, c);
      kw[k] = weight ? ld1<T>(weight, c) : 1.f;
      kd[k] = d[c];
    }
    auto sums = [&](float v, float w, float g) {
      const float z = v * w;
      s[0] += v * v;
      s[1] += z * z;
      s[2] += z * g;
    };
#pragma unroll
    for (int k = 0; k < PB_KEPT; ++k)
      if ((int)threadIdx.x + 256 * k < dim) sums(kx[k], kw[k], kd[k]);
    for (int c = threadIdx.x + 256 * PB_KEPT; c < dim; c += 256) sums(ld1<T>(x, c), weight ? ld1<T>(weight, c) : 1.f, d[c]);
    wg_sums<3>(s, red);
    const float xx = s[0], zz = s[1], zd = s[2];
    const float inv = 1.0f / sqrtf(xx / (float)dim + eps);
    const float s2 = inv * inv * zz + PB_UNIT_EPS, is = 1.0f / sqrtf(s2);
    const float along = inv * zd / s2;                                              // y . d / size
    const float mean = inv * zd * is * (PB_UNIT_EPS / s2) / (float)dim;             // of dn x / rms
    auto put = [&](int c, float v, float w, float g) {
      const float hat = v * inv;
      const float dz = is * (g - hat * w * along);
      st1<TO>(out, row * os + c, inv * (dz * w - hat * mean));
      if (dw) dw[c] = dz * hat;
    };
#pragma unroll
    for (int k = 0; k < PB_KEPT; ++k) {
      const int c = threadIdx.x + 256 * k;
      if (c < dim) put(c, kx[k], kw[k], kd[k]);
    }
    for (int c = threadIdx.x + 256 * PB_KEPT; c < dim; c += 256) put(c, ld1<T>(x, c), weight ? ld1<T>(weight, c) : 1.f, d[c]);
    return;
  }
  __shared__ int taken[PB_ROWS];
  const int64_t first = (int64_t)(blockIdx.x - n_texts) * PB_ROWS, last = min(first + PB_ROWS, rows);
  if (threadIdx.x < PB_ROWS) taken[threadIdx.x] = 0;
  __syncthreads();
  // texts that end in these rows: entries cu[b + 1] in (first, last]
  const int b0 = n_texts ? max(cu_upto(cu, n_texts, first) - 1, 0) : 0;
  for (int b = b0 + (int)threadIdx.x; b < n_texts; b += 256) {
    const int64_t end = cu[b + 1];
    if (end > last) break;
    if (end > cu[b] && end > first) taken[end - 1 - first] = 1;
  }
  __syncthreads();
  const int lanes = dim / V;                         // lanes of a row; short rows are written side by side
  const int pass = max(1, 256 / lanes), sub = lanes <= 256 ? threadIdx.x / lanes : 0;
  const int l0 = lanes <= 256 ? threadIdx.x - sub * lanes : threadIdx.x;
  const float zero[8] = {};
  if (sub >= pass) return;
  for (int64_t i = first + sub; i < last; i += pass) {
    if (taken[i - first]) continue;
    for (int l = l0; l < lanes; l += 256) {
      if constexpr (V == 8) store8<TO>(out + (i * os + (int64_t)l * 8) * (int64_t)sizeof(TO), zero);
      else st1<TO>(out, i * os + l, 0.f);
    }
  }
}

int pool_bwd_check(const char* what, int32_t n_texts, const int32_t* cu, int32_t dim, int64_t rows, int64_t stride,
                   int32_t dtype, const float* dp, const void* out) {
  const std::string w(what);
  if (n_texts < 0 || dim <= 0 || rows < 0 || !dtype_ok(dtype)) return fail(INL_E_INVALID, w + ": bad n_texts, hidden_dim, rows or dtype");
  // (a grid has fewer than 2^32 threads: 256 for a text, and for PB_ROWS rows)
  if (n_texts + (rows + PB_ROWS - 1) / PB_ROWS >= (int64_t)1 << 24)
    return fail(INL_E_UNSUPPORTED, w + ": n_texts + rows / 32 must stay below 2^24");
  if (stride < dim) return fail(INL_E_INVALID, w + ": the row stride must cover hidden_dim");
  if (rows && (!out || (n_texts && (!cu || !dp)))) return fail(INL_E_INVALID, w + ": NULL pointer");
  if ((((uintptr_t)cu | (uintptr_t)dp) & 3) || ((uintptr_t)out % dtype_size(dtype)))
    return fail(INL_E_INVALID, w + ": misaligned pointer");
  return INL_OK;
}

bool pool_vec(const void* out, int32_t dim, int64_t stride, int32_t dtype) {
  return dim % 8 == 0 && ((uintptr_t)out & 15) == 0 && (stride * dtype_size(dtype)) % 16 == 0;
}

}  // namespace

}  // namespace inl

extern "C" int inl_pool_mean_bwd(int32_t n_texts, const int32_t* cu, int32_t dim, int64_t rows, int64_t row_stride,
                                 int32_t dtype, const float* dpooled, const float* mean, void* dhidden, void* stream) {
  using namespace inl;
  const int64_t stride = row_stride ? row_stride : dim;
  int rc = pool_bwd_check("pool_mean_bwd", n_texts, cu, dim, rows, stride, dtype, dpooled, dhidden);
  if (rc) return rc;
  if ((uintptr_t)mean & 3) return fail(INL_E_INVALID, "pool_mean_bwd: misaligned pointer");
  const int64_t es = dtype_size(dtype), in = (int64_t)n_texts * dim * 4;
  const Rows o{dhidden, rows, dim * es, stride * es};
  if (rows_meet(o, {dpooled, 1, in, in}) || rows_meet(o, {mean, 1, in, in}) ||
      rows_meet(o, {cu, 1, ((int64_t)n_texts + 1) * 4, ((int64_t)n_texts + 1) * 4}))
    return fail(INL_E_INVALID, "pool_mean_bwd: dhidden overlaps an input");
  if (rows == 0) return INL_OK;
  const dim3 grid((unsigned)((rows + PB_ROWS - 1) / PB_ROWS)), block(256);
  hipStream_t st = (hipStream_t)stream;
#define INL_POOL(T, V)                                                                                                     \
  hipLaunchKernelGGL((pool_mean_bwd_kernel<T, V>), grid, block, 0, st, cu, n_texts, dim, rows, dpooled, mean, (char*)dhidden, stride)
  if (pool_vec(dhidden, dim, stride, dtype)) {
    if (dtype == INL_BF16) INL_POOL(bf16, 8);
    else INL_POOL(float, 8);
  } else {
    if (dtype == INL_BF16) INL_POOL(bf16, 1);
    else INL_POOL(float, 1);
  }
#undef INL_POOL
  INL_HIP_TRY(hipGetLastError());
  return INL_OK;
}

extern "C" int inl_pool_last_bwd_workspace_size(int32_t n_texts, int32_t dim, size_t* bytes) {
  using namespace inl;
  if (!bytes || n_texts < 0 || dim <= 0) return fail(INL_E_INVALID, "pool_last_bwd: bad arguments");
  *bytes = (size_t)n_texts * (size_t)dim * 4;
  return INL_OK;
}

extern "C" int inl_pool_last_bwd(int32_t n_texts, const int32_t* cu, int32_t dim, int64_t rows, int64_t row_stride,
                                 int32_t dtype, const float* dpooled, const void* hidden, const void* weight, float eps,
                                 int64_t dx_stride, int32_t dx_dtype, void* dhidden, float* dweight, void* ws,
                                 size_t ws_bytes, void* stream) {
  using namespace inl;
  hipStream_t st = (hipStream_t)stream;
  const int64_t stride = row_stride ? row_stride : dim, os = dx_stride ? dx_stride : dim;
  int rc = pool_bwd_check("pool_last_bwd", n_texts, cu, dim, rows, os, dx_dtype, dpooled, dhidden);
  if (rc) return rc;
  if (!dtype_ok(dtype) || stride < dim || !(eps >= 0.f)) return fail(INL_E_INVALID, "pool_last_bwd: bad dtype, row stride or eps");
  if (rows && n_texts && !hidden) return fail(INL_E_INVALID, "pool_last_bwd: NULL pointer");
  const int64_t es = dtype_size(dtype), eo = dtype_size(dx_dtype), in = (int64_t)n_texts * dim * 4;
  if (((uintptr_t)hidden | (uintptr_t)weight) % es || ((uintptr_t)dweight & 3))
    return fail(INL_E_INVALID, "pool_last_bwd: misaligned pointer");
  const Rows o{dhidden, rows, dim * eo, os * eo}, hid{hidden, rows, dim * es, stride * es}, gr{dpooled, 1, in, in},
      wt{weight, 1, dim * es, dim * es}, dwr{dweight, 1, (int64_t)dim * 4, (int64_t)dim * 4},
      tab{cu, 1, ((int64_t)n_texts + 1) * 4, ((int64_t)n_texts + 1) * 4};
  for (const Rows& out : {o, dwr})
    if (rows_meet(out, hid) || rows_meet(out, gr) || rows_meet(out, wt) || rows_meet(out, tab))
      return fail(INL_E_INVALID, "pool_last_bwd: an output overlaps an input");
  if (rows_meet(o, dwr)) return fail(INL_E_INVALID, "pool_last_bwd: dhidden overlaps dweight");
  if (dweight && (rows == 0 || n_texts == 0) && (rc = fill_zero(dweight, 1, dim, dim, INL_F32, st))) return rc;
  if (rows == 0) return INL_OK;   // (a text without rows has no gradient)
  const bool join = dweight && n_texts > 1;
  if (join && (rc = check_workspace("pool_last_bwd", ws, ws_bytes, (size_t)n_texts * (size_t)dim * 4))) return rc;
  float* part = join ? (float*)ws : dweight;
  const int64_t fills = (rows + PB_ROWS - 1) / PB_ROWS;
  const dim3 grid((unsigned)(n_texts + fills)), block(256);
#define INL_POOL(T, TO, V)                                                                                            \
  hipLaunchKernelGGL((pool_last_bwd_kernel<T, TO, V>), grid, block, 0, st, cu, n_texts, dim, rows, (const char*)hidden, \
                     stride, (const char*)weight, eps, dpooled, (char*)dhidden, os, part)
  const bool vec = pool_vec(dhidden, dim, os, dx_dtype);
  auto launch = [&](auto t, auto to) {
    using T = decltype(t);
    using TO = decltype(to);
    if (vec) INL_POOL(T, TO, 8);
    else INL_POOL(T, TO, 1);
  };
#undef INL_POOL
  if (dtype == INL_BF16 && dx_dtype == INL_BF16) launch(bf16{}, bf16{});
  else if (dtype == INL_BF16) launch(bf16{}, float{});
  else if (dx_dtype == INL_BF16) launch(float{}, bf16{});
  else launch(float{}, float{});
  INL_HIP_TRY(hipGetLastError());
  return join ? colsum_join(part, n_texts, dim, dweight, dim, nullptr, st) : INL_OK;
}
