// The residual stream's addition, with dropout, and the RMSNorm behind it, with their
// gradients (inl_add_rms_norm_fwd, inl_add_rms_norm_bwd):
//
//   h = residual + drop(x),  y = h / rms(h) * weight,  rms(h) = sqrt(mean(h^2) + eps)
//   dn = dy weight,  g = (dn - h / rms mean(dn h / rms)) / rms + dh
//   dresidual = g,  dx = drop(g),  dweight = sum over rows of dy h / rms
//
// Bound by memory: every input is read once and every output written once. A row stays in
// registers between its sums and its outputs, 8 values per lane and chunk: one wave per row up to 2,048
// columns, a workgroup per row above. Both sums of the backward (h^2 and dn h) are one pass. Its lanes
// keep their columns of dweight in f32 over all rows of a workgroup; the workgroups meet in
// a second kernel, in a fixed order.
//
// The dropout's mask is drawn again wherever it is needed and never stored: Philox 4x32-10 (Salmon,
// Moraes, Dror and Shaw, "Parallel random numbers: as easy as 1, 2, 3", 2011), one draw of 128
// bits for 8 elements, 16 bits each: with 32 bits an element the generator's multiplications
// would take longer than the memory does.
//
// 20,011 x 768, f32 stream, dropout 0.1: forward 36.5 us a call (5.0 TB/s), backward 51 and 5 for
// the join of dweight (4.8 TB/s without it); 65,536 x 1,024 in bf16, backward 107 us in all (5.0 TB/s). One row: 2.5.
// Wide rows, 2^26 values, bf16 x and y, dropout, kernel alone, TB/s of forward and backward in a bf16 / f32
// stream: 2,048 columns 5.6 and 4.4 / 5.5 and 5.1, 4,096 5.8 and 5.0 / 5.7 and 5.4, 8,192 5.5 and 4.6 / 5.5 and 5.1,
// 16,384 5.1 and 4.2 / 5.2 and 4.0: a row of more than 8,192 fills up to 336 registers of a lane in the backward, so
// one wave is on a SIMD in an f32 stream, and two in a bf16 one. The join of dweight takes 5 us to 4,096 columns, 7
// to 9 at 8,192, 14 to 15 at 16,384.
#include <algorithm>

#include "norm_rope.hpp"
#include "train_ops.hpp"

#include "inl_train.h"

namespace inl {

namespace {

struct AddNormParams {
  const char* x;         // forward: x; backward: dy
  const char* res;       // forward: residual; backward: dh
  const char* hin;       // backward: h
  const char* w;
  const int64_t* rng;
  char* h;               // forward: h; backward: dresidual
  char* y;               // forward: y; backward: dx
  float* part;           // backward: [workgroups][n], or null
  int64_t m, xs, rs, his, hs, ys;   // elements
  int32_t n, w16, drop, tag;
  float eps, keep_scale;
};

struct Draw {
  uint32_t w[4];
};

__device__ __forceinline__ Draw philox(uint64_t at, uint32_t tag, uint32_t step, uint32_t k0, uint32_t k1) {
  uint32_t c0 = (uint32_t)at, c1 = (uint32_t)(at >> 32), c2 = tag, c3 = step;
#pragma unroll
  for (int i = 0; i < 10; ++i) {
    const uint64_t a = (uint64_t)0xD2511F53u * c0, b = (uint64_t)0xCD9E8D57u * c2;
    c0 = (uint32_t)(b >> 32) ^ c1 ^ k0;
    c1 = (uint32_t)b;
    c2 = (uint32_t)(a >> 32) ^ c3 ^ k1;
    c3 = (uint32_t)a;
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
  return {{c0, c1, c2, c3}};
}

// The 8 values of group `at` of the row-major matrix, dropped or scaled.
__device__ __forceinline__ void drop8(const AddNormParams& p, uint64_t at, uint32_t step, uint32_t k0, uint32_t k1,
                                      float (&v)[8]) {
  const Draw d = philox(at, (uint32_t)p.tag, step, k0, k1);
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const uint32_t bits = e & 1 ? d.w[e >> 1] >> 16 : d.w[e >> 1] & 0xffffu;
    v[e] = bits >= (uint32_t)p.drop ? v[e] * p.keep_scale : 0.f;
  }
}

__device__ __forceinline__ void weight8(const AddNormParams& p, int col, float (&v)[8]) {
  if (!p.w) {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = 1.f;
  } else if (p.w16) {
    load8<bf16>(p.w + (int64_t)col * 2, v);
  } else {
    load8<float>(p.w + (int64_t)col * 4, v);
  }
}

// Sum of x over the W waves of a row, in all of them.
template <int W>
__device__ __forceinline__ float row_sum(float x, float* red) {
  x = wave_sum(x);
  if constexpr (W > 1) {
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = x;
    __syncthreads();
    x = 0.f;
#pragma unroll
    for (int i = 0; i < W; ++i) x += red[i];
  }
  return x;
}

// W waves per row (1 or 4), K chunks of 512 W columns.
template <typename TX, typename TR, typename TY, int W, int K>
__global__ __launch_bounds__(256) void add_norm_kernel(AddNormParams p) {
  constexpr int ROWS = 4 / W;
  __shared__ float red[4];
  const int64_t r = ((int64_t)blockIdx.y * gridDim.x + blockIdx.x) * ROWS + (W == 1 ? threadIdx.x >> 6 : 0);
  if (r >= p.m) return;   // uniform over the waves of a row
  const int j = W == 1 ? threadIdx.x & 63 : threadIdx.x;
  const char* xr = p.x + r * p.xs * (int64_t)sizeof(TX);
  const char* rr = p.res + r * p.rs * (int64_t)sizeof(TR);
  Raw8 rx[K], rres[K];
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const int c = min(8 * (j + 64 * W * k), p.n - 8);   // (past the row: loaded, not used)
    load_raw<TX>(xr + c * (int)sizeof(TX), rx[k]);
    if (p.res) load_raw<TR>(rr + c * (int)sizeof(TR), rres[k]);
  }
  uint32_t k0 = 0, k1 = 0, step = 0;
  if (p.drop) {
    const uint64_t seed = (uint64_t)p.rng[0];
    k0 = (uint32_t)seed;
    k1 = (uint32_t)(seed >> 32);
    step = (uint32_t)(uint64_t)p.rng[1];
  }
  float h[K][8], ss = 0.f;
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const int c = 8 * (j + 64 * W * k);
    unpack8<TX>(rx[k], h[k]);
    if (p.drop) drop8(p, (uint64_t)(r * p.n + c) >> 3, step, k0, k1, h[k]);
    if (p.res) {
      float v[8];
      unpack8<TR>(rres[k], v);
#pragma unroll
      for (int e = 0; e < 8; ++e) h[k][e] += v[e];
    }
    if (c < p.n)
#pragma unroll
      for (int e = 0; e < 8; ++e) ss += h[k][e] * h[k][e];
  }
  const float inv = 1.0f / sqrtf(row_sum<W>(ss, red) / (float)p.n + p.eps);
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const int c = 8 * (j + 64 * W * k);
    if (c >= p.n) break;
    if (p.h) store8<TR>(p.h + (r * p.hs + c) * (int64_t)sizeof(TR), h[k]);
    // y from the sum before its rounding to the stream's type
    float w[8];
    weight8(p, c, w);
#pragma unroll
    for (int e = 0; e < 8; ++e) h[k][e] = h[k][e] * inv * w[e];
    store8<TY>(p.y + (r * p.ys + c) * (int64_t)sizeof(TY), h[k]);
  }
}

template <typename TX, typename TR, typename TY, int W, int K>
__global__ __launch_bounds__(256) void add_norm_bwd_kernel(AddNormParams p) {
  constexpr int ROWS = 4 / W;
  __shared__ float red[4];
  __shared__ float cols[W == 1 ? 4 : 1][W == 1 ? 512 * K : 1];
  const int wave = threadIdx.x >> 6;
  const int j = W == 1 ? threadIdx.x & 63 : threadIdx.x;
  float dw[K][8] = {};
  uint32_t k0 = 0, k1 = 0, step = 0;
  if (p.drop && p.y) {
    const uint64_t seed = (uint64_t)p.rng[0];
    k0 = (uint32_t)seed;
    k1 = (uint32_t)(seed >> 32);
    step = (uint32_t)(uint64_t)p.rng[1];
  }
  for (int64_t r = (int64_t)blockIdx.x * ROWS + (W == 1 ? wave : 0); r < p.m; r += (int64_t)gridDim.x * ROWS) {
    const char* yr = p.x + r * p.xs * (int64_t)sizeof(TY);
    const char* hr = p.hin + r * p.his * (int64_t)sizeof(TR);
    const char* rr = p.res + r * p.rs * (int64_t)sizeof(TR);
    Raw8 rh[K], ry[K], rres[K];
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int c = min(8 * (j + 64 * W * k), p.n - 8);
      load_raw<TR>(hr + c * (int)sizeof(TR), rh[k]);
      load_raw<TY>(yr + c * (int)sizeof(TY), ry[k]);
      if (p.res) load_raw<TR>(rr + c * (int)sizeof(TR), rres[k]);
    }
    float ss = 0.f, dot = 0.f;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int c = 8 * (j + 64 * W * k);
      if (c < p.n) {
        float h[8], d[8], w[8];
        unpack8<TR>(rh[k], h);
        unpack8<TY>(ry[k], d);
        weight8(p, c, w);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          ss += h[e] * h[e];
          dot += d[e] * w[e] * h[e];
        }
      }
    }
    const float inv = 1.0f / sqrtf(row_sum<W>(ss, red) / (float)p.n + p.eps);
    const float mean = row_sum<W>(dot, red) * inv / (float)p.n;   // of dn h / rms
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int c = 8 * (j + 64 * W * k);
      if (c < p.n) {
        float h[8], d[8], w[8], g[8];
        unpack8<TR>(rh[k], h);
        unpack8<TY>(ry[k], d);
        weight8(p, c, w);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float hat = h[e] * inv;
          dw[k][e] += d[e] * hat;
          g[e] = inv * (d[e] * w[e] - hat * mean);
        }
        if (p.res) {
          float v[8];
          unpack8<TR>(rres[k], v);
#pragma unroll
          for (int e = 0; e < 8; ++e) g[e] += v[e];
        }
        if (p.h) store8<TR>(p.h + (r * p.hs + c) * (int64_t)sizeof(TR), g);
        if (p.y) {
          if (p.drop) drop8(p, (uint64_t)(r * p.n + c) >> 3, step, k0, k1, g);
          store8<TX>(p.y + (r * p.ys + c) * (int64_t)sizeof(TX), g);
        }
      }
    }
  }
  if (!p.part) return;   // uniform
  float* out = p.part + (int64_t)blockIdx.x * p.n;
  if constexpr (W == 1) {
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int e = 0; e < 8; ++e) cols[wave][8 * (j + 64 * k) + e] = dw[k][e];
    __syncthreads();
    for (int c = threadIdx.x; c < p.n; c += 256) out[c] = (cols[0][c] + cols[1][c]) + (cols[2][c] + cols[3][c]);
  } else {
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int c = 8 * (j + 256 * k);
      if (c < p.n) store8<float>((char*)(out + c), dw[k]);
    }
  }
}

constexpr int64_t ADD_NORM_WIDEST = 16384;   // columns: 8 chunks of a workgroup

int64_t norm_bwd_groups(int64_t m, int64_t n, int cus) {
  const int64_t rows = n <= 2048 ? 4 : 1;
  return std::max<int64_t>(1, std::min<int64_t>((m + rows - 1) / rows, (int64_t)cus * 4));
}

int add_norm_check(const inl_add_norm_desc* d) {
  if (!d) return fail(INL_E_INVALID, "add_rms_norm: desc is NULL");
  if (d->m < 0 || d->n <= 0) return fail(INL_E_INVALID, "add_rms_norm: m must be >= 0, n > 0");
  if (d->n % 8 || d->n > ADD_NORM_WIDEST)
    return fail(INL_E_UNSUPPORTED, "add_rms_norm: n must be a multiple of 8, at most 16384");
  if (d->m >= (int64_t)1 << 31) return fail(INL_E_UNSUPPORTED, "add_rms_norm: m must stay below 2^31");
  if (!dtype_ok(d->x_dtype) || !dtype_ok(d->stream_dtype) || !dtype_ok(d->out_dtype) || !dtype_ok(d->weight_dtype))
    return fail(INL_E_INVALID, "add_rms_norm: dtypes must be INL_F32 or INL_BF16");
  if (d->drop < 0 || d->drop > 65535) return fail(INL_E_INVALID, "add_rms_norm: drop must be in [0, 65535]");
  if (!(d->eps >= 0.f)) return fail(INL_E_INVALID, "add_rms_norm: eps must be >= 0");
  return INL_OK;
}

struct NormMat {
  const char* what;
  const void* at;
  int64_t stride;
  int32_t dtype;
  bool needed;
};

// Checks matrices [m, n]; those from `outs` on are written, each at another matrix's own place (same
// address, stride and size of element: every lane reads what it overwrites) or away from all.
int norm_mats(const inl_add_norm_desc* d, const NormMat* t, int count, int outs) {
  Rows r[8];
  for (int i = 0; i < count; ++i) {
    const int64_t es = dtype_size(t[i].dtype);
    if (t[i].needed && !t[i].at && d->m)
      return fail(INL_E_INVALID, std::string("add_rms_norm: ") + t[i].what + " is NULL");
    if (t[i].at && (((uintptr_t)t[i].at & 15) || t[i].stride < d->n || (t[i].stride * es) % 16))
      return fail(INL_E_INVALID, std::string("add_rms_norm: ") + t[i].what +
                                     " must be 16-byte aligned, its row stride cover n and be a multiple of 16 bytes");
    r[i] = {t[i].at, d->m, d->n * es, t[i].stride * es};
  }
  for (int i = outs; i < count; ++i)
    for (int j = 0; j < i; ++j) {
      const bool place = j < outs && t[i].at == t[j].at && t[i].dtype == t[j].dtype && (t[i].stride == t[j].stride || d->m == 1);
      if (!place && rows_meet(r[i], r[j]))
        return fail(INL_E_INVALID, std::string("add_rms_norm: ") + t[i].what + " overlaps " + t[j].what);
    }
  return INL_OK;
}

int norm_weight(const inl_add_norm_desc* d, const void* weight, const void* rng, bool draws, const NormMat* outs, int count) {
  if ((uintptr_t)weight & 15) return fail(INL_E_INVALID, "add_rms_norm: weight must be 16-byte aligned");
  if (draws && (!rng || ((uintptr_t)rng & 7)))
    return fail(INL_E_INVALID, "add_rms_norm: dropout needs rng (two int64 on the device)");
  const int64_t len = d->n * dtype_size(d->weight_dtype);
  for (int i = 0; i < count; ++i) {
    const int64_t es = dtype_size(outs[i].dtype);
    const Rows o{outs[i].at, d->m, d->n * es, outs[i].stride * es};
    if (rows_meet(o, {weight, 1, len, len}) || (draws && rows_meet(o, {rng, 1, 16, 16})))
      return fail(INL_E_INVALID, std::string("add_rms_norm: ") + outs[i].what + " overlaps weight or rng");
  }
  return INL_OK;
}

template <typename TX, typename TR, typename TY, bool BWD>
void add_norm_launch(const AddNormParams& p, unsigned groups, hipStream_t st) {
  // (a dimension of a grid has fewer than 2^32 threads)
  auto grid = [&](int64_t n) {
    const int64_t x = std::min<int64_t>(n, 1 << 22);
    return BWD ? dim3(groups) : dim3((unsigned)x, (unsigned)((n + x - 1) / x));
  };
  const dim3 block(256), rows = grid((p.m + 3) / 4), wide = grid(p.m);
#define INL_NORM(W, K)                                                                                        \
  do {                                                                                                        \
    if constexpr (BWD) hipLaunchKernelGGL((add_norm_bwd_kernel<TX, TR, TY, W, K>), W == 1 ? rows : wide, block, 0, st, p); \
    else hipLaunchKernelGGL((add_norm_kernel<TX, TR, TY, W, K>), W == 1 ? rows : wide, block, 0, st, p);      \
  } while (0)
  if (p.n <= 512) INL_NORM(1, 1);
  else if (p.n <= 1024) INL_NORM(1, 2);
  else if (p.n <= 2048) INL_NORM(1, 4);
  else if (p.n <= 4096) INL_NORM(4, 2);
  else if (p.n <= 8192) INL_NORM(4, 4);
  else INL_NORM(4, 8);
#undef INL_NORM
}

template <bool BWD>
int add_norm_run(const inl_add_norm_desc* d, const AddNormParams& p, unsigned groups, hipStream_t st) {
  auto by_y = [&](auto tx, auto tr) {
    using TX = decltype(tx);
    using TR = decltype(tr);
    if (d->out_dtype == INL_BF16) add_norm_launch<TX, TR, bf16, BWD>(p, groups, st);
    else add_norm_launch<TX, TR, float, BWD>(p, groups, st);
  };
  auto by_r = [&](auto tx) {
    if (d->stream_dtype == INL_BF16) by_y(tx, bf16{});
    else by_y(tx, float{});
  };
  if (d->x_dtype == INL_BF16) by_r(bf16{});
  else by_r(float{});
  INL_HIP_TRY(hipGetLastError());
  return INL_OK;
}

AddNormParams norm_params(const inl_add_norm_desc* d, const void* weight, const int64_t* rng) {
  AddNormParams p{};
  p.w = (const char*)weight;
  p.w16 = d->weight_dtype == INL_BF16;
  p.rng = rng;
  p.m = d->m;
  p.n = (int32_t)d->n;
  p.drop = d->drop;
  p.tag = d->tag;
  p.eps = d->eps;
  p.keep_scale = 65536.0f / (float)(65536 - d->drop);
  return p;
}

int64_t or_packed(int64_t stride, int64_t n) { return stride ? stride : n; }

}  // namespace

}  // namespace inl

extern "C" int inl_add_rms_norm_fwd(const inl_add_norm_desc* d, const void* x, const void* residual, const void* weight,
                                    const int64_t* rng, void* h, void* y, void* stream) {
  using namespace inl;
  int rc = add_norm_check(d);
  if (rc) return rc;
  const int64_t xs = or_packed(d->x_stride, d->n), rs = or_packed(d->residual_stride, d->n);
  const int64_t hs = or_packed(d->h_stride, d->n), ys = or_packed(d->y_stride, d->n);
  const NormMat t[4] = {{"x", x, xs, d->x_dtype, true}, {"residual", residual, rs, d->stream_dtype, false},
                        {"h", h, hs, d->stream_dtype, false}, {"y", y, ys, d->out_dtype, true}};
  if ((rc = norm_mats(d, t, 4, 2)) || (rc = norm_weight(d, weight, rng, d->drop != 0, t + 2, 2))) return rc;
  if (d->m == 0) return INL_OK;
  AddNormParams p = norm_params(d, weight, rng);
  p.x = (const char*)x;
  p.res = (const char*)residual;
  p.h = (char*)h;
  p.y = (char*)y;
  p.xs = xs;
  p.rs = rs;
  p.hs = hs;
  p.ys = ys;
  return add_norm_run<false>(d, p, 0, (hipStream_t)stream);
}

extern "C" int inl_add_rms_norm_bwd_workspace_size(const inl_add_norm_desc* d, size_t* bytes) {
  using namespace inl;
  if (!bytes) return fail(INL_E_INVALID, "add_rms_norm: bytes is NULL");
  int rc = add_norm_check(d);
  if (rc) return rc;
  int cus = 0;
  if ((rc = device_cus(&cus))) return rc;
  *bytes = d->m == 0 ? 0 : (size_t)norm_bwd_groups(d->m, d->n, cus) * (size_t)d->n * 4;
  return INL_OK;
}

extern "C" int inl_add_rms_norm_bwd(const inl_add_norm_desc* d, const void* dy, const void* h, const void* dh,
                                    const void* weight, const int64_t* rng, void* dx, void* dresidual, float* dweight,
                                    void* ws, size_t ws_bytes, void* stream) {
  using namespace inl;
  hipStream_t st = (hipStream_t)stream;
  int rc = add_norm_check(d);
  if (rc) return rc;
  const int64_t ys = or_packed(d->y_stride, d->n), hs = or_packed(d->h_stride, d->n);
  const int64_t dhs = or_packed(d->dh_stride, d->n), xs = or_packed(d->x_stride, d->n);
  const int64_t rs = or_packed(d->residual_stride, d->n);
  const NormMat t[5] = {{"dy", dy, ys, d->out_dtype, true}, {"h", h, hs, d->stream_dtype, true},
                        {"dh", dh, dhs, d->stream_dtype, false}, {"dx", dx, xs, d->x_dtype, false},
                        {"dresidual", dresidual, rs, d->stream_dtype, false}};
  if ((rc = norm_mats(d, t, 5, 3)) || (rc = norm_weight(d, weight, rng, d->drop != 0 && dx, t + 3, 2))) return rc;
  if ((uintptr_t)dweight & 15) return fail(INL_E_INVALID, "add_rms_norm: dweight must be 16-byte aligned");
  const Rows dwr{dweight, 1, d->n * 4, d->n * 4};
  for (int i = 0; i < 5; ++i) {
    const int64_t es = dtype_size(t[i].dtype);
    if (rows_meet(dwr, {t[i].at, d->m, d->n * es, t[i].stride * es}))
      return fail(INL_E_INVALID, std::string("add_rms_norm: dweight overlaps ") + t[i].what);
  }
  if (d->m == 0) return dweight ? fill_zero(dweight, 1, d->n, d->n, INL_F32, st) : INL_OK;
  if (!dx && !dresidual && !dweight) return INL_OK;
  int cus = 0;
  if ((rc = device_cus(&cus))) return rc;
  const int64_t groups = norm_bwd_groups(d->m, d->n, cus);
  if (dweight && (rc = check_workspace("add_rms_norm", ws, ws_bytes, (size_t)groups * (size_t)d->n * 4))) return rc;
  AddNormParams p = norm_params(d, weight, rng);
  p.x = (const char*)dy;
  p.hin = (const char*)h;
  p.res = (const char*)dh;
  p.y = (char*)dx;
  p.h = (char*)dresidual;
  p.xs = ys;
  p.his = hs;
  p.rs = dhs;
  p.ys = xs;
  p.hs = rs;
  p.part = !dweight ? nullptr : groups == 1 ? dweight : (float*)ws;
  if ((rc = add_norm_run<true>(d, p, (unsigned)groups, st))) return rc;
  return dweight && groups > 1 ? colsum_join((const float*)ws, groups, (int32_t)d->n, dweight, (int32_t)d->n, nullptr, st)
                               : INL_OK;
}
