// The linear layer with bias, activation and residual, and its gradients.
//
//   forward   pre = x . w^T + bias, y = act(pre) + residual      2 m n k flops
//   backward  dz = dy act'(pre);  dx = dz . w, dw = dz^T . x, dbias = column sums of dz
//                                                                4 m n k flops
//
// The products are the tiled ones of tile_gemm.hpp; here are the few-row
// forward and the element-wise half of the backward.
#include "train_ops.hpp"
#include "lanes.hpp"

namespace inl {

namespace {

// ---- one to four rows ----
//
// Bound by the weights, read once: a wave takes one output column (or the gate
// and up rows of one) and walks its row of w in contiguous KiB, 16 bytes per
// lane, next to the same k of the M rows of x (from L1 after the first wave);
// f32 products and sums, one cross-lane sum at the end. (The instruction that adds
// two bf16 products rounds too coarsely.) One row through 1,024 x 1,024 takes 2.6 us,
// through 50,000 x 768 13.5 us (5.7 TB/s). Its vector instructions grow with M.
template <int M, int R, bool OUT16>
__global__ __launch_bounds__(256) void row_dense_kernel(TileParams p) {
  const int lane = threadIdx.x & 63;
  const int c = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (c >= p.n) return;   // a whole wave
  const int m = (int)p.m;
  const char* wr[R];
#pragma unroll
  for (int r = 0; r < R; ++r) wr[r] = p.w + ((int64_t)c + (int64_t)r * p.n) * p.ws_b;
  float acc[M][R] = {};
  const u32x4 none = {};
#pragma unroll 2
  for (int k0 = 0; k0 < p.k; k0 += 512) {
    const int k = k0 + lane * 8;
    const bool in = k < p.k;
    const int64_t off = (int64_t)(in ? k : 0) * 2;
    u32x4 wv[R], xv[M];
#pragma unroll
    for (int r = 0; r < R; ++r) wv[r] = *reinterpret_cast<const u32x4*>(wr[r] + off);
#pragma unroll
    for (int i = 0; i < M; ++i) xv[i] = *reinterpret_cast<const u32x4*>(p.x + min(i, m - 1) * p.xs_b + off);
#pragma unroll
    for (int r = 0; r < R; ++r) wv[r] = in ? wv[r] : none;
    if (!in)
#pragma unroll
      for (int i = 0; i < M; ++i) xv[i] = none;
#pragma unroll
    for (int i = 0; i < M; ++i)
#pragma unroll
      for (int r = 0; r < R; ++r)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const uint32_t a = xv[i][e], b = wv[r][e];
          acc[i][r] = __builtin_fmaf(__builtin_bit_cast(float, a << 16), __builtin_bit_cast(float, b << 16), acc[i][r]);
          acc[i][r] = __builtin_fmaf(__builtin_bit_cast(float, a & 0xffff0000u),
                                     __builtin_bit_cast(float, b & 0xffff0000u), acc[i][r]);
        }
  }
  float v[R] = {};
#pragma unroll
  for (int i = 0; i < M; ++i)
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const float s = wave_sum(acc[i][r]);
      if (lane == i) v[r] = s;
    }
  if (lane >= m) return;
  const int64_t row = lane;
  float y;
  if constexpr (R == 2) {
    if (p.pre) {
      *reinterpret_cast<bf16*>(p.pre + (row * p.ps + c) * 2) = (bf16)v[0];
      *reinterpret_cast<bf16*>(p.pre + (row * p.ps + p.n + c) * 2) = (bf16)v[1];
    }
    y = act_apply(p.act, v[0]) * v[1];
  } else {
    y = v[0];
    if (p.bias) y += p.bias[c];
    if (p.pre) *reinterpret_cast<bf16*>(p.pre + (row * p.ps + c) * 2) = (bf16)y;
    y = act_apply(p.act, y);
    if (p.res)
      y += p.beta * (p.res_bf16 ? (float)*reinterpret_cast<const bf16*>(p.res + (row * p.rs + c) * 2)
                                : *reinterpret_cast<const float*>(p.res + (row * p.rs + c) * 4));
  }
  if constexpr (OUT16) *reinterpret_cast<bf16*>(p.y + (row * p.ys + c) * 2) = (bf16)y;
  else *reinterpret_cast<float*>(p.y + (row * p.ys + c) * 4) = y;
}

// ---- up to 16 XB rows ----
//
// Bound by latency, and by what one CU can load: no LDS stage, no ring. A workgroup
// takes 16 output columns (R = 2: their gate and up rows), its waves share k in units
// of 64 (whole 128-byte lines of 16 rows of w). Operands go from memory to
// v_mfma_f32_16x16x32_bf16 as they lie, U units asked for at a time (x from L2 after
// the first workgroups); the waves' sums meet in LDS, in order. 8 rows through 1,024 x
// 1,024 take 3.8 us, 16 take 4.1 (tiled product: 7.2).
constexpr int FEW_WAVES = 4;   // (eight: 5.8 us instead of 4.0 for 16 rows, 1,024 x 1,024)

template <int R, int XB, bool OUT16>
__global__ __launch_bounds__(FEW_WAVES * 64) void few_dense_kernel(TileParams p) {
  constexpr int U = XB == 1 ? 4 : 2;
  __shared__ f32x4 red[FEW_WAVES][R * XB][64];
  const int lane = threadIdx.x & 63, l16 = lane & 15, quad = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int c0 = blockIdx.x * 16, m = (int)p.m;
  const char* wr[R];
  const char* xr[XB];
#pragma unroll
  for (int r = 0; r < R; ++r) wr[r] = p.w + (min(c0 + l16, p.n - 1) + (int64_t)r * p.n) * p.ws_b;
#pragma unroll
  for (int b = 0; b < XB; ++b) xr[b] = p.x + min(b * 16 + l16, m - 1) * p.xs_b;
  f32x4 acc[R][XB] = {};
  const u32x4 none = {};
  for (int k0 = wave * 64; k0 < p.k; k0 += FEW_WAVES * 64 * U) {
    u32x4 wv[U][2][R], xv[U][2][XB];
#pragma unroll
    for (int i = 0; i < U; ++i)
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        const int k = k0 + i * FEW_WAVES * 64 + s * 32 + quad * 8;
        const bool in = k < p.k;
        const int64_t off = in ? (int64_t)k * 2 : 0;
#pragma unroll
        for (int r = 0; r < R; ++r) wv[i][s][r] = *reinterpret_cast<const u32x4*>(wr[r] + off);
#pragma unroll
        for (int b = 0; b < XB; ++b) xv[i][s][b] = *reinterpret_cast<const u32x4*>(xr[b] + off);
      }
#pragma unroll
    for (int i = 0; i < U; ++i)
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        const bool in = k0 + i * FEW_WAVES * 64 + s * 32 + quad * 8 < p.k;
#pragma unroll
        for (int r = 0; r < R; ++r) wv[i][s][r] = in ? wv[i][s][r] : none;
#pragma unroll
        for (int b = 0; b < XB; ++b) {
          const u32x4 x = in ? xv[i][s][b] : none;
#pragma unroll
          for (int r = 0; r < R; ++r)
            acc[r][b] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, wv[i][s][r]),
                                                                __builtin_bit_cast(bf16x8, x), acc[r][b], 0, 0, 0);
        }
      }
  }
#pragma unroll
  for (int r = 0; r < R; ++r)
#pragma unroll
    for (int b = 0; b < XB; ++b) red[wave][r * XB + b][lane] = acc[r][b];
  __syncthreads();
  // element e: row b 16 + l16, column c0 + 4 quad + e; a wave per block of rows
  if (wave >= XB) return;
  const int row = wave * 16 + l16, c = c0 + 4 * quad;
  if (row >= m || c >= p.n) return;
  f32x4 v[R];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    v[r] = red[0][r * XB + wave][lane];
#pragma unroll
    for (int i = 1; i < FEW_WAVES; ++i) {
      const f32x4 q = red[i][r * XB + wave][lane];
#pragma unroll
      for (int e = 0; e < 4; ++e) v[r][e] += q[e];
    }
  }
  auto put16 = [](char* at, const f32x4& z) {
    bf16x4 o;
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] = (bf16)z[e];
    *reinterpret_cast<bf16x4*>(at) = o;
  };
  f32x4 y = v[0];
  if constexpr (R == 2) {
    if (p.pre) {
      put16(p.pre + (row * p.ps + c) * 2, v[0]);
      put16(p.pre + (row * p.ps + p.n + c) * 2, v[1]);
    }
    y = act_apply4(p.act, y);
#pragma unroll
    for (int e = 0; e < 4; ++e) y[e] *= v[1][e];
  } else {
    if (p.bias) {
      const f32x4 b = *reinterpret_cast<const f32x4*>(p.bias + c);
#pragma unroll
      for (int e = 0; e < 4; ++e) y[e] += b[e];
    }
    if (p.pre) put16(p.pre + (row * p.ps + c) * 2, y);
    y = act_apply4(p.act, y);
    if (p.res && p.res_bf16) {
      const bf16x4 q = *reinterpret_cast<const bf16x4*>(p.res + (row * p.rs + c) * 2);
#pragma unroll
      for (int e = 0; e < 4; ++e) y[e] += p.beta * (float)q[e];
    } else if (p.res) {
      const f32x4 q = *reinterpret_cast<const f32x4*>(p.res + (row * p.rs + c) * 4);
#pragma unroll
      for (int e = 0; e < 4; ++e) y[e] += p.beta * q[e];
    }
  }
  if constexpr (OUT16) put16(p.y + (row * p.ys + c) * 2, y);
  else *reinterpret_cast<f32x4*>(p.y + (row * p.ys + c) * 4) = y;
}

// ---- dz and column sums ----
//
// Bound by memory: dy and pre read once, dz written once (20,011 x 768: 19.4 us, 4.75 TB/s).
// A thread takes 8 columns of every 8th row of its block's CS_ROWS rows; the 8 row groups
// meet in LDS, the blocks in a second kernel that adds their sums in order. dz is rounded
// to bf16, the type of the products' operands, which dx and dw feel as much as their own
// rounding (2.4e-3 of their norm from 64 bits, 1.7e-3 without); the sums take it unrounded.
constexpr int CS_ROWS = 64, CS_COLS = 256;
int64_t colsum_blocks(int64_t m) { return std::min<int64_t>((m + CS_ROWS - 1) / CS_ROWS, 65535); }

struct ActBwdParams {
  const char* dy;
  const char* pre;
  char* dz;
  float* part;
  int64_t m, dys, ps;
  int32_t n, act;
};

template <bool PRE, bool SUM>
__global__ __launch_bounds__(256) void act_bwd_kernel(ActBwdParams p) {
  __shared__ float red[8][CS_COLS + 4];
  const int tc = threadIdx.x & 31, tr = threadIdx.x >> 5;
  const int col = blockIdx.x * CS_COLS + tc * 8;
  const bool in = col < p.n;
  float s[8] = {};
  for (int64_t row0 = (int64_t)blockIdx.y * CS_ROWS; row0 < p.m; row0 += (int64_t)gridDim.y * CS_ROWS)
#pragma unroll 4
  for (int i = 0; i < CS_ROWS / 8; ++i) {
    const int64_t row = row0 + tr + 8 * i;
    if (!in || row >= p.m) continue;
    const bf16x8 d = *reinterpret_cast<const bf16x8*>(p.dy + (row * p.dys + col) * 2);
    float v[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = (float)d[e];
    if constexpr (PRE) {
      const bf16x8 z = *reinterpret_cast<const bf16x8*>(p.pre + (row * p.ps + col) * 2);
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] *= act_pair(p.act, (float)z[e]).slope;
      if (p.dz) {
        bf16x8 o;
#pragma unroll
        for (int e = 0; e < 8; ++e) o[e] = (bf16)v[e];
        *reinterpret_cast<bf16x8*>(p.dz + (row * p.n + col) * 2) = o;
      }
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) s[e] += v[e];
  }
  if constexpr (SUM) {
#pragma unroll
    for (int e = 0; e < 8; ++e) red[tr][tc * 8 + e] = s[e];
    __syncthreads();
    const int c = threadIdx.x;
    if (blockIdx.x * CS_COLS + c < p.n) {
      float t = 0.f;
#pragma unroll
      for (int r = 0; r < 8; ++r) t += red[r][c];
      p.part[(int64_t)blockIdx.y * p.n + blockIdx.x * CS_COLS + c] = t;
    }
  }
}

// out[c] = sum over blocks of part[block][c], columns from `cut` on to out2.
__global__ __launch_bounds__(1024) void colsum_join_kernel(const float* part, int64_t blocks, int32_t n, float* out,
                                                           int32_t cut, float* out2) {
  __shared__ float red[16][64];
  const int tc = threadIdx.x & 63, tr = threadIdx.x >> 6;
  const int c = blockIdx.x * 64 + tc;
  float s = 0.f;
  if (c < n)
#pragma unroll 8
    for (int64_t b = tr; b < blocks; b += 16) s += part[b * n + c];
  red[tr][tc] = s;
  __syncthreads();
  if (tr == 0 && c < n) {
    float t = 0.f;
#pragma unroll
    for (int r = 0; r < 16; ++r) t += red[r][tc];
    float* o = c < cut ? out : out2;
    if (o) o[c < cut ? c : c - cut] = t;
  }
}

__global__ __launch_bounds__(256) void fill_zero_kernel(char* p, int64_t rows, int64_t words, int64_t stride_b) {
  for (int64_t i = blockIdx.x * (int64_t)256 + threadIdx.x; i < rows * words; i += (int64_t)gridDim.x * 256)
    reinterpret_cast<uint32_t*>(p + i / words * stride_b)[i % words] = 0;
}

template <int R, bool OUT16>
int few_launch(const TileParams& p, hipStream_t stream) {
  const dim3 rows((unsigned)((p.n + 3) / 4)), blocks((unsigned)((p.n + 15) / 16)), t(256), tb(FEW_WAVES * 64);
  if (p.m == 1) hipLaunchKernelGGL((row_dense_kernel<1, R, OUT16>), rows, t, 0, stream, p);
  else if (p.m == 2) hipLaunchKernelGGL((row_dense_kernel<2, R, OUT16>), rows, t, 0, stream, p);
  else if (p.m <= 4) hipLaunchKernelGGL((row_dense_kernel<4, R, OUT16>), rows, t, 0, stream, p);
  else if (p.m <= 16) hipLaunchKernelGGL((few_dense_kernel<R, 1, OUT16>), blocks, tb, 0, stream, p);
  else hipLaunchKernelGGL((few_dense_kernel<R, 2, OUT16>), blocks, tb, 0, stream, p);
  INL_HIP_TRY(hipGetLastError());
  return INL_OK;
}

}  // namespace

// Measured, us, few rows against the tiled product, by (n, k), six sets of weights in turn:
//   2 rows   (8,192, 256) 3.5 / 4.2   (16,384, 512) 6.4 / 6.0    (16,384, 1,024) 7.8 / 8.3   (50,000, 768) 18.8 / 18.3
//   4        (8,192, 512) 5.2 / 5.6   (8,192, 2,048) 9.0 / 10.1  (12,288, 1,024) 8.2 / 7.8   (4,096, 8,192) 21.6 / 20.6
//   5        (1,024, 1,024) 3.6 / 7.1 (8,192, 512) 5.4 / 5.7     (8,192, 2,048) 9.5 / 10.1   (1,024, 4,096) 8.2 / 9.5
//   16       (1,024, 1,024) 4.1 / 7.2 (8,192, 256) 5.9 / 4.3     (8,192, 1,024) 6.4 / 7.8    (16,384, 1,024) 9.8 / 8.3
//            (4,096, 2,048) 7.0 / 8.9 (4,096, 4,096) 10.4 / 10.8 (2,048, 8,192) 16.9 / 12.1
//   32       (4,096, 2,048) 8.6 / 9.6 (8,192, 512) 5.6 / 6.0     (8,192, 768) 8.5 / 6.9      (1,024, 4,096) 13.3 / 9.8
// Gate and up rows (n of each), few less tiled:
//   2 rows   (16,384, 512) -1.4       (8,192, 2,048) -4.2
//   4        (4,096, 512) -1.2        (8,192, 512) +0.4          (8,192, 1,024) -1.3         (12,288, 1,024) -0.8
//   16       (4,096, 1,024) -1.8      (4,096, 2,048) -1.3        (6,144, 1,024) +0.6         (8,192, 512) +2.2
//   32       (4,096, 2,048) -0.5      (1,024, 4,096) +4.5        (8,192, 512) +0.7           (8,192, 1,024) +2.3
// (One row through 50,000 x 768: 13.5 / 16. A workgroup's time goes with k and its blocks of
// rows; 256 workgroups of the kernel from 5 rows on are 4,096 columns, a round.)
bool few_rows(int64_t m, int64_t n, int64_t k, bool gated) {
  if (m <= 1) return true;
  if (m == 2) return gated || n <= 8192 || n <= 16 * k;
  if (m <= 4) return gated ? n <= 6144 || (k >= 1024 && n <= 12288) : n <= 8192 && n * k <= ((int64_t)1 << 24);
  const int64_t rounds = (n + 4095) / 4096;
  if (m <= 16) return rounds * k <= 4096 && (rounds == 1 || (rounds == 2 && k >= (gated ? 1024 : 768)));
  return m <= 32 && ((rounds == 1 && k <= 2048) || (rounds == 2 && !gated && k <= 512));
}

int few_dense(const TileParams& p, bool gated, bool out_bf16, hipStream_t stream) {
  if (gated) return few_launch<2, true>(p, stream);
  return out_bf16 ? few_launch<1, true>(p, stream) : few_launch<1, false>(p, stream);
}

int device_cus(int* cus) {
  int dev = 0;
  INL_HIP_TRY(hipGetDevice(&dev));
  INL_HIP_TRY(hipDeviceGetAttribute(cus, hipDeviceAttributeMultiprocessorCount, dev));
  return INL_OK;
}

int check_rows(const char* what, const void* p, int64_t cols, int64_t stride, int32_t dtype) {
  const std::string w(what);
  if (!p) return fail(INL_E_INVALID, w + " is NULL");
  if ((uintptr_t)p & 15) return fail(INL_E_INVALID, w + " must be 16-byte aligned");
  if (stride < cols) return fail(INL_E_INVALID, w + ": the row stride is shorter than the row");
  if (stride % 8) return fail(INL_E_UNSUPPORTED, w + ": the row stride must be a multiple of 8 elements");
  // a tile's descriptor spans at most 256 rows, below 2^31 bytes
  if (stride > ((int64_t)1 << 21)) return fail(INL_E_UNSUPPORTED, w + ": the row stride is above 2^21 elements");
  if (!dtype_ok(dtype)) return fail(INL_E_INVALID, w + ": dtype must be INL_F32 or INL_BF16");
  return INL_OK;
}

bool rows_meet(const Rows& a, const Rows& b) {
  if (!a.at || !b.at || a.rows <= 0 || b.rows <= 0) return false;
  const int64_t d = (int64_t)((uintptr_t)b.at - (uintptr_t)a.at);   // b's start from a's
  if (d >= (a.rows - 1) * a.step + a.len || -d >= (b.rows - 1) * b.step + b.len) return false;
  auto floor_div = [](int64_t x, int64_t y) { return x / y - (x % y < 0); };
  // rows j of b meet row i of a where i a.step - b.len < d + j b.step < i a.step + a.len
  auto met = [&](int64_t at) {   // a row of a that starts `at` bytes after a's start
    const int64_t lo = floor_div(at - b.len - d, b.step) + 1, hi = -floor_div(d - at - a.len, b.step) - 1;
    return std::max<int64_t>(lo, 0) <= std::min(hi, b.rows - 1);
  };
  if (a.step == b.step) {   // columns of one buffer, say: only j - i counts
    const int64_t lo = floor_div(-b.len - d, b.step) + 1, hi = -floor_div(d - a.len, b.step) - 1;
    return std::max(lo, 1 - a.rows) <= std::min(hi, b.rows - 1);
  }
  for (int64_t i = 0; i < a.rows; ++i)
    if (met(i * a.step)) return true;
  return false;
}

int check_workspace(const char* what, const void* ws, size_t have, size_t need) {
  if (!need) return INL_OK;
  if (!ws || ((uintptr_t)ws & 15)) return fail(INL_E_INVALID, std::string(what) + ": the workspace must be 16-byte aligned");
  if (have < need)
    return fail(INL_E_INVALID, std::string(what) + ": workspace of " + std::to_string(have) + " bytes, need " + std::to_string(need));
  return INL_OK;
}

size_t colsum_bytes(int64_t m, int64_t n) { return (size_t)colsum_blocks(m) * (size_t)n * 4; }

int colsum_join(const float* part, int64_t blocks, int32_t n, float* out, int32_t cut, float* out2,
                hipStream_t stream) {
  hipLaunchKernelGGL(colsum_join_kernel, dim3((unsigned)((n + 63) / 64)), dim3(1024), 0, stream, part, blocks, n, out,
                     cut, out2);
  INL_HIP_TRY(hipGetLastError());
  return INL_OK;
}

int act_bwd(int64_t m, int64_t n, const void* dy, int64_t dys, const void* pre, int64_t pres, int32_t act, void* dz,
            float* colsum, float* part, hipStream_t stream) {
  ActBwdParams p{(const char*)dy, (const char*)pre, (char*)dz, part, m, dys, pres, (int32_t)n, act};
  const int64_t blocks = colsum_blocks(m);
  if (colsum && blocks == 1) p.part = colsum;   // nothing to join
  const dim3 grid((unsigned)((n + CS_COLS - 1) / CS_COLS), (unsigned)blocks), block(256);
  if (pre && colsum) hipLaunchKernelGGL((act_bwd_kernel<true, true>), grid, block, 0, stream, p);
  else if (pre) hipLaunchKernelGGL((act_bwd_kernel<true, false>), grid, block, 0, stream, p);
  else hipLaunchKernelGGL((act_bwd_kernel<false, true>), grid, block, 0, stream, p);
  INL_HIP_TRY(hipGetLastError());
  return colsum && blocks > 1 ? colsum_join(part, blocks, (int32_t)n, colsum, (int32_t)n, nullptr, stream) : INL_OK;
}

int fill_zero(void* p, int64_t rows, int64_t cols, int64_t stride, int32_t dtype, hipStream_t stream) {
  const int64_t words = cols * dtype_size(dtype) / 4;
  if (rows * words == 0) return INL_OK;
  hipLaunchKernelGGL(fill_zero_kernel, dim3((unsigned)std::min<int64_t>((rows * words + 255) / 256, 4096)), dim3(256),
                     0, stream, (char*)p, rows, words, stride * dtype_size(dtype));
  INL_HIP_TRY(hipGetLastError());
  return INL_OK;
}

namespace {

int dense_check(const inl_dense_desc* d) {
  if (!d) return fail(INL_E_INVALID, "dense: desc is NULL");
  if (d->m < 0 || d->n <= 0 || d->k <= 0) return fail(INL_E_INVALID, "dense: m must be >= 0, n and k > 0");
  if (d->n % 8 || d->k % 8) return fail(INL_E_UNSUPPORTED, "dense: n and k must be multiples of 8");
  if (d->m >= ((int64_t)1 << 31) - 256 || d->n > (1 << 21) || d->k > (1 << 21))
    return fail(INL_E_UNSUPPORTED, "dense: m must stay below 2^31 - 256, n and k at most 2^21");
  if (d->act < INL_ACT_NONE || d->act > INL_ACT_GELU_ERF) return fail(INL_E_INVALID, "dense: unknown act");
  return INL_OK;
}

struct DenseStrides {
  int64_t x, w, y, res, pre, dx, dw;
  explicit DenseStrides(const inl_dense_desc& d)
      : x(d.x_stride ? d.x_stride : d.k), w(d.w_stride ? d.w_stride : d.k), y(d.y_stride ? d.y_stride : d.n),
        res(d.residual_stride ? d.residual_stride : d.n), pre(d.pre_stride ? d.pre_stride : d.n),
        dx(d.dx_stride ? d.dx_stride : d.k), dw(d.dw_stride ? d.dw_stride : d.k) {}
};

constexpr int MAX_SPLITS = 32;

struct DensePlan {
  TilePlan y, dx, dw;
  size_t need(const inl_dense_desc& d, bool backward) const {
    if (!backward) return few_rows(d.m, d.n, d.k, false) ? 0 : tile_part_bytes(y, d.m, d.n);
    Carve c(nullptr);
    if (d.act != INL_ACT_NONE) c.take((size_t)d.m * d.n * 2);
    c.take(colsum_bytes(d.m, d.n));
    c.take(std::max(tile_part_bytes(dx, d.m, d.k), tile_part_bytes(dw, d.n, d.k)));
    return c.used;
  }
};

int dense_plan(const inl_dense_desc& d, bool backward, DensePlan* p, int* cus) {
  if (!backward && few_rows(d.m, d.n, d.k, false)) return INL_OK;
  int rc = device_cus(cus);
  if (rc) return rc;
  if (!backward) {
    p->y = tile_plan(d.m, d.n, d.k, 0, false, MAX_SPLITS, *cus);
    return INL_OK;
  }
  p->dx = tile_plan(d.m, d.k, d.n, 1, false, MAX_SPLITS, *cus);
  p->dw = tile_plan(d.n, d.k, d.m, 2, false, MAX_SPLITS, *cus);
  return INL_OK;
}

}  // namespace

}  // namespace inl

extern "C" int inl_dense_workspace_size(const inl_dense_desc* d, int32_t backward, size_t* bytes) {
  using namespace inl;
  if (!bytes) return fail(INL_E_INVALID, "dense: bytes is NULL");
  int rc = dense_check(d);
  if (rc) return rc;
  DensePlan plan;
  int cus = 0;
  if ((rc = dense_plan(*d, backward != 0, &plan, &cus))) return rc;
  *bytes = plan.need(*d, backward != 0);
  return INL_OK;
}

extern "C" int inl_dense_fwd(const inl_dense_desc* d, const void* x, const void* w, const float* bias,
                             const void* residual, void* y, void* pre, void* ws, size_t ws_bytes, void* stream) {
  using namespace inl;
  int rc = dense_check(d);
  if (rc) return rc;
  if (d->m == 0) return INL_OK;
  const DenseStrides s(*d);
  if ((rc = check_rows("dense: x", x, d->k, s.x, INL_BF16))) return rc;
  if ((rc = check_rows("dense: w", w, d->k, s.w, INL_BF16))) return rc;
  if ((rc = check_rows("dense: y", y, d->n, s.y, d->out_dtype))) return rc;
  if (residual && (rc = check_rows("dense: residual", residual, d->n, s.res, d->residual_dtype))) return rc;
  if (pre && (rc = check_rows("dense: pre", pre, d->n, s.pre, INL_BF16))) return rc;
  if ((uintptr_t)bias & 15) return fail(INL_E_INVALID, "dense: bias must be 16-byte aligned");
  // tiles are written while others still read x and w
  auto rows = [](const void* at, int64_t n, int64_t cols, int64_t stride, int32_t dtype) {
    return Rows{at, n, cols * dtype_size(dtype), stride * dtype_size(dtype)};
  };
  const Rows rx = rows(x, d->m, d->k, s.x, INL_BF16), rw = rows(w, d->n, d->k, s.w, INL_BF16);
  const Rows ry = rows(y, d->m, d->n, s.y, d->out_dtype), rp = rows(pre, d->m, d->n, s.pre, INL_BF16);
  const Rows rr = rows(residual, d->m, d->n, s.res, residual ? d->residual_dtype : INL_BF16);
  const bool in_place = residual == y && d->residual_dtype == d->out_dtype && (s.res == s.y || d->m == 1);
  auto meet = [](const char* what, const Rows& a, const Rows& b) {
    return rows_meet(a, b) ? fail(INL_E_INVALID, std::string("dense: overlap of ") + what) : INL_OK;
  };
  if ((rc = meet("y and x", ry, rx)) || (rc = meet("y and w", ry, rw)) || (rc = meet("pre and x", rp, rx)) ||
      (rc = meet("pre and w", rp, rw)) || (rc = meet("pre and y", rp, ry)) || (rc = meet("pre and residual", rp, rr)))
    return rc;
  if (!in_place && (rc = meet("y and residual, which are not the same rows", ry, rr))) return rc;
  DensePlan plan;
  int cus = 0;
  if ((rc = dense_plan(*d, false, &plan, &cus))) return rc;
  if ((rc = check_workspace("dense", ws, ws_bytes, plan.need(*d, false)))) return rc;
  TileParams p{};
  p.x = (const char*)x;
  p.w = (const char*)w;
  p.xs_b = s.x * 2;
  p.ws_b = s.w * 2;
  p.m = d->m;
  p.n = (int32_t)d->n;
  p.k = (int32_t)d->k;
  p.y = (char*)y;
  p.ys = s.y;
  p.res = (const char*)residual;
  p.rs = s.res;
  p.res_bf16 = d->residual_dtype == INL_BF16;
  p.alpha = p.beta = 1.f;
  p.bias = bias;
  p.pre = (char*)pre;
  p.ps = s.pre;
  p.act = d->act;
  const bool out16 = d->out_dtype == INL_BF16;
  if (few_rows(d->m, d->n, d->k, false)) return few_dense(p, false, out16, (hipStream_t)stream);
  return tile_nt_linear(p, plan.y, out16, (float*)ws, cus, (hipStream_t)stream);
}

extern "C" int inl_dense_bwd(const inl_dense_desc* d, const void* dy, const void* x, const void* w, const void* pre,
                             void* dx, void* dw, float* dbias, void* ws, size_t ws_bytes, void* stream) {
  using namespace inl;
  hipStream_t st = (hipStream_t)stream;
  int rc = dense_check(d);
  if (rc) return rc;
  const DenseStrides s(*d);
  if (dx && !dtype_ok(d->dx_dtype)) return fail(INL_E_INVALID, "dense: dx_dtype must be INL_F32 or INL_BF16");
  if (dw && (rc = check_rows("dense: dw", dw, d->k, s.dw, d->dw_dtype))) return rc;
  if ((uintptr_t)dbias & 15) return fail(INL_E_INVALID, "dense: dbias must be 16-byte aligned");
  if (d->m == 0) {
    if (dw && (rc = fill_zero(dw, d->n, d->k, s.dw, d->dw_dtype, st))) return rc;
    return dbias ? fill_zero(dbias, 1, d->n, d->n, INL_F32, st) : INL_OK;
  }
  if ((rc = check_rows("dense: dy", dy, d->n, s.y, INL_BF16))) return rc;
  if (dx && (rc = check_rows("dense: dx", dx, d->k, s.dx, d->dx_dtype))) return rc;
  if (dx && (rc = check_rows("dense: w", w, d->k, s.w, INL_BF16))) return rc;
  if (dw && (rc = check_rows("dense: x", x, d->k, s.x, INL_BF16))) return rc;
  const bool acts = d->act != INL_ACT_NONE;
  if (acts && (rc = check_rows("dense: pre", pre, d->n, s.pre, INL_BF16))) return rc;
  DensePlan plan;
  int cus = 0;
  if ((rc = dense_plan(*d, true, &plan, &cus))) return rc;
  if ((rc = check_workspace("dense", ws, ws_bytes, plan.need(*d, true)))) return rc;
  Carve c(ws);
  char* dzb = acts ? c.take((size_t)d->m * d->n * 2) : nullptr;
  float* sums = (float*)c.take(colsum_bytes(d->m, d->n));
  float* part = (float*)c.take(0);
  if (acts || dbias)
    if ((rc = act_bwd(d->m, d->n, dy, s.y, acts ? pre : nullptr, s.pre, d->act, dx || dw ? dzb : nullptr, dbias, sums,
                      st)))
      return rc;
  const char* dz = acts ? dzb : (const char*)dy;
  const int64_t dzs = acts ? d->n : s.y;
  TileParams p{};
  p.alpha = p.beta = 1.f;
  p.act = ACT_NONE;
  if (dx) {
    p.x = dz;
    p.xs_b = dzs * 2;
    p.w = (const char*)w;
    p.ws_b = s.w * 2;
    p.m = d->m;
    p.n = (int32_t)d->k;
    p.k = (int32_t)d->n;
    p.y = (char*)dx;
    p.ys = s.dx;
    if ((rc = tile_nn_linear(p, plan.dx, d->dx_dtype == INL_BF16, part, cus, st))) return rc;
  }
  if (dw) {
    p.x = dz;
    p.xs_b = dzs * 2;
    p.w = (const char*)x;
    p.ws_b = s.x * 2;
    p.m = d->n;
    p.n = (int32_t)d->k;
    p.k = (int32_t)d->m;
    p.y = (char*)dw;
    p.ys = s.dw;
    if ((rc = tile_tn_linear(p, plan.dw, d->dw_dtype == INL_BF16, part, cus, st))) return rc;
  }
  return INL_OK;
}
