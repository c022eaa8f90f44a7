// Tiled bf16 matrix products with the operands in either storage order and an
// epilogue per use: the products of the linear layer, the gated feed-forward
// block and the softmax cross entropy, forward and backward.
//
//   c[m, n] = sum_k X(m, k) W(n, k),   f32 accumulation
//
// An operand is stored as rows of k (OP_ROWS: x [M, K], w [N, K], the forward
// products) or as rows of m or n (OP_COLS: [K, M], [K, N]; dx = dz . W reads
// W that way, dW = dz^T . x both). Nothing is transposed in memory: a stage of
// an OP_COLS operand sits in LDS as it is stored (32 rows of k) and its MFMA
// operands are read with ds_read_b64_tr_b16, which hands lane j of 16 the four
// k values of column j.
//
// Pipeline: 8 or 4 waves, each WNB x WMB blocks of v_mfma_f32_32x32x16_bf16; a
// ring of 32-wide k slices in LDS filled by direct loads; operands read one
// 16-wide k step ahead. A workgroup is persistent: its units (tile, k range)
// form one stream of stages, so the next unit's first loads are in flight
// while a unit's epilogue runs.
//
// Units: a tile's k range may be cut into `splits` parts of `kper` stages
// (EPI_PART writes f32 partial tiles, a second kernel adds them in order), so
// that dW of a 768 x 768 layer over 20,000 tokens (9 tiles) fills 256 CUs.
//
// Unit order: split-major, then groups of GROUP m-tiles, n outer and m inner
// within a group, cut into 8 contiguous ranges, one per XCD (workgroup b runs
// on XCD b % 8). The ~32 units an XCD runs at one time form a rectangle of 8 x
// 4 tiles, 12 operand slices per stage instead of 33 for a row of tiles.
#pragma once

#include <algorithm>
#include <type_traits>

#include "activations.hpp"
#include "attn_stream.hpp"

namespace inl {

enum TileOperand { OP_ROWS = 0, OP_COLS = 1 };

enum TileEpi {
  EPI_PART = 0,      // f32 partial tiles [split][m][n]
  EPI_LINEAR = 1,    // y = act(alpha c + bias) + beta res; pre = alpha c + bias
  EPI_GATED = 2,     // w = n gate rows then n up rows: y = act(gate) * up; pre = gate, up
  EPI_DGATED = 3,    // c = dh, pre = [g u]: y = [dh u act'(g), dh act(g)]
  EPI_XENT = 4,      // scores alpha c + bias: row maxima and sums of exponentials per 32 WNB columns
  EPI_DXENT = 5,     // y = dl (softmax - onehot)
};

struct TileParams {
  const char* x;
  const char* w;
  int64_t xs_b, ws_b;       // bytes between stored rows
  int64_t m;
  int32_t n, k;
  char* y;
  int64_t ys;               // row strides in elements
  const char* res;          // added rows (f32 or bf16)
  int64_t rs;
  int32_t res_bf16;
  float alpha, beta;
  const float* bias;        // [n] or null
  char* pre;                // bf16 rows or null
  int64_t ps;
  int32_t act;
  // cross entropy
  const int32_t* target;    // [m]
  const float* lse;         // [m]
  const float* dl;          // [m]
  float* at;                // [m] the target's score
  float2* part;             // [column block][m] (maximum, sum)
  int32_t col0;             // vocabulary id of column 0
  int32_t ignore;
  int32_t n_store;          // columns of y, past n zeros (EPI_DXENT)
  // schedule
  int32_t tiles_m, tiles_n, group;
  int32_t units, per_xcd, wg_per_xcd;
  int32_t kper;             // stages per unit
};

constexpr int TG_BK = 32;
constexpr int TG_STG = 4096;   // per-wave epilogue staging: 32 rows x 128 bytes
constexpr int TG_XCDS = 8;
constexpr int TG_GROUP = 8;

template <int NWN_, int NWM_, int WNB_, int WMB_, int STAGES_, int WPC_>
struct TileShape {
  static constexpr int NWN = NWN_, NWM = NWM_, WNB = WNB_, WMB = WMB_;
  static constexpr int NW = NWN * NWM;
  static constexpr int BN = NWN * WNB * 32, BM = NWM * WMB * 32;
  static constexpr int STAGES = STAGES_, WPC = WPC_;
  static constexpr int W = BN * 64, X = BM * 64;
  static constexpr int STAGE = W + X;
  static constexpr int PER_WAVE = STAGE / 1024 / NW;
  static constexpr int W_PER_WAVE = W / 1024 / NW;
  static constexpr int RING = STAGES * STAGE;
  static constexpr int LDS = RING + NW * TG_STG;
  static_assert((STAGE / 1024) % NW == 0 && (W / 1024) % NW == 0, "the direct loads split evenly over the waves");
  static_assert(NW % 2 == 0, "w blocks of one wave share its parity (EPI_GATED)");
  static_assert(STAGES >= 2 && (STAGES - 1) * PER_WAVE <= 63, "vmcnt range");
};
// 0: 256 x 256, one workgroup of 8 waves per CU. 1: 128 x 128, two of 4 waves
// per CU. 2: 64 x 64, for outputs that would leave most of the chip idle.
template <int SH>
using TileShapeOf = std::conditional_t<SH == 0, TileShape<2, 4, 4, 2, 3, 1>,
                    std::conditional_t<SH == 1, TileShape<2, 2, 2, 2, 4, 2>, TileShape<2, 2, 1, 1, 6, 2>>>;
constexpr int TG_SHAPES = 3;

struct TilePlan {
  int shape;
  int splits;
  int32_t kper;
};
// The shape and k split with the least estimated time. `gated`: w has 2n rows.
// max_splits 1 keeps every tile in one unit.
TilePlan tile_plan(int64_t m, int64_t n, int64_t k, bool gated, int max_splits, int cus);

// f32 partials of a plan (0 for one split).
inline size_t tile_part_bytes(const TilePlan& t, int64_t m, int64_t n) {
  return t.splits > 1 ? (size_t)t.splits * (size_t)m * (size_t)n * 4 : 0;
}

namespace {

// 16-byte chunk c of stored row r of an operand stage, R = rows of m or n per
// tile. OP_ROWS: 64-byte rows, the 16 rows of one ds_read_b128 pass cover all
// banks. OP_COLS: 2 R-byte rows, the 4 rows x 64 bytes that 32 lanes of a
// transposed read touch cover all banks.
template <int L, int R>
__device__ __forceinline__ int tg_swz(int r, int c) {
  if constexpr (L == OP_ROWS) return c ^ ((r >> 2) & 3);
  if constexpr (R >= 128) return c ^ ((r & 3) << 2);
  return c ^ (((r >> 1) & 1) << 2);
}
template <int L, int R>
constexpr int tg_chunks() { return L == OP_ROWS ? 4 : R / 8; }

template <int SH, int LX, int LW, int EPI, bool OUT16, bool RES>
__global__ __launch_bounds__(TileShapeOf<SH>::NW * 64, TileShapeOf<SH>::WPC) void tile_gemm_kernel(TileParams p) {
  using C = TileShapeOf<SH>;
  constexpr int NW = C::NW, BM = C::BM, BN = C::BN, STAGES = C::STAGES, STAGE = C::STAGE;
  constexpr int PER_WAVE = C::PER_WAVE, WNB = C::WNB, WMB = C::WMB;
  constexpr int BNO = EPI == EPI_GATED ? BN / 2 : BN;   // output columns per tile
  static_assert(EPI != EPI_GATED || LW == OP_ROWS, "gate and up rows");
  extern __shared__ __attribute__((aligned(1024))) char smem[];
  const int xcd = blockIdx.x % TG_XCDS, slot = blockIdx.x / TG_XCDS;
  const int first = xcd * p.per_xcd;
  const int last = min(first + p.per_xcd, p.units);
  const int u0 = first + slot;
  if (u0 >= last) return;
  const int my_units = (last - 1 - u0) / p.wg_per_xcd + 1;
  const int kst = (p.k + TG_BK - 1) / TG_BK;

  const uint32_t lds0 = lds_addr(smem);
  const int tid = threadIdx.x;
  const int lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wn = wave / C::NWM, wm = wave % C::NWM;
  const int l32 = lane & 31, hf = lane >> 5;

  // ---- units ----
  struct Unit {
    int mt, nt, s;
  };
  const int tiles = p.tiles_m * p.tiles_n;
  auto unit_of = [&](int j) __attribute__((always_inline)) {
    const int u = u0 + j * p.wg_per_xcd;
    const int s = u / tiles, t = u - s * tiles;
    const int per_group = p.group * p.tiles_n;
    const int g = t / per_group, r = t - g * per_group;
    const int gm = min(p.group, p.tiles_m - g * p.group);
    const int nt = r / gm;
    Unit q;
    q.mt = g * p.group + (r - nt * gm);
    q.nt = nt;
    q.s = s;
    return q;
  };

  // ---- loads ----
  // Per-lane byte offsets of this wave's 1 KiB blocks {wave, wave + NW, ...} of
  // a stage (w first). The chunk of a lane is the same in all blocks of an
  // OP_ROWS operand.
  uint32_t goff[PER_WAVE];
#pragma unroll
  for (int i = 0; i < PER_WAVE; ++i) {
    const bool is_w = i < C::W_PER_WAVE;
    const int blk = wave + NW * i - (is_w ? 0 : C::W / 1024);
    const int cpr = is_w ? tg_chunks<LW, BN>() : tg_chunks<LX, BM>();
    const int b = EPI == EPI_GATED && is_w ? blk >> 1 : blk;   // 16 gate (even) or up (odd) rows
    const int at = b * 64 + lane, r = at / cpr, cp = at % cpr;
    const int c = is_w ? tg_swz<LW, BN>(r, cp) : tg_swz<LX, BM>(r, cp);
    goff[i] = (uint32_t)r * (uint32_t)(is_w ? p.ws_b : p.xs_b) + c * 16;
  }
  const int my_chunk = (lane & 3) ^ ((lane >> 4) & 3);   // k chunk of an OP_ROWS load

  // Descriptors start at a unit's first row and at the stage's k, so that no
  // offset exceeds 31 bits; rows past the end read as zero, and so does k past
  // the end: OP_COLS by the range, OP_ROWS by an offset out of it.
  int ld_j = 0, ld_ks = 0, ld_end = 0, ld_slot = 0;
  const char* xp = nullptr;
  const char* wp = nullptr;
  uint32_t x_rows = 0, w_rows = 0;   // rows (OP_ROWS) or columns (OP_COLS) of this unit
  auto ld_unit = [&]() __attribute__((always_inline)) {
    const Unit q = unit_of(ld_j);
    ld_ks = q.s * p.kper;
    ld_end = min(ld_ks + p.kper, kst);
    const int64_t k0 = (int64_t)ld_ks * TG_BK;
    const int64_t r0 = (int64_t)q.mt * BM;
    x_rows = (uint32_t)min((int64_t)BM, p.m - r0);
    xp = p.x + (LX == OP_ROWS ? r0 * p.xs_b + k0 * 2 : k0 * p.xs_b + r0 * 2);
    const int c0 = q.nt * BNO;
    w_rows = (uint32_t)min(BNO, p.n - c0);
    const int64_t c1 = EPI == EPI_GATED && (wave & 1) ? (int64_t)p.n + c0 : (int64_t)c0;
    wp = p.w + (LW == OP_ROWS ? c1 * p.ws_b + k0 * 2 : k0 * p.ws_b + c1 * 2);
  };
  auto range = [&](int L, uint32_t rows, int64_t stride, int left) __attribute__((always_inline)) {
    // (whole 16-byte chunks: an odd row end lies inside its padded row)
    return L == OP_ROWS ? (uint32_t)((rows - 1) * stride) + (uint32_t)((left + 7) & ~7) * 2
                        : (uint32_t)((min(left, TG_BK) - 1) * stride) + ((rows + 7) & ~7u) * 2;
  };
  const i32x4 none = pp_rsrc_words(p.x, 0);
  auto issue = [&]() __attribute__((always_inline)) {
    const uint32_t st = lds0 + (uint32_t)ld_slot * STAGE;
    if (++ld_slot == STAGES) ld_slot = 0;
    if (ld_j < my_units) {
      const int left = p.k - ld_ks * TG_BK;   // k from this stage on
      const i32x4 xrs = pp_rsrc_words(xp, range(LX, x_rows, p.xs_b, left));
      const i32x4 wrs = pp_rsrc_words(wp, range(LW, w_rows, p.ws_b, left));
      uint32_t kill = 0;
      if ((LX == OP_ROWS || LW == OP_ROWS) && left < TG_BK) kill = my_chunk * 8 >= left ? 0x80000000u : 0u;
#pragma unroll
      for (int i = 0; i < PER_WAVE; ++i) {
        const bool is_w = i < C::W_PER_WAVE;
        const bool rows = (is_w ? LW : LX) == OP_ROWS;
        dma_b128(is_w ? wrs : xrs, st + (wave + NW * i) * 1024, rows ? goff[i] | kill : goff[i]);
      }
      xp += LX == OP_ROWS ? TG_BK * 2 : TG_BK * p.xs_b;
      wp += LW == OP_ROWS ? TG_BK * 2 : TG_BK * p.ws_b;
      if (++ld_ks == ld_end) {
        if (++ld_j < my_units) ld_unit();
      }
    } else {   // past the last stage: zeros, so that every stage counts the same loads
#pragma unroll
      for (int i = 0; i < PER_WAVE; ++i) dma_b128(none, st + (wave + NW * i) * 1024, goff[i]);
    }
  };

  // ---- fragments: w rows (wn WNB + a) 32 + l32, x rows (wm WMB + b) 32 + l32, k = 16 ks + 8 hf .. + 7 ----
  auto frag_addr = [&](int L, int R, int blk, int ks) __attribute__((always_inline)) {
    if (L == OP_ROWS) {
      const int r = blk * 32 + l32, c = 2 * ks + hf;
      return (uint32_t)(r * 64 + ((c ^ ((r >> 2) & 3)) << 4));
    }
    const int a16 = lane & 15, e = a16 >> 2;
    const int col = blk * 32 + (lane & 16) + 4 * (a16 & 3);
    const int sw = R >= 128 ? e << 2 : (e >> 1) << 2;
    return (uint32_t)((16 * ks + 8 * hf + e) * (2 * R) + (((col >> 3) ^ sw) << 4) + (a16 & 1) * 8);
  };
  // OP_COLS: the second k step is a constant offset from the first
  uint32_t fa[WNB][LW == OP_ROWS ? 2 : 1], fb[WMB][LX == OP_ROWS ? 2 : 1];
#pragma unroll
  for (int ks = 0; ks < 2; ++ks) {
#pragma unroll
    for (int a = 0; a < WNB; ++a)
      if (LW == OP_ROWS || ks == 0) fa[a][ks] = opaque(lds0 + frag_addr(LW, BN, wn * WNB + a, ks));
#pragma unroll
    for (int b = 0; b < WMB; ++b)
      if (LX == OP_ROWS || ks == 0) fb[b][ks] = opaque(lds0 + C::W + frag_addr(LX, BM, wm * WMB + b, ks));
  }
  auto tr_read = [&](uint32_t at, int pitch) __attribute__((always_inline)) {
    const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(size_t)at);
    const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
        (__attribute__((address_space(3))) s16x4*)(size_t)(at + 4 * pitch));
    const u32x2 l = __builtin_bit_cast(u32x2, lo), h = __builtin_bit_cast(u32x2, hi);
    return (u32x4){l[0], l[1], h[0], h[1]};
  };

  f32x16 acc[WNB][WMB];
  const f32x16 zero = {};
#pragma unroll
  for (int a = 0; a < WNB; ++a)
#pragma unroll
    for (int b = 0; b < WMB; ++b) acc[a][b] = zero;

  struct Half {
    u32x4 a[WNB], b[WMB];
  };
  int rd_slot = 0;
  auto read_half = [&](int ks, Half& f) __attribute__((always_inline)) {
    const uint32_t so = (uint32_t)rd_slot * STAGE;
#pragma unroll
    for (int a = 0; a < WNB; ++a) {
      if constexpr (LW == OP_ROWS) f.a[a] = lds_load<u32x4>(fa[a][ks] + so);
      else f.a[a] = tr_read(fa[a][0] + so + ks * 16 * 2 * BN, 2 * BN);
    }
#pragma unroll
    for (int b = 0; b < WMB; ++b) {
      if constexpr (LX == OP_ROWS) f.b[b] = lds_load<u32x4>(fb[b][ks] + so);
      else f.b[b] = tr_read(fb[b][0] + so + ks * 16 * 2 * BM, 2 * BM);
    }
  };
  auto mfmas = [&](const Half& f) __attribute__((always_inline)) {
#pragma unroll
    for (int a = 0; a < WNB; ++a)
#pragma unroll
      for (int b = 0; b < WMB; ++b)
        acc[a][b] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, f.a[a]),
                                                            __builtin_bit_cast(bf16x8, f.b[b]), acc[a][b], 0, 0, 0);
  };

  // ---- epilogue: acc[a][b][4 g + e] is row (wm WMB + b) 32 + l32, w row (wn WNB + a) 32 + 8 g + 4 hf + e ----
  // Staging of one wave: 32 rows x 128 bytes, 16-byte chunk c of row r at
  // r * 128 + ((c ^ ((r >> 1) & 7)) << 4); 64 bf16 columns, or 32 f32 ones where
  // the value still meets memory (RES, EPI_DGATED) or is stored in f32.
  const uint32_t stg = lds0 + C::RING + (uint32_t)wave * TG_STG;
  auto stg_at = [&](int r, int c) __attribute__((always_inline)) {
    return stg + (uint32_t)r * 128 + (((uint32_t)c ^ (((uint32_t)r >> 1) & 7)) << 4);
  };
  auto put16 = [&](int c, f32x4 v) __attribute__((always_inline)) {
    const f32x2 lo = {v[0], v[1]}, hi = {v[2], v[3]};
    const u32x2 q = {__builtin_bit_cast(uint32_t, __builtin_convertvector(lo, bf16x2)),
                     __builtin_bit_cast(uint32_t, __builtin_convertvector(hi, bf16x2))};
    lds_store<u32x2>(stg_at(l32, c >> 3) + ((c & 7) << 1), q);
  };
  auto put32 = [&](int c, f32x4 v) __attribute__((always_inline)) {
    lds_store<u32x4>(stg_at(l32, c >> 2), __builtin_bit_cast(u32x4, v));
  };
  // The staged rows row0 .. + 31, columns col0 .. + width, to bf16 rows at dst
  auto flush16 = [&](char* dst, int64_t stride, int64_t row0, int64_t col0, int width, int64_t end)
      __attribute__((always_inline)) {
    const int c = lane & 7;
    const int64_t col = col0 + c * 8;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int r = (lane >> 3) + 8 * j;
      const u32x4 v = lds_load<u32x4>(stg_at(r, c));
      const int64_t row = row0 + r;
      if (row < p.m && col < end && c * 8 < width) *reinterpret_cast<u32x4*>(dst + (row * stride + col) * 2) = v;
    }
  };
  // The same from f32 staging, with what the value meets in memory
  auto flush32 = [&](char* dst, int64_t row0, int col0, int width) __attribute__((always_inline)) {
    const int c = lane & 7;
    const int col = col0 + c * 4;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int r = (lane >> 3) + 8 * j;
      f32x4 t = __builtin_bit_cast(f32x4, lds_load<u32x4>(stg_at(r, c)));
      const int64_t row = row0 + r;
      if (row < p.m && col < p.n && c * 4 < width) {
        if constexpr (EPI == EPI_DGATED) {
          const char* g0 = p.pre + (row * p.ps + col) * 2;
          const bf16x4 gv = *reinterpret_cast<const bf16x4*>(g0);
          const bf16x4 uv = *reinterpret_cast<const bf16x4*>(g0 + (int64_t)p.n * 2);
          bf16x4 dg, du;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const ActPair q = act_pair(p.act, (float)gv[e]);
            dg[e] = (bf16)(t[e] * (float)uv[e] * q.slope);
            du[e] = (bf16)(t[e] * q.value);
          }
          char* o = dst + (row * p.ys + col) * 2;
          *reinterpret_cast<bf16x4*>(o) = dg;
          *reinterpret_cast<bf16x4*>(o + (int64_t)p.n * 2) = du;
        } else {
          if constexpr (RES) {
            if (p.res_bf16) {
              const bf16x4 o = *reinterpret_cast<const bf16x4*>(p.res + (row * p.rs + col) * 2);
#pragma unroll
              for (int e = 0; e < 4; ++e) t[e] += p.beta * (float)o[e];
            } else {
              const f32x4 o = *reinterpret_cast<const f32x4*>(p.res + (row * p.rs + col) * 4);
#pragma unroll
              for (int e = 0; e < 4; ++e) t[e] += p.beta * o[e];
            }
          }
          if constexpr (OUT16) {
            bf16x4 o;
#pragma unroll
            for (int e = 0; e < 4; ++e) o[e] = (bf16)t[e];
            *reinterpret_cast<bf16x4*>(dst + (row * p.ys + col) * 2) = o;
          } else {
            *reinterpret_cast<f32x4*>(dst + (row * p.ys + col) * 4) = t;
          }
        }
      }
    }
  };
  constexpr bool STG16 = EPI == EPI_GATED || EPI == EPI_DXENT || (EPI == EPI_LINEAR && OUT16 && !RES);

  auto tile_end = [&](const Unit& q) __attribute__((always_inline)) {
    const int ncol0 = q.nt * BNO;
#pragma unroll
    for (int b = 0; b < WMB; ++b) {
      const int64_t row0 = (int64_t)q.mt * BM + (wm * WMB + b) * 32;
      if constexpr (EPI == EPI_GATED) {
        // block wn WNB + a: 16 gate rows and their 16 up rows, output columns 16 (wn WNB + a) ..
        constexpr int PER = WNB < 4 ? WNB : 4;
#pragma unroll
        for (int a0 = 0; a0 < WNB; a0 += PER) {
          const int col = ncol0 + (wn * WNB + a0) * 16;
          if (p.pre) {
#pragma unroll
            for (int part = 0; part < 2; ++part) {
#pragma unroll
              for (int a = a0; a < a0 + PER; ++a)
#pragma unroll
                for (int g = 0; g < 2; ++g) {
                  f32x4 v;
#pragma unroll
                  for (int e = 0; e < 4; ++e) v[e] = acc[a][b][4 * (g + 2 * part) + e];
                  put16((a - a0) * 16 + 8 * g + 4 * hf, v);
                }
              flush16(p.pre + (part ? (int64_t)p.n * 2 : 0), p.ps, row0, col, PER * 16, p.n);
            }
          }
#pragma unroll
          for (int a = a0; a < a0 + PER; ++a)
#pragma unroll
            for (int g = 0; g < 2; ++g) {
              f32x4 v;
#pragma unroll
              for (int e = 0; e < 4; ++e) v[e] = acc[a][b][4 * g + e];
              v = act_apply4(p.act, v);
#pragma unroll
              for (int e = 0; e < 4; ++e) v[e] *= acc[a][b][4 * (g + 2) + e];
              put16((a - a0) * 16 + 8 * g + 4 * hf, v);
            }
          flush16(p.y, p.ys, row0, col, PER * 16, p.n);
        }
      } else if constexpr (EPI == EPI_XENT || EPI == EPI_DXENT) {
        const int64_t row = row0 + l32;
        const bool in = row < p.m;
        const int colb = ncol0 + wn * WNB * 32 + 4 * hf;   // this lane's first column
        const int t = in ? p.target[row] : p.ignore;
        const int tc = t == p.ignore ? -1 : t - p.col0;    // the target's column, if it is in [0, n)
        // Scores in place of the products, columns past n -inf. (One block of
        // columns at a time: with all bias loads in flight at once the 256 x 256
        // shape spills.)
        const bool whole = ncol0 + BN <= p.n;
#pragma unroll
        for (int a = 0; a < WNB; ++a) {
          if (p.bias) {
            f32x4 bv[4];
            if (whole) {   // (uniform)
#pragma unroll
              for (int g = 0; g < 4; ++g) bv[g] = *reinterpret_cast<const f32x4*>(p.bias + colb + a * 32 + 8 * g);
            } else {
#pragma unroll
              for (int g = 0; g < 4; ++g)
#pragma unroll
                for (int e = 0; e < 4; ++e) bv[g][e] = p.bias[min(colb + a * 32 + 8 * g + e, p.n - 1)];
            }
#pragma unroll
            for (int g = 0; g < 4; ++g)
#pragma unroll
              for (int e = 0; e < 4; ++e) acc[a][b][4 * g + e] = __builtin_fmaf(p.alpha, acc[a][b][4 * g + e], bv[g][e]);
          } else {
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[a][b][e] *= p.alpha;
          }
          if (!whole) {
#pragma unroll
            for (int g = 0; g < 4; ++g)
#pragma unroll
              for (int e = 0; e < 4; ++e)
                if (colb + a * 32 + 8 * g + e >= p.n) acc[a][b][4 * g + e] = -INFINITY;
          }
          __builtin_amdgcn_sched_barrier(0);
        }
        if constexpr (EPI == EPI_XENT) {
          if (__any(tc >= colb && tc < colb + WNB * 32)) {
#pragma unroll
            for (int a = 0; a < WNB; ++a)
#pragma unroll
              for (int g = 0; g < 4; ++g)
#pragma unroll
                for (int e = 0; e < 4; ++e)
                  if (in && tc == colb + a * 32 + 8 * g + e && tc < p.n) p.at[row] = acc[a][b][4 * g + e];
          }
          float top = -INFINITY;
#pragma unroll
          for (int a = 0; a < WNB; ++a)
#pragma unroll
            for (int e = 0; e < 16; ++e) top = fmaxf(top, acc[a][b][e]);
          top = fmaxf(top, __shfl_xor(top, 32, 64));
          const float base = top == -INFINITY ? 0.f : top;
          float sum = 0.f;
#pragma unroll
          for (int a = 0; a < WNB; ++a) {
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int e = 0; e < 16; ++e) sum += __builtin_amdgcn_exp2f((acc[a][b][e] - base) * 1.44269504088896f);
          }
          sum += __shfl_xor(sum, 32, 64);
          if (in && hf == 0) p.part[(int64_t)(q.nt * C::NWN + wn) * p.m + row] = make_float2(top, sum);
        } else {
          const float lse = in ? p.lse[row] : 0.f;
          const float f = in && t != p.ignore ? p.dl[row] : 0.f;
          // (an ignored row is zeros whatever its scores are)
          const bool live = f != 0.f || f != f;
#pragma unroll
          for (int a0 = 0; a0 < WNB; a0 += (WNB < 2 ? 1 : 2)) {
            constexpr int PER = WNB < 2 ? 1 : 2;
#pragma unroll
            for (int a = a0; a < a0 + PER; ++a)
#pragma unroll
              for (int g = 0; g < 4; ++g) {
                __builtin_amdgcn_sched_barrier(0);
                const int col = colb + a * 32 + 8 * g;
                f32x4 v;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                  float pr = __builtin_amdgcn_exp2f((acc[a][b][4 * g + e] - lse) * 1.44269504088896f);
                  if (col + e == tc) pr -= 1.f;
                  v[e] = live && (whole || col + e < p.n) ? pr * f : 0.f;
                }
                put16((a - a0) * 32 + 8 * g + 4 * hf, v);
              }
            flush16(p.y, p.ys, row0, ncol0 + (wn * WNB + a0) * 32, PER * 32, p.n_store);
          }
        }
      } else {
        constexpr int COLS = STG16 ? 64 : 32;
        constexpr int PER = COLS / 32 < WNB ? COLS / 32 : WNB;
        char* dst = EPI == EPI_PART ? p.y + (int64_t)q.s * p.m * p.n * 4 : p.y;
#pragma unroll
        for (int a0 = 0; a0 < WNB; a0 += PER) {
          const int col0 = ncol0 + (wn * WNB + a0) * 32;
          f32x4 z[PER * 4];
#pragma unroll
          for (int a = 0; a < PER; ++a)
#pragma unroll
            for (int g = 0; g < 4; ++g)
#pragma unroll
              for (int e = 0; e < 4; ++e)
                z[a * 4 + g][e] = EPI == EPI_LINEAR ? p.alpha * acc[a0 + a][b][4 * g + e] : acc[a0 + a][b][4 * g + e];
          if constexpr (EPI == EPI_LINEAR) {
            if (p.bias) {
#pragma unroll
              for (int i = 0; i < PER * 4; ++i) {
                const int col = min(col0 + i * 8 + 4 * hf, p.n - 4);
                const f32x4 bv = *reinterpret_cast<const f32x4*>(p.bias + col);
#pragma unroll
                for (int e = 0; e < 4; ++e) z[i][e] += bv[e];
              }
            }
            if (p.pre) {
#pragma unroll
              for (int i = 0; i < PER * 4; ++i) put16(i * 8 + 4 * hf, z[i]);
              flush16(p.pre, p.ps, row0, col0, PER * 32, p.n);
            }
            if (p.act != ACT_NONE) {
#pragma unroll
              for (int i = 0; i < PER * 4; ++i) z[i] = act_apply4(p.act, z[i]);
            }
          }
          if constexpr (STG16) {
#pragma unroll
            for (int i = 0; i < PER * 4; ++i) put16(i * 8 + 4 * hf, z[i]);
            flush16(dst, p.ys, row0, col0, PER * 32, p.n);
          } else {
#pragma unroll
            for (int i = 0; i < PER * 4; ++i) put32(i * 8 + 4 * hf, z[i]);
            flush32(dst, row0, col0, PER * 32);
          }
        }
      }
    }
#pragma unroll
    for (int a = 0; a < WNB; ++a)
#pragma unroll
      for (int b = 0; b < WMB; ++b) acc[a][b] = zero;
  };

  // The cross entropy epilogues need the registers of the next unit's first
  // operands: they are read after it.
  constexpr bool LATE = EPI == EPI_XENT || EPI == EPI_DXENT;
  // One iteration per stage: read its second k step while the first one's
  // MFMAs run; wait for the next stage (vmcnt) and for every wave to have read
  // this one (barrier), refill its slot, and read the next stage's first step
  // while the second step's MFMAs run.
  ld_unit();
  Half h0, h1;
#pragma unroll
  for (int i = 0; i < STAGES; ++i) issue();
  asm volatile("s_waitcnt vmcnt(%0)" :: "n"((STAGES - 1) * PER_WAVE) : "memory");
  lds_barrier();
  read_half(0, h0);
  for (int j = 0; j < my_units; ++j) {
    const Unit q = unit_of(j);
    const int stages = min(p.kper, kst - q.s * p.kper);
    for (int s = 0; s < stages; ++s) {
      read_half(1, h1);
      mfmas(h0);
      asm volatile("s_waitcnt vmcnt(%0)" :: "n"((STAGES - 2) * PER_WAVE) : "memory");
      lds_barrier();
      issue();
      if (++rd_slot == STAGES) rd_slot = 0;
      if (!LATE || s + 1 < stages) read_half(0, h0);
      mfmas(h1);
    }
    tile_end(q);
    if (LATE) read_half(0, h0);
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");   // the dummy loads past the end
}

template <int SH, int LX, int LW, int EPI, bool OUT16, bool RES>
int tile_launch_shape(TileParams p, const TilePlan& plan, int cus, hipStream_t stream) {
  using C = TileShapeOf<SH>;
  const int bno = EPI == EPI_GATED ? C::BN / 2 : C::BN;
  const int64_t tm = (p.m + C::BM - 1) / C::BM, tn = (p.n + bno - 1) / bno;
  const int64_t units = tm * tn * plan.splits;
  if (units >= ((int64_t)1 << 30)) return fail(INL_E_UNSUPPORTED, "too many output tiles");
  p.tiles_m = (int32_t)tm;
  p.tiles_n = (int32_t)tn;
  p.group = TG_GROUP;
  p.units = (int32_t)units;
  p.per_xcd = (int32_t)((units + TG_XCDS - 1) / TG_XCDS);
  p.wg_per_xcd = std::max(1, std::min(cus / TG_XCDS * C::WPC, p.per_xcd));
  p.kper = plan.kper;
  const void* fn = (const void*)tile_gemm_kernel<SH, LX, LW, EPI, OUT16, RES>;
  int rc = set_max_dynamic_lds(fn, C::LDS);
  if (rc) return rc;
  void* args[] = {&p};
  INL_HIP_TRY(hipLaunchKernel(fn, dim3((unsigned)(p.wg_per_xcd * TG_XCDS)), dim3(C::NW * 64), args, C::LDS, stream));
  return INL_OK;
}

template <int LX, int LW, int EPI, bool OUT16, bool RES>
int tile_launch(const TileParams& p, const TilePlan& plan, int cus, hipStream_t stream) {
  switch (plan.shape) {
    case 0: return tile_launch_shape<0, LX, LW, EPI, OUT16, RES>(p, plan, cus, stream);
    case 1: return tile_launch_shape<1, LX, LW, EPI, OUT16, RES>(p, plan, cus, stream);
    default: return tile_launch_shape<2, LX, LW, EPI, OUT16, RES>(p, plan, cus, stream);
  }
}

}  // namespace

// The launches that the operators use (one file per operand order). out_bf16:
// dtype of y; a residual when p.res is set. With plan.splits > 1 the product
// goes to `part` and tile_finish applies the epilogue.
int tile_nt_linear(TileParams p, const TilePlan& plan, bool out_bf16, float* part, int cus, hipStream_t stream);
int tile_nt_gated(TileParams p, const TilePlan& plan, float* part, int cus, hipStream_t stream);
int tile_nt_xent(const TileParams& p, const TilePlan& plan, int cus, hipStream_t stream);
int tile_nt_dxent(const TileParams& p, const TilePlan& plan, int cus, hipStream_t stream);
int tile_nn_linear(TileParams p, const TilePlan& plan, bool out_bf16, float* part, int cus, hipStream_t stream);
int tile_nn_dgated(TileParams p, const TilePlan& plan, float* part, int cus, hipStream_t stream);
int tile_tn_linear(TileParams p, const TilePlan& plan, bool out_bf16, float* part, int cus, hipStream_t stream);

// Adds the partial tiles [splits][m][n] (EPI_GATED: [splits][m][2n]) in split
// order and applies the epilogue (EPI_LINEAR, EPI_GATED, EPI_DGATED).
int tile_finish(const TileParams& p, int epi, int splits, const float* part, bool out_bf16, hipStream_t stream);

}  // namespace inl
