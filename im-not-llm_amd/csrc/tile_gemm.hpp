// Tiled bf16 matrix products with the operands in either storage order and an
// epilogue per use: the products of the linear layer, the gated feed-forward
// block and the softmax cross entropy, forward and backward.
//
//   c[m, n] = sum_k X(m, k) W(n, k),   f32 accumulation
//
// An operand is stored as rows of k (OP_ROWS: x [M, K], w [N, K], the forward
// products) or as rows of m or n (OP_COLS: [K, M], [K, N]; dx = dz . W reads
// W that way, dW = dz^T . x both). Nothing is transposed in memory: a stage of
// an OP_COLS operand sits in LDS as it is stored (64 rows of k) and its MFMA
// operands are read with ds_read_b64_tr_b16, which hands lane j of 16 the four
// k values of column j.
//
// Pipeline: 8 or 4 waves, each WNB x WMB blocks of v_mfma_f32_16x16x32_bf16; a
// ring of 64-wide k slices in LDS (128-byte rows: whole cache lines) filled by direct
// loads, operands read a phase ahead (see the k loop). A workgroup is persistent: its
// units (tile, k range) form one stream of stages, so the next unit's first loads
// are in flight while a unit's epilogue runs.
//
// Rates on random values, 8,192^3, TFLOP/s: 1,472 with both operands as rows of k, 1,453
// with W as rows of n, about 1,430 with both as rows of m and n (a large library
// product reached 1,422 on the card): bound by power (matrix cores 72 to 74 % busy at
// 1.5 to 1.6 GHz of 2.4). Products of one to three rounds of tiles are bound by their first
// loads and epilogues, which nothing hides (20,011 x 768 x 768 takes 27 us for 17, matrix
// cores 31 % busy). In 128 x 128 tiles two stages of a CU take 0.94 us for 0.43 of products
// (8,192 x 1,024 x 2,048: matrix cores 35 % busy, LDS 20 %; of the waves' time 30 % goes to
// barriers and loads, 33 % to waiting for an instruction slot, 6 % for LDS's): no unit is
// full, the pieces of a stage stand in line.
//
// The 16 x 16 x 32 instruction and not 32 x 32 x 16: both run at the same rate, but a large
// product is bound by the card's power, and on values that toggle (normal
// random bf16) a loop of the former alone held 2,022 TFLOP/s and of the latter 1,748
// (on zeros 2,448 and 2,329).
//
// Units: a tile's k range may be cut into `splits` parts of `kper` stages
// (EPI_PART writes f32 partial tiles, a second kernel adds them in order), so
// that dW of a 768 x 768 layer over 20,000 tokens (9 tiles) fills 256 CUs.
//
// Unit order: split-major, then groups of GROUP m-tiles, n outer and m inner
// within a group, cut into 8 contiguous ranges, one per XCD (workgroup b runs
// on XCD b % 8). The ~32 units an XCD runs at one time form a rectangle of 4 x
// 8 tiles: 12 operand slices per stage instead of 33 for a row of tiles, and output
// rows of 4 KiB at a time (8 x 4 tiles: the gate gradients of 16,384 x 4,096 took 8 % longer).
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
  EPI_XENT = 4,      // scores alpha c + bias: row maxima and sums of exponentials per 16 WNB columns
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
  int32_t col0, vocab;      // vocabulary id of column 0, and their number
  int32_t ignore;
  int32_t n_store;          // columns of y, past n zeros (EPI_DXENT)
  // schedule
  int32_t tiles_m, tiles_n, group;
  int32_t units, per_xcd, wg_per_xcd;
  int32_t kper;             // stages per unit
};

constexpr int TG_BK = 64;      // k per LDS stage
constexpr int TG_KS = TG_BK / 32;   // MFMA k steps of it
constexpr int TG_ROW = TG_BK * 2;
constexpr int TG_STG = 4096;   // per-wave epilogue staging: 32 rows x 128 bytes
constexpr int TG_XCDS = 8;
constexpr int TG_GROUP = 4;

template <int NWN_, int NWM_, int WNB_, int WMB_, int STAGES_, int WPC_>
struct TileShape {
  static constexpr int NWN = NWN_, NWM = NWM_, WNB = WNB_, WMB = WMB_;
  static constexpr int NW = NWN * NWM;
  static constexpr int BN = NWN * WNB * 16, BM = NWM * WMB * 16;
  static constexpr int STAGES = STAGES_, WPC = WPC_;
  static constexpr int W = BN * TG_ROW, X = BM * TG_ROW;
  static constexpr int STAGE = W + X;
  // Direct loads of 1 KiB per wave and stage. With four or more w blocks per wave
  // a stage's w comes in H = 2 halves (each wave's lower and upper blocks).
  static constexpr int H = WNB >= 4 ? 2 : 1;
  static constexpr int WH = WNB / H;
  static constexpr int PX = X / 1024 / NW, PW = W / 1024 / NW / H;
  static constexpr int PER_WAVE = PX + H * PW;
  static constexpr int RING = STAGES * STAGE;
  static constexpr int LDS = RING + NW * TG_STG;
  static_assert(X % (1024 * NW) == 0 && W % (1024 * NW * H) == 0, "the direct loads split evenly over the waves");
  static_assert(NW % 4 == 0, "w blocks of one wave are all gate or all up rows (EPI_GATED)");
  static_assert(H == 1 || (WH * 2 == NW && STAGES == 2), "a half is the waves' next blocks");
  static_assert((STAGES - 1) * PER_WAVE <= 63, "vmcnt range");
};
// 0: 256 x 256, one workgroup of 8 waves per CU. 1: 128 x 128, two of 4 waves
// per CU. 2: 64 x 64, for outputs that would leave most of the chip idle.
template <int SH>
using TileShapeOf = std::conditional_t<SH == 0, TileShape<2, 4, 8, 4, 2, 1>,
                    std::conditional_t<SH == 1, TileShape<2, 2, 4, 4, 2, 2>, TileShape<2, 2, 2, 2, 3, 2>>>;
constexpr int TG_SHAPES = 3;

struct TilePlan {
  int shape;
  int splits;
  int32_t kper;
};
// The shape and k split with the least estimated time. by_cols: operands stored by
// columns (0 to 2); `gated`: w has 2n rows. max_splits 1 keeps every tile in one unit.
TilePlan tile_plan(int64_t m, int64_t n, int64_t k, int by_cols, bool gated, int max_splits, int cus);

// f32 partials of a plan (0 for one split).
inline size_t tile_part_bytes(const TilePlan& t, int64_t m, int64_t n) {
  return t.splits > 1 ? (size_t)t.splits * (size_t)m * (size_t)n * 4 : 0;
}

namespace {

// 16-byte chunk c of stored row r of an operand stage, R = rows of m or n per
// tile. OP_ROWS: 128-byte rows, the 16 rows of one ds_read_b128 pass cover all
// banks. OP_COLS: 2 R-byte rows, the 8 rows x 32 bytes that 32 lanes of a
// transposed read touch cover all banks.
template <int L, int R>
__device__ __forceinline__ int tg_swz(int r, int c) {
  if constexpr (L == OP_ROWS) return c ^ ((r >> 1) & 7);
  if constexpr (R >= 128) return c ^ ((r & 3) << 2) ^ (((r >> 3) & 1) << 1);
  return c ^ (((r >> 1) & 1) << 2) ^ (((r >> 3) & 1) << 1);
}
template <int L, int R>
constexpr int tg_chunks() { return L == OP_ROWS ? TG_ROW / 16 : R / 8; }

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
  const int l16 = lane & 15, quad = lane >> 4;

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
  // Per-lane byte offset of this wave's first 1 KiB block of x and of w; the
  // following blocks are uniform steps away (added at each load: eight offsets
  // held in registers would not fit beside the operands).
  // OP_ROWS: LDS row r of an operand is its row r; a half of w is every other
  // block. OP_COLS: [64 k][columns]; w's halves are tiles of their own, each
  // with the half's columns of both waves along n.
  constexpr int NWH = BN / C::H;   // columns of an OP_COLS half of w
  uint32_t xo, wo;
  {
    constexpr int cpr = tg_chunks<LX, BM>();
    const int at = wave * 64 + lane, r = at / cpr;
    xo = (uint32_t)r * (uint32_t)p.xs_b + tg_swz<LX, BM>(r, at % cpr) * 16;
  }
  {
    constexpr int cpr = tg_chunks<LW, NWH>();
    const int at = wave * 64 + lane;
    int r = at / cpr;
    int c = tg_swz<LW, NWH>(r, at % cpr);
    if (LW == OP_COLS) c = c / (C::WH * 2) * (WNB * 2) + c % (C::WH * 2);   // chunk of 8 columns
    // EPI_GATED: LDS rows are 16 gate rows, then their 16 up rows, and so on
    if (EPI == EPI_GATED) r = (r >> 5) * 16 + (r & 15);
    wo = (uint32_t)r * (uint32_t)p.ws_b + c * 16;
  }
  const uint32_t xstep = (LX == OP_ROWS ? NW * 8 : NW * 64 / tg_chunks<LX, BM>()) * (uint32_t)p.xs_b;
  const uint32_t wstep = (LW == OP_COLS ? NW * 64 / tg_chunks<LW, NWH>() : EPI == EPI_GATED ? NW * 4 : NW * 8) * (uint32_t)p.ws_b;

  // Descriptors start at a unit's first row and at the stage's k, so that no
  // offset exceeds 31 bits; rows past the end read as zero, and so does k past
  // the end: OP_COLS by the range, OP_ROWS by an offset out of it. They, the
  // offsets and the LDS base are kept from stage to stage and only moved on: the
  // scalar instructions of a stage's loads stand in line with its products.
  const int tail = p.k - (kst - 1) * TG_BK;   // k of the last stage
  const uint32_t xnext = LX == OP_ROWS ? TG_ROW : TG_BK * (uint32_t)p.xs_b;
  const uint32_t wnext = LW == OP_ROWS ? TG_ROW : TG_BK * (uint32_t)p.ws_b;
  int ld_j = 0, ld_ks = 0, ld_end = 0;
  i32x4 xrs, wrs;
  uint32_t x_bytes = 0, w_bytes = 0, x_cut = 0, w_cut = 0;   // ranges, and by how much the last stage's are shorter
  // (whole 16-byte chunks: an odd row end lies inside its padded row)
  auto range = [&](int L, uint32_t rows, int64_t stride, int ks) __attribute__((always_inline)) {
    return L == OP_ROWS ? (rows - 1) * (uint32_t)stride + (uint32_t)((ks + 7) & ~7) * 2
                        : (uint32_t)(ks - 1) * (uint32_t)stride + ((rows + 7) & ~7u) * 2;
  };
  auto ld_tail = [&]() __attribute__((always_inline)) {
    x_bytes -= x_cut;
    w_bytes -= w_cut;
    if (LX == OP_ROWS || LW == OP_ROWS) {
      // (the lane's chunk anew: this is rare, and a register less in the loop)
      const int l = (int)opaque((uint32_t)lane);
      const int chunk = (l & 7) ^ ((wave * 4 + (l >> 4)) & 7);
      const uint32_t kill = chunk * 8 >= tail ? 0x80000000u : 0u;
      if (LX == OP_ROWS) xo |= kill;
      if (LW == OP_ROWS) wo |= kill;
    }
  };
  auto ld_unit = [&]() __attribute__((always_inline)) {
    const Unit q = unit_of(ld_j);
    ld_ks = q.s * p.kper;
    ld_end = min(ld_ks + p.kper, kst);
    const int64_t k0 = (int64_t)ld_ks * TG_BK;
    const int64_t r0 = (int64_t)q.mt * BM;
    // (a 64-bit minimum is vector code)
    const uint32_t x_rows = (uint32_t)__builtin_amdgcn_readfirstlane((int)min((int64_t)BM, p.m - r0));
    const int c0 = q.nt * BNO;
    const uint32_t w_rows = (uint32_t)min(BNO, p.n - c0);
    const int64_t c1 = EPI == EPI_GATED && (wave & 2) ? (int64_t)p.n + c0 : (int64_t)c0;
    const uint32_t xr = range(LX, x_rows, p.xs_b, TG_BK), wr = range(LW, w_rows, p.ws_b, TG_BK);
    x_bytes = xr;
    w_bytes = wr;
    x_cut = (uint32_t)__builtin_amdgcn_readfirstlane((int)(xr - range(LX, x_rows, p.xs_b, tail)));
    w_cut = (uint32_t)__builtin_amdgcn_readfirstlane((int)(wr - range(LW, w_rows, p.ws_b, tail)));
    xrs = pp_rsrc_words(p.x + (LX == OP_ROWS ? r0 * p.xs_b + k0 * 2 : k0 * p.xs_b + r0 * 2), xr);
    wrs = pp_rsrc_words(p.w + (LW == OP_ROWS ? c1 * p.ws_b + k0 * 2 : k0 * p.ws_b + c1 * 2), wr);
    xo &= 0x7fffffffu;
    wo &= 0x7fffffffu;
    if (ld_ks + 1 == kst) ld_tail();
    xrs[2] = (int)x_bytes;
    wrs[2] = (int)w_bytes;
  };
  auto move_on = [&](i32x4& rs, uint32_t by) __attribute__((always_inline)) {
    const uint64_t at = (((uint64_t)(uint32_t)rs[1] << 32) | (uint32_t)rs[0]) + by;
    rs[0] = (int)(uint32_t)at;
    rs[1] = (int)(uint32_t)(at >> 32);
  };
  // Loads of the cursor's stage in two parts: x with the first half of w (h = 0),
  // then the other half, then move the cursor on (end). Past the last stage:
  // zeros, so that every stage counts the same loads.
  uint32_t ld_at = lds0 + (uint32_t)wave * 1024, ld_slot = 0;
  auto load = [&](int h, int i) __attribute__((always_inline)) {
    if (h == 0 && i < C::PX) {
      dma_b128_at(xrs, ld_at + C::W + NW * 1024 * i, xo, i * xstep);
      return;
    }
    if (h == 0) i -= C::PX;
    const uint32_t half = LW == OP_ROWS ? h * wstep : h * C::WH * 32;
    const int blk = LW == OP_ROWS ? NW * (C::H * i + h) : h * (NWH / 8) + NW * i;
    dma_b128_at(wrs, ld_at + blk * 1024, wo, half + i * (LW == OP_ROWS ? C::H * wstep : wstep));
  };
  auto end = [&](int h) __attribute__((always_inline)) {
    if (h + 1 < C::H) return;
    ld_slot = ld_slot + 1 == STAGES ? 0 : ld_slot + 1;
    ld_at = lds0 + (uint32_t)wave * 1024 + ld_slot * STAGE;
    move_on(xrs, xnext);
    move_on(wrs, wnext);
    if (++ld_ks >= ld_end) {   // (past the last unit, too)
      if (++ld_j < my_units) {
        ld_unit();
      } else {
        x_bytes = w_bytes = 0;
      }
    } else if (ld_ks + 1 == kst) {
      ld_tail();
    }
    // (set apart from the branches: a choice between whole descriptors is made in
    // vector registers)
    xrs[2] = (int)x_bytes;
    wrs[2] = (int)w_bytes;
    asm volatile("" : "+s"(xrs), "+s"(wrs));
  };
  constexpr int L0 = C::PX + C::PW, L1 = C::H == 2 ? C::PW : 0;   // loads of the two parts
  auto issue = [&](int h) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < (h ? L1 : L0); ++i) load(h, i);
    end(h);
  };

  // ---- fragments: w rows (wn WNB + a) 16 + l16, x rows (wm WMB + b) 16 + l16, k = 32 ks + 8 quad .. + 7 ----
  // OP_ROWS: blocks are 16 rows apart, a multiple of the swizzle's period, so a
  // block is a constant offset from the first. OP_COLS: so is a k step; of x, blocks
  // 2 and 3 are 0 and 1 with chunk bit 2 the other way (two registers less).
  auto frag_addr = [&](int L, int R, int blk, int ks) __attribute__((always_inline)) {
    if (L == OP_ROWS) {
      const int r = blk * 16 + l16, c = 4 * ks + quad;
      return (uint32_t)(r * TG_ROW + ((c ^ ((r >> 1) & 7)) << 4));
    }
    // lane 4 e + j of 16 addresses columns 4 j .. + 3 of k row e and receives
    // column 4 e + j of k rows 0 .. 3; a second read takes rows 4 .. 7
    const int e = l16 >> 2, r = 8 * quad + e;
    const int c = blk * 2 + ((l16 & 3) >> 1);
    const int sw = (R >= 128 ? e << 2 : (e >> 1) << 2) ^ ((quad & 1) << 1);
    return (uint32_t)(r * (2 * R) + ((c ^ sw) << 4) + (l16 & 1) * 8);
  };
  constexpr int NFA = LW == OP_ROWS ? TG_KS : C::WH, NFB = 2;
  static_assert(TG_KS == 2 && (WMB == 2 || WMB == 4), "two address registers for x");
  uint32_t fa[NFA], fb[NFB];
#pragma unroll
  for (int i = 0; i < NFA; ++i)
    fa[i] = opaque(lds0 + (LW == OP_ROWS ? frag_addr(LW, BN, wn * WNB, i) : frag_addr(LW, NWH, wn * C::WH + i, 0)));
#pragma unroll
  for (int i = 0; i < NFB; ++i)
    fb[i] = opaque(lds0 + C::W + (LX == OP_ROWS ? frag_addr(LX, BM, wm * WMB, i) : frag_addr(LX, BM, wm * WMB + i, 0)));
  auto tr_read = [&](uint32_t at, int pitch) __attribute__((always_inline)) {
    const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(size_t)at);
    const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
        (__attribute__((address_space(3))) s16x4*)(size_t)(at + 4 * pitch));
    const u32x2 l = __builtin_bit_cast(u32x2, lo), h = __builtin_bit_cast(u32x2, hi);
    return (u32x4){l[0], l[1], h[0], h[1]};
  };
  // (the addresses move from slot to slot, so that what is left is a constant
  // offset of the read)
  int rd_slot = 0;
  auto rd_next = [&]() __attribute__((always_inline)) {
    const bool wrap = ++rd_slot == STAGES;
    if (wrap) rd_slot = 0;
    const uint32_t by = wrap ? (uint32_t)-(int)((STAGES - 1) * STAGE) : (uint32_t)STAGE;
#pragma unroll
    for (uint32_t& a : fa) a = opaque(a + by);
#pragma unroll
    for (uint32_t& b : fb) b = opaque(b + by);
  };
  auto read_w = [&](int h, int i, int ks) __attribute__((always_inline)) {
    if constexpr (LW == OP_ROWS) return lds_load<u32x4>(fa[ks] + (h * C::WH + i) * 16 * TG_ROW);
    else return tr_read(fa[i] + h * (C::W / C::H) + ks * 32 * 2 * NWH, 2 * NWH);
  };
  auto read_x = [&](int b, int ks) __attribute__((always_inline)) {
    if constexpr (LX == OP_ROWS) return lds_load<u32x4>(fb[ks] + b * 16 * TG_ROW);
    else return tr_read((b < 2 ? fb[b] : opaque(fb[b & 1]) ^ 64u) + ks * 32 * 2 * BM, 2 * BM);
  };

  f32x4 acc[WNB][WMB];
  const f32x4 zero = {};
#pragma unroll
  for (int a = 0; a < WNB; ++a)
#pragma unroll
    for (int b = 0; b < WMB; ++b) acc[a][b] = zero;

  auto mfma = [&](int a, int b, const u32x4& w, const u32x4& x) __attribute__((always_inline)) {
    acc[a][b] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, w), __builtin_bit_cast(bf16x8, x),
                                                        acc[a][b], 0, 0, 0);
  };

  // ---- epilogue: acc[a][b][e] is row (wm WMB + b) 16 + l16, w row (wn WNB + a) 16 + 4 quad + e ----
  // Staging of one wave: 32 rows (two x blocks) x 128 bytes, 16-byte chunk c of row r at
  // r * 128 + ((c ^ ((r >> 1) & 7)) << 4); 64 bf16 columns, or 32 f32 ones.
  const uint32_t stg = lds0 + C::RING + (uint32_t)wave * TG_STG;
  // (the lane anew for each tile: what an epilogue derives from it would otherwise
  // be kept in registers through the k loop)
  int el = lane;
  auto stg_at = [&](int r, int c) __attribute__((always_inline)) {
    return stg + (uint32_t)r * 128 + (((uint32_t)c ^ (((uint32_t)r >> 1) & 7)) << 4);
  };
  // 4 values of row r, columns c .. + 3
  auto put16 = [&](int r, int c, f32x4 v) __attribute__((always_inline)) {
    const f32x2 lo = {v[0], v[1]}, hi = {v[2], v[3]};
    const u32x2 q = {__builtin_bit_cast(uint32_t, __builtin_convertvector(lo, bf16x2)),
                     __builtin_bit_cast(uint32_t, __builtin_convertvector(hi, bf16x2))};
    lds_store<u32x2>(stg_at(r, c >> 3) + ((c & 7) << 1), q);
  };
  auto put32 = [&](int r, int c, f32x4 v) __attribute__((always_inline)) {
    lds_store<u32x4>(stg_at(r, c >> 2), __builtin_bit_cast(u32x4, v));
  };
  // The staged rows row0 .. + 31, columns col0 .. + width, to bf16 rows at dst
  auto flush16 = [&](char* dst, int64_t stride, int64_t row0, int64_t col0, int width, int64_t end)
      __attribute__((always_inline)) {
    const int c = el & 7;
    const int64_t col = col0 + c * 8;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int r = (el >> 3) + 8 * j;
      const u32x4 v = lds_load<u32x4>(stg_at(r, c));
      const int64_t row = row0 + r;
      if (row < p.m && col < end && c * 8 < width) *reinterpret_cast<u32x4*>(dst + (row * stride + col) * 2) = v;
    }
  };
  // f32 rows (32 x 32): 128-byte row segments, plus a residual that was asked for
  // before (res_load): a load behind the last block's stores would wait for them
  struct Res {
    f32x4 v[4];
    f32x4 bias[2];   // of the block's columns (here and not with the tile's: registers)
  };
  auto res_load = [&](int64_t row0, int col0, int width, Res& q) __attribute__((always_inline)) {
    const int c = (el & 7) * 4, col = col0 + c;
#pragma unroll
    for (int a = 0; a < 2; ++a) {
      q.bias[a] = zero;
      if (p.bias) q.bias[a] = *reinterpret_cast<const f32x4*>(p.bias + min(col0 + a * 16 + 4 * (el >> 4), p.n - 4));
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int64_t row = row0 + (el >> 3) + 8 * j;
      q.v[j] = zero;
      if (row >= p.m || col >= p.n || c >= width) continue;
      if (p.res_bf16) {
        const bf16x4 o = *reinterpret_cast<const bf16x4*>(p.res + (row * p.rs + col) * 2);
#pragma unroll
        for (int e = 0; e < 4; ++e) q.v[j][e] = (float)o[e];
      } else {
        q.v[j] = *reinterpret_cast<const f32x4*>(p.res + (row * p.rs + col) * 4);
      }
    }
  };
  auto flush32 = [&](char* dst, int64_t row0, int col0, int width, const Res& q) __attribute__((always_inline)) {
    const int c = el & 7;
    const int col = col0 + c * 4;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int r = (el >> 3) + 8 * j;
      f32x4 t = __builtin_bit_cast(f32x4, lds_load<u32x4>(stg_at(r, c)));
      const int64_t row = row0 + r;
      if constexpr (RES) {
#pragma unroll
        for (int e = 0; e < 4; ++e) t[e] += p.beta * q.v[j][e];
      }
      if (row < p.m && col < p.n && c * 4 < width) *reinterpret_cast<f32x4*>(dst + (row * p.ys + col) * 4) = t;
    }
  };
  // bf16 rows of values that meet others in memory first (MEET): 16 rows x 64 f32
  // columns are staged, so that both are read and written in 128-byte row segments,
  // 8 values per lane; chunk c of 16 of row r at r * 256 + ((c ^ r) << 4). The
  // other values are asked for some blocks ahead (meet_load).
  constexpr bool MEET = EPI == EPI_DGATED || (EPI == EPI_LINEAR && OUT16 && RES);
  struct Met {
    u32x4 v[2][2];
  };
  auto meet_row = [&](int64_t row0, int j) __attribute__((always_inline)) { return row0 + (el >> 3) + 8 * j; };
  auto meet_load = [&](int64_t row0, int col0, int width, Met& q) __attribute__((always_inline)) {
    const int c = (el & 7) * 8, col = col0 + c;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int64_t row = meet_row(row0, j);
      if (row >= p.m || col >= p.n || c >= width) continue;
      if constexpr (EPI == EPI_DGATED) {
        const char* g0 = p.pre + (row * p.ps + col) * 2;
        q.v[j][0] = *reinterpret_cast<const u32x4*>(g0);
        q.v[j][1] = *reinterpret_cast<const u32x4*>(g0 + (int64_t)p.n * 2);
      } else if (p.res_bf16) {
        q.v[j][0] = *reinterpret_cast<const u32x4*>(p.res + (row * p.rs + col) * 2);
      } else {
        const char* r0 = p.res + (row * p.rs + col) * 4;
        q.v[j][0] = *reinterpret_cast<const u32x4*>(r0);
        q.v[j][1] = *reinterpret_cast<const u32x4*>(r0 + 16);
      }
    }
  };
  auto meet_at = [&](int r, int c) __attribute__((always_inline)) {
    return stg + (uint32_t)r * 256 + (((uint32_t)c ^ (uint32_t)r) << 4);
  };
  auto meet_flush = [&](char* dst, int64_t row0, int col0, int width, const Met& q) __attribute__((always_inline)) {
    const int c = (el & 7) * 8, col = col0 + c;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int r = (el >> 3) + 8 * j;
      float t[8];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const f32x4 v = __builtin_bit_cast(f32x4, lds_load<u32x4>(meet_at(r, (el & 7) * 2 + i)));
#pragma unroll
        for (int e = 0; e < 4; ++e) t[4 * i + e] = v[e];
      }
      const int64_t row = meet_row(row0, j);
      if (row >= p.m || col >= p.n || c >= width) continue;
      const bf16x8 a = __builtin_bit_cast(bf16x8, q.v[j][0]), b = __builtin_bit_cast(bf16x8, q.v[j][1]);
      bf16x8 o;
      char* at = dst + (row * p.ys + col) * 2;
      if constexpr (EPI == EPI_DGATED) {
        bf16x8 du;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const ActPair s = act_pair(p.act, (float)a[e]);
          o[e] = (bf16)(t[e] * (float)b[e] * s.slope);
          du[e] = (bf16)(t[e] * s.value);
        }
        *reinterpret_cast<bf16x8*>(at + (int64_t)p.n * 2) = du;
      } else if (p.res_bf16) {
#pragma unroll
        for (int e = 0; e < 8; ++e) o[e] = (bf16)(t[e] + p.beta * (float)a[e]);
      } else {
        const f32x4 lo = __builtin_bit_cast(f32x4, q.v[j][0]), hi = __builtin_bit_cast(f32x4, q.v[j][1]);
#pragma unroll
        for (int e = 0; e < 8; ++e) o[e] = (bf16)(t[e] + p.beta * (e < 4 ? lo[e & 3] : hi[e & 3]));
      }
      *reinterpret_cast<bf16x8*>(at) = o;
    }
  };
  constexpr bool STG16 = EPI == EPI_GATED || EPI == EPI_DXENT || (EPI == EPI_LINEAR && OUT16 && !RES);

  auto tile_end = [&](const Unit& q) __attribute__((always_inline)) {
    el = (int)opaque((uint32_t)lane);
    const int ncol0 = q.nt * BNO;
    const int er = el & 15, ec = 4 * (el >> 4);   // this lane's row and first column of a block
    // What the epilogue reads of vectors comes first: a load behind a store waits
    // for the store (one counter, in order).
    constexpr bool XENT = EPI == EPI_XENT || EPI == EPI_DXENT;
    f32x4 bv[WNB];
#pragma unroll
    for (int a = 0; a < WNB; ++a) bv[a] = zero;
    if constexpr ((EPI == EPI_LINEAR && !(RES && !OUT16)) || XENT) {
      if (p.bias) {
        const int c0 = ncol0 + wn * WNB * 16 + ec;
        if (!XENT || ncol0 + BN <= p.n) {
#pragma unroll
          for (int a = 0; a < WNB; ++a) bv[a] = *reinterpret_cast<const f32x4*>(p.bias + min(c0 + a * 16, p.n - 4));
        } else {   // any number of columns
#pragma unroll
          for (int a = 0; a < WNB; ++a)
#pragma unroll
            for (int e = 0; e < 4; ++e) bv[a][e] = p.bias[min(c0 + a * 16 + e, p.n - 1)];
        }
      }
    }
    int tcol[WMB];          // the target's column, if it is in [0, n)
    float row_lse[WMB], row_dl[WMB];
#pragma unroll
    for (int b = 0; b < WMB; ++b) {
      tcol[b] = -1;
      row_lse[b] = row_dl[b] = 0.f;
      if constexpr (XENT) {
        const int64_t row = (int64_t)q.mt * BM + (wm * WMB + b) * 16 + er;
        if (row < p.m) {
          const int t = p.target[row];
          if (t != p.ignore) tcol[b] = t - p.col0;
          if constexpr (EPI == EPI_DXENT) {
            row_lse[b] = p.lse[row];
            // (another target outside the vocabulary: NaN in the whole row)
            if (t != p.ignore) row_dl[b] = (uint32_t)t < (uint32_t)p.vocab ? p.dl[row] : __builtin_nanf("");
          }
        }
      }
    }
    Res res[2];   // (RES, f32 rows)
    if constexpr (MEET) {
      // 16 rows x 64 columns at a time, what they meet asked for DEPTH blocks ahead
      constexpr int PER = WNB < 4 ? WNB : 4, WIDE = WNB / PER, STEPS = WMB * WIDE, DEPTH = STEPS < 4 ? STEPS : EPI == EPI_DGATED ? 4 : 2;
      auto step_row = [&](int i) __attribute__((always_inline)) { return (int64_t)q.mt * BM + (wm * WMB + i / WIDE) * 16; };
      auto step_col = [&](int i) __attribute__((always_inline)) { return ncol0 + (wn * WNB + i % WIDE * PER) * 16; };
      Met met[DEPTH];
#pragma unroll
      for (int i = 0; i < DEPTH; ++i) meet_load(step_row(i), step_col(i), PER * 16, met[i]);
#pragma unroll
      for (int i = 0; i < STEPS; ++i) {
        const int b = i / WIDE, a0 = i % WIDE * PER;
#pragma unroll
        for (int a = 0; a < PER; ++a) {
          f32x4 z = acc[a0 + a][b];
          if constexpr (EPI == EPI_LINEAR) {
#pragma unroll
            for (int e = 0; e < 4; ++e) z[e] *= p.alpha;
#pragma unroll
            for (int e = 0; e < 4; ++e) z[e] += bv[a0 + a][e];
            if (p.pre) {   // straight from the accumulators, 8 bytes per lane
              const int64_t row = step_row(i) + er;
              const int col = step_col(i) + a * 16 + ec;
              if (row < p.m && col < p.n) {
                bf16x4 o;
#pragma unroll
                for (int e = 0; e < 4; ++e) o[e] = (bf16)z[e];
                *reinterpret_cast<bf16x4*>(p.pre + (row * p.ps + col) * 2) = o;
              }
            }
            if constexpr (LW == OP_ROWS) z = act_apply4(p.act, z);
          }
          lds_store<u32x4>(meet_at(er, a * 4 + (el >> 4)), __builtin_bit_cast(u32x4, z));
        }
        meet_flush(p.y, step_row(i), step_col(i), PER * 16, met[i % DEPTH]);
        if (i + DEPTH < STEPS) meet_load(step_row(i + DEPTH), step_col(i + DEPTH), PER * 16, met[i % DEPTH]);
        __builtin_amdgcn_sched_barrier(0);
      }
    } else
#pragma unroll
    for (int b0 = 0; b0 < WMB; b0 += 2) {
      const int64_t row0 = (int64_t)q.mt * BM + (wm * WMB + b0) * 16;
      if constexpr (EPI == EPI_GATED) {
        // blocks 2 i and 2 i + 1: 16 gate rows and their up rows, output columns 16 (wn WNB / 2 + i) ..
        constexpr int NG = WNB / 2;
        const int col = ncol0 + wn * NG * 16;
        if (p.pre) {
#pragma unroll
          for (int part = 0; part < 2; ++part) {
#pragma unroll
            for (int i = 0; i < NG; ++i)
#pragma unroll
              for (int b = 0; b < 2; ++b) put16(b * 16 + er, i * 16 + ec, acc[2 * i + part][b0 + b]);
            flush16(p.pre + (part ? (int64_t)p.n * 2 : 0), p.ps, row0, col, NG * 16, p.n);
          }
        }
#pragma unroll
        for (int i = 0; i < NG; ++i)
#pragma unroll
          for (int b = 0; b < 2; ++b) {
            f32x4 v = act_apply4(p.act, acc[2 * i][b0 + b]);
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] *= acc[2 * i + 1][b0 + b][e];
            put16(b * 16 + er, i * 16 + ec, v);
          }
        flush16(p.y, p.ys, row0, col, NG * 16, p.n);
      } else if constexpr (EPI == EPI_XENT || EPI == EPI_DXENT) {
        const int colb = ncol0 + wn * WNB * 16 + ec;   // this lane's first column
        const bool whole = ncol0 + BN <= p.n;
        constexpr float LOG2E = 1.44269504088896f;
        if constexpr (EPI == EPI_XENT) {
          // Scores in place of the products, columns past n -inf. (Not in units of
          // ln 2, which would save a product each: a bias of the lowest float would
          // leave the range.)
#pragma unroll
          for (int a = 0; a < WNB; ++a) {
#pragma unroll
            for (int b = b0; b < b0 + 2; ++b)
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                float s = __builtin_fmaf(p.alpha, acc[a][b][e], bv[a][e]);
                if (!whole && colb + a * 16 + e >= p.n) s = -INFINITY;
                acc[a][b][e] = s;
              }
            __builtin_amdgcn_sched_barrier(0);
          }
#pragma unroll
          for (int b = b0; b < b0 + 2; ++b) {
            const int64_t row = row0 + (b - b0) * 16 + er;
            const bool in = row < p.m;
            const int tc = tcol[b];
            if (__any(tc >= colb - ec && tc < colb - ec + WNB * 16)) {
#pragma unroll
              for (int a = 0; a < WNB; ++a)
#pragma unroll
                for (int e = 0; e < 4; ++e)
                  if (in && tc == colb + a * 16 + e && tc < p.n) p.at[row] = acc[a][b][e];
            }
            float top = -INFINITY;
#pragma unroll
            for (int a = 0; a < WNB; ++a)
#pragma unroll
              for (int e = 0; e < 4; ++e) top = fmaxf(top, acc[a][b][e]);
            top = fmaxf(top, __shfl_xor(top, 16, 64));
            top = fmaxf(top, __shfl_xor(top, 32, 64));
            const float base = top == -INFINITY ? 0.f : top;
            float sum = 0.f;
#pragma unroll
            for (int a = 0; a < WNB; ++a)
#pragma unroll
              for (int e = 0; e < 4; ++e) sum += __builtin_amdgcn_exp2f((acc[a][b][e] - base) * LOG2E);
            sum += __shfl_xor(sum, 16, 64);
            sum += __shfl_xor(sum, 32, 64);
            if (in && el < 16) p.part[(int64_t)(q.nt * C::NWN + wn) * p.m + row] = make_float2(top, sum);
          }
        } else {
          const float lse[2] = {row_lse[b0], row_lse[b0 + 1]}, f[2] = {row_dl[b0], row_dl[b0 + 1]};
          const int tc[2] = {tcol[b0], tcol[b0 + 1]};
          bool live[2];   // (an ignored row is zeros whatever its scores are)
          bool hit = false;
#pragma unroll
          for (int b = 0; b < 2; ++b) {
            hit |= tc[b] >= colb - ec && tc[b] < colb - ec + WNB * 16;
            live[b] = f[b] != 0.f || f[b] != f[b];
          }
          // the common case has no target, end or dead row among the wave's columns
          const bool plain = whole && !__any(hit) && __all(live[0] && live[1]);
          constexpr int PER = WNB < 4 ? WNB : 4;
#pragma unroll
          for (int a0 = 0; a0 < WNB; a0 += PER) {
#pragma unroll
            for (int a = a0; a < a0 + PER; ++a) {
#pragma unroll
              for (int b = 0; b < 2; ++b) {
                f32x4 v;
#pragma unroll
                for (int e = 0; e < 4; ++e)
                  v[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(p.alpha, acc[a][b0 + b][e], bv[a][e] - lse[b]) * LOG2E);
                if (!plain) {
#pragma unroll
                  for (int e = 0; e < 4; ++e) {
                    const int col = colb + a * 16 + e;
                    if (col == tc[b]) v[e] -= 1.f;
                    if (!live[b] || col >= p.n) v[e] = 0.f;
                  }
                }
#pragma unroll
                for (int e = 0; e < 4; ++e) v[e] = live[b] ? v[e] * f[b] : 0.f;
                put16(b * 16 + er, (a - a0) * 16 + ec, v);
                __builtin_amdgcn_sched_barrier(0);
              }
            }
            flush16(p.y, p.ys, row0, ncol0 + (wn * WNB + a0) * 16, PER * 16, p.n_store);
          }
        }
      } else {
        constexpr int COLS = STG16 ? 64 : 32;
        constexpr int PER = COLS / 16 < WNB ? COLS / 16 : WNB;
        char* dst = EPI == EPI_PART ? p.y + (int64_t)q.s * p.m * p.n * 4 : p.y;
        if constexpr (RES) {
          if (b0 == 0) res_load(row0, ncol0 + wn * WNB * 16, PER * 16, res[0]);
        }
#pragma unroll
        for (int a0 = 0; a0 < WNB; a0 += PER) {
          constexpr int NA = WNB / PER;
          const int step = b0 / 2 * NA + a0 / PER;
          const int col0 = ncol0 + (wn * WNB + a0) * 16;
          f32x4 z[PER][2];
#pragma unroll
          for (int a = 0; a < PER; ++a)
#pragma unroll
            for (int b = 0; b < 2; ++b)
#pragma unroll
              for (int e = 0; e < 4; ++e)
                z[a][b][e] = EPI == EPI_LINEAR ? p.alpha * acc[a0 + a][b0 + b][e] : acc[a0 + a][b0 + b][e];
          if constexpr (EPI == EPI_LINEAR) {
#pragma unroll
            for (int a = 0; a < PER; ++a)
#pragma unroll
              for (int b = 0; b < 2; ++b)
#pragma unroll
                for (int e = 0; e < 4; ++e) z[a][b][e] += RES ? res[step & 1].bias[a & 1][e] : bv[a0 + a][e];
            if (p.pre) {
#pragma unroll
              for (int a = 0; a < PER; ++a)
#pragma unroll
                for (int b = 0; b < 2; ++b) put16(b * 16 + er, a * 16 + ec, z[a][b]);
              flush16(p.pre, p.ps, row0, col0, PER * 16, p.n);
            }
            if (LW == OP_ROWS && p.act != ACT_NONE) {   // (the gradients' products have none)
#pragma unroll
              for (int a = 0; a < PER; ++a)
#pragma unroll
                for (int b = 0; b < 2; ++b) z[a][b] = act_apply4(p.act, z[a][b]);
            }
          }
#pragma unroll
          for (int a = 0; a < PER; ++a)
#pragma unroll
            for (int b = 0; b < 2; ++b) {
              if constexpr (STG16) put16(b * 16 + er, a * 16 + ec, z[a][b]);
              else put32(b * 16 + er, a * 16 + ec, z[a][b]);
            }
          if constexpr (RES) {   // the next block's, in front of this one's stores
            __builtin_amdgcn_sched_barrier(0);
            if (step + 1 < WMB / 2 * NA)
              res_load(row0 + (a0 + PER == WNB ? 32 : 0), ncol0 + (wn * WNB + (a0 + PER) % WNB) * 16, PER * 16,
                       res[(step + 1) & 1]);
          }
          if constexpr (STG16) flush16(dst, p.ys, row0, col0, PER * 16, p.n);
          else flush32(dst, row0, col0, PER * 16, res[step & 1]);
          __builtin_amdgcn_sched_barrier(0);
        }
      }
    }
#pragma unroll
    for (int a = 0; a < WNB; ++a)
#pragma unroll
      for (int b = 0; b < WMB; ++b) acc[a][b] = zero;
  };

  ld_unit();
  u32x4 fx[TG_KS][WMB], fw[C::H][TG_KS][C::WH];   // operands of a stage
  if constexpr (C::H == 2) {
    // Two phases per stage, the products of the lower and of the upper w blocks.
    // The operands of a phase are read from LDS in the one before: during phase A the
    // upper w blocks of its stage, during phase B x and the lower w blocks of the
    // next (x into the registers that the step's products have just read). So
    // x and the lower half of a slot are free one phase into its stage, the upper half two, and
    // their refills have three of the four phases of a two-slot ring to arrive.
    auto boundary = [&]() __attribute__((always_inline)) {
      // every wave's loads of what the next phase reads have landed, and its
      // reads of what is refilled now are done
      asm volatile("s_waitcnt vmcnt(%0)" :: "n"(C::PER_WAVE) : "memory");
      lds_barrier();
      __builtin_amdgcn_sched_barrier(0);
    };
    auto read_first = [&]() __attribute__((always_inline)) {
#pragma unroll
      for (int ks = 0; ks < TG_KS; ++ks) {
#pragma unroll
        for (int i = 0; i < C::WH; ++i) fw[0][ks][i] = read_w(0, i, ks);
#pragma unroll
        for (int b = 0; b < WMB; ++b) fx[ks][b] = read_x(b, ks);
      }
    };
    // The products of a phase (h: lower or upper w blocks), each followed by a read or a
    // refill at most: a product keeps its matrix core busy for four issue slots of
    // the wave, which hide that many instructions and not a dozen at once. With the
    // reads and refills in groups a stage of 4,096 rows of zeros took 1.11 us, so 1.02.
    // AHEAD: read the other w blocks, and in phase B x, for the next phase.
    auto phase = [&](auto hc, auto ahead) __attribute__((always_inline)) {
      constexpr int h = decltype(hc)::value;
      constexpr bool AHEAD = decltype(ahead)::value;
      constexpr int L = h ? L1 : L0;
      constexpr int NP = TG_KS * WMB * C::WH;            // products
      constexpr int XR = h && AHEAD ? WMB * TG_KS : 0;   // x reads, one behind each block's last product of a step
#pragma unroll
      for (int t = 0; t < NP; ++t) {
        const int ks = t / (WMB * C::WH), b = t / C::WH % WMB, i = t % C::WH;
        mfma(h * C::WH + i, b, fw[h][ks][i], fx[ks][b]);
        if constexpr (XR > 0) {
          if (i == C::WH - 1) fx[ks][b] = read_x(b, ks);
        }
        // w reads of a k step in the first half of the step's products: the registers
        // of the steps before are free by then
        if constexpr (AHEAD) {
          const int u = t % (WMB * C::WH);
          const int r = u % 2 == 1 && u / 2 < C::WH ? ks * C::WH + u / 2 : -1;
          if (r >= 0) fw[1 - h][r / C::WH][r % C::WH] = read_w(1 - h, r % C::WH, r / C::WH);
        }
        // refills: spread over the rest
        {
          constexpr int first = h == 0 ? 2 : NP / 2 + 2, step = h == 0 ? (NP - 4) / L0 : NP / 8;
          if ((t - first) >= 0 && (t - first) % step == 0 && (t - first) / step < L) load(h, (t - first) / step);
          static_assert(first + (L > 0 ? L - 1 : 0) * step < NP, "every refill of a phase has a place");
          if (t == NP - 3) {
            if (h == 0 && AHEAD) rd_next();
            end(h);
          }
        }
        __builtin_amdgcn_sched_barrier(0);
      }
    };
    const std::integral_constant<int, 0> A{};
    const std::integral_constant<int, 1> B{};
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      issue(0);
      issue(1);
    }
    asm volatile("s_waitcnt vmcnt(%0)" :: "n"(C::PER_WAVE + C::PW) : "memory");
    lds_barrier();
    for (int j = 0; j < my_units; ++j) {
      const Unit q = unit_of(j);
      const int stages = min(p.kper, kst - q.s * p.kper);
      read_first();
      for (int s = 1; s < stages; ++s) {
        boundary();
        phase(A, std::true_type{});
        boundary();
        phase(B, std::true_type{});
      }
      // the last stage reads nothing past itself: the epilogue needs the registers
      boundary();
      phase(A, std::true_type{});
      boundary();
      phase(B, std::false_type{});
      tile_end(q);
    }
  } else {
    // Small tiles: whole stages, STAGES - 1 of them in flight.
    auto read_stage = [&]() __attribute__((always_inline)) {
#pragma unroll
      for (int ks = 0; ks < TG_KS; ++ks) {
#pragma unroll
        for (int i = 0; i < C::WH; ++i) fw[0][ks][i] = read_w(0, i, ks);
#pragma unroll
        for (int b = 0; b < WMB; ++b) fx[ks][b] = read_x(b, ks);
      }
    };
#pragma unroll
    for (int i = 0; i < STAGES - 1; ++i) issue(0);
    for (int j = 0; j < my_units; ++j) {
      const Unit q = unit_of(j);
      const int stages = min(p.kper, kst - q.s * p.kper);
      for (int s = 0; s < stages; ++s) {
        asm volatile("s_waitcnt vmcnt(%0)" :: "n"((STAGES - 2) * C::PER_WAVE) : "memory");
        lds_barrier();   // this stage is in LDS, and every wave has read the one before
        issue(0);        // ... whose slot this refills
        read_stage();
        rd_next();
#pragma unroll
        for (int ks = 0; ks < TG_KS; ++ks)
#pragma unroll
          for (int i = 0; i < C::WH; ++i)
#pragma unroll
            for (int b = 0; b < WMB; ++b) mfma(i, b, fw[0][ks][i], fx[ks][b]);
      }
      tile_end(q);
    }
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
