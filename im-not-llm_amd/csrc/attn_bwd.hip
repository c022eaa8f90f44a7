// Gradients of packed varlen attention (inl_attn_varlen_bwd), bf16 on gfx950.
//
//   S = scale q k^T, P = softmax(S) over the visible keys, dP = dO v^T,
//   delta = rowsum(dO o), dS = P (dP - delta);
//   dq = scale dS k,  dk = scale dS^T q,  dv = P^T dO  (k, v: summed over their heads)
//
// Two kernels and no atomics, so equal calls give equal bits: one owns query rows and
// streams keys (dq), the other owns keys and streams the queries of every head of the
// group (dk, dv). S and dP are computed in both: 14 flops per (pair, feature) where
// one pass with atomics would take 10 and as many f32 additions to memory as there are
// (query, key block) pairs. The probabilities are recomputed: the dq kernel runs the
// forward's online softmax (its sum of exponentials and running maximum are per query
// row, so dq is scaled once at the end), and leaves log-sum-exp and delta, f32 per (head,
// row), for the other.
//
// Both kernels are one: a wave owns 32 rows whose two operands (q and dO, or k and v)
// stay in registers as B operands, and streams tiles of the other pair through LDS:
// X (k, or q) and Y (v, or dO).
//   T1[s][o] = X own0^T  (S^T or S),  T2[s][o] = Y own1^T  (dP^T or dP)
//   acc[d][o] += X^T dS  (dq^T or dk^T),  and for keys accv[d][o] += Y^T P
// An own row is a lane (lane & 31), stream rows are the accumulators' registers, so P
// and dS leave the first products in the layout in which the second ones read them: the
// k index of a product is summed over, and both operands take it in the same order. X
// and Y are stored once, row-major, and read both ways (ds_read_b128 for the first
// products, ds_read_b64_tr_b16 for the second); the swizzle serves both.
//
// P and dS are rounded to bf16 before the second products. A matrix instruction takes one type for both operands,
// and the others are the caller's bf16 q, k and dO: fp16, in which the forward keeps its P, would lose bits of
// gradients below 6e-5 and all of those below 6e-8, and a mean over a large batch makes them that small; two bf16 terms
// would double the second products (20 flops for 14). The two roundings put 0.0016 to 0.0017 of the gradients' norm
// on them (what grad_dtype f32 is off by); with bf16 outputs, whose rounding alone is 0.0017, it is 0.0023 to 0.0024.
//
// Bound by its products where texts are long: 8 x 2,048 tokens, 16/8 heads of 128, full: dq 1,050, dk and dv
// 1,120 TFLOP/s of those that they do; 4 x 4,096 causal, 16/2 heads of 256: 0.90 and 1.20 ms, matrix cores 38 % busy
// in both, as one wave or a pair has a SIMD to itself and its exponentials stand between its products. By
// bytes and the start of workgroups where they are short: 64 x 256 tokens of 16 heads of 64 take 50 to 57 and 55 to
// 62 us, for 42 us of bytes each at 4.84 TB/s; 48 texts to 1,021 with a window of 64 and 12 heads 74 and 68 for 53.
#include <algorithm>
#include <new>
#include <vector>

#include "attn_bwd.hpp"
#include "attn_stream.hpp"
#include "train_ops.hpp"

namespace inl {

namespace {

constexpr uint32_t BWD_NOWHERE = 0xffff0000u;   // beyond every text's range: reads 0, not written

// QS parts of a workgroup's four waves take different rows of every stream tile for the same own rows.
template <int D, bool KV, int QS>
struct BwdShape {
  static constexpr int KG = 4 / QS;               // waves with own rows of their own
  static constexpr int OWN = 32 * KG;             // own rows of a workgroup
  static constexpr int BN = D <= 64 || QS == 2 ? 64 : 32;    // stream rows of a tile
  static constexpr int TILE = BN * D * 2;         // bytes of X, and of Y
  static constexpr int STAT = KV ? 2 * BN * 4 : 0;   // log-sum-exp and delta of the stream rows
  static constexpr int STAGE = 2 * TILE + STAT;
  static constexpr int NS = D <= 64 ? 3 : BN == 32 ? 4 : 2;  // tiles in LDS: one in use, the others loading
  static constexpr int LDS = NS * STAGE;
};

// A tile of BN rows lies in groups of 64 features (a 128-byte line): 16-byte chunk c of row r at
//   ((c / 8) BN + r) 128 + ((c % 8) ^ bwd_swz(r)) 16.
// 16 rows at one chunk (a row read) fill 256 bytes, and so do 4 rows at 4 chunks (a transposed read): no
// bank conflicts; and an address is one of four of a lane plus a constant, for every k-step and
// every block of features.
__device__ __forceinline__ int bwd_swz(int r) { return (((r >> 1) & 1) << 2) | ((r >> 2) & 3); }

__device__ __forceinline__ bf16x8 pack8(const float* x) {
  u32x4 o;
#pragma unroll
  for (int e = 0; e < 4; ++e)
    o[e] = __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2){x[2 * e], x[2 * e + 1]}, bf16x2));
  return __builtin_bit_cast(bf16x8, o);
}

// Rows r0 .. r0 + 31 of an output from acc[d][row] (D / 32 blocks of 32 features): one
// v_permlane32_swap per register pair puts 8 consecutive features of a row into a lane.
template <int D, bool OUT16>
__device__ __forceinline__ void bwd_store(const f32x16 (&acc)[D / 32], float by, __amdgpu_buffer_rsrc_t rs, uint32_t at,
                                          int hf, int head_dim) {
#pragma unroll
  for (int db = 0; db < D / 32; ++db) {
    if constexpr (OUT16) {
#pragma unroll
      for (int gp = 0; gp < 2; ++gp) {
        uint32_t w[4];
#pragma unroll
        for (int h = 0; h < 4; ++h) {
          const f32x2 x = {acc[db][8 * gp + 2 * h] * by, acc[db][8 * gp + 2 * h + 1] * by};
          w[h] = __builtin_bit_cast(uint32_t, __builtin_convertvector(x, bf16x2));
        }
        swap_lanes_32(w[0], w[2]);
        swap_lanes_32(w[1], w[3]);
        const int col = db * 32 + 16 * gp + 8 * hf;
        __builtin_amdgcn_raw_buffer_store_b128((u32x4){w[0], w[1], w[2], w[3]}, rs,
                                               col < head_dim ? at + col * 2 : BWD_NOWHERE, 0, 0);
      }
    } else {
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const int col = db * 32 + 8 * g + 4 * hf;
        u32x4 val;
#pragma unroll
        for (int e = 0; e < 4; ++e) val[e] = __builtin_bit_cast(uint32_t, acc[db][4 * g + e] * by);
        __builtin_amdgcn_raw_buffer_store_b128(val, rs, col < head_dim ? at + col * 4 : BWD_NOWHERE, 0, 0);
      }
    }
  }
}

// What a workgroup works on: a block of own rows of a text, for a key head and one of its query heads (of
// `members`; all of them for members = 1).
struct BwdUnit {
  int start, len, block, kvh, member;
};
// False where there is nothing (classes have unequal numbers of units).
__device__ __forceinline__ bool bwd_unit(const AttnBwdParams& p, int members, int lane, BwdUnit* out) {
  const int width = p.h_kv * p.classes;
  const uint32_t wg = blockIdx.y * gridDim.x + blockIdx.x;
  const int rest = wg / width, x = wg - rest * width;
  const int cls = x / p.h_kv, u = rest / members;
  out->kvh = x - cls * p.h_kv;
  out->member = rest - u * members;
  if (u >= p.units[cls]) return false;
  // the class's first units ascend: the text is the last one whose is not above u
  const BwdText* const texts = p.texts ? p.texts : p.own;
  const int n = p.first[cls + 1];
  int at = p.first[cls];
  for (int i = at; i < n; i += 64) {
    const int first = i + lane < n ? texts[i + lane].unit : 0x7fffffff;
    const int below = __builtin_popcountll(__builtin_amdgcn_ballot_w64(first <= u));
    at = below ? i + below - 1 : at;
    if (below < 64) break;
  }
  const BwdText t = texts[at];
  out->start = __builtin_amdgcn_readfirstlane(t.start);
  out->len = __builtin_amdgcn_readfirstlane(t.len);
  out->block = u - __builtin_amdgcn_readfirstlane(t.unit);
  return true;
}

// acc += rows . opnd over the features of 32 stream rows, at base[step % 4] (a lane's row and chunk) + off;
// fragments are read RD - 1 products ahead, so that a product waits for its own read only. `first`: what
// acc starts from.
template <int D, int BN, int RD>
__device__ __forceinline__ void rows_product(f32x16& acc, const f32x16& first, const uint32_t (&base)[4], uint32_t off,
                                             const bf16x8 (&opnd)[D / 16]) {
  constexpr int KST = D / 16;
  u32x4 fr[RD];
  auto read = [&](int st) __attribute__((always_inline)) {
    fr[st % RD] = lds_load<u32x4>(base[st & 3] + off + (st >> 2) * BN * 128);
  };
#pragma unroll
  for (int st = 0; st < RD - 1 && st < KST; ++st) read(st);
#pragma unroll
  for (int st = 0; st < KST; ++st) {
    if (st + RD - 1 < KST) read(st + RD - 1);
    __builtin_amdgcn_sched_barrier(0);
    acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, fr[st % RD]), opnd[st],
                                                  st == 0 ? first : acc, 0, 0, 0);
    __builtin_amdgcn_sched_barrier(0);
  }
}

// Two such products beside one another, of rows at base + off and base + off2: neither waits for its own
// last step. dq, one after the other / so: 4 x 4,096 tokens of 16/2 heads of 256 0.92 / 0.92 ms, 8 x 2,048 of 16/8 x
// 128 387 / 392 us, 64 x 256 of 16 heads of 64 53 / 51.5, 8 x 2,048 of them 226 / 225.
template <int D, int BN, int RD>
__device__ __forceinline__ void rows_products(f32x16& a, f32x16& b, const f32x16& first, const uint32_t (&base)[4], uint32_t off,
                                              uint32_t off2, const bf16x8 (&opnd)[D / 16], const bf16x8 (&opnd2)[D / 16]) {
  constexpr int KST = D / 16;
  u32x4 fr[RD], fr2[RD];
  auto read = [&](int st) __attribute__((always_inline)) {
    fr[st % RD] = lds_load<u32x4>(base[st & 3] + off + (st >> 2) * BN * 128);
    fr2[st % RD] = lds_load<u32x4>(base[st & 3] + off2 + (st >> 2) * BN * 128);
  };
#pragma unroll
  for (int st = 0; st < RD - 1 && st < KST; ++st) read(st);
#pragma unroll
  for (int st = 0; st < KST; ++st) {
    if (st + RD - 1 < KST) read(st + RD - 1);
    __builtin_amdgcn_sched_barrier(0);
    a = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, fr[st % RD]), opnd[st], st == 0 ? (f32x16){} : a, 0, 0, 0);
    b = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, fr2[st % RD]), opnd2[st], st == 0 ? first : b, 0, 0, 0);
    __builtin_amdgcn_sched_barrier(0);
  }
}

// acc[d][own] += (32 stream rows, transposed) . x, likewise: base[2 (block of 32 features % 2) + (8 rows of 16)].
template <int D, int BN, int RD>
__device__ __forceinline__ void cols_product(f32x16 (&acc)[D / 32], const uint32_t (&base)[4], uint32_t off,
                                             const bf16x8 (&x)[2]) {
  constexpr int NDB = D / 32;
  typedef short s16x8 __attribute__((ext_vector_type(8)));
  s16x8 fr[RD];
  auto read = [&](int i) __attribute__((always_inline)) {
    const int ks = i / NDB, db = i % NDB;
    s16x4 a[2];
#pragma unroll
    for (int h = 0; h < 2; ++h)
      a[h] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(size_t)(
          base[2 * (db & 1) + h] + off + (db >> 1) * BN * 128 + (ks * 16 + 8 * h) * 128));
    fr[i % RD] = (s16x8){a[0][0], a[0][1], a[0][2], a[0][3], a[1][0], a[1][1], a[1][2], a[1][3]};
  };
#pragma unroll
  for (int i = 0; i < RD - 1; ++i) read(i);
#pragma unroll
  for (int i = 0; i < 2 * NDB; ++i) {
    if (i + RD - 1 < 2 * NDB) read(i + RD - 1);
    __builtin_amdgcn_sched_barrier(0);
    acc[i % NDB] =
        __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, fr[i % RD]), x[i / NDB], acc[i % NDB], 0, 0, 0);
    __builtin_amdgcn_sched_barrier(0);
  }
}

// 16 values, one per accumulator register, of 32 f32 values at `at` (+ 4 hf, a lane's)
__device__ __forceinline__ f32x16 rows_stat(uint32_t at) {
  f32x16 s;
#pragma unroll
  for (int g = 0; g < 4; ++g) {
    const f32x4 a = lds_load<f32x4>(at + g * 32);
#pragma unroll
    for (int e = 0; e < 4; ++e) s[4 * g + e] = a[e];
  }
  return s;
}

// 16 bytes a lane at rsrc + voff + off to LDS at lds + 16 lane. The instruction adds its offset to both
// addresses. The s_nop stands for two waits that the compiler does not see into asm to make: one state
// from the write of M0, and five from a v_readfirstlane that wrote a word of the descriptor (with
// fewer the load has taken the old word, and its address from it).
__device__ __forceinline__ void bwd_dma(i32x4 rsrc, uint32_t lds, uint32_t voff, int off) {
  asm volatile("s_nop 4\n\tbuffer_load_dwordx4 %0, %1, 0 offen offset:%3 lds"
               :: "v"(voff), "s"(rsrc), "{m0}"(lds - off), "n"(off) : "memory");
}

// A lane's LDS addresses in a tile at `tile`, from row `row0` on: row reads (k-steps of 16 features, modulo 4), and
// transposed ones (blocks of 32 features modulo 2, rows 0-7 and 8-15 of 16): there 16 lanes read
// 4 rows x 16 features, in the order of rows that the accumulators' registers have.
__device__ __forceinline__ void bwd_row_reads(uint32_t (&at)[4], uint32_t tile, int row0, int lane) {
  const int row = lane & 31, hf = lane >> 5;
#pragma unroll
  for (int i = 0; i < 4; ++i) at[i] = tile + (row0 + row) * 128 + (((2 * i + hf) ^ bwd_swz(row)) << 4);
}
__device__ __forceinline__ void bwd_col_reads(uint32_t (&at)[4], uint32_t tile, int row0, int lane) {
  const int g16 = lane >> 4, j16 = lane & 15, row = 4 * (lane >> 5) + (j16 >> 2);
  const int c = 2 * (g16 & 1) + ((j16 & 3) >> 1);
#pragma unroll
  for (int i = 0; i < 4; ++i)
    at[i] = tile + (row0 + row) * 128 + (((4 * (i >> 1) + c) ^ bwd_swz(row + 8 * (i & 1))) << 4) + ((j16 & 1) << 3);
}

// Tile loads by NW waves: 1 KB blocks of 8 rows x 128 bytes, the group's rows first; a wave's i-th
// instruction loads block i NW + wave. Lanes whose chunk is behind the head load nothing, and find zeros there.
template <int D, int BN, int NW>
struct BwdLoad {
  static constexpr int RBN = BN / 8;                              // blocks of a group
  static constexpr int RP = RBN > NW ? RBN / NW : 1;              // a wave's blocks of one group
  static constexpr int GP = D / 64 * RBN / NW / RP;               // groups that a wave takes part in
  static constexpr int GSTEP = NW > RBN ? NW / RBN : 1;           // from one to the next
  static_assert(RP * GP * NW == D / 64 * RBN && (NW * 8) % 16 == 0, "blocks of a tile");
  uint32_t x, y;      // byte offset of this lane's chunk in X and Y, less the tile's first row
  int chunk, g0;      // of the group; the wave's first group
  __device__ __forceinline__ BwdLoad(int wave, int lane, uint32_t xst, uint32_t yst) {
    const int row = 8 * (wave % RBN) + (lane >> 3);
    g0 = wave / RBN;
    chunk = (lane & 7) ^ bwd_swz(row);   // (the swizzle repeats every 16 rows)
    x = row * xst + g0 * 128 + chunk * 16;
    y = row * yst + g0 * 128 + chunk * 16;
  }
  __device__ __forceinline__ void issue(const i32x4& xrs, const i32x4& yrs, uint32_t at, uint32_t row, uint32_t xst,
                                        uint32_t yst, uint32_t off, int head_dim) const {
#pragma unroll
    for (int r = 0; r < RP; ++r) {
      const uint32_t xa = x + ((row + r * NW * 8) * xst + off), ya = y + ((row + r * NW * 8) * yst + off);
#pragma unroll
      for (int g = 0; g < GP; ++g)
        if (head_dim == D || (8 * (g0 + g * GSTEP) + chunk) * 8 < head_dim) {
          const uint32_t lds = at + (g * GSTEP * RBN + r * NW) * 1024;
          bwd_dma(xrs, lds, xa, g * GSTEP * 128);
          bwd_dma(yrs, lds + D * 2 * BN, ya, g * GSTEP * 128);
        }
    }
  }
};

// The statistics of one head (log-sum-exp, or those of delta h_q behind) of a text's rows.
__device__ __forceinline__ i32x4 bwd_stat_rsrc(const AttnBwdParams& p, int64_t h, const BwdUnit& txt) {
  const uint64_t a = (uint64_t)(p.stat + h * p.rows + txt.start);
  return (i32x4){(int)(uint32_t)a, (int)((uint32_t)(a >> 32) & 0xffffu), txt.len * 4, 0x00020000};
}

// KV: own rows are keys (dk, dv); otherwise queries (dq, and the row statistics).
template <int D, bool KV, int QS, bool OUT16>
__global__ __launch_bounds__(256, D <= 128 ? 2 : 1) void attn_bwd_kernel(AttnBwdParams p) {
  using S = BwdShape<D, KV, QS>;
  constexpr int KST = D / 16;            // k-steps of the products over features
  constexpr int NDB = D / 32;            // 32-feature blocks of an accumulator
  constexpr int NKB = S::BN / 32 / QS;   // 32-row blocks of a tile for a wave
  static_assert(QS == 1 || NKB == 1, "parts of a tile");
  constexpr int RR = D == 128 && KV ? 3 : 4, RC = 4;   // fragments in flight (eight are no faster)
  constexpr int RB = 2;                                // of each of two products (three are no faster)
  extern __shared__ __attribute__((aligned(1024))) char smem[];

  const int tid = threadIdx.x;
  const int lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int lq = lane & 31;
  const int hf = lane >> 5;
  const uint32_t lds0 = lds_addr(smem);
  BwdUnit txt;
  if (!bwd_unit(p, KV ? 1 : p.group, lane, &txt)) return;
  const int kvh = txt.kvh, head = KV ? kvh : kvh * p.group + txt.member;   // own head
  const int T = txt.len;
  const int kg = QS == 1 ? wave : wave % S::KG, qg = QS == 1 ? 0 : wave / S::KG;
  const int b0 = txt.block * S::OWN;                // first own row of the workgroup
  const int r0 = b0 + kg * 32;                      // and of this wave
  const bool active = r0 < T;
  const int blast = min(b0 + S::OWN - 1, T - 1), rlast = min(r0 + 31, T - 1);
  const int own = r0 + lq;

  const char* const base_q = p.q + txt.start * p.q_stride;
  const char* const base_k = p.k + txt.start * p.k_stride + (int64_t)kvh * p.head_dim * 2;
  const char* const base_v = p.v + txt.start * p.v_stride + (int64_t)kvh * p.head_dim * 2;
  const char* const base_do = p.dout + txt.start * p.do_stride;

  // ---- the stream: tiles [t_lo, t_hi) of every head that the own rows meet ----
  int s_lo = 0, s_hi = T;
  if (p.window >= 0) {
    s_lo = max(0, b0 - p.window);
    s_hi = min(T, blast + p.window + 1);
  }
  if (p.causal) {
    if (KV) s_lo = max(s_lo, b0);
    else s_hi = min(s_hi, blast + 1);
  }
  const int t_lo = s_lo / S::BN, t_hi = (s_hi + S::BN - 1) / S::BN;
  const int n_tiles = (t_hi - t_lo) * (KV ? p.group : 1);

  const uint32_t xst = (uint32_t)(KV ? p.q_stride : p.k_stride), yst = (uint32_t)(KV ? p.do_stride : p.v_stride);
  const BwdLoad<D, S::BN, 4> load(wave, lane, xst, yst);
  if (p.head_dim < D) {
    for (int i = tid; i < S::LDS / 16; i += 256) lds_store<u32x4>(lds0 + i * 16, (u32x4){0u, 0u, 0u, 0u});
    __syncthreads();
  }
  int dh = 0, dt = t_lo;   // load cursor: head of the group (its heads take a tile after one another), tile
  const int64_t h0 = (int64_t)kvh * p.group;
  const i32x4 xrs = pp_rsrc_words(KV ? base_q + h0 * p.head_dim * 2 : base_k, (uint32_t)T * xst);
  const i32x4 yrs = pp_rsrc_words(KV ? base_do + h0 * p.head_dim * 2 : base_v, (uint32_t)T * yst);
  uint32_t put = lds0;     // the stage it goes to
  auto issue = [&]() __attribute__((always_inline)) {
    const uint32_t s0 = (uint32_t)(dt * S::BN);
    load.issue(xrs, yrs, put + wave * 1024, s0, xst, yst, dh * p.head_dim * 2, p.head_dim);
    if constexpr (KV) {
      // BN / 2 statistics per wave, 4 bytes a lane
      if (lane < S::BN / 2) {
        const uint32_t dst = put + 2 * S::TILE + wave * (S::BN * 2);
        const i32x4 rs = bwd_stat_rsrc(p, h0 + dh + (wave < 2 ? 0 : p.h_q), txt);
        asm volatile("s_nop 4\n\tbuffer_load_dword %0, %1, 0 offen lds"
                     :: "v"((s0 + (wave & 1) * (S::BN / 2) + lane) * 4), "s"(rs), "{m0}"(dst) : "memory");
      }
      if (++dh == p.group) {
        dh = 0;
        ++dt;
      }
    } else {
      ++dt;
    }
    put = put == lds0 + (S::NS - 1) * S::STAGE ? lds0 : put + S::STAGE;
  };

  // The first tiles are under way while the own operands are loaded.
#pragma unroll
  for (int i = 0; i < S::NS - 1; ++i)
    if (i < n_tiles) issue();

  // ---- own operands: lane lq's row, chunks 2 i + hf ----
  bf16x8 own0[KST], own1[KST];
  float delta = 0.f;
  {
    const int64_t ho = (int64_t)head * p.head_dim * 2;
    const uint32_t st0 = (uint32_t)(KV ? p.k_stride : p.q_stride), st1 = (uint32_t)(KV ? p.v_stride : p.do_stride);
    const __amdgpu_buffer_rsrc_t rs0 = pp_rsrc(KV ? base_k : base_q + ho, (uint32_t)T * st0);
    const __amdgpu_buffer_rsrc_t rs1 = pp_rsrc(KV ? base_v : base_do + ho, (uint32_t)T * st1);
    const bool in = own < T;
#pragma unroll
    for (int i = 0; i < KST; ++i) {
      const int c = 2 * i + hf;
      const bool ok = in && c * 8 < p.head_dim;
      own0[i] = __builtin_bit_cast(bf16x8, __builtin_amdgcn_raw_buffer_load_b128(rs0, ok ? own * st0 + c * 16 : BWD_NOWHERE, 0, 0));
      own1[i] = __builtin_bit_cast(bf16x8, __builtin_amdgcn_raw_buffer_load_b128(rs1, ok ? own * st1 + c * 16 : BWD_NOWHERE, 0, 0));
    }
    if constexpr (!KV) {
      const uint32_t st2 = (uint32_t)p.o_stride;
      const __amdgpu_buffer_rsrc_t rs2 = pp_rsrc(p.o + txt.start * p.o_stride + ho, (uint32_t)T * st2);
#pragma unroll
      for (int i = 0; i < KST; ++i) {
        const int c = 2 * i + hf;
        const bool ok = in && c * 8 < p.head_dim;
        const bf16x8 ov =
            __builtin_bit_cast(bf16x8, __builtin_amdgcn_raw_buffer_load_b128(rs2, ok ? own * st2 + c * 16 : BWD_NOWHERE, 0, 0));
#pragma unroll
        for (int e = 0; e < 8; ++e) delta += (float)ov[e] * (float)own1[i][e];
      }
      delta = half_sum(delta);
    }
  }

  // ---- per-lane LDS addresses in stage 0 ----
  uint32_t xa[4], ta[4];
  bwd_row_reads(xa, lds0, qg * 32, lane);
  bwd_col_reads(ta, lds0, qg * 32, lane);
  uint32_t la = lds0 + 2 * S::TILE + 16 * hf + qg * 128;

  f32x16 acc[NDB], accv[KV ? NDB : 1];
#pragma unroll
  for (int i = 0; i < NDB; ++i) {
    acc[i] = (f32x16){};
    if constexpr (KV) accv[i] = (f32x16){};
  }
  float m_i = -INFINITY, l_i = 0.f;
  // dP^T - delta starts from -delta, where registers hold it 16 times
  constexpr bool LESS = !KV && D <= 128;
  f32x16 less = {};
  if constexpr (LESS)
#pragma unroll
    for (int r = 0; r < 16; ++r) less[r] = -delta;

  // One 32-row block of the stream against this wave's rows.
  auto block = [&](int kb, int s0) __attribute__((always_inline)) {
    const uint32_t X = kb * 32 * 128, Y = S::TILE + X;
    f32x16 s, dp;
    if constexpr (KV) rows_product<D, S::BN, RR>(s, rows_stat(la + kb * 128), xa, X, own0);
    else rows_products<D, S::BN, RB>(s, dp, less, xa, X, Y, own0, own1);
    // masks: stream row s0 + c of register r, c = 8 (r / 4) + 4 hf + r % 4
    const bool whole = (KV || s0 + 31 < T) && (!p.causal || (KV ? s0 >= rlast : s0 + 31 <= r0)) &&
                       (p.window < 0 || (s0 + 31 - r0 <= p.window && rlast - s0 <= p.window));
    if (!whole) {
      const int sb = s0 + 4 * hf;
      int hi = KV ? 0x3fffffff : T - 1, lo = 0;
      if (p.causal) {
        if (KV) lo = own;
        else hi = min(hi, own);
      }
      if (p.window >= 0) {
        lo = max(lo, own - p.window);
        hi = min(hi, own + p.window);
      }
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const int at = sb + 8 * (r >> 2) + (r & 3);
        s[r] = at >= lo && at <= hi ? s[r] : -INFINITY;
      }
    }
    float pr[16], ds[16];
    if constexpr (KV) {
#pragma unroll
      for (int r = 0; r < 16; ++r) pr[r] = __builtin_amdgcn_exp2f(s[r] * p.c);
      const bf16x8 pb[2] = {pack8(pr), pack8(pr + 8)};
      cols_product<D, S::BN, RC>(accv, ta, Y, pb);
      rows_product<D, S::BN, RR>(dp, rows_stat(la + S::BN * 4 + kb * 128), xa, Y, own1);
#pragma unroll
      for (int r = 0; r < 16; ++r) ds[r] = pr[r] * dp[r];
    } else {
      auto mx2 = [](float a, float b) __attribute__((always_inline)) { return __builtin_elementwise_maximum(a, b); };
      float m4[4];
#pragma unroll
      for (int c = 0; c < 4; ++c) m4[c] = mx2(mx2(s[4 * c], s[4 * c + 1]), mx2(s[4 * c + 2], s[4 * c + 3]));
      float mx = mx2(mx2(m4[0], m4[1]), mx2(m4[2], m4[3]));
      mx = half_max(mx) * p.c;
      // the reference maximum moves only when a row's grows by more than 2^8
      if (__builtin_amdgcn_ballot_w64(!(mx <= m_i + 8.0f)) != 0) {
        const float m_new = mx2(m_i, mx);
        const float alpha = m_i == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m_i - m_new);
        m_i = m_new;
        l_i *= alpha;
#pragma unroll
        for (int i = 0; i < NDB; ++i)
#pragma unroll
          for (int r = 0; r < 16; ++r) acc[i][r] *= alpha;
      }
      const float base = m_i == -INFINITY ? 0.f : m_i;
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        pr[r] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[r], p.c, -base));
        l_i += pr[r];
        ds[r] = pr[r] * (LESS ? dp[r] : dp[r] - delta);
      }
    }
    const bf16x8 db[2] = {pack8(ds), pack8(ds + 8)};
    cols_product<D, S::BN, RC>(acc, ta, X, db);
  };

  // stream rows that some row of this wave sees
  int w_lo = 0, w_hi = T;
  if (p.window >= 0) {
    w_lo = max(0, r0 - p.window);
    w_hi = min(T, rlast + p.window + 1);
  }
  if (p.causal) {
    if (KV) w_lo = max(w_lo, r0);
    else w_hi = min(w_hi, rlast + 1);
  }
  if (!active) w_hi = 0;

  using Load = BwdLoad<D, S::BN, 4>;
  constexpr int LOADS = 2 * Load::RP * Load::GP + (KV ? 1 : 0);
  int t = t_lo, th = 0, at = 0;
  for (int i = 0; i < n_tiles; ++i) {
    // this wave's loads of tile i are done once no more than those of the tiles behind it are in
    // flight (a wave that loads no feature of a narrow head has fewer)
    if (i + S::NS - 2 < n_tiles && p.head_dim == D)
      asm volatile("s_waitcnt vmcnt(%0)" ::"n"((S::NS - 2) * LOADS) : "memory");
    else
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    lds_barrier();
    if (i + S::NS - 1 < n_tiles) issue();
#pragma unroll
    for (int kb = 0; kb < NKB; ++kb) {
      const int s0 = t * S::BN + (kb + qg) * 32;
      if (s0 < w_hi && s0 + 32 > w_lo) block(kb, s0);
    }
    if (!KV || ++th == p.group) {
      th = 0;
      ++t;
    }
    const uint32_t step = at == S::NS - 1 ? (uint32_t)(-(S::NS - 1) * S::STAGE) : S::STAGE;
    at = at == S::NS - 1 ? 0 : at + 1;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      xa[e] += step;
      ta[e] += step;
    }
    la += step;
  }

  if constexpr (QS > 1) {
    // The parts' sums meet in LDS, where the stages were. Queries' are brought to one maximum first: a part
    // that saw no key of a row has none (-inf) and counts 0.
    constexpr int PART = (KV ? 8 : 4) * NDB * 1024;   // a wave's
    static_assert(QS == 2 && S::KG * (PART + 512) <= S::LDS, "sums of the second part fit");
    const uint32_t to = lds0 + kg * PART + lane * 16, stat = lds0 + S::KG * PART + kg * 512 + lane * 4;
    auto each = [&](auto&& f) __attribute__((always_inline)) {
#pragma unroll
      for (int db = 0; db < NDB; ++db)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          f(acc[db], g, to + (db * 4 + g) * 1024);
          if constexpr (KV) f(accv[db], g, to + ((NDB + db) * 4 + g) * 1024);
        }
    };
    lds_barrier();
    if (qg == 1) {
      each([&](f32x16& a, int g, uint32_t at) __attribute__((always_inline)) {
        lds_store<f32x4>(at, (f32x4){a[4 * g], a[4 * g + 1], a[4 * g + 2], a[4 * g + 3]});
      });
      if constexpr (!KV) {
        lds_store<float>(stat, m_i);
        lds_store<float>(stat + 256, l_i);
      }
    }
    lds_barrier();
    if (qg == 1) return;
    float by0 = 1.f, by1 = 1.f;
    if constexpr (!KV) {
      const float m1 = lds_load<float>(stat), m = __builtin_elementwise_maximum(m_i, m1);
      by0 = m_i == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m_i - m);
      by1 = m1 == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m1 - m);
      l_i = l_i * by0 + lds_load<float>(stat + 256) * by1;
      m_i = m;
    }
    each([&](f32x16& a, int g, uint32_t at) __attribute__((always_inline)) {
      const f32x4 v = lds_load<f32x4>(at);
#pragma unroll
      for (int e = 0; e < 4; ++e) a[4 * g + e] = KV ? a[4 * g + e] + v[e] : a[4 * g + e] * by0 + v[e] * by1;
    });
  }

  // ---- results ----
  const int osz = OUT16 ? 2 : 4;
  const int64_t ho = (int64_t)head * p.head_dim * osz;
  auto out = [&](char* at, int64_t stride, const f32x16 (&a)[NDB], float by) __attribute__((always_inline)) {
    const __amdgpu_buffer_rsrc_t rs = pp_rsrc(at + txt.start * stride + ho, (uint32_t)T * (uint32_t)stride);
    bwd_store<D, OUT16>(a, by, rs, own < T ? (uint32_t)own * (uint32_t)stride : BWD_NOWHERE, hf, p.head_dim);
  };
  if constexpr (KV) {
    out(p.dk, p.dk_stride, acc, p.scale);
    out(p.dv, p.dv_stride, accv, 1.f);
  } else {
    const float l = half_sum(l_i);
    if (p.dq) out(p.dq, p.dq_stride, acc, p.scale / l);
    if (hf == 0 && own < T) {
      float* st = p.stat + (int64_t)head * p.rows + txt.start + own;
      st[0] = -(m_i + log2f(l)) / p.c;
      st[(int64_t)p.h_q * p.rows] = -delta;
    }
  }
}

// dk and dv of wide heads. One wave's registers do not hold the accumulators of both beside k
// and v, so two waves share 32 keys, on one SIMD: the first makes P (from q and its k) and
// accumulates dv, the second makes dP (from dO and its v), takes P from the first through LDS, and
// accumulates dk. A stream tile is two phases with a barrier between: S and P beside dP, then dv
// beside dS and dk; the first wave goes ahead of the second in the first phase (s_setprio), so
// that its exponentials run under the other's products.
// Two of a workgroup's four pairs own 32 keys each, the others take other rows of the stream for
// the same keys, and the sums meet in LDS at the end. Four pairs with keys of their own read half the tiles, but
// make half as many workgroups of twice the length. As here / so: 4 x 4,096 tokens, causal, of 16/2 heads 1.21 / 1.91
// ms, 24 x 1,024 of 3/1 heads with a window of 512 155 / 162 us; but full, whose blocks are of equal length, 24 x
// 1,024 199 / 172 and 64 x 1,024 501 / 403.
template <int D>
struct PairShape {
  static constexpr int QS = 2, KG = 2;            // parts of a stream tile, blocks of own keys
  static constexpr int BN = 32 * QS;
  static constexpr int ROW = D * 2;
  static constexpr int TILE = BN * ROW;
  static constexpr int STAGE = 2 * TILE;
  static constexpr int SWAP = 2 * STAGE;          // P of every pair, f32
  static constexpr int STATS = SWAP + 4 * 4096;
  static constexpr int STAT = 2 * BN * 4;
  static constexpr int LDS = STATS + 2 * STAT;
  static_assert((STAGE & (STAGE - 1)) == 0, "stages differ in one bit of an address");
};

template <int D, bool OUT16>
__global__ __launch_bounds__(512, 2) void attn_bwd_pair_kernel(AttnBwdParams p) {
  using S = PairShape<D>;
  constexpr int KG = S::KG;
  constexpr int KST = D / 16;
  constexpr int NDB = D / 32;
  constexpr int RR = 4, RC = 4;
  extern __shared__ __attribute__((aligned(1024))) char smem[];

  const int tid = threadIdx.x;
  const int lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int pair = wave & 3;
  const bool second = wave >= 4;
  const int kg = pair % KG, qg = pair / KG;
  const int lq = lane & 31;
  const int hf = lane >> 5;
  const uint32_t lds0 = lds_addr(smem);
  BwdUnit txt;
  if (!bwd_unit(p, 1, lane, &txt)) return;
  const int head = txt.kvh;
  const int T = txt.len;
  const int b0 = txt.block * (32 * KG);
  const int r0 = b0 + kg * 32;
  const int blast = min(b0 + 32 * KG - 1, T - 1), rlast = min(r0 + 31, T - 1);
  const int own = r0 + lq;

  const char* const base_q = p.q + txt.start * p.q_stride;
  const char* const base_do = p.dout + txt.start * p.do_stride;

  int s_lo = 0, s_hi = T;
  if (p.window >= 0) {
    s_lo = max(0, b0 - p.window);
    s_hi = min(T, blast + p.window + 1);
  }
  if (p.causal) s_lo = max(s_lo, b0);
  const int t_lo = s_lo / S::BN, t_hi = (s_hi + S::BN - 1) / S::BN;
  const int n_tiles = (t_hi - t_lo) * p.group;

  const uint32_t xst = (uint32_t)p.q_stride, yst = (uint32_t)p.do_stride;
  const BwdLoad<D, S::BN, 8> load(wave, lane, xst, yst);
  if (p.head_dim < D) {
    for (int i = tid; i < S::SWAP / 16; i += 512) lds_store<u32x4>(lds0 + i * 16, (u32x4){0u, 0u, 0u, 0u});
    __syncthreads();
  }
  // From the last rows on, the heads of a tile after one another: so the blocks of a text, in their causal
  // triangle too, stream the same rows at about the same time, and find them in L2. That counts where they do not share
  // one already (bwd_classes): 4 x 4,096 tokens of 16/2 heads, whose q and dO are 32 MB a key head, take 1.91 ms in
  // one class, 1.21 in four; and there 1.12 head by head from the diagonal on. One key head: both the same.
  int dh = 0, dt = t_hi - 1;
  const int64_t h0 = (int64_t)head * p.group;
  const i32x4 xrs = pp_rsrc_words(base_q + h0 * p.head_dim * 2, (uint32_t)T * xst);
  const i32x4 yrs = pp_rsrc_words(base_do + h0 * p.head_dim * 2, (uint32_t)T * yst);
  auto issue = [&](int stage) __attribute__((always_inline)) {
    const uint32_t at = lds0 + stage * S::STAGE + wave * 1024;
    const uint32_t s0 = (uint32_t)(dt * S::BN);
    load.issue(xrs, yrs, at, s0, xst, yst, dh * p.head_dim * 2, p.head_dim);
    if (pair == 0 && lane < S::BN) {
      const uint32_t dst = lds0 + S::STATS + stage * S::STAT + (second ? S::BN * 4 : 0);
      const i32x4 rs = bwd_stat_rsrc(p, h0 + dh + (second ? p.h_q : 0), txt);
      asm volatile("s_nop 4\n\tbuffer_load_dword %0, %1, 0 offen lds"
                   :: "v"((s0 + lane) * 4), "s"(rs), "{m0}"(dst) : "memory");
    }
    if (++dh == p.group) {
      dh = 0;
      --dt;
    }
  };

  // (the first tile is under way while the operand is loaded)
  if (n_tiles > 0) issue(0);

  // this wave's operand: k or v
  bf16x8 opnd[KST];
  {
    const int64_t ho = (int64_t)head * p.head_dim * 2;
    const uint32_t st = (uint32_t)(second ? p.v_stride : p.k_stride);
    const __amdgpu_buffer_rsrc_t rs =
        pp_rsrc((second ? p.v + txt.start * p.v_stride : p.k + txt.start * p.k_stride) + ho, (uint32_t)T * st);
#pragma unroll
    for (int i = 0; i < KST; ++i) {
      const int c = 2 * i + hf;
      const bool ok = own < T && c * 8 < p.head_dim;
      opnd[i] = __builtin_bit_cast(bf16x8, __builtin_amdgcn_raw_buffer_load_b128(rs, ok ? own * st + c * 16 : BWD_NOWHERE, 0, 0));
    }
  }

  // per-lane addresses in stage 0: row reads of q, or dO; transposed reads of dO, or q; statistics
  uint32_t xa[4], ta[4];
  bwd_row_reads(xa, lds0 + (second ? S::TILE : 0), qg * 32, lane);
  bwd_col_reads(ta, lds0 + (second ? 0 : S::TILE), qg * 32, lane);
  uint32_t la = lds0 + S::STATS + ((second ? S::BN : 0) + qg * 32 + 4 * hf) * 4;

  f32x16 acc[NDB];
#pragma unroll
  for (int i = 0; i < NDB; ++i) acc[i] = (f32x16){};
  const uint32_t swap = lds0 + S::SWAP + pair * 4096 + lane * 16;

  // stream rows that some row of this wave sees
  int w_lo = 0, w_hi = T;
  if (p.window >= 0) {
    w_lo = max(0, r0 - p.window);
    w_hi = min(T, rlast + p.window + 1);
  }
  if (p.causal) w_lo = max(w_lo, r0);
  if (r0 >= T) w_hi = 0;

  int t = t_hi - 1, th = 0;
  for (int i = 0; i < n_tiles; ++i) {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    lds_barrier();
    if (i + 1 < n_tiles) issue((i + 1) & 1);
    const int s0 = t * S::BN + qg * 32;
    const bool seen = s0 < w_hi && s0 + 32 > w_lo;
    bf16x8 x[2];
    f32x16 s;
    if (seen) {
      if (!second) __builtin_amdgcn_s_setprio(1);
      rows_product<D, S::BN, RR>(s, rows_stat(la), xa, 0, opnd);
      if (!second) {
        __builtin_amdgcn_s_setprio(0);
        const bool whole = (!p.causal || s0 >= rlast) && (p.window < 0 || (s0 + 31 - r0 <= p.window && rlast - s0 <= p.window));
        if (!whole) {
          const int sb = s0 + 4 * hf;
          int hi = 0x3fffffff, lo = 0;
          if (p.causal) lo = own;
          if (p.window >= 0) {
            lo = max(lo, own - p.window);
            hi = own + p.window;
          }
#pragma unroll
          for (int r = 0; r < 16; ++r) {
            const int at = sb + 8 * (r >> 2) + (r & 3);
            s[r] = at >= lo && at <= hi ? s[r] : -INFINITY;
          }
        }
        float pr[16];
#pragma unroll
        for (int r = 0; r < 16; ++r) pr[r] = __builtin_amdgcn_exp2f(s[r] * p.c);
#pragma unroll
        for (int g = 0; g < 4; ++g) lds_store<f32x4>(swap + g * 1024, (f32x4){pr[4 * g], pr[4 * g + 1], pr[4 * g + 2], pr[4 * g + 3]});
        x[0] = pack8(pr);
        x[1] = pack8(pr + 8);
      }
    }
    lds_barrier();
    if (seen) {
      if (second) {
        float ds[16];
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const f32x4 a = lds_load<f32x4>(swap + g * 1024);
#pragma unroll
          for (int e = 0; e < 4; ++e) ds[4 * g + e] = a[e] * s[4 * g + e];
        }
        x[0] = pack8(ds);
        x[1] = pack8(ds + 8);
      }
      cols_product<D, S::BN, RC>(acc, ta, 0, x);
    }
    if (++th == p.group) {
      th = 0;
      --t;
    }
    // to the other stage: a stage is a power of two and the first one begins at LDS address 0 (the build refuses
    // static LDS in this kernel, which would go before it)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      xa[e] ^= S::STAGE;
      ta[e] ^= S::STAGE;
    }
    la = (i & 1) ? la - S::STAT : la + S::STAT;
  }

  if constexpr (S::QS > 1) {
    // the parts' sums: part 1 into the stages (16 KB per 64 features and pair), part 0 adds
    static_assert(S::QS == 2 && 2 * KG * NDB * 4096 <= S::SWAP, "sums of the second half fit the stages");
    const uint32_t at = lds0 + (kg * 2 + (second ? 1 : 0)) * NDB * 4096 + lane * 16;
    lds_barrier();
#pragma unroll
    for (int db = 0; db < NDB; ++db)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const uint32_t a = at + (db * 4 + g) * 1024;
        if (qg == 1) lds_store<f32x4>(a, (f32x4){acc[db][4 * g], acc[db][4 * g + 1], acc[db][4 * g + 2], acc[db][4 * g + 3]});
      }
    lds_barrier();
    if (qg == 1) return;
#pragma unroll
    for (int db = 0; db < NDB; ++db)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const f32x4 v = lds_load<f32x4>(at + (db * 4 + g) * 1024);
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[db][4 * g + e] += v[e];
      }
  }
  char* const dst = second ? p.dk : p.dv;
  const int64_t stride = second ? p.dk_stride : p.dv_stride;
  const __amdgpu_buffer_rsrc_t rs =
      pp_rsrc(dst + txt.start * stride + (int64_t)head * p.head_dim * (OUT16 ? 2 : 4), (uint32_t)T * (uint32_t)stride);
  bwd_store<D, OUT16>(acc, second ? p.scale : 1.f, rs, own < T ? (uint32_t)own * (uint32_t)stride : BWD_NOWHERE, hf, p.head_dim);
}

struct BwdTable {
  BwdText at[BWD_INLINE];
};
__global__ __launch_bounds__(BWD_INLINE) void bwd_table_kernel(BwdTable t, BwdText* out, int n) {
  if ((int)threadIdx.x < n) out[threadIdx.x] = t.at[threadIdx.x];
}

}  // namespace

}  // namespace inl

namespace inl {

namespace {

typedef void (*AttnBwdFn)(AttnBwdParams);

struct BwdLaunch {
  const char* name;
  AttnBwdFn fn;
  int own;       // own rows of a workgroup
  int threads, lds;
};

template <int D, bool KV, int QS>
BwdLaunch bwd_plain(const char* name, bool out16) {
  using S = BwdShape<D, KV, QS>;
  return {name, out16 ? attn_bwd_kernel<D, KV, QS, true> : attn_bwd_kernel<D, KV, QS, false>, S::OWN, 256, S::LDS};
}
template <int D>
BwdLaunch bwd_pair(const char* name, bool out16) {
  using S = PairShape<D>;
  return {name, out16 ? attn_bwd_pair_kernel<D, true> : attn_bwd_pair_kernel<D, false>, 32 * S::KG, 512, S::LDS};
}

// How many times the average load of a place for a workgroup (`places` per CU) the longest workgroup's stream
// is, with blocks of 128 own rows: above 1 it is what the kernel takes. 0: nothing to share between parts.
double bwd_longest(const inl_attn_desc& d, const std::vector<BwdText>& texts, bool kv, int cus, int places) {
  double longest = 0, all = 0;
  for (const BwdText& x : texts) {
    const double rows = d.window >= 0 ? std::min<double>(x.len, 2.0 * d.window + 128) : x.len;
    longest = std::max(longest, rows);
    all += rows * ((x.len + 127) / 128) * (d.causal && d.window < 0 ? 0.5 : 1.0);
  }
  if (longest <= 64) return 0;
  // (a key block streams its group of heads, a query block is one of as many)
  return longest * cus * places / (all * (kv ? d.h_kv : d.h_q));
}

// Two parts of the waves (QS = 2) halve the longest workgroup's stream and make twice the
// workgroups, for twice the tiles read. us with one part / two (texts x tokens, query / key heads x features;
// average loads of the longest):
//   dq:     two above 2.5: 1 x 1,024 causal 16/8 x 128 (8) 36 / 23, 1 x 2,048 12/12 x 64 (4) 47 / 39,
//           8 x 512 causal 16/8 x 128 (2) 34 / 40, 64 ragged causal passages 16/8 x 128 (1.6) 109 / 131,
//           8 x 1,024 3/1 x 256 (1.3) 63 / 78, 16 x 256 16/16 x 64 (1.5) 17 / 20
//   dk, dv: x 64, two above 2: 1 x 2,048 12/12 (4) 57 / 47, 2 x 2,048 16/16 (1.5) 81 / 93;
//           x 128, two above 1.2: 8 x 512 16/8 (2) 54 / 45, 4 x 2,048 (1) 256 / 275;
//           x 128, causal, whose blocks are of unequal length, two: the passages (3.3) 179 / 123, 8 x 2,048 (1)
//           374 / 323, 64 x 180 (1) 64 / 56; with a window, which makes long texts' equal: 64 x 180, 32 and 128:
//           56 / 53 and 64 / 57; 32 x 512, 64 and 256: 75 / 77 and 113 / 110; 8 x 2,048, 64 and 512: 74 / 77 and
//           176 / 172; 16 x 1,024, 16: 68 / 77; 4 x 4,096, 128: 90 / 92
BwdLaunch bwd_launch(const inl_attn_desc& d, const std::vector<BwdText>& texts, bool kv, int cus, bool out16) {
  const int dim = d.head_dim <= 64 ? 64 : d.head_dim <= 128 ? 128 : 256;
#define INL_BWD(D, KV, QS) bwd_plain<D, KV, QS>("attn_bwd_kernel<" #D ", " #KV ", " #QS ">", out16)
  if (kv && dim == 256) return bwd_pair<256>("attn_bwd_pair_kernel<256>", out16);
  const double over = bwd_longest(d, texts, kv, cus, dim == 64 ? 3 : dim == 128 ? 2 : 1);
  const bool two = !kv ? over > 2.5 : dim == 64 ? over > 2 : (d.causal && over > 0) || over > 1.2;
  if (dim == 64) return kv ? (two ? INL_BWD(64, true, 2) : INL_BWD(64, true, 1))
                           : (two ? INL_BWD(64, false, 2) : INL_BWD(64, false, 1));
  if (dim == 128) return kv ? (two ? INL_BWD(128, true, 2) : INL_BWD(128, true, 1))
                            : (two ? INL_BWD(128, false, 2) : INL_BWD(128, false, 1));
  return two ? INL_BWD(256, false, 2) : INL_BWD(256, false, 1);
#undef INL_BWD
}

// Which texts a workgroup finds its unit among, longest first within a class, so that the last workgroups
// are short ones. Workgroup i runs on XCD i mod 8, each with an L2 of its own: with the texts dealt to as many
// classes as make key heads x classes a multiple of 8, all blocks of a (text, key head), which
// stream the same rows, share one. Texts that do not fill the classes evenly, to 1.15 of the mean, run in
// one class: an XCD without work costs more than L2 misses. us (dq, and dk and dv) in one class / several:
//   4 x 4,096 causal 16/2 x 256 (1.0 of the mean) 940 / 909, 1,908 / 1,207; 24 x 1,024 3/1 x 256 (1.0) 174 / 171,
//   205 / 195; 24 texts to 2,048 of them, window 512 (1.1) 141 / 136, 178 / 164; 14 x 1,024 16/2 x 256 (1.14) 432 / 479,
//   627 / 618; 28 x 1,024 8/1 x 128 (1.14) 190 / 204, 262 / 251; 5 x 1,024 12/12 x 64 (1.2) 38 / 45, 44 / 50;
//   18 x 1,024 3/1 x 256 (1.33) 118 / 169, 203 / 194; 3 x 4,096 16/2 x 256 (1.33) 1,211 / 1,558, 2,322 / 2,048;
//   6 x 4,096 (1.33) 2,402 / 3,145, 3,584 / 4,667; 1 x 4,096 (4) 417 / 1,542, 925 / 1,964
void bwd_classes(const inl_attn_desc& d, std::vector<BwdText>* texts, AttnBwdParams* p) {
  std::sort(texts->begin(), texts->end(), [](const BwdText& a, const BwdText& b) {
    return a.len != b.len ? a.len > b.len : a.start < b.start;
  });
  const int h = d.h_kv;
  p->classes = h % 8 == 0 ? 1 : h % 4 == 0 ? 2 : h % 2 == 0 ? 4 : 8;
  p->first[1] = (int32_t)texts->size();
  if (p->classes == 1) return;
  std::vector<BwdText> in[BWD_CLASSES];
  double load[BWD_CLASSES] = {}, all = 0;
  for (const BwdText& x : *texts) {   // the next longest to the least loaded
    const int c = (int)(std::min_element(load, load + p->classes) - load);
    const double cost = (double)x.len * (d.window >= 0 ? std::min<double>(x.len, 2.0 * d.window + 128) : x.len);
    in[c].push_back(x);
    load[c] += cost;
    all += cost;
  }
  if (*std::max_element(load, load + p->classes) * p->classes > 1.15 * all) {
    p->classes = 1;
    return;
  }
  int32_t at = 0;
  for (int c = 0; c < p->classes; ++c) {
    p->first[c] = at;
    for (const BwdText& x : in[c]) (*texts)[at++] = x;
    p->first[c + 1] = at;
  }
}

size_t bwd_stat_bytes(const inl_attn_desc& d, int64_t rows) { return ((size_t)2 * d.h_q * rows * 4 + 255) & ~(size_t)255; }

// Checks what the forward's desc leaves open, and lists the texts that have tokens.
int bwd_texts(const inl_attn_desc* d, int64_t* rows, std::vector<BwdText>* texts) {
  int rc = attn_check(d, rows);
  if (rc) return rc;
  if (d->dtype != INL_BF16 || d->out_dtype != INL_BF16)
    return fail(INL_E_UNSUPPORTED, "attention backward: q, k, v, out and dout must be bf16");
  texts->reserve(d->n_texts);
  for (int32_t b = 0; b < d->n_texts; ++b) {
    const int32_t at = d->cu_seqlens_host[b], len = d->cu_seqlens_host[b + 1] - at;
    if (len > 0) texts->push_back({d->seq_starts_host ? d->seq_starts_host[b] : at, len, 0});
  }
  if (d->seq_starts_host) {   // a row of two texts would get two gradients
    std::vector<BwdText> by(*texts);
    std::sort(by.begin(), by.end(), [](const BwdText& a, const BwdText& b) { return a.start < b.start; });
    for (size_t i = 1; i < by.size(); ++i)
      if (by[i].start < by[i - 1].start + by[i - 1].len)
        return fail(INL_E_INVALID, "attention backward: texts overlap (seq_starts_host)");
  }
  return INL_OK;
}

size_t bwd_bytes(const inl_attn_desc& d, int64_t rows, size_t texts) {
  return texts == 0 ? 0 : bwd_stat_bytes(d, rows) + (texts > (size_t)BWD_INLINE ? texts * sizeof(BwdText) : 0);
}

struct BwdTensor {
  const char* what;
  const void* at;
  int64_t heads, stride;   // elements
  int32_t dtype;
};

int bwd_run(const inl_attn_desc* d, const inl_attn_grads* g, const void* q, const void* k, const void* v, const void* o,
            const void* dout, void* dq, void* dk, void* dv, void* ws, size_t ws_bytes, hipStream_t st) {
  if (!g) return fail(INL_E_INVALID, "attention backward: grads is NULL");
  int64_t rows = 0;
  std::vector<BwdText> texts;
  int rc = bwd_texts(d, &rows, &texts);
  if (rc) return rc;
  if (!dtype_ok(g->grad_dtype)) return fail(INL_E_INVALID, "attention backward: grad_dtype must be INL_F32 or INL_BF16");
  if (!dk != !dv) return fail(INL_E_INVALID, "attention backward: dk and dv are computed together (or both NULL)");
  const int64_t qr = (int64_t)d->h_q * d->head_dim, kr = (int64_t)d->h_kv * d->head_dim;
  const BwdTensor t[8] = {{"q", q, d->h_q, d->q_row_stride ? d->q_row_stride : qr, INL_BF16},
                          {"k", k, d->h_kv, d->k_row_stride ? d->k_row_stride : kr, INL_BF16},
                          {"v", v, d->h_kv, d->v_row_stride ? d->v_row_stride : kr, INL_BF16},
                          {"out", o, d->h_q, d->o_row_stride ? d->o_row_stride : qr, INL_BF16},
                          {"dout", dout, d->h_q, g->do_row_stride ? g->do_row_stride : qr, INL_BF16},
                          {"dq", dq, d->h_q, g->dq_row_stride ? g->dq_row_stride : qr, g->grad_dtype},
                          {"dk", dk, d->h_kv, g->dk_row_stride ? g->dk_row_stride : kr, g->grad_dtype},
                          {"dv", dv, d->h_kv, g->dv_row_stride ? g->dv_row_stride : kr, g->grad_dtype}};
  int64_t longest = 0;
  int64_t blocks = 0;
  for (const BwdText& x : texts) {
    longest = std::max<int64_t>(longest, x.len);
    blocks += (x.len + 63) / 64;
  }
  // (all classes are numbered like the one with the most blocks)
  if (blocks * d->h_q * BWD_CLASSES > INT32_MAX)
    return fail(INL_E_UNSUPPORTED, "attention backward: more than 2^28 blocks of 64 rows and a head");
  Rows r[8];
  for (int i = 0; i < 8; ++i) {
    const int64_t es = dtype_size(t[i].dtype), len = t[i].heads * d->head_dim;
    if (t[i].stride < len || (t[i].stride * es) % 16)
      return fail(INL_E_INVALID, std::string("attention backward: ") + t[i].what +
                                     ": the row stride must cover all heads and be a multiple of 16 bytes");
    if ((!t[i].at && i < 5 && rows) || ((uintptr_t)t[i].at & 15))
      return fail(INL_E_INVALID, std::string("attention backward: ") + t[i].what + " must be non-null and 16-byte aligned");
    // rows of a text, and those of its last tile behind it, are addressed with 32 bits
    if (t[i].stride >= (int64_t)BWD_NOWHERE || (longest + 128) * t[i].stride * es >= (int64_t)BWD_NOWHERE)
      return fail(INL_E_UNSUPPORTED, std::string("attention backward: a text's rows of ") + t[i].what + " span 4 GiB or more");
    r[i] = {t[i].at, rows, len * es, t[i].stride * es};
  }
  for (int i = 5; i < 8; ++i)
    for (int j = 0; j < i; ++j)
      if (rows_meet(r[i], r[j]))
        return fail(INL_E_INVALID, std::string("attention backward: ") + t[i].what + " overlaps " + t[j].what);
  if (texts.empty() || (!dq && !dk)) return INL_OK;
  if ((rc = check_workspace("attention backward", ws, ws_bytes, bwd_bytes(*d, rows, texts.size())))) return rc;

  AttnBwdParams p{};
  p.q = (const char*)q;
  p.k = (const char*)k;
  p.v = (const char*)v;
  p.o = (const char*)o;
  p.dout = (const char*)dout;
  p.dq = (char*)dq;
  p.dk = (char*)dk;
  p.dv = (char*)dv;
  int64_t* const strides[8] = {&p.q_stride, &p.k_stride, &p.v_stride, &p.o_stride,
                               &p.do_stride, &p.dq_stride, &p.dk_stride, &p.dv_stride};
  for (int i = 0; i < 8; ++i) *strides[i] = t[i].stride * dtype_size(t[i].dtype);
  p.stat = (float*)ws;
  p.rows = rows;
  p.h_q = d->h_q;
  p.h_kv = d->h_kv;
  p.group = d->h_q / d->h_kv;
  p.head_dim = d->head_dim;
  p.causal = d->causal;
  p.window = (int32_t)std::min<int64_t>(d->window, longest);   // (own + window stays in 32 bits)
  // (the statistics are divided by c, and must stay finite; scores times less than this are 0)
  p.c = std::max(d->scale * kLog2e, 1e-30f);
  p.scale = d->scale;
  const bool out16 = g->grad_dtype == INL_BF16;
  int cus = 0;
  if ((rc = device_cus(&cus))) return rc;
  bwd_classes(*d, &texts, &p);
  for (int kv = 0; kv < (dk ? 2 : 1); ++kv) {
    const BwdLaunch l = bwd_launch(*d, texts, kv, cus, out16);
    int64_t most = 0;
    for (int c = 0; c < p.classes; ++c) {
      int64_t units = 0;
      for (int i = p.first[c]; i < p.first[c + 1]; ++i) {
        texts[i].unit = (int32_t)units;
        units += (texts[i].len + l.own - 1) / l.own;
      }
      p.units[c] = (int32_t)units;
      most = std::max(most, units);
    }
    const int64_t groups = most * p.h_kv * p.classes * (kv ? 1 : p.group);
    // (a dimension of a grid has fewer than 2^32 threads; a multiple of 8 keeps workgroups on their XCDs)
    const int64_t across = std::min<int64_t>(groups, 1 << 22);
    if (texts.size() <= (size_t)BWD_INLINE) {
      std::copy(texts.begin(), texts.end(), p.own);
    } else {
      // More texts go through the workspace, by launches that carry them as arguments: a copy from
      // host memory could not be captured, nor its source freed.
      BwdText* table = (BwdText*)((char*)ws + bwd_stat_bytes(*d, rows));
      for (size_t i = 0; i < texts.size(); i += BWD_INLINE) {
        BwdTable part{};
        const int n = (int)std::min<size_t>(BWD_INLINE, texts.size() - i);
        std::copy(texts.begin() + i, texts.begin() + i + n, part.at);
        hipLaunchKernelGGL(bwd_table_kernel, dim3(1), dim3(BWD_INLINE), 0, st, part, table + i, n);
      }
      p.texts = table;
    }
    if ((rc = set_max_dynamic_lds((const void*)l.fn, l.lds))) return rc;
    hipLaunchKernelGGL(l.fn, dim3((unsigned)across, (unsigned)((groups + across - 1) / across)), dim3(l.threads), l.lds, st, p);
    INL_HIP_TRY(hipGetLastError());
  }
  return INL_OK;
}

}  // namespace

}  // namespace inl

extern "C" int inl_attn_bwd_workspace_size(const inl_attn_desc* d, size_t* bytes) {
  using namespace inl;
  if (!bytes) return fail(INL_E_INVALID, "attention backward: bytes is NULL");
  try {
    int64_t rows = 0;
    std::vector<BwdText> texts;
    int rc = bwd_texts(d, &rows, &texts);
    if (rc) return rc;
    *bytes = bwd_bytes(*d, rows, texts.size());
    return INL_OK;
  } catch (const std::bad_alloc&) {
    return fail(INL_E_NOMEM, "attention backward: out of host memory");
  }
}

extern "C" int inl_attn_bwd_kernel_name(const inl_attn_desc* d, int32_t kv, const char** name) {
  using namespace inl;
  if (!name) return fail(INL_E_INVALID, "attention backward: name out-pointer is NULL");
  *name = nullptr;
  if (kv != 0 && kv != 1) return fail(INL_E_INVALID, "attention backward: kv must be 0 (dq) or 1 (dk, dv)");
  try {
    int64_t rows = 0;
    std::vector<BwdText> texts;
    int rc = bwd_texts(d, &rows, &texts);
    if (rc) return rc;
    int cus = 0;
    if (device_cus(&cus)) {   // (no device: as an MI355X has them)
      (void)hipGetLastError();
      cus = 256;
    }
    *name = texts.empty() ? "none" : bwd_launch(*d, texts, kv != 0, cus, true).name;
    return INL_OK;
  } catch (const std::bad_alloc&) {
    return fail(INL_E_NOMEM, "attention backward: out of host memory");
  }
}

extern "C" int inl_attn_varlen_bwd(const inl_attn_desc* d, const inl_attn_grads* g, const void* q, const void* k,
                                   const void* v, const void* out, const void* dout, void* dq, void* dk, void* dv,
                                   void* ws, size_t ws_bytes, void* stream) {
  using namespace inl;
  try {
    return bwd_run(d, g, q, k, v, out, dout, dq, dk, dv, ws, ws_bytes, (hipStream_t)stream);
  } catch (const std::bad_alloc&) {
    return fail(INL_E_NOMEM, "attention backward: out of host memory");
  }
}
