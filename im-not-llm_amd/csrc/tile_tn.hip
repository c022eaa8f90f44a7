// The tiled products whose operands are both stored along the summed axis:
// dw = dz^T . x, summed over the token rows. And the plan of a tiled product,
// and the kernel that joins a split one.
#include "tile_gemm.hpp"

namespace inl {

namespace {

struct FinishParams {
  TileParams t;
  const float* part;
  int splits;
  int64_t quads;   // groups of 4 output columns
};

// One thread: 4 output columns of one row, the partials added in split order. Bound by
// memory (splits 4-byte reads per output).
template <int EPI, bool OUT16>
__global__ __launch_bounds__(256) void tile_finish_kernel(FinishParams f) {
  const TileParams& p = f.t;
  const int nq = p.n / 4;
  const int64_t cols = EPI == EPI_GATED ? 2 * (int64_t)p.n : p.n;
  const int64_t plane = p.m * cols;
  for (int64_t i = blockIdx.x * 256LL + threadIdx.x; i < f.quads; i += gridDim.x * 256LL) {
    const int64_t row = i / nq;
    const int col = (int)(i - row * nq) * 4;
    auto sum = [&](int64_t at) {
      f32x4 t = *reinterpret_cast<const f32x4*>(f.part + at);
      for (int s = 1; s < f.splits; ++s) {
        const f32x4 q = *reinterpret_cast<const f32x4*>(f.part + at + s * plane);
#pragma unroll
        for (int e = 0; e < 4; ++e) t[e] += q[e];
      }
      return t;
    };
    auto put16 = [](char* dst, const f32x4& v) {
      bf16x4 o;
#pragma unroll
      for (int e = 0; e < 4; ++e) o[e] = (bf16)v[e];
      *reinterpret_cast<bf16x4*>(dst) = o;
    };
    f32x4 t = sum(row * cols + col);
    if constexpr (EPI == EPI_GATED) {
      const f32x4 up = sum(row * cols + p.n + col);
      if (p.pre) {
        put16(p.pre + (row * p.ps + col) * 2, t);
        put16(p.pre + (row * p.ps + p.n + col) * 2, up);
      }
      t = act_apply4(p.act, t);
#pragma unroll
      for (int e = 0; e < 4; ++e) t[e] *= up[e];
      put16(p.y + (row * p.ys + col) * 2, t);
    } else if constexpr (EPI == EPI_DGATED) {
      const char* g0 = p.pre + (row * p.ps + col) * 2;
      const bf16x4 gv = *reinterpret_cast<const bf16x4*>(g0);
      const bf16x4 uv = *reinterpret_cast<const bf16x4*>(g0 + (int64_t)p.n * 2);
      f32x4 dg, du;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const ActPair q = act_pair(p.act, (float)gv[e]);
        dg[e] = t[e] * (float)uv[e] * q.slope;
        du[e] = t[e] * q.value;
      }
      put16(p.y + (row * p.ys + col) * 2, dg);
      put16(p.y + (row * p.ys + p.n + col) * 2, du);
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) t[e] *= p.alpha;
      if (p.bias) {
        const f32x4 b = *reinterpret_cast<const f32x4*>(p.bias + col);
#pragma unroll
        for (int e = 0; e < 4; ++e) t[e] += b[e];
      }
      if (p.pre) put16(p.pre + (row * p.ps + col) * 2, t);
      t = act_apply4(p.act, t);
      if (p.res) {
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
      if constexpr (OUT16) put16(p.y + (row * p.ys + col) * 2, t);
      else *reinterpret_cast<f32x4*>(p.y + (row * p.ys + col) * 4) = t;
    }
  }
}

int part_tn(TileParams p, const TilePlan& plan, float* part, int cus, hipStream_t stream) {
  p.y = (char*)part;
  p.ys = p.n;
  return tile_launch<OP_COLS, OP_COLS, EPI_PART, false, false>(p, plan, cus, stream);
}

}  // namespace

int tile_finish(const TileParams& p, int epi, int splits, const float* part, bool out_bf16, hipStream_t stream) {
  FinishParams f;
  f.t = p;
  f.part = part;
  f.splits = splits;
  f.quads = p.m * (p.n / 4);
  const dim3 grid((unsigned)std::min<int64_t>((f.quads + 255) / 256, 8192)), block(256);
  if (epi == EPI_GATED) hipLaunchKernelGGL((tile_finish_kernel<EPI_GATED, true>), grid, block, 0, stream, f);
  else if (epi == EPI_DGATED) hipLaunchKernelGGL((tile_finish_kernel<EPI_DGATED, true>), grid, block, 0, stream, f);
  else if (out_bf16) hipLaunchKernelGGL((tile_finish_kernel<EPI_LINEAR, true>), grid, block, 0, stream, f);
  else hipLaunchKernelGGL((tile_finish_kernel<EPI_LINEAR, false>), grid, block, 0, stream, f);
  INL_HIP_TRY(hipGetLastError());
  return INL_OK;
}

int tile_tn_linear(TileParams p, const TilePlan& plan, bool out_bf16, float* part, int cus, hipStream_t stream) {
  if (plan.splits > 1) {
    int rc = part_tn(p, plan, part, cus, stream);
    return rc ? rc : tile_finish(p, EPI_LINEAR, plan.splits, part, out_bf16, stream);
  }
  return out_bf16 ? tile_launch<OP_COLS, OP_COLS, EPI_LINEAR, true, false>(p, plan, cus, stream)
                  : tile_launch<OP_COLS, OP_COLS, EPI_LINEAR, false, false>(p, plan, cus, stream);
}

// Estimated us of a launch: `start`, then the units of the fullest CU one after
// another, each kper stages and `drain`. A stage of the largest shape is slower on a
// full chip than on a few CUs (the clock goes down under load), 1.05 to 1.42 us.
// Fitted to x . w^T in bf16, us of the shapes 0 / 1 / 2, one split:
//   (1,024 rows, 1,024 outputs, k 8,192): 141 / 60 / 35    (8,192, 1,024, 1,024): 29 / 21 / 34
//   (8,192, 1,024, 2,048): 45 / 35 / 58                    (12,000, 768, 768): 24 / 24 / 29
//   (20,011, 768, 768): 27 / 30 / 46                       (16,384, 2,304, 768): 63 / 60 / 103
//   (16,384, 4,096, 1,024): 114 / 137 / 226                (2,048, 4,096, 1,024): 29 / 21 / 34
// Joining s splits: a launch, a little for each (206 x 184 outputs, k 1,392: 9.3 us with
// 11, 8.0 with 6; 64 x 1,024, k 4,096: 11.7 with 16, 10.2 with 8), and the partials
// written and read.
// An operand by columns costs two reads per fragment, which the smaller shapes
// feel: `cols` us a stage more for each.
TilePlan tile_plan(int64_t m, int64_t n, int64_t k, int by_cols, bool gated, int max_splits, int cus) {
  struct Cost {
    int bn, bm;
    float stage, full, drain, start, cols;
  };
  static const Cost costs[TG_SHAPES] = {{TileShapeOf<0>::BN, TileShapeOf<0>::BM, 1.05f, 1.42f, 4.5f, 4.f, 0.f},
                                        {TileShapeOf<1>::BN, TileShapeOf<1>::BM, 0.44f, 0.47f, 1.f, 4.5f, 0.045f},
                                        {TileShapeOf<2>::BN, TileShapeOf<2>::BM, 0.25f, 0.21f, 0.4f, 3.5f, 0.02f}};
  const int64_t kst = std::max<int64_t>(1, (k + TG_BK - 1) / TG_BK);
  TilePlan best{0, 1, (int32_t)kst};
  float least = -1.f;
  for (int i = 0; i < TG_SHAPES; ++i) {
    const Cost& c = costs[i];
    const int64_t bno = gated ? c.bn / 2 : c.bn;
    const int64_t tiles = ((m + c.bm - 1) / c.bm) * ((n + bno - 1) / bno);
    // (past two units per CU a split only adds partials)
    for (int s = 1; s <= max_splits && s <= kst && (s == 1 || tiles * (s - 1) < 2 * cus); ++s) {
      const int64_t kper = (kst + s - 1) / s;
      if ((kst + kper - 1) / kper != s) continue;   // a split would have no work
      const int64_t units = tiles * s;
      const float fill = std::min(1.f, (float)units / (float)cus);
      const float stage = c.stage + fill * (c.full - c.stage) + (float)by_cols * c.cols;
      float t = c.start + (float)((units + cus - 1) / cus) * ((float)kper * stage + c.drain);
      if (s > 1) t += 3.f + 0.15f * (float)s + (float)m * (float)n * (gated ? 2.f : 1.f) * 8.f * (float)s / 7e6f;
      if (least < 0.f || t < least) {
        least = t;
        best = {i, s, (int32_t)kper};
      }
    }
  }
  return best;
}

}  // namespace inl
