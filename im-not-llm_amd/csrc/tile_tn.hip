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

// One thread: 4 output columns of one row, the partials added in split order.
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

TilePlan tile_plan(int64_t m, int64_t n, int64_t k, bool gated, int max_splits, int cus) {
  struct Cost {
    int bn, bm;
    float stage, drain, start;   // us
  };
  static const Cost costs[TG_SHAPES] = {{TileShapeOf<0>::BN, TileShapeOf<0>::BM, 0.56f, 9.f, 2.f},
                                        {TileShapeOf<1>::BN, TileShapeOf<1>::BM, 0.25f, 2.2f, 2.9f},
                                        {TileShapeOf<2>::BN, TileShapeOf<2>::BM, 0.13f, 0.5f, 3.7f}};
  const int64_t kst = std::max<int64_t>(1, (k + TG_BK - 1) / TG_BK);
  TilePlan best{0, 1, (int32_t)kst};
  float least = -1.f;
  for (int i = 0; i < TG_SHAPES; ++i) {
    const Cost& c = costs[i];
    const int64_t bno = gated ? c.bn / 2 : c.bn;
    const int64_t tiles = ((m + c.bm - 1) / c.bm) * ((n + bno - 1) / bno);
    for (int s = 1; s <= max_splits && s <= kst; s = s < 4 ? s + 1 : s + s / 4) {
      const int64_t kper = (kst + s - 1) / s;
      const int64_t used = (kst + kper - 1) / kper;   // splits that have work
      if (used != s) continue;
      float t = c.start + (float)((tiles * s + cus - 1) / cus) * ((float)kper * c.stage + c.drain);
      // joining: the partials written and read at some 3.5 TB/s, and a launch
      if (s > 1) t += 3.f + (float)m * (float)n * (gated ? 2.f : 1.f) * 8.f * (float)s / 3.5e6f;
      if (least < 0.f || t < least) {
        least = t;
        best = {i, s, (int32_t)kper};
      }
    }
  }
  return best;
}

}  // namespace inl
