// The tiled products whose operands are both rows of k: y = x . w^T and its
// epilogues (linear, gated, cross entropy).
#include "tile_gemm.hpp"

namespace inl {

namespace {
template <bool OUT16>
int linear(const TileParams& p, const TilePlan& plan, int cus, hipStream_t stream) {
  return p.res ? tile_launch<OP_ROWS, OP_ROWS, EPI_LINEAR, OUT16, true>(p, plan, cus, stream)
               : tile_launch<OP_ROWS, OP_ROWS, EPI_LINEAR, OUT16, false>(p, plan, cus, stream);
}
int part_nt(TileParams p, const TilePlan& plan, float* part, int cus, hipStream_t stream) {
  p.y = (char*)part;
  p.ys = p.n;
  return tile_launch<OP_ROWS, OP_ROWS, EPI_PART, false, false>(p, plan, cus, stream);
}
}  // namespace

int tile_nt_linear(TileParams p, const TilePlan& plan, bool out_bf16, float* part, int cus, hipStream_t stream) {
  if (plan.splits > 1) {
    int rc = part_nt(p, plan, part, cus, stream);
    return rc ? rc : tile_finish(p, EPI_LINEAR, plan.splits, part, out_bf16, stream);
  }
  return out_bf16 ? linear<true>(p, plan, cus, stream) : linear<false>(p, plan, cus, stream);
}

int tile_nt_gated(TileParams p, const TilePlan& plan, float* part, int cus, hipStream_t stream) {
  if (plan.splits > 1) {
    TileParams q = p;
    q.n = 2 * p.n;
    int rc = part_nt(q, plan, part, cus, stream);
    return rc ? rc : tile_finish(p, EPI_GATED, plan.splits, part, true, stream);
  }
  return tile_launch<OP_ROWS, OP_ROWS, EPI_GATED, true, false>(p, plan, cus, stream);
}

int tile_nt_xent(const TileParams& p, const TilePlan& plan, int cus, hipStream_t stream) {
  return tile_launch<OP_ROWS, OP_ROWS, EPI_XENT, false, false>(p, plan, cus, stream);
}

int tile_nt_dxent(const TileParams& p, const TilePlan& plan, int cus, hipStream_t stream) {
  return tile_launch<OP_ROWS, OP_ROWS, EPI_DXENT, true, false>(p, plan, cus, stream);
}

}  // namespace inl
