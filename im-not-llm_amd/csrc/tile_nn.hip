// The tiled products whose second operand is stored along the summed axis:
// dx = dz . w with w [n, k] rows, summed over n.
#include "tile_gemm.hpp"

namespace inl {

namespace {
template <bool OUT16>
int linear(const TileParams& p, const TilePlan& plan, int cus, hipStream_t stream) {
  return p.res ? tile_launch<OP_ROWS, OP_COLS, EPI_LINEAR, OUT16, true>(p, plan, cus, stream)
               : tile_launch<OP_ROWS, OP_COLS, EPI_LINEAR, OUT16, false>(p, plan, cus, stream);
}
int part_nn(TileParams p, const TilePlan& plan, float* part, int cus, hipStream_t stream) {
  p.y = (char*)part;
  p.ys = p.n;
  return tile_launch<OP_ROWS, OP_COLS, EPI_PART, false, false>(p, plan, cus, stream);
}
}  // namespace

int tile_nn_linear(TileParams p, const TilePlan& plan, bool out_bf16, float* part, int cus, hipStream_t stream) {
  if (plan.splits > 1) {
    int rc = part_nn(p, plan, part, cus, stream);
    return rc ? rc : tile_finish(p, EPI_LINEAR, plan.splits, part, out_bf16, stream);
  }
  return out_bf16 ? linear<true>(p, plan, cus, stream) : linear<false>(p, plan, cus, stream);
}

int tile_nn_dgated(TileParams p, const TilePlan& plan, float* part, int cus, hipStream_t stream) {
  if (plan.splits > 1) {
    int rc = part_nn(p, plan, part, cus, stream);
    return rc ? rc : tile_finish(p, EPI_DGATED, plan.splits, part, true, stream);
  }
  return tile_launch<OP_ROWS, OP_COLS, EPI_DGATED, true, false>(p, plan, cus, stream);
}

}  // namespace inl
