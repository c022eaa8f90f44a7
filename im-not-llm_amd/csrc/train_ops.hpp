// What the entry points of inl_train.h share: argument checks, workspace
// carving, and the memory-bound kernels beside the tiled products.
#pragma once

#include "tile_gemm.hpp"

namespace inl {

// Compute units of the current device.
int device_cus(int* cus);

// One matrix argument: rows of `cols` elements, `stride` apart (0 = packed),
// 16-byte aligned; `what` names it in the error.
int check_rows(const char* what, const void* p, int64_t cols, int64_t stride, int32_t dtype);

// Whether two matrices share a byte: rows of `len` bytes, `step` apart.
struct Rows {
  const void* at;
  int64_t rows, len, step;
};
bool rows_meet(const Rows& a, const Rows& b);

// Pieces of a workspace, each on a 256-byte boundary.
struct Carve {
  char* base;
  size_t used = 0;
  explicit Carve(void* p) : base((char*)p) {}
  char* take(size_t bytes) {
    char* at = base ? base + used : nullptr;
    used += (bytes + 255) & ~(size_t)255;
    return at;
  }
};
int check_workspace(const char* what, const void* ws, size_t have, size_t need);

// y[m, n] = act(x . w^T + bias) + residual, and act(x . w_gate^T) * (x . w_up^T), for
// few rows of x: where few_rows says that they beat the tiled product.
bool few_rows(int64_t m, int64_t n, int64_t k, bool gated);
int few_dense(const TileParams& p, bool gated, bool out_bf16, hipStream_t stream);

// dz = dy * act'(pre) (bf16, packed [m, n]; NULL = not stored) and the column sums of the
// unrounded dz (f32 [n]; NULL = none); pre NULL: dz = dy. `part` holds
// colsum_bytes(m, n). dy may hold any bf16 rows with act NONE.
size_t colsum_bytes(int64_t m, int64_t n);
int act_bwd(int64_t m, int64_t n, const void* dy, int64_t dys, const void* pre, int64_t pres, int32_t act, void* dz,
            float* colsum, float* part, hipStream_t stream);

// out[c] = sum over blocks, in order, of part[block][c], c < n; columns from
// `cut` on go to out2 (either may be NULL).
int colsum_join(const float* part, int64_t blocks, int32_t n, float* out, int32_t cut, float* out2,
                hipStream_t stream);

// Zeros in rows of `cols` elements (an even number in bf16), by a kernel: a
// memset node in a captured graph has given wrong results on replays.
int fill_zero(void* p, int64_t rows, int64_t cols, int64_t stride, int32_t dtype, hipStream_t stream);

}  // namespace inl
