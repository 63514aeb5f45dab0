// Windowed and tree decode of f16 caches on the matrix cores: the
// instances of tree_kernels.h.

#include "tree_kernels.h"

int qd_tree_mfma_launch_f16(const TreeParams& p, int dp, int grid, void* stream) {
  hipStream_t st = static_cast<hipStream_t>(stream);
  switch (dp) {
    case 64: return tree_launch_rows<QD_DTYPE_F16, 64, 16>(p, grid, st);
    case 96: return tree_launch_rows<QD_DTYPE_F16, 96, 16>(p, grid, st);
    case 128: return tree_launch_rows<QD_DTYPE_F16, 128, 16>(p, grid, st);
    case 192: return tree_launch_rows<QD_DTYPE_F16, 192, 16>(p, grid, st);
    case 256: return tree_launch_rows<QD_DTYPE_F16, 256, 16>(p, grid, st);
    default: return hipErrorInvalidValue;
  }
}
