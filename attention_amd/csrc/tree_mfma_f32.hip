// Windowed and tree decode of f32 caches on the matrix cores: the
// instances of tree_kernels.h.

#include "tree_kernels.h"

int qd_tree_mfma_launch_f32(const TreeParams& p, int dp, int grid, void* stream) {
  hipStream_t st = static_cast<hipStream_t>(stream);
  switch (dp) {
    case 64: return tree_launch_rows<QD_DTYPE_F32, 64, 16>(p, grid, st);
    case 96: return tree_launch_rows<QD_DTYPE_F32, 96, 16>(p, grid, st);
    case 128: return tree_launch_rows<QD_DTYPE_F32, 128, 16>(p, grid, st);
    case 256: return tree_launch_rows<QD_DTYPE_F32, 256, 32>(p, grid, st);
    default: return hipErrorInvalidValue;
  }
}
