// Prompt attention of f32 tensors on the matrix cores: the instances of
// prefill_kernels.h.

#include "prefill_kernels.h"

int qd_prefill_mfma_launch_f32(const PrefillParams& p, int dp, int rows, uint32_t grid, void* stream) {
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (rows != 128) return hipErrorInvalidValue;
  switch (dp) {
    case 64: return prefill_launch<QD_DTYPE_F32, 64, 1, 4>(p, grid, st);
    case 128: return prefill_launch<QD_DTYPE_F32, 128, 1, 4>(p, grid, st);
    case 256: return prefill_launch<QD_DTYPE_F32, 256, 1, 4>(p, grid, st);
    default: return hipErrorInvalidValue;
  }
}
