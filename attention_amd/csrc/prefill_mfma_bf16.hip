// Prompt attention of bf16 tensors on the matrix cores: the instances of
// prefill_kernels.h.

#include "prefill_kernels.h"

namespace {

template <int DP>
hipError_t run(const PrefillParams& p, int rows, uint32_t grid, hipStream_t st) {
  if (rows == 128) return prefill_launch<QD_DTYPE_BF16, DP, 1, 4>(p, grid, st);
  if constexpr (DP == 64)
    if (rows == 256) return prefill_launch<QD_DTYPE_BF16, DP, 2, 4>(p, grid, st);
  return hipErrorInvalidValue;
}

}  // namespace

int qd_prefill_mfma_launch_bf16(const PrefillParams& p, int dp, int rows, uint32_t grid, void* stream) {
  hipStream_t st = static_cast<hipStream_t>(stream);
  switch (dp) {
    case 64: return run<64>(p, rows, grid, st);
    case 96: return run<96>(p, rows, grid, st);
    case 128: return run<128>(p, rows, grid, st);
    case 192: return run<192>(p, rows, grid, st);
    case 256: return run<256>(p, rows, grid, st);
    default: return hipErrorInvalidValue;
  }
}
