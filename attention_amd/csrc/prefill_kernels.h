// Device code of prompt attention shared by the VALU kernel (prefill.hip) and
// the matrix-core kernels (prefill_mfma_*.hip).
#ifndef QD_PREFILL_KERNELS_H
#define QD_PREFILL_KERNELS_H

#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include "packed.h"
#include "qd_attention.h"
#include "qd_device.h"

// Arguments of the kernels, passed between translation units.
struct PrefillParams {
  const void* q;
  const void* k;
  const void* v;
  const int32_t* cu;
  const int32_t* cu_k;
  void* out;
  int64_t q_stride, k_stride, v_stride;  // elements from token to token
  int B, Tq, Tk, Hq, Hkv, D, G;          // G q-heads per kv-head
  int window, sinks;
  float sl2;  // scale * log2(e)
};

#endif  // QD_PREFILL_KERNELS_H
