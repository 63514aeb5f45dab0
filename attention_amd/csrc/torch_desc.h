// Tensor descriptors of the C ABI from torch tensors; shared by the files that
// register torch ops.
#ifndef QD_TORCH_DESC_H
#define QD_TORCH_DESC_H

#include <ATen/ATen.h>

#include "qd_attention.h"

namespace {

int dtype_code(const at::Tensor& t) {
  switch (t.scalar_type()) {
    case at::kFloat: return QD_DTYPE_F32;
    case at::kHalf: return QD_DTYPE_F16;
    case at::kBFloat16: return QD_DTYPE_BF16;
    case at::kInt: return QD_DTYPE_I32;
    case at::kLong: return QD_DTYPE_I64;
    default: return QD_DTYPE_OTHER;
  }
}

qd_tensor_desc describe(const at::Tensor& t) {
  qd_tensor_desc d{};
  if (!t.defined()) return d;
  d.defined = 1;
  d.is_device = t.is_cuda() ? 1 : 0;
  d.device_index = t.is_cuda() ? t.get_device() : -1;
  d.contiguous = t.is_contiguous() ? 1 : 0;
  d.dtype = dtype_code(t);
  d.ndim = static_cast<int32_t>(t.dim());
  for (int64_t i = 0; i < t.dim() && i < 8; ++i) d.sizes[i] = t.size(i);
  return d;
}

}  // namespace

#endif  // QD_TORCH_DESC_H
