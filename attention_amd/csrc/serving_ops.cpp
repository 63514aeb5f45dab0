// Torch ops of the operators without a counterpart in the reference: a
// namespace of their own (qd_serving), because qd_attention holds exactly the
// reference's schemas.  Same host path as torch_ops.cpp: validation, device
// guard, output, launch on the current stream, no host synchronization.

#include <ATen/ATen.h>
#include <ATen/hip/impl/HIPGuardImplMasqueradingAsCUDA.h>
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>
#include <hip/hip_runtime_api.h>
#include <torch/library.h>

#include <vector>

#include "qd_attention.h"
#include "torch_desc.h"

namespace {

// Windowed decode (no mask, q [B, Hq, D]) and tree decode (q [B, T, Hq, D]).
// Workspaces come from the caching allocator per call: they need no zeroing,
// and calls on other streams or in captured graphs get their own.
at::Tensor tree_impl(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, const at::Tensor& table,
                     const at::Tensor& lens, const at::Tensor* mask, double scale, int64_t window, int64_t sinks) {
  const qd_tensor_desc dq = describe(q), dk = describe(k), dv = describe(v), dt = describe(table),
                       dl = describe(lens), dm = mask ? describe(*mask) : qd_tensor_desc{};
  char msg[256];
  int st = qd_gqa_decode_tree_validate(&dq, &dk, &dv, &dt, &dl, mask ? &dm : nullptr, scale, window, sinks, msg,
                                       sizeof(msg));
  TORCH_CHECK(st == QD_OK, msg);
  c10::hip::HIPGuardMasqueradingAsCUDA guard(q.device());
  auto out = at::empty_like(q);
  if (q.size(0) == 0) return out;
  const int B = static_cast<int>(q.size(0));
  const int T = mask ? static_cast<int>(q.size(1)) : 1;
  const int Hq = static_cast<int>(q.size(mask ? 2 : 1));
  const int D = static_cast<int>(k.size(3));
  const int P = static_cast<int>(k.size(1));
  const int Hkv = static_cast<int>(k.size(2));
  const int maxP = static_cast<int>(table.size(1));
  const int has_mask = mask ? 1 : 0, win = static_cast<int>(window), snk = static_cast<int>(sinks);
  const size_t bytes =
      qd_gqa_decode_tree_workspace_bytes(B, T, Hq, Hkv, D, P, maxP, has_mask, win, snk, dq.dtype, 0);
  at::Tensor ws;
  if (bytes > 0) ws = at::empty({static_cast<int64_t>(bytes)}, q.options().dtype(at::kByte));
  hipStream_t stream = c10::hip::getCurrentHIPStreamMasqueradingAsCUDA(q.get_device()).stream();
  st = qd_gqa_decode_tree(q.data_ptr(), k.data_ptr(), v.data_ptr(), table.data_ptr<int32_t>(),
                          lens.data_ptr<int32_t>(), mask ? mask->data_ptr<int64_t>() : nullptr, out.data_ptr(),
                          ws.defined() ? ws.data_ptr() : nullptr, bytes, B, T, Hq, Hkv, D, P, maxP, k.size(0),
                          dq.dtype, static_cast<float>(scale), win, snk, 0, stream);
  TORCH_CHECK(st == QD_OK, qd_error_string(st));
  return out;
}

at::Tensor gqa_decode_window_hip(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v,
                                 const at::Tensor& table, const at::Tensor& lens, double scale, int64_t window,
                                 int64_t sinks) {
  return tree_impl(q, k, v, table, lens, nullptr, scale, window, sinks);
}

at::Tensor gqa_decode_tree_hip(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v,
                               const at::Tensor& table, const at::Tensor& lens, const at::Tensor& mask, double scale,
                               int64_t window, int64_t sinks) {
  return tree_impl(q, k, v, table, lens, &mask, scale, window, sinks);
}

// Descriptor of q, key or value [N, heads, D]: contiguous where the heads of
// each token are, whatever the stride from one token to the next.
qd_tensor_desc describe_tokens(const at::Tensor& t) {
  qd_tensor_desc d = describe(t);
  if (t.dim() == 3)
    d.contiguous = (t.size(2) <= 1 || t.stride(2) == 1) && (t.size(1) <= 1 || t.stride(1) == t.size(2)) ? 1 : 0;
  return d;
}

at::Tensor qk_norm_rope_write_hip(const at::Tensor& q, const at::Tensor& key, const at::Tensor& value,
                                  const at::Tensor& cos_sin, const at::Tensor& positions, at::Tensor k_cache,
                                  at::Tensor v_cache, const at::Tensor& slots,
                                  const c10::optional<at::Tensor>& q_weight,
                                  const c10::optional<at::Tensor>& k_weight, double eps, bool interleaved) {
  const qd_tensor_desc dq = describe_tokens(q), dk = describe_tokens(key), dv = describe_tokens(value),
                       dc = describe(cos_sin), dp = describe(positions), dkc = describe(k_cache),
                       dvc = describe(v_cache), ds = describe(slots),
                       dqw = q_weight.has_value() ? describe(*q_weight) : qd_tensor_desc{},
                       dkw = k_weight.has_value() ? describe(*k_weight) : qd_tensor_desc{};
  char msg[256];
  int st = qd_qk_norm_rope_write_validate(&dq, &dk, &dv, &dc, &dp, &dkc, &dvc, &ds, &dqw, &dkw, eps, msg,
                                          sizeof(msg));
  TORCH_CHECK(st == QD_OK, msg);
  c10::hip::HIPGuardMasqueradingAsCUDA guard(q.device());
  auto out = at::empty({q.size(0), q.size(1), q.size(2)}, q.options());
  if (q.size(0) == 0) return out;
  hipStream_t stream = c10::hip::getCurrentHIPStreamMasqueradingAsCUDA(q.get_device()).stream();
  const int wdt = dqw.defined ? dqw.dtype : dkw.defined ? dkw.dtype : dq.dtype;
  st = qd_qk_norm_rope_write(q.data_ptr(), key.data_ptr(), value.data_ptr(), cos_sin.data_ptr<float>(),
                             positions.data_ptr<int32_t>(), k_cache.data_ptr(), v_cache.data_ptr(),
                             slots.data_ptr<int64_t>(), dqw.defined ? q_weight->data_ptr() : nullptr,
                             dkw.defined ? k_weight->data_ptr() : nullptr, out.data_ptr(), q.size(0),
                             static_cast<int>(q.size(1)), static_cast<int>(key.size(1)), static_cast<int>(q.size(2)),
                             static_cast<int>(cos_sin.size(1)), q.stride(0), key.stride(0), value.stride(0),
                             cos_sin.size(0), k_cache.size(0) * k_cache.size(1), dq.dtype, wdt,
                             static_cast<float>(eps), interleaved ? 1 : 0, stream);
  TORCH_CHECK(st == QD_OK, qd_error_string(st));
  return out;
}

void kv_compact_hip(at::TensorList caches, const at::Tensor& table, const at::Tensor& lens,
                    const at::Tensor& accepted) {
  if (caches.empty()) return;
  const at::Tensor& first = caches[0];
  const qd_tensor_desc dc = describe(first), dt = describe(table), dl = describe(lens), da = describe(accepted);
  char msg[256];
  int st = qd_kv_compact_validate(&dc, &dt, &dl, &da, msg, sizeof(msg));
  TORCH_CHECK(st == QD_OK, msg);
  std::vector<void*> pointers;
  pointers.reserve(caches.size());
  for (const at::Tensor& c : caches) {
    TORCH_CHECK(c.sizes() == first.sizes() && c.scalar_type() == first.scalar_type() && c.device() == first.device() &&
                    c.is_contiguous(),
                "all caches must be contiguous, of one shape and dtype, on one device");
    pointers.push_back(c.data_ptr());
  }
  c10::hip::HIPGuardMasqueradingAsCUDA guard(first.device());
  hipStream_t stream = c10::hip::getCurrentHIPStreamMasqueradingAsCUDA(first.get_device()).stream();
  const int64_t rows = first.size(0) * first.size(1);
  st = qd_kv_compact(pointers.data(), static_cast<int>(pointers.size()), table.data_ptr<int32_t>(),
                     lens.data_ptr<int32_t>(), accepted.data_ptr<int32_t>(), static_cast<int>(accepted.size(0)),
                     static_cast<int>(accepted.size(1)), static_cast<int>(first.size(1)),
                     static_cast<int>(table.size(1)), first.size(0),
                     first.numel() / rows * static_cast<int64_t>(first.element_size()), stream);
  TORCH_CHECK(st == QD_OK, qd_error_string(st));
}

}  // namespace

TORCH_LIBRARY(qd_serving, m) {
  m.def(
      "gqa_decode_window(Tensor q, Tensor k_cache, Tensor v_cache, Tensor block_table, Tensor context_lens, "
      "float scale, int window, int sinks) -> Tensor");
  m.def(
      "gqa_decode_tree(Tensor q, Tensor k_cache, Tensor v_cache, Tensor block_table, Tensor context_lens, "
      "Tensor tree_mask, float scale, int window, int sinks) -> Tensor");
  m.def(
      "qk_norm_rope_write(Tensor q, Tensor key, Tensor value, Tensor cos_sin, Tensor positions, "
      "Tensor(a!) k_cache, Tensor(b!) v_cache, Tensor slots, Tensor? q_weight, Tensor? k_weight, float eps, "
      "bool interleaved) -> Tensor");
  m.def("kv_compact(Tensor(a!)[] caches, Tensor block_table, Tensor context_lens, Tensor accepted) -> ()");
}

TORCH_LIBRARY_IMPL(qd_serving, CUDA, m) {
  m.impl("gqa_decode_window", TORCH_FN(gqa_decode_window_hip));
  m.impl("gqa_decode_tree", TORCH_FN(gqa_decode_tree_hip));
  m.impl("qk_norm_rope_write", TORCH_FN(qk_norm_rope_write_hip));
  m.impl("kv_compact", TORCH_FN(kv_compact_hip));
}
