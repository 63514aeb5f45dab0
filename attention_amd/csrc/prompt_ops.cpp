// Torch ops of prompts and 8-bit caches, in the namespace of the operators
// without a counterpart in the reference (serving_ops.cpp).

#include <ATen/ATen.h>
#include <ATen/hip/impl/HIPGuardImplMasqueradingAsCUDA.h>
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>
#include <hip/hip_runtime_api.h>
#include <torch/library.h>

#include "qd_attention.h"
#include "torch_desc.h"

namespace {

// Descriptor of q, key or value [T, heads, D]: contiguous where the heads of
// each token are, whatever the stride from one token to the next.
qd_tensor_desc describe_tokens(const at::Tensor& t) {
  qd_tensor_desc d = describe(t);
  if (t.dim() == 3)
    d.contiguous = (t.size(2) <= 1 || t.stride(2) == 1) && (t.size(1) <= 1 || t.stride(1) == t.size(2)) ? 1 : 0;
  return d;
}

qd_tensor_desc describe_cache(const at::Tensor& t) {
  qd_tensor_desc d = describe(t);
  if (t.scalar_type() == at::kFloat8_e4m3fn) d.dtype = QD_DTYPE_E4M3;
  if (t.scalar_type() == at::kChar) d.dtype = QD_DTYPE_I8;
  return d;
}

qd_tensor_desc describe_optional(const c10::optional<at::Tensor>& t) {
  return t.has_value() ? describe(*t) : qd_tensor_desc{};
}

hipStream_t current_stream(const at::Tensor& t) {
  return c10::hip::getCurrentHIPStreamMasqueradingAsCUDA(t.get_device()).stream();
}

// Workspaces come from the caching allocator per call: they need no zeroing,
// and calls on other streams or in captured graphs get their own.
at::Tensor workspace(const at::Tensor& like, size_t bytes) {
  return bytes > 0 ? at::empty({static_cast<int64_t>(bytes)}, like.options().dtype(at::kByte)) : at::Tensor();
}

at::Tensor gqa_prefill_hip(const at::Tensor& q, const at::Tensor& key, const at::Tensor& value, const at::Tensor& cu,
                           const c10::optional<at::Tensor>& cu_k, double scale, int64_t window, int64_t sinks) {
  const qd_tensor_desc dq = describe_tokens(q), dk = describe_tokens(key), dv = describe_tokens(value),
                       dc = describe(cu), dck = describe_optional(cu_k);
  char msg[256];
  int st = qd_gqa_prefill_validate(&dq, &dk, &dv, &dc, &dck, scale, window, sinks, msg, sizeof(msg));
  TORCH_CHECK(st == QD_OK, msg);
  c10::hip::HIPGuardMasqueradingAsCUDA guard(q.device());
  auto out = at::empty({q.size(0), q.size(1), q.size(2)}, q.options());
  if (q.size(0) == 0) return out;
  const int B = static_cast<int>(cu.size(0)) - 1, Hq = static_cast<int>(q.size(1)), Hkv = static_cast<int>(key.size(1)),
            D = static_cast<int>(q.size(2)), win = static_cast<int>(window);
  const size_t bytes = qd_gqa_prefill_workspace_bytes(B, q.size(0), key.size(0), Hq, Hkv, D, dq.dtype, win,
                                                      static_cast<int>(sinks), 0);
  const at::Tensor ws = workspace(q, bytes);
  st = qd_gqa_prefill(q.data_ptr(), key.data_ptr(), value.data_ptr(), cu.data_ptr<int32_t>(),
                      dck.defined ? cu_k->data_ptr<int32_t>() : nullptr, out.data_ptr(),
                      ws.defined() ? ws.data_ptr() : nullptr, bytes, B, q.size(0), key.size(0), Hq, Hkv, D, q.stride(0),
                      key.stride(0), value.stride(0), dq.dtype, static_cast<float>(scale), win,
                      static_cast<int>(sinks), 0, current_stream(q));
  TORCH_CHECK(st == QD_OK, qd_error_string(st));
  return out;
}

void kv_append_q8_hip(const at::Tensor& key, const at::Tensor& value, at::Tensor k_cache, at::Tensor v_cache,
                      at::Tensor k_scales, at::Tensor v_scales, const at::Tensor& table, const at::Tensor& positions,
                      const c10::optional<at::Tensor>& cu) {
  const qd_tensor_desc dk = describe_tokens(key), dv = describe_tokens(value), dkc = describe_cache(k_cache),
                       dvc = describe_cache(v_cache), dks = describe(k_scales), dvs = describe(v_scales),
                       dt = describe(table), dp = describe(positions), dc = describe_optional(cu);
  char msg[256];
  int st = qd_kv_append_q8_validate(&dk, &dv, &dkc, &dvc, &dks, &dvs, &dt, &dp, &dc, msg, sizeof(msg));
  TORCH_CHECK(st == QD_OK, msg);
  c10::hip::HIPGuardMasqueradingAsCUDA guard(key.device());
  st = qd_kv_append_q8(key.data_ptr(), value.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(),
                       k_scales.data_ptr<float>(), v_scales.data_ptr<float>(), table.data_ptr<int32_t>(),
                       positions.data_ptr<int32_t>(), dc.defined ? cu->data_ptr<int32_t>() : nullptr,
                       static_cast<int>(positions.size(0)), key.size(0), static_cast<int>(key.size(1)),
                       static_cast<int>(key.size(2)), static_cast<int>(k_cache.size(1)),
                       static_cast<int>(table.size(1)), k_cache.size(0), key.stride(0), value.stride(0), dk.dtype,
                       dkc.dtype, current_stream(key));
  TORCH_CHECK(st == QD_OK, qd_error_string(st));
}

void kv_gather_q8_hip(at::Tensor key, at::Tensor value, const at::Tensor& k_cache, const at::Tensor& v_cache,
                      const at::Tensor& k_scales, const at::Tensor& v_scales, const at::Tensor& table,
                      const at::Tensor& lens, const at::Tensor& cu) {
  const qd_tensor_desc dk = describe_tokens(key), dv = describe_tokens(value), dkc = describe_cache(k_cache),
                       dvc = describe_cache(v_cache), dks = describe(k_scales), dvs = describe(v_scales),
                       dt = describe(table), dl = describe(lens), dc = describe(cu);
  char msg[256];
  int st = qd_kv_gather_q8_validate(&dk, &dv, &dkc, &dvc, &dks, &dvs, &dt, &dl, &dc, msg, sizeof(msg));
  TORCH_CHECK(st == QD_OK, msg);
  c10::hip::HIPGuardMasqueradingAsCUDA guard(key.device());
  st = qd_kv_gather_q8(key.data_ptr(), value.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(),
                       k_scales.data_ptr<float>(), v_scales.data_ptr<float>(), table.data_ptr<int32_t>(),
                       lens.data_ptr<int32_t>(), cu.data_ptr<int32_t>(), static_cast<int>(lens.size(0)), key.size(0),
                       static_cast<int>(key.size(1)), static_cast<int>(key.size(2)), static_cast<int>(k_cache.size(1)),
                       static_cast<int>(table.size(1)), k_cache.size(0), key.stride(0), value.stride(0), dk.dtype,
                       dkc.dtype, current_stream(key));
  TORCH_CHECK(st == QD_OK, qd_error_string(st));
}

at::Tensor gqa_decode_q8_hip(const at::Tensor& q, const at::Tensor& k_cache, const at::Tensor& v_cache,
                             const at::Tensor& k_scales, const at::Tensor& v_scales, const at::Tensor& table,
                             const at::Tensor& lens, double scale) {
  const qd_tensor_desc dq = describe(q), dkc = describe_cache(k_cache), dvc = describe_cache(v_cache),
                       dks = describe(k_scales), dvs = describe(v_scales), dt = describe(table), dl = describe(lens);
  char msg[256];
  int st = qd_gqa_decode_q8_validate(&dq, &dkc, &dvc, &dks, &dvs, &dt, &dl, scale, msg, sizeof(msg));
  TORCH_CHECK(st == QD_OK, msg);
  c10::hip::HIPGuardMasqueradingAsCUDA guard(q.device());
  auto out = at::empty_like(q);
  if (q.size(0) == 0) return out;
  const int B = static_cast<int>(q.size(0)), Hq = static_cast<int>(q.size(1)), D = static_cast<int>(q.size(2)),
            P = static_cast<int>(k_cache.size(1)), Hkv = static_cast<int>(k_cache.size(2)),
            maxP = static_cast<int>(table.size(1));
  const size_t bytes = qd_gqa_decode_q8_workspace_bytes(B, Hq, Hkv, D, P, maxP, dq.dtype, 0);
  const at::Tensor ws = workspace(q, bytes);
  st = qd_gqa_decode_q8(q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), k_scales.data_ptr<float>(),
                        v_scales.data_ptr<float>(), table.data_ptr<int32_t>(), lens.data_ptr<int32_t>(),
                        out.data_ptr(), ws.defined() ? ws.data_ptr() : nullptr, bytes, B, Hq, Hkv, D, P, maxP,
                        k_cache.size(0), dq.dtype, dkc.dtype, static_cast<float>(scale), 0, current_stream(q));
  TORCH_CHECK(st == QD_OK, qd_error_string(st));
  return out;
}

}  // namespace

TORCH_LIBRARY_FRAGMENT(qd_serving, m) {
  m.def(
      "gqa_prefill(Tensor q, Tensor key, Tensor value, Tensor cu_seqlens, Tensor? cu_seqlens_k, float scale, "
      "int window, int sinks) -> Tensor");
  m.def(
      "kv_append_q8(Tensor key, Tensor value, Tensor(a!) k_cache, Tensor(b!) v_cache, Tensor(c!) k_scales, "
      "Tensor(d!) v_scales, Tensor block_table, Tensor positions, Tensor? cu_seqlens) -> ()");
  m.def(
      "kv_gather_q8(Tensor(a!) key, Tensor(b!) value, Tensor k_cache, Tensor v_cache, Tensor k_scales, "
      "Tensor v_scales, Tensor block_table, Tensor context_lens, Tensor cu_seqlens) -> ()");
  m.def(
      "gqa_decode_q8(Tensor q, Tensor k_cache, Tensor v_cache, Tensor k_scales, Tensor v_scales, "
      "Tensor block_table, Tensor context_lens, float scale) -> Tensor");
}

TORCH_LIBRARY_IMPL(qd_serving, CUDA, m) {
  m.impl("gqa_prefill", TORCH_FN(gqa_prefill_hip));
  m.impl("kv_append_q8", TORCH_FN(kv_append_q8_hip));
  m.impl("kv_gather_q8", TORCH_FN(kv_gather_q8_hip));
  m.impl("gqa_decode_q8", TORCH_FN(gqa_decode_q8_hip));
}
