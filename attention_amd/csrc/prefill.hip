// Attention over whole prompts, packed, causal, with grouped heads, for MI355X
// (gfx950): the VALU kernel, argument checks and the C entries.  C ABI in
// include/qd_attention.h.

#include <hip/hip_runtime.h>

#include <math.h>
#include <stdint.h>
#include <string.h>

#include <algorithm>
#include <atomic>
#include <string>

#include "prefill_kernels.h"

void qd_set_last_error(int status, const std::string& msg);

namespace {

// Any head_dim, alignment and type, on the VALU: a workgroup per query head of a
// token; its four waves take 64 keys in turn, a lane per key for the scores and
// a lane per 64th column for the values.  Keys that the query does not see are
// not read at all.  For what the matrix-core kernel does not take, and as its
// check: it reads K and V once per query and head.
// grid Tq * Hq, block 256.
template <int DT>
__global__ __launch_bounds__(256) void prefill_generic_kernel(PrefillParams p) {
  using E = Elem<DT>;
  using S = typename E::S;
  __shared__ float qs[256];
  __shared__ float weight[4][64];
  __shared__ int32_t keys[4][64];
  __shared__ float acc_s[4][256];
  __shared__ float ml_s[4][2];
  const int tid = static_cast<int>(threadIdx.x), lane = tid & 63, wv = tid >> 6;
  const int64_t row = blockIdx.x;
  const int hq = static_cast<int>(row % p.Hq), t = static_cast<int>(row / p.Hq);
  const int h = hq / p.G;
  const S* q = static_cast<const S*>(p.q) + t * p.q_stride + static_cast<int64_t>(hq) * p.D;
  for (int d = tid; d < p.D; d += 256) qs[d] = E::to_f(q[d]);
  const int b = packed_find(p.cu, p.B, p.Tq, 1, 1, 0, t);
  const int next = min(b + 1, p.B);  // no sequences: cu has one entry, and no row sees anything
  const int q0 = packed_start(p.cu, b, p.Tq), q1 = packed_start(p.cu, next, p.Tq);
  const int k0 = packed_start(p.cu_k, b, p.Tk), k1 = packed_start(p.cu_k, next, p.Tk);
  // Keys [0, sinks) and [lo, at] are seen; none by rows outside the sequences.
  const int at = t < q1 ? max(max(k1 - k0, 0) - (q1 - q0) + (t - q0), -1) : -1;
  const int lo = p.window > 0 ? max(at - p.window + 1, 0) : 0;
  const int sinks = min(p.sinks, lo);
  const int count = sinks + max(at + 1 - lo, 0);
  __syncthreads();
  float m = -INFINITY, l = 0.f, acc[4] = {0.f, 0.f, 0.f, 0.f};
  for (int first = 64 * wv; first < count; first += 256) {
    const int v = first + lane;
    const bool seen = v < count;
    const int key = k0 + (v < sinks ? v : lo + (v - sinks));
    float x = -INFINITY;
    if (seen) {
      const S* k = static_cast<const S*>(p.k) + key * p.k_stride + static_cast<int64_t>(h) * p.D;
      float dot = 0.f;
      for (int d = 0; d < p.D; ++d) dot = fmaf(qs[d], E::to_f(k[d]), dot);
      x = dot * p.sl2;
    }
    const float mx = fmaxf(m, wave_max(x));
    const float use = mx == -INFINITY ? 0.f : mx;
    const float alpha = fast_exp2(m - use);  // m = -inf: 0
    const float w = seen ? fast_exp2(x - use) : 0.f;
    m = mx;
    l = l * alpha + wave_sum(w);
    for (int e = 0; e < 4; ++e) acc[e] *= alpha;
    weight[wv][lane] = w;
    keys[wv][lane] = key;
    __builtin_amdgcn_wave_barrier();
    for (int j = 0; j < min(64, count - first); ++j) {
      const float wj = weight[wv][j];
      const S* val = static_cast<const S*>(p.v) + keys[wv][j] * p.v_stride + static_cast<int64_t>(h) * p.D;
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (lane + 64 * e < p.D) acc[e] = fmaf(wj, E::to_f(val[lane + 64 * e]), acc[e]);
    }
    __builtin_amdgcn_wave_barrier();
  }
  for (int e = 0; e < 4; ++e) acc_s[wv][lane + 64 * e] = acc[e];
  if (lane == 0) {
    ml_s[wv][0] = m;
    ml_s[wv][1] = l;
  }
  __syncthreads();
  float mx = -INFINITY;
  for (int w = 0; w < 4; ++w) mx = fmaxf(mx, ml_s[w][0]);
  const float use = mx == -INFINITY ? 0.f : mx;
  float sum = 0.f, f[4];
  for (int w = 0; w < 4; ++w) {
    f[w] = fast_exp2(ml_s[w][0] - use);
    sum += f[w] * ml_s[w][1];
  }
  if (tid < p.D) {
    float a = 0.f;
    for (int w = 0; w < 4; ++w) a += f[w] * acc_s[w][tid];
    static_cast<S*>(p.out)[row * p.D + tid] = E::from_f(sum > 0.f || sum != sum ? a / sum : 0.f);
  }
}

int prefill_fail(char* msg, size_t cap, const char* text) {
  qd_set_last_error(QD_ERR_INVALID_VALUE, text);
  if (msg && cap) {
    size_t n = strlen(text);
    if (n >= cap) n = cap - 1;
    memcpy(msg, text, n);
    msg[n] = '\0';
  }
  return QD_ERR_INVALID_VALUE;
}

bool float_dtype(int dt) { return dt == QD_DTYPE_F32 || dt == QD_DTYPE_F16 || dt == QD_DTYPE_BF16; }

bool prefill_shape_ok(int batch, int64_t q_tokens, int64_t k_tokens, int q_heads, int kv_heads, int head_dim,
                      int dtype) {
  return batch >= 0 && batch < (1 << 24) && q_tokens >= 0 && k_tokens >= 0 && k_tokens <= INT32_MAX - 255 &&
         q_heads > 0 && kv_heads > 0 && q_heads % kv_heads == 0 && head_dim >= 1 && head_dim <= 256 &&
         float_dtype(dtype) && q_heads < (1 << 24) && q_tokens < (int64_t{1} << 31) / q_heads;
}

struct PrefillPlan {
  bool mfma;
  int dp;        // padded head_dim
  int rows;      // rows of a workgroup
  int64_t grid;  // workgroups, of which `splits` share an item's keys
  int splits;
  size_t bytes;
};

int prefill_cu_count() {
  static std::atomic<int> cached[16];
  int dev = 0;
  if (hipGetDevice(&dev) != hipSuccess || dev < 0 || dev >= 16) {
    (void)hipGetLastError();
    dev = 0;
  }
  int n = cached[dev].load(std::memory_order_relaxed);
  if (n > 0) return n;
  if (hipDeviceGetAttribute(&n, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess || n <= 0) {
    (void)hipGetLastError();
    return 256;  // no device: MI355X
  }
  cached[dev].store(n, std::memory_order_relaxed);
  return n;
}

PrefillPlan prefill_plan(int batch, int64_t q_tokens, int64_t k_tokens, int q_heads, int kv_heads, int head_dim, int dtype,
                         int window, int sinks, int flags) {
  PrefillPlan pl{};
  pl.splits = 1;
  pl.rows = 1;
  pl.grid = q_tokens * q_heads;
  const int group = q_heads / kv_heads;
  const int es = dtype == QD_DTYPE_F32 ? 4 : 2;
  if (head_dim * es % 16 != 0 || static_cast<int64_t>(q_heads) * head_dim > (1 << 21) || (flags & QD_FLAG_FORCE_GENERIC))
    return pl;
  const auto grid_of = [&](int rows) { return (q_tokens * group / rows + batch + 1) * kv_heads; };
  pl.dp = es == 4 ? (head_dim <= 64 ? 64 : head_dim <= 128 ? 128 : 256)
                  : (head_dim <= 64 ? 64 : head_dim <= 96 ? 96 : head_dim <= 128 ? 128 : head_dim <= 192 ? 192 : 256);
  // 64 rows per wave where the registers hold two such waves per SIMD, and there are
  // rows for two rounds of workgroups: K and V are read from LDS half as often.
  // Heads of 64 with 32 / 64 rows per wave: 16 prompts of 1000 tokens, 32 heads, 129 /
  // 118 us; one of 8192, 16 heads, 180 / 187 us; one of 4096 63 / 92 us.
  const int rows = es == 2 && pl.dp == 64 && q_tokens * q_heads >= 512 * 512 ? 256 : 128;
  if (grid_of(rows) > INT32_MAX) return pl;
  pl.mfma = true;
  pl.rows = rows;
  pl.grid = grid_of(rows);
  // Few rows with many keys: the items' keys are split until the card has a
  // workgroup for every CU, as long as each keeps 128 keys on average (fp32, eight
  // times slower per key: 64), and two where they fit beside each other (fp32: one
  // after the other), with 256 each.  Items and keys are what static shapes tell: an
  // item per 128 or 256 rows, at least one per sequence; the keys that a sequence's
  // queries see on average.  Below 384 keys the merge's launch costs more than it
  // saves (fp32: 128).  Measured, 32 heads over 8 of 128, bf16: one query over 2000
  // keys 22 -> 14 us, 16 over 30000 557 -> 35 us, 4 x 64 over 8000 158 -> 58 us; 300
  // queries over their own 300 keys would go from 13 to 18 us.  fp32, 16 heads over
  // 4: a prompt of 500 tokens 87 -> 48 us.
  const int64_t items = std::max((q_tokens * group + rows - 1) / rows, std::min<int64_t>(batch, q_tokens)) * kv_heads;
  int64_t keys = std::max<int64_t>(k_tokens - q_tokens / 2, 0) / std::max(batch, 1);
  if (window > 0) keys = std::min(keys, static_cast<int64_t>(window) + sinks + rows / group);
  if (keys < (es == 4 ? 128 : 384)) return pl;
  const int64_t cus = prefill_cu_count(), slots = es == 4 || pl.dp <= 128 ? 2 * cus : cus;
  const int64_t splits = std::min<int64_t>(std::max(std::min(cus / std::max<int64_t>(items, 1), keys / (es == 4 ? 64 : 128)),
                                                    std::min(slots / std::max<int64_t>(items, 1), keys / 256)), 32);
  if (splits >= 2 && pl.grid * splits <= INT32_MAX) {
    pl.splits = static_cast<int>(splits);
    pl.grid *= splits;
    pl.bytes = sizeof(float) * static_cast<size_t>(splits) * q_tokens * q_heads * (head_dim + 4);
  }
  return pl;
}

template <int DT>
void launch_generic(const PrefillParams& p, hipStream_t st) {
  hipLaunchKernelGGL(prefill_generic_kernel<DT>, dim3(static_cast<uint32_t>(p.Tq) * static_cast<uint32_t>(p.Hq)),
                     dim3(256), 0, st, p);
}

}  // namespace

extern "C" {

int qd_gqa_prefill_validate(const qd_tensor_desc* q, const qd_tensor_desc* key, const qd_tensor_desc* value,
                            const qd_tensor_desc* cu, const qd_tensor_desc* cu_k, double scale, int64_t window,
                            int64_t sinks, char* msg, size_t msg_cap) {
  const qd_tensor_desc* all[5] = {q, key, value, cu, cu_k};
  const bool has_k = cu_k && cu_k->defined;
  for (int i = 0; i < (has_k ? 5 : 4); ++i) {
    if (!all[i]) return prefill_fail(msg, msg_cap, "null tensor descriptor");
    if (!all[i]->defined || !all[i]->is_device) return prefill_fail(msg, msg_cap, "all tensors must be CUDA tensors");
    if (all[i]->device_index != q->device_index) return prefill_fail(msg, msg_cap, "all tensors must share a device");
    if (!all[i]->contiguous)
      return prefill_fail(msg, msg_cap,
                          i < 3 ? "the heads of a token must be contiguous in q, key and value"
                                : "cu_seqlens must be contiguous");
  }
  if (q->ndim != 3) return prefill_fail(msg, msg_cap, "q must be [Tq, Hq, D]");
  if (key->ndim != 3) return prefill_fail(msg, msg_cap, "key/value must be [Tk, Hkv, D]");
  for (int i = 0; i < 3; ++i)
    if (value->ndim != 3 || value->sizes[i] != key->sizes[i])
      return prefill_fail(msg, msg_cap, "key/value must be [Tk, Hkv, D]");
  if (key->sizes[2] != q->sizes[2]) return prefill_fail(msg, msg_cap, "q and key head_dim must match");
  if (key->sizes[1] <= 0 || q->sizes[1] <= 0 || q->sizes[1] % key->sizes[1] != 0)
    return prefill_fail(msg, msg_cap, "Hq must be divisible by Hkv");
  if (q->sizes[2] < 1 || q->sizes[2] > 256) return prefill_fail(msg, msg_cap, "supported head_dim is [1, 256]");
  if (!float_dtype(q->dtype)) return prefill_fail(msg, msg_cap, "q/key/value must be float32/float16/bfloat16");
  if (key->dtype != q->dtype || value->dtype != q->dtype)
    return prefill_fail(msg, msg_cap, "q/key/value dtype must match");
  if (cu->ndim != 1 || cu->dtype != QD_DTYPE_I32 || cu->sizes[0] < 1)
    return prefill_fail(msg, msg_cap, "cu_seqlens must be int32 [B + 1]");
  if (has_k && (cu_k->ndim != 1 || cu_k->dtype != QD_DTYPE_I32 || cu_k->sizes[0] != cu->sizes[0]))
    return prefill_fail(msg, msg_cap, "cu_seqlens_k must be int32 [B + 1]");
  if (!has_k && key->sizes[0] != q->sizes[0])
    return prefill_fail(msg, msg_cap, "without cu_seqlens_k there must be a key for every query");
  if (!(scale > 0.0) || !isfinite(scale)) return prefill_fail(msg, msg_cap, "scale must be positive and finite");
  if (window < 0 || window > 2147483647) return prefill_fail(msg, msg_cap, "window must be in [0, 2^31)");
  if (sinks < 0 || sinks > 2147483647 || (window == 0 && sinks > 0))
    return prefill_fail(msg, msg_cap, "sinks must be in [0, 2^31) and need a window");
  if (cu->sizes[0] > (1 << 24) || key->sizes[0] > 2147483647 - 255 || q->sizes[1] >= (1 << 24) ||
      q->sizes[0] >= (int64_t{1} << 31) / q->sizes[1])
    return prefill_fail(msg, msg_cap, "tensor sizes exceed int32 CUDA launch limits");
  if (msg && msg_cap) msg[0] = '\0';
  return QD_OK;
}

int qd_gqa_prefill_info(int batch, int64_t q_tokens, int64_t k_tokens, int q_heads, int kv_heads, int head_dim,
                        int dtype, int flags, int* workgroups, int* rows) {
  if (!prefill_shape_ok(batch, q_tokens, k_tokens, q_heads, kv_heads, head_dim, dtype)) return -1;
  const PrefillPlan pl = prefill_plan(batch, q_tokens, k_tokens, q_heads, kv_heads, head_dim, dtype, 0, 0, flags);
  if (workgroups) *workgroups = static_cast<int>(pl.grid);
  if (rows) *rows = pl.rows;
  return pl.mfma ? QD_PREFILL_MFMA : QD_PREFILL_VALU;
}

size_t qd_gqa_prefill_workspace_bytes(int batch, int64_t q_tokens, int64_t k_tokens, int q_heads, int kv_heads,
                                      int head_dim, int dtype, int window, int sinks, int flags) {
  if (!prefill_shape_ok(batch, q_tokens, k_tokens, q_heads, kv_heads, head_dim, dtype) || window < 0 || sinks < 0) return 0;
  return prefill_plan(batch, q_tokens, k_tokens, q_heads, kv_heads, head_dim, dtype, window, sinks, flags).bytes;
}

int qd_gqa_prefill(const void* q, const void* key, const void* value, const int32_t* cu, const int32_t* cu_k,
                   void* out, void* workspace, size_t workspace_bytes, int batch, int64_t q_tokens, int64_t k_tokens,
                   int q_heads, int kv_heads, int head_dim, int64_t q_stride, int64_t k_stride, int64_t v_stride,
                   int dtype, float scale, int window, int sinks, int flags, void* stream) {
  if (!prefill_shape_ok(batch, q_tokens, k_tokens, q_heads, kv_heads, head_dim, dtype) || q_stride < 0 ||
      k_stride < 0 || v_stride < 0 || (!cu_k && k_tokens != q_tokens))
    return prefill_fail(nullptr, 0, "invalid dimensions");
  if (!(scale > 0.f) || !isfinite(scale)) return prefill_fail(nullptr, 0, "scale must be positive and finite");
  if (window < 0 || sinks < 0 || (window == 0 && sinks > 0))
    return prefill_fail(nullptr, 0, "sinks must not be negative and need a window");
  if (q_tokens == 0) return QD_OK;
  if (!q || !cu || !out || (k_tokens > 0 && (!key || !value))) return prefill_fail(nullptr, 0, "null tensor pointer");
  const int64_t es = dtype == QD_DTYPE_F32 ? 4 : 2;
  // The matrix-core kernel loads 16 bytes at a time, at 32-bit offsets within a
  // tile of at most 256 tokens.
  if (((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(key) | reinterpret_cast<uintptr_t>(value) |
        reinterpret_cast<uintptr_t>(out) | static_cast<uintptr_t>(q_stride * es) |
        static_cast<uintptr_t>(k_stride * es) | static_cast<uintptr_t>(v_stride * es)) &
       15u) != 0 ||
      std::max({q_stride, k_stride, v_stride}) > (int64_t{1} << 21))
    flags |= QD_FLAG_FORCE_GENERIC;
  const PrefillPlan pl =
      prefill_plan(batch, q_tokens, k_tokens, q_heads, kv_heads, head_dim, dtype, window, sinks, flags);
  // Threads of a launch are counted in 32 bits.
  if (pl.grid >= (1 << 24)) return prefill_fail(nullptr, 0, "tensor sizes exceed int32 CUDA launch limits");
  if (pl.bytes > 0 && (!workspace || workspace_bytes < pl.bytes || (reinterpret_cast<uintptr_t>(workspace) & 15u)))
    return prefill_fail(nullptr, 0, "workspace too small or not 16-byte aligned");
  PrefillParams p;
  p.q = q;
  p.k = key;
  p.v = value;
  p.cu = cu;
  p.cu_k = cu_k ? cu_k : cu;
  p.out = out;
  p.q_stride = q_stride;
  p.k_stride = k_stride;
  p.v_stride = v_stride;
  p.B = batch;
  p.Tq = static_cast<int>(q_tokens);
  p.Tk = static_cast<int>(k_tokens);
  p.Hq = q_heads;
  p.Hkv = kv_heads;
  p.D = head_dim;
  p.G = q_heads / kv_heads;
  p.window = window;
  p.sinks = sinks;
  p.sl2 = scale * kLog2e;
  p.inv_g = 1.f / static_cast<float>(p.G);
  p.by_g = packed_divide_by(static_cast<uint32_t>(p.G));
  p.by_hkv = packed_divide_by(static_cast<uint32_t>(kv_heads));
  p.groups = pl.mfma ? static_cast<int>(pl.grid / pl.splits / kv_heads) : 0;
  p.splits = pl.splits;
  p.by_splits = packed_divide_by(static_cast<uint32_t>(pl.splits));
  p.part = static_cast<float*>(workspace);
  hipStream_t st = static_cast<hipStream_t>(stream);
  (void)hipGetLastError();
  hipError_t e = hipSuccess;
  if (pl.mfma) {
    const auto run = dtype == QD_DTYPE_F32   ? qd_prefill_mfma_launch_f32
                     : dtype == QD_DTYPE_F16 ? qd_prefill_mfma_launch_f16
                                             : qd_prefill_mfma_launch_bf16;
    e = static_cast<hipError_t>(run(p, pl.dp, pl.rows, static_cast<uint32_t>(pl.grid), stream));
  } else {
    switch (dtype) {
      case QD_DTYPE_F32: launch_generic<QD_DTYPE_F32>(p, st); break;
      case QD_DTYPE_F16: launch_generic<QD_DTYPE_F16>(p, st); break;
      default: launch_generic<QD_DTYPE_BF16>(p, st); break;
    }
    e = hipGetLastError();
  }
  if (e != hipSuccess) {
    qd_set_last_error(static_cast<int>(e), std::string("gqa_prefill kernel launch failed: ") + hipGetErrorString(e));
    return static_cast<int>(e);
  }
  return QD_OK;
}

}  // extern "C"
