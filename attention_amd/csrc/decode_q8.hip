// Paged grouped-query decode over a cache in 8 bits with a scale per page and
// kv-head, for MI355X (gfx950).  C ABI in include/qd_attention.h.

#include <hip/hip_runtime.h>

#include <math.h>
#include <stdint.h>
#include <string.h>

#include <algorithm>
#include <atomic>
#include <string>
#include <type_traits>

#include "qd_device.h"

void qd_set_last_error(int status, const std::string& msg);

namespace {

// Most tokens of a table row: token numbers and the ends of their tiles fit 32
// bits.
constexpr int32_t kQ8Capacity = INT32_MAX - 255;

struct Q8Params {
  const void* q;
  const uint8_t* k;
  const uint8_t* v;
  const float* ks;
  const float* vs;
  const int32_t* table;
  const int32_t* lens;
  void* out;
  float* part;
  int64_t num_blocks;
  int B, Hq, Hkv, D, P, maxP, G;
  int32_t capacity;
  int splits;
  float sl2;  // scale * log2(e)
};

__device__ __forceinline__ int q8_len(const Q8Params& p, int b) { return min(max(p.lens[b], 0), p.capacity); }

template <int KIND>
__device__ __forceinline__ float q8_value(uint8_t x) {
  if constexpr (KIND == QD_DTYPE_E4M3)
    return __builtin_amdgcn_cvt_f32_fp8(static_cast<int>(x), 0);
  else
    return static_cast<float>(static_cast<int8_t>(x));
}

// Any head_dim, page and alignment, on the VALU: a workgroup per (query head,
// split); its four waves take 64 tokens in turn, a lane per token for the scores
// and a lane per 64th column for the values.  For what the matrix-core kernel
// does not take, and as its check.
// grid (B * Hq, splits), block 256.
template <int DT, int KIND>
__global__ __launch_bounds__(256) void q8_generic_kernel(Q8Params p) {
  using E = Elem<DT>;
  using S = typename E::S;
  __shared__ float qs[256];
  __shared__ float weight[4][64];
  __shared__ int64_t rows[4][64];
  __shared__ float acc_s[4][256];
  __shared__ float ml_s[4][2];
  const int tid = static_cast<int>(threadIdx.x), lane = tid & 63, wv = tid >> 6;
  const int64_t row = blockIdx.x;
  const int hq = static_cast<int>(row % p.Hq), b = static_cast<int>(row / p.Hq), h = hq / p.G;
  const S* q = static_cast<const S*>(p.q) + row * p.D;
  for (int d = tid; d < p.D; d += 256) qs[d] = E::to_f(q[d]);
  __syncthreads();
  const int len = q8_len(p, b);
  const int blocks = (len + 63) / 64, s = static_cast<int>(blockIdx.y);
  const int first = static_cast<int>(static_cast<int64_t>(blocks) * s / p.splits);
  const int last = static_cast<int>(static_cast<int64_t>(blocks) * (s + 1) / p.splits);
  float m = -INFINITY, l = 0.f, acc[4] = {0.f, 0.f, 0.f, 0.f};
  for (int blk = first + wv; blk < last; blk += 4) {
    const int tok = 64 * blk + lane;
    const bool seen = tok < len;
    float x = -INFINITY, vscale = 0.f;
    int64_t at = 0;
    if (seen) {
      const int page = tok / p.P;
      const int64_t id = p.table[static_cast<int64_t>(b) * p.maxP + page];
      const int64_t phys = min(max(id, int64_t{0}), p.num_blocks - 1);
      at = ((phys * p.P + (tok - page * p.P)) * p.Hkv + h) * p.D;
      const uint8_t* k = p.k + at;
      float dot = 0.f;
      for (int d = 0; d < p.D; ++d) dot = fmaf(qs[d], q8_value<KIND>(k[d]), dot);
      x = dot * p.ks[phys * p.Hkv + h] * p.sl2;
      vscale = p.vs[phys * p.Hkv + h];
    }
    const float mx = fmaxf(m, wave_max(x));
    const float use = mx == -INFINITY ? 0.f : mx;
    const float alpha = fast_exp2(m - use);  // m = -inf: 0
    const float w = seen ? fast_exp2(x - use) : 0.f;
    m = mx;
    l = l * alpha + wave_sum(w);
    for (int e = 0; e < 4; ++e) acc[e] *= alpha;
    weight[wv][lane] = w * vscale;
    rows[wv][lane] = at;
    __builtin_amdgcn_wave_barrier();
    for (int j = 0; j < min(64, len - 64 * blk); ++j) {
      const float wj = weight[wv][j];
      const uint8_t* val = p.v + rows[wv][j];
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (lane + 64 * e < p.D) acc[e] = fmaf(wj, q8_value<KIND>(val[lane + 64 * e]), acc[e]);
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
    if (p.splits == 1) {
      static_cast<S*>(p.out)[row * p.D + tid] = E::from_f(sum > 0.f || sum != sum ? a / sum : 0.f);
    } else {
      float* part = p.part + (row * p.splits + s) * (p.D + 2);
      part[2 + tid] = a;
      if (tid == 0) {
        part[0] = mx;
        part[1] = sum;
      }
    }
  }
}

// Log-sum-exp merge of [row][split]{m, l, acc[D]}.  grid rows, block 256.
template <int DT>
__global__ __launch_bounds__(256) void q8_combine_kernel(Q8Params p) {
  using E = Elem<DT>;
  const int64_t row = blockIdx.x;
  const float* part = p.part + row * p.splits * (p.D + 2);
  float mx = -INFINITY;
  for (int s = 0; s < p.splits; ++s) mx = fmaxf(mx, part[s * (p.D + 2)]);
  const float use = mx == -INFINITY ? 0.f : mx;
  const int d = static_cast<int>(threadIdx.x);
  if (d >= p.D) return;
  float sum = 0.f, a = 0.f;
  for (int s = 0; s < p.splits; ++s) {
    const float* x = part + s * (p.D + 2);
    const float f = fast_exp2(x[0] - use);
    sum += f * x[1];
    a += f * x[2 + d];
  }
  static_cast<typename E::S*>(p.out)[row * p.D + d] = E::from_f(sum > 0.f || sum != sum ? a / sum : 0.f);
}

int q8_fail(char* msg, size_t cap, const char* text) {
  qd_set_last_error(QD_ERR_INVALID_VALUE, text);
  if (msg && cap) {
    size_t n = strlen(text);
    if (n >= cap) n = cap - 1;
    memcpy(msg, text, n);
    msg[n] = '\0';
  }
  return QD_ERR_INVALID_VALUE;
}

bool q8_shape_ok(int batch, int q_heads, int kv_heads, int head_dim, int block_size, int max_pages, int dtype) {
  return batch >= 0 && batch < (1 << 24) && q_heads > 0 && q_heads < (1 << 24) && kv_heads > 0 &&
         q_heads % kv_heads == 0 && head_dim >= 1 && head_dim <= 256 && block_size > 0 && max_pages > 0 &&
         (dtype == QD_DTYPE_F16 || dtype == QD_DTYPE_BF16) && static_cast<int64_t>(batch) * q_heads < (1 << 24);
}

int64_t q8_capacity(int block_size, int max_pages) {
  return std::min<int64_t>(static_cast<int64_t>(block_size) * max_pages, kQ8Capacity);
}

// Context splits of the VALU kernel: enough workgroups to fill the card, at
// least 512 tokens each.
int generic_splits(int batch, int q_heads, int64_t capacity) {
  const int64_t rows = std::max<int64_t>(1, static_cast<int64_t>(batch) * q_heads);
  const int64_t want = (2048 + rows - 1) / rows;
  return static_cast<int>(std::max<int64_t>(1, std::min({want, (capacity + 511) / 512, int64_t{64}})));
}

struct Q8Plan {
  int splits;  // VALU kernel
  size_t bytes;
};

Q8Plan q8_plan(int batch, int q_heads, int head_dim, int block_size, int max_pages) {
  Q8Plan pl{};
  pl.splits = generic_splits(batch, q_heads, q8_capacity(block_size, max_pages));
  if (pl.splits > 1) pl.bytes = sizeof(float) * static_cast<size_t>(batch) * q_heads * pl.splits * (head_dim + 2);
  return pl;
}

template <int DT>
void launch_generic(const Q8Params& p, int cache_dtype, hipStream_t st) {
  const uint32_t rows = static_cast<uint32_t>(p.B * p.Hq);
  const dim3 grid(rows, static_cast<uint32_t>(p.splits));
  if (cache_dtype == QD_DTYPE_E4M3)
    hipLaunchKernelGGL((q8_generic_kernel<DT, QD_DTYPE_E4M3>), grid, dim3(256), 0, st, p);
  else
    hipLaunchKernelGGL((q8_generic_kernel<DT, QD_DTYPE_I8>), grid, dim3(256), 0, st, p);
  if (p.splits > 1) hipLaunchKernelGGL(q8_combine_kernel<DT>, dim3(rows), dim3(256), 0, st, p);
}

}  // namespace

extern "C" {

int qd_gqa_decode_q8_validate(const qd_tensor_desc* q, const qd_tensor_desc* k_cache, const qd_tensor_desc* v_cache,
                              const qd_tensor_desc* k_scales, const qd_tensor_desc* v_scales,
                              const qd_tensor_desc* block_table, const qd_tensor_desc* context_lens, double scale,
                              char* msg, size_t msg_cap) {
  const qd_tensor_desc* all[7] = {q, k_cache, v_cache, k_scales, v_scales, block_table, context_lens};
  static const char* const device_text[7] = {
      "q must be a CUDA tensor",        "k_cache must be a CUDA tensor",  "v_cache must be a CUDA tensor",
      "k_scales must be a CUDA tensor", "v_scales must be a CUDA tensor", "block_table must be a CUDA tensor",
      "context_lens must be a CUDA tensor"};
  static const char* const contiguous_text[7] = {
      "q must be contiguous",        "k_cache must be contiguous",  "v_cache must be contiguous",
      "k_scales must be contiguous", "v_scales must be contiguous", "block_table must be contiguous",
      "context_lens must be contiguous"};
  for (int i = 0; i < 7; ++i) {
    if (!all[i]) return q8_fail(msg, msg_cap, "null tensor descriptor");
    if (!all[i]->defined || !all[i]->is_device) return q8_fail(msg, msg_cap, device_text[i]);
    if (!all[i]->contiguous) return q8_fail(msg, msg_cap, contiguous_text[i]);
  }
  if (q->ndim != 3) return q8_fail(msg, msg_cap, "q must be [B, Hq, D]");
  if (k_cache->ndim != 4) return q8_fail(msg, msg_cap, "k_cache must be [Nblocks, BlockSize, Hkv, D]");
  if (v_cache->ndim != 4) return q8_fail(msg, msg_cap, "v_cache shape mismatch");
  for (int i = 0; i < 4; ++i)
    if (v_cache->sizes[i] != k_cache->sizes[i]) return q8_fail(msg, msg_cap, "v_cache shape mismatch");
  for (const qd_tensor_desc* s : {k_scales, v_scales})
    if (s->ndim != 2 || s->dtype != QD_DTYPE_F32 || s->sizes[0] != k_cache->sizes[0] || s->sizes[1] != k_cache->sizes[2])
      return q8_fail(msg, msg_cap, "scales must be float32 [Nblocks, Hkv]");
  if (block_table->ndim != 2) return q8_fail(msg, msg_cap, "block_table must be [B, MaxPages]");
  if (context_lens->ndim != 1) return q8_fail(msg, msg_cap, "context_lens must be [B]");
  for (int i = 0; i < 7; ++i)
    if (all[i]->device_index != q->device_index)
      return q8_fail(msg, msg_cap, "all tensors must use one CUDA device");
  if (q->dtype != QD_DTYPE_F16 && q->dtype != QD_DTYPE_BF16)
    return q8_fail(msg, msg_cap, "q must be float16/bfloat16");
  if ((k_cache->dtype != QD_DTYPE_E4M3 && k_cache->dtype != QD_DTYPE_I8) || v_cache->dtype != k_cache->dtype)
    return q8_fail(msg, msg_cap, "caches must both be float8_e4m3fn or int8");
  if (block_table->dtype != QD_DTYPE_I32 || context_lens->dtype != QD_DTYPE_I32)
    return q8_fail(msg, msg_cap, "block_table and context_lens must be int32");
  if (block_table->sizes[0] != q->sizes[0] || context_lens->sizes[0] != q->sizes[0])
    return q8_fail(msg, msg_cap, "batch sizes must match");
  if (q->sizes[2] != k_cache->sizes[3]) return q8_fail(msg, msg_cap, "q head_dim and cache head_dim must match");
  if (k_cache->sizes[2] <= 0 || q->sizes[1] <= 0 || q->sizes[1] % k_cache->sizes[2] != 0)
    return q8_fail(msg, msg_cap, "Hq must be divisible by Hkv");
  if (q->sizes[2] < 1 || q->sizes[2] > 256) return q8_fail(msg, msg_cap, "supported head_dim is [1, 256]");
  if (k_cache->sizes[0] <= 0 || k_cache->sizes[1] <= 0)
    return q8_fail(msg, msg_cap, "cache must have positive blocks and block_size");
  if (block_table->sizes[1] <= 0) return q8_fail(msg, msg_cap, "block_table must have at least one page");
  if (!(scale > 0.0) || !isfinite(scale)) return q8_fail(msg, msg_cap, "scale must be positive and finite");
  if (q->sizes[1] >= (1 << 24) || q->sizes[0] >= (1 << 24) || q->sizes[0] * q->sizes[1] >= (1 << 24) ||
      k_cache->sizes[0] > 2147483647 || k_cache->sizes[1] > 2147483647 || block_table->sizes[1] > 2147483647)
    return q8_fail(msg, msg_cap, "tensor sizes exceed int32 CUDA launch limits");
  if (msg && msg_cap) msg[0] = '\0';
  return QD_OK;
}

size_t qd_gqa_decode_q8_workspace_bytes(int batch, int q_heads, int kv_heads, int head_dim, int block_size,
                                        int max_pages, int dtype, int flags) {
  (void)flags;
  if (!q8_shape_ok(batch, q_heads, kv_heads, head_dim, block_size, max_pages, dtype) || batch == 0) return 0;
  return q8_plan(batch, q_heads, head_dim, block_size, max_pages).bytes;
}

int qd_gqa_decode_q8_info(int batch, int q_heads, int kv_heads, int head_dim, int block_size, int max_pages,
                          int dtype, int flags, int* workgroups) {
  (void)flags;
  if (!q8_shape_ok(batch, q_heads, kv_heads, head_dim, block_size, max_pages, dtype)) return -1;
  if (workgroups) *workgroups = batch * q_heads * q8_plan(batch, q_heads, head_dim, block_size, max_pages).splits;
  return QD_Q8_VALU;
}

int qd_gqa_decode_q8(const void* q, const void* k_cache, const void* v_cache, const float* k_scales,
                     const float* v_scales, const int32_t* block_table, const int32_t* context_lens, void* out,
                     void* workspace, size_t workspace_bytes, int batch, int q_heads, int kv_heads, int head_dim,
                     int block_size, int max_pages, int64_t num_blocks, int dtype, int cache_dtype, float scale,
                     int flags, void* stream) {
  (void)flags;
  if (!q8_shape_ok(batch, q_heads, kv_heads, head_dim, block_size, max_pages, dtype) || num_blocks <= 0 ||
      num_blocks > INT32_MAX || (cache_dtype != QD_DTYPE_E4M3 && cache_dtype != QD_DTYPE_I8))
    return q8_fail(nullptr, 0, "invalid dimensions");
  if (!(scale > 0.f) || !isfinite(scale)) return q8_fail(nullptr, 0, "scale must be positive and finite");
  if (batch == 0) return QD_OK;
  if (!q || !k_cache || !v_cache || !k_scales || !v_scales || !block_table || !context_lens || !out)
    return q8_fail(nullptr, 0, "null tensor pointer");
  const Q8Plan pl = q8_plan(batch, q_heads, head_dim, block_size, max_pages);
  if (pl.bytes > 0 && (!workspace || workspace_bytes < pl.bytes || (reinterpret_cast<uintptr_t>(workspace) & 15u)))
    return q8_fail(nullptr, 0, "workspace too small or not 16-byte aligned");
  Q8Params p;
  p.q = q;
  p.k = static_cast<const uint8_t*>(k_cache);
  p.v = static_cast<const uint8_t*>(v_cache);
  p.ks = k_scales;
  p.vs = v_scales;
  p.table = block_table;
  p.lens = context_lens;
  p.out = out;
  p.part = static_cast<float*>(workspace);
  p.num_blocks = num_blocks;
  p.B = batch;
  p.Hq = q_heads;
  p.Hkv = kv_heads;
  p.D = head_dim;
  p.P = block_size;
  p.maxP = max_pages;
  p.G = q_heads / kv_heads;
  p.capacity = static_cast<int32_t>(q8_capacity(block_size, max_pages));
  p.splits = pl.splits;
  p.sl2 = scale * kLog2e;
  hipStream_t st = static_cast<hipStream_t>(stream);
  (void)hipGetLastError();
  if (dtype == QD_DTYPE_F16)
    launch_generic<QD_DTYPE_F16>(p, cache_dtype, st);
  else
    launch_generic<QD_DTYPE_BF16>(p, cache_dtype, st);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) {
    qd_set_last_error(static_cast<int>(e), std::string("gqa_decode_q8 kernel launch failed: ") + hipGetErrorString(e));
    return static_cast<int>(e);
  }
  return QD_OK;
}

}  // extern "C"
