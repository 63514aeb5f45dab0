// Paged grouped-query attention of several drafted tokens per sequence (a
// tree given by ancestor masks), with an optional sliding window and a few
// first tokens that stay visible, for MI355X (gfx950).  One query without a
// mask is windowed decode.  C ABI in include/qd_attention.h.
//
// What a query sees (Row below): context tokens [0, sinks) and [lo, len), and
// the drafted tokens of its mask.  The tokens that it sees without the mask
// are numbered through ("virtual" tokens): v < sinks is token v, the others
// are lo + v - sinks, so tiles of 64 never cover the gap between the first
// tokens and the window.

#include <hip/hip_runtime.h>

#include <math.h>
#include <stdint.h>
#include <string.h>

#include <algorithm>
#include <string>

#include "qd_attention.h"
#include "qd_device.h"

void qd_set_last_error(int status, const std::string& msg);

namespace {

struct TreeParams {
  const void* q;
  const void* k;
  const void* v;
  const int32_t* table;
  const int32_t* lens;
  const int64_t* mask;  // null: one query per sequence, the last of its tokens
  void* out;
  float* part;          // partials of split contexts
  int B, T, Hq, Hkv, D, P, maxP;
  int64_t num_blocks;
  int window, sinks;
  float sl2;  // scale * log2(e)
  int splits;
};

// Tokens of sequence b in its table.
__device__ __forceinline__ int context_len(const TreeParams& p, int b) {
  const int64_t cap = static_cast<int64_t>(p.maxP) * p.P;
  const int64_t len = max(p.lens[b], 0);
  return static_cast<int>(len < cap ? len : cap);
}

__device__ __forceinline__ uint64_t draft_bits(const TreeParams& p, int b, int t) {
  const uint64_t m = static_cast<uint64_t>(p.mask[static_cast<int64_t>(b) * p.T + t]);
  return p.T >= 64 ? m : m & ((uint64_t{1} << p.T) - 1);
}

// What query t of sequence b sees: context tokens [0, sinks) and [lo, len),
// sinks <= lo <= len, and drafted token j (token len + j) where bit j of `seen`
// is set.
struct Row {
  int len, lo, sinks;
  uint64_t seen;
};

__device__ __forceinline__ Row row_view(const TreeParams& p, int b, int t) {
  Row r;
  r.len = context_len(p, b);
  r.seen = 0;
  int depth = -1;
  if (p.mask) {
    const uint64_t m = draft_bits(p, b, t);
    if (m == 0) {  // padding
      r.len = r.lo = r.sinks = 0;
      return r;
    }
    depth = __builtin_popcountll(m) - 1;
    // Drafted tokens past the table are not seen.
    const int64_t room = static_cast<int64_t>(p.maxP) * p.P - r.len;
    r.seen = room >= 64 ? m : room > 0 ? m & ((uint64_t{1} << room) - 1) : 0;
    // The window hides drafted tokens only where it is shorter than a path.
    if (p.window > 0 && p.window <= depth + 1)
      for (uint64_t left = r.seen; left; left &= left - 1) {
        const int j = __builtin_ctzll(left);
        const int dj = __builtin_popcountll(draft_bits(p, b, j)) - 1;
        if (dj <= depth - p.window && r.len + static_cast<int64_t>(dj) >= p.sinks) r.seen &= ~(uint64_t{1} << j);
      }
  }
  int64_t lo = p.window > 0 ? static_cast<int64_t>(r.len) + depth - p.window + 1 : 0;
  lo = lo < 0 ? 0 : lo;
  r.lo = static_cast<int>(lo < r.len ? lo : r.len);
  r.sinks = min(p.sinks, r.lo);
  return r;
}

// Pool row of token `tok`; page ids are clamped to the pool.
__device__ __forceinline__ int64_t pool_row(const TreeParams& p, int b, int tok) {
  const int page = tok / p.P;
  int64_t phys = p.table[static_cast<int64_t>(b) * p.maxP + page];
  phys = phys < 0 ? 0 : phys >= p.num_blocks ? p.num_blocks - 1 : phys;
  return phys * p.P + (tok - page * p.P);
}

// Any head_dim, alignment and type, on the VALU: a workgroup per (query head,
// split); its four waves take 64-token blocks in turn, a lane per token for
// the scores and a lane per 64th column for the values.  Tokens that the query
// does not see are not read at all.
// grid (B * T * Hq, splits), block 256.
template <int DT>
__global__ __launch_bounds__(256) void tree_generic_kernel(TreeParams p) {
  using E = Elem<DT>;
  using S = typename E::S;
  __shared__ float qs[256];
  __shared__ float weight[4][64];
  __shared__ int64_t rows[4][64];
  __shared__ float acc_s[4][256];
  __shared__ float ml_s[4][2];
  const int tid = static_cast<int>(threadIdx.x), lane = tid & 63, wv = tid >> 6;
  const int64_t row = blockIdx.x;
  const int hq = static_cast<int>(row % p.Hq);
  const int64_t bt = row / p.Hq;
  const int b = static_cast<int>(bt / p.T), t = static_cast<int>(bt % p.T);
  const int h = hq / (p.Hq / p.Hkv);
  const S* q = static_cast<const S*>(p.q) + row * p.D;
  for (int d = tid; d < p.D; d += 256) qs[d] = E::to_f(q[d]);
  const Row r = row_view(p, b, t);
  __syncthreads();
  const int drafts = r.seen ? 64 - __builtin_clzll(r.seen) : 0;
  const int context = r.sinks + r.len - r.lo;
  const int blocks = (context + drafts + 63) / 64;
  const int s = static_cast<int>(blockIdx.y);
  const int first = static_cast<int>(static_cast<int64_t>(blocks) * s / p.splits);
  const int last = static_cast<int>(static_cast<int64_t>(blocks) * (s + 1) / p.splits);
  float m = -INFINITY, l = 0.f, acc[4] = {0.f, 0.f, 0.f, 0.f};
  for (int blk = first + wv; blk < last; blk += 4) {
    const int v = 64 * blk + lane;
    const int tok = v < r.sinks ? v : r.lo + (v - r.sinks);
    const bool seen = v < context || (v - context < drafts && ((r.seen >> (v - context)) & 1));
    float x = -INFINITY;
    int64_t at = 0;
    if (seen) {
      at = (pool_row(p, b, tok) * p.Hkv + h) * p.D;
      const S* k = static_cast<const S*>(p.k) + at;
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
    rows[wv][lane] = seen ? at : -1;
    __builtin_amdgcn_wave_barrier();
    for (int j = 0; j < 64; ++j) {
      const int64_t vr = rows[wv][j];
      if (vr < 0) continue;
      const float wj = weight[wv][j];
      const S* val = static_cast<const S*>(p.v) + vr;
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
__global__ __launch_bounds__(256) void tree_combine_kernel(TreeParams p) {
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

int tree_fail(char* msg, size_t cap, const char* text) {
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

bool tree_shape_ok(int batch, int q_len, int q_heads, int kv_heads, int head_dim, int block_size, int max_pages,
                   int has_mask, int window, int sinks, int dtype) {
  return batch >= 0 && q_len >= 1 && q_len <= QD_TREE_MAX_DRAFTS && (has_mask || q_len == 1) && q_heads > 0 &&
         kv_heads > 0 && q_heads % kv_heads == 0 && head_dim >= 1 && head_dim <= 256 && block_size > 0 &&
         max_pages > 0 && window >= 0 && sinks >= 0 && (window > 0 || sinks == 0) && float_dtype(dtype) &&
         static_cast<int64_t>(batch) * q_len * q_heads < (1 << 24);
}

// The most tokens that a query of the batch can see.
int64_t visible_capacity(int q_len, int block_size, int max_pages, int has_mask, int window, int sinks) {
  const int64_t cap = static_cast<int64_t>(block_size) * max_pages;
  if (window <= 0) return cap;
  return std::min(cap, static_cast<int64_t>(window) + sinks + (has_mask ? q_len : 0));
}

// Context splits of the VALU kernel: enough workgroups to fill the card, at
// least 512 tokens each.
int generic_splits(int batch, int q_len, int q_heads, int64_t capacity) {
  const int64_t rows = std::max<int64_t>(1, static_cast<int64_t>(batch) * q_len * q_heads);
  const int64_t want = (2048 + rows - 1) / rows;
  return static_cast<int>(std::max<int64_t>(1, std::min({want, (capacity + 511) / 512, int64_t{64}})));
}

template <int DT>
void launch_generic(const TreeParams& p, hipStream_t st) {
  const uint32_t rows = static_cast<uint32_t>(p.B * p.T * p.Hq);
  hipLaunchKernelGGL(tree_generic_kernel<DT>, dim3(rows, static_cast<uint32_t>(p.splits)), dim3(256), 0, st, p);
  if (p.splits > 1) hipLaunchKernelGGL(tree_combine_kernel<DT>, dim3(rows), dim3(256), 0, st, p);
}

}  // namespace

extern "C" {

int qd_gqa_decode_tree_validate(const qd_tensor_desc* q, const qd_tensor_desc* k_cache,
                                const qd_tensor_desc* v_cache, const qd_tensor_desc* block_table,
                                const qd_tensor_desc* context_lens, const qd_tensor_desc* tree_mask, double scale,
                                int64_t window, int64_t sinks, char* msg, size_t msg_cap) {
  const qd_tensor_desc* all[6] = {q, k_cache, v_cache, block_table, context_lens, tree_mask};
  static const char* const device_text[6] = {
      "q must be a CUDA tensor",           "k_cache must be a CUDA tensor",      "v_cache must be a CUDA tensor",
      "block_table must be a CUDA tensor", "context_lens must be a CUDA tensor", "tree_mask must be a CUDA tensor"};
  static const char* const contiguous_text[6] = {
      "q must be contiguous",           "k_cache must be contiguous",      "v_cache must be contiguous",
      "block_table must be contiguous", "context_lens must be contiguous", "tree_mask must be contiguous"};
  const bool tree = tree_mask && tree_mask->defined;
  for (int i = 0; i < 6; ++i) {
    if (i == 5 && !tree) break;
    if (!all[i]) return tree_fail(msg, msg_cap, "null tensor descriptor");
    if (!all[i]->defined || !all[i]->is_device) return tree_fail(msg, msg_cap, device_text[i]);
    if (!all[i]->contiguous) return tree_fail(msg, msg_cap, contiguous_text[i]);
  }
  const int heads = tree ? 2 : 1;
  if (q->ndim != heads + 2) return tree_fail(msg, msg_cap, tree ? "q must be [B, T, Hq, D]" : "q must be [B, Hq, D]");
  if (k_cache->ndim != 4) return tree_fail(msg, msg_cap, "k_cache must be [Nblocks, BlockSize, Hkv, D]");
  if (v_cache->ndim != 4) return tree_fail(msg, msg_cap, "v_cache shape mismatch");
  for (int i = 0; i < 4; ++i)
    if (v_cache->sizes[i] != k_cache->sizes[i]) return tree_fail(msg, msg_cap, "v_cache shape mismatch");
  if (block_table->ndim != 2) return tree_fail(msg, msg_cap, "block_table must be [B, MaxPages]");
  if (context_lens->ndim != 1) return tree_fail(msg, msg_cap, "context_lens must be [B]");
  if (tree && (tree_mask->ndim != 2 || tree_mask->dtype != QD_DTYPE_I64 || tree_mask->sizes[0] != q->sizes[0] ||
               tree_mask->sizes[1] != q->sizes[1]))
    return tree_fail(msg, msg_cap, "tree_mask must be int64 [B, T]");
  for (int i = 0; i < (tree ? 6 : 5); ++i)
    if (all[i]->device_index != q->device_index)
      return tree_fail(msg, msg_cap, "all tensors must use one CUDA device");
  if (k_cache->dtype != q->dtype || v_cache->dtype != q->dtype)
    return tree_fail(msg, msg_cap, "q/k/v dtype must match");
  if (!float_dtype(q->dtype)) return tree_fail(msg, msg_cap, "q/k/v must be float32/float16/bfloat16");
  if (block_table->dtype != QD_DTYPE_I32 || context_lens->dtype != QD_DTYPE_I32)
    return tree_fail(msg, msg_cap, "block_table and context_lens must be int32");
  if (block_table->sizes[0] != q->sizes[0] || context_lens->sizes[0] != q->sizes[0])
    return tree_fail(msg, msg_cap, "batch sizes must match");
  if (tree && (q->sizes[1] < 1 || q->sizes[1] > QD_TREE_MAX_DRAFTS))
    return tree_fail(msg, msg_cap, "supported drafted tokens per sequence are [1, 64]");
  if (q->sizes[heads + 1] != k_cache->sizes[3])
    return tree_fail(msg, msg_cap, "q head_dim and cache head_dim must match");
  if (k_cache->sizes[2] <= 0 || q->sizes[heads] <= 0 || q->sizes[heads] % k_cache->sizes[2] != 0)
    return tree_fail(msg, msg_cap, "Hq must be divisible by Hkv");
  if (q->sizes[heads + 1] < 1 || q->sizes[heads + 1] > 256)
    return tree_fail(msg, msg_cap, "supported head_dim is [1, 256]");
  if (k_cache->sizes[0] <= 0 || k_cache->sizes[1] <= 0)
    return tree_fail(msg, msg_cap, "cache must have positive blocks and block_size");
  if (block_table->sizes[1] <= 0) return tree_fail(msg, msg_cap, "block_table must have at least one page");
  if (!(scale > 0.0) || !isfinite(scale)) return tree_fail(msg, msg_cap, "scale must be positive and finite");
  if (window < 0 || window > 2147483647 || (!tree && window == 0))
    return tree_fail(msg, msg_cap, "window must be in [1, 2^31)");
  if (sinks < 0 || sinks > 2147483647 || (window == 0 && sinks > 0))
    return tree_fail(msg, msg_cap, "sinks must be in [0, 2^31) and need a window");
  const int64_t rows_per_seq = (tree ? q->sizes[1] : 1) * q->sizes[heads];
  if (q->sizes[heads] >= (1 << 24) || k_cache->sizes[1] > 2147483647 || block_table->sizes[1] > 2147483647 ||
      q->sizes[0] > (1 << 24) || q->sizes[0] * rows_per_seq >= (1 << 24))
    return tree_fail(msg, msg_cap, "tensor sizes exceed int32 CUDA launch limits");
  if (msg && msg_cap) msg[0] = '\0';
  return QD_OK;
}

size_t qd_gqa_decode_tree_workspace_bytes(int batch, int q_len, int q_heads, int kv_heads, int head_dim,
                                          int block_size, int max_pages, int has_mask, int window, int sinks,
                                          int dtype, int flags) {
  (void)flags;
  if (!tree_shape_ok(batch, q_len, q_heads, kv_heads, head_dim, block_size, max_pages, has_mask, window, sinks, dtype))
    return 0;
  const int splits =
      generic_splits(batch, q_len, q_heads, visible_capacity(q_len, block_size, max_pages, has_mask, window, sinks));
  if (splits == 1) return 0;
  return sizeof(float) * static_cast<size_t>(batch) * q_len * q_heads * splits * (head_dim + 2);
}

int qd_gqa_decode_tree_info(int batch, int q_len, int q_heads, int kv_heads, int head_dim, int block_size,
                            int max_pages, int has_mask, int window, int sinks, int dtype, int flags,
                            int* workgroups, int* rows) {
  (void)flags;
  if (!tree_shape_ok(batch, q_len, q_heads, kv_heads, head_dim, block_size, max_pages, has_mask, window, sinks, dtype))
    return -1;
  if (workgroups)
    *workgroups = batch * q_len * q_heads *
                  generic_splits(batch, q_len, q_heads,
                                 visible_capacity(q_len, block_size, max_pages, has_mask, window, sinks));
  if (rows) *rows = 1;
  return QD_TREE_VALU;
}

int qd_gqa_decode_tree(const void* q, const void* k_cache, const void* v_cache, const int32_t* block_table,
                       const int32_t* context_lens, const int64_t* tree_mask, void* out, void* workspace,
                       size_t workspace_bytes, int batch, int q_len, int q_heads, int kv_heads, int head_dim,
                       int block_size, int max_pages, int64_t num_blocks, int dtype, float scale, int window,
                       int sinks, int flags, void* stream) {
  const int has_mask = tree_mask != nullptr;
  if (!tree_shape_ok(batch, q_len, q_heads, kv_heads, head_dim, block_size, max_pages, has_mask, window, sinks,
                     dtype) ||
      num_blocks <= 0 || (!has_mask && window == 0))
    return tree_fail(nullptr, 0, "invalid dimensions");
  if (!(scale > 0.f) || !isfinite(scale)) return tree_fail(nullptr, 0, "scale must be positive and finite");
  if (batch == 0) return QD_OK;
  if (!q || !k_cache || !v_cache || !block_table || !context_lens || !out)
    return tree_fail(nullptr, 0, "null tensor pointer");
  const size_t need = qd_gqa_decode_tree_workspace_bytes(batch, q_len, q_heads, kv_heads, head_dim, block_size,
                                                         max_pages, has_mask, window, sinks, dtype, flags);
  if (need > 0 && (!workspace || workspace_bytes < need || (reinterpret_cast<uintptr_t>(workspace) & 15u)))
    return tree_fail(nullptr, 0, "workspace too small or not 16-byte aligned");
  TreeParams p;
  p.q = q;
  p.k = k_cache;
  p.v = v_cache;
  p.table = block_table;
  p.lens = context_lens;
  p.mask = tree_mask;
  p.out = out;
  p.part = static_cast<float*>(workspace);
  p.B = batch;
  p.T = q_len;
  p.Hq = q_heads;
  p.Hkv = kv_heads;
  p.D = head_dim;
  p.P = block_size;
  p.maxP = max_pages;
  p.num_blocks = num_blocks;
  p.window = window;
  p.sinks = sinks;
  p.sl2 = scale * kLog2e;
  p.splits =
      generic_splits(batch, q_len, q_heads, visible_capacity(q_len, block_size, max_pages, has_mask, window, sinks));
  hipStream_t st = static_cast<hipStream_t>(stream);
  (void)hipGetLastError();
  switch (dtype) {
    case QD_DTYPE_F32: launch_generic<QD_DTYPE_F32>(p, st); break;
    case QD_DTYPE_F16: launch_generic<QD_DTYPE_F16>(p, st); break;
    default: launch_generic<QD_DTYPE_BF16>(p, st); break;
  }
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) {
    qd_set_last_error(static_cast<int>(e),
                      std::string("gqa_decode_tree kernel launch failed: ") + hipGetErrorString(e));
    return static_cast<int>(e);
  }
  return QD_OK;
}

}  // extern "C"
