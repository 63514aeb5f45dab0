// Paged grouped-query attention of several drafted tokens per sequence (a
// tree given by ancestor masks), with an optional sliding window and a few
// first tokens that stay visible, for MI355X (gfx950).  One query without a
// mask is windowed decode.  C ABI in include/qd_attention.h.
//
// What a query sees (Row below): context tokens [0, sinks) and [lo, len), and
// the drafted tokens of its mask.  The tokens that it sees without the mask
// are numbered through ("virtual" tokens): v < sinks is token v, the others
// are lo + v - sinks, so no tile covers the gap between the first tokens and
// the window.

#include <hip/hip_runtime.h>

#include <math.h>
#include <stdint.h>
#include <string.h>

#include <algorithm>
#include <atomic>
#include <string>

#include "tree_kernels.h"

void qd_set_last_error(int status, const std::string& msg);

namespace {

// Any head_dim, alignment and type, on the VALU: a workgroup per (query head,
// split); its four waves take 64-token blocks in turn, a lane per token for
// the scores and a lane per 64th column for the values.  Tokens that the query
// does not see are not read at all.  For what the matrix-core kernel does not
// take, and as its check: it reads K and V once per query and head, a lane a
// whole row (8 sequences, trees of 64, 64 heads of 128: 33 ms against 270 us;
// trees of 16 over 32 sequences 4.5 ms / 75 us; 4 short windows 17.6 / 9.5 us).
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
  const Row r = row_view(p, b, context_len(p, b), p.mask ? draft_bits(p, b, t) : 0);
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
         batch < (1 << 24) && q_heads < (1 << 24) &&  // each, so that the product fits 64 bits
         static_cast<int64_t>(batch) * q_len * q_heads < (1 << 24);
}

// The most tokens that a query of the batch can see by the width of the table
// and the window: lengths are not known on the host.
int64_t visible_capacity(int q_len, int block_size, int max_pages, int has_mask, int window, int sinks) {
  // As the kernels clamp it: products with the items of a batch fit 64 bits.
  const int64_t cap = std::min<int64_t>(static_cast<int64_t>(block_size) * max_pages, kTreeCapacity);
  if (window <= 0) return cap;
  // Widened to whole groups of 16 tokens at three ends (item_span).
  return std::min(cap, static_cast<int64_t>(window) + sinks + (has_mask ? q_len : 0) + 48);
}

// Context splits of the VALU kernel: enough workgroups to fill the card, at
// least 512 tokens each.
int generic_splits(int batch, int q_len, int q_heads, int64_t capacity) {
  const int64_t rows = std::max<int64_t>(1, static_cast<int64_t>(batch) * q_len * q_heads);
  const int64_t want = (2048 + rows - 1) / rows;
  return static_cast<int>(std::max<int64_t>(1, std::min({want, (capacity + 511) / 512, int64_t{64}})));
}

int tree_cu_count() {
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

// How a call runs.  All from static shapes and the device: without a window, the
// table's width stands for the longest context.  Short contexts in a wide table
// therefore run as long ones would, us with a table of the longest context's
// pages / of 2048 pages of 16: 8 sequences of 489 tokens, 64 drafts x 8 heads of
// 128, 23.7 / 47.5 (rows in chunks of 64 / 256); 122 of up to 115, 20 x 4 heads,
// 14.5 / 24.3; 64 of 100 to 500, 16 x 8 heads, 24.1 / 31.1; one of 300, 24 x 4
// heads of 96, 16.7 / 21.0; 32 of 512 to 4096, 16 x 4 heads on 8 kv-heads, 73.2 /
// 72.5.
struct TreePlan {
  bool mfma;
  int splits;                                  // VALU kernel
  int dp, chunks, chunk_rows, W, grid;         // matrix-core kernel
  size_t meta_bytes, bytes;
};

// One workgroup per item, without a merge, or the items' tiles cut into equal
// ranges, one per resident workgroup, with a merge kernel (about 5 us, and a
// start of 4 tiles for every item that a range begins)?  By what is left idle
// if every context fills its table or window, in units of 64 tokens with rows
// of 256 bytes per resident workgroup (longer rows count as more units: fp32,
// 22 items of 230 tokens x 256, 25.5 us in ranges, 38.3 us whole), and by how
// uneven contexts without a window can be.  bf16, 8 kv-heads of 128, one
// workgroup per item against equal ranges, us:
// 512 items of 18 units (a window of 1024) 48.6 / 54.6, 320 of them 40.0 / 38.9,
// 128 of them 32.7 / 25.1; 1024 items of 9 units 56.4 / 60.1, 1600 of them 98 /
// 93.6; without a window, 512 items of 2 to 16 units 40.5 / 52.6, 1024 items of
// 2 to 32 units 126 / 115, 256 items of 8 to 64 units 107 / 77.
constexpr int kTreeIdleUnits = 5;
constexpr int kTreeUnevenUnits = 20;

// Up to 128 rows run as two chunks on four waves each, rather than as one on
// eight, while the table (or the window) holds at most this many tokens.  Two chunks / one, us: 80
// rows, 122 sequences of up to 115 tokens 64.1 / 84.9; 128 rows, 64 sequences of
// 100 to 500 tokens 53.5 / 60.7; 80 rows, 32 sequences of 1000 to 3000 98.9 /
// 96.2; 128 rows, 8 sequences of 2000 to 8000 76.5 / 72.1; heads of 64, 96 rows,
// 16 sequences of 2000 to 8000 66.4 / 58.0.
constexpr int64_t kTreeShortContext = 1024;

bool tree_direct(int64_t items, int64_t units, int64_t resident, bool windowed) {
  const int64_t rounds = (items + resident - 1) / resident;
  if (!windowed && rounds * units > kTreeUnevenUnits) return false;
  return rounds * units * resident - items * units <= kTreeIdleUnits * resident;
}

TreePlan tree_plan(int batch, int q_len, int q_heads, int kv_heads, int head_dim, int block_size, int max_pages,
                   int has_mask, int window, int sinks, int dtype, int flags) {
  TreePlan pl{};
  const int64_t cap = visible_capacity(q_len, block_size, max_pages, has_mask, window, sinks);
  // The matrix-core kernel's page and row offsets are 32 bits wide.
  pl.mfma = head_dim % 8 == 0 && !(flags & QD_FLAG_FORCE_GENERIC) &&
            static_cast<int64_t>(kv_heads) * head_dim * 4 <= INT32_MAX / std::max(block_size, 16);
  if (!pl.mfma) {
    pl.splits = generic_splits(batch, q_len, q_heads, cap);
    if (pl.splits > 1)
      pl.bytes = sizeof(float) * static_cast<size_t>(batch) * q_len * q_heads * pl.splits * (head_dim + 2);
    return pl;
  }
  const int es = dtype == QD_DTYPE_F32 ? 4 : 2;
  pl.dp = tree_padded(es, head_dim);
  const int slots = tree_slots(es, pl.dp);
  const int R = q_len * (q_heads / kv_heads);
  TreeWaves wv{};
  int64_t items = 0, tiles = 0, units = 0, resident = 0;
  // The largest chunks that still give every resident workgroup a tile if the
  // contexts fill the table or the window: K and V are read once per chunk, but a
  // tile of 256 rows takes 8 times as long as one of 16 (one sequence of 8000 to 16000 tokens, 24 drafts x 4 heads of 96:
  // chunks of 16 rows 20.6 us, one chunk 30.5 us; 8 sequences of 489 tokens, 64
  // drafts x 8 heads of 128: 23.6 us, chunks of 256 rows 41.3 us).
  int most = tree_most_rows(slots);
  if (R <= 128 && cap <= kTreeShortContext) most = std::min(most, 64);
  for (;; most /= 2) {
    pl.chunks = (R + most - 1) / most;
    pl.chunk_rows = (R + pl.chunks - 1) / pl.chunks;
    wv = tree_waves(slots, pl.chunk_rows);
    const int tt = tree_tile(slots, wv.nw);
    items = static_cast<int64_t>(batch) * kv_heads * pl.chunks;
    tiles = (cap + tt - 1) / tt;
    units = std::max<int64_t>(1, tiles * tt / 64) * std::max(1, slots / 16);
    resident = static_cast<int64_t>(tree_cu_count()) * tree_occupancy(slots, wv.nw);
    if (pl.chunk_rows <= 16 || items * tiles >= resident) break;
  }
  if (batch > kTreeMaxBalanced || items * (tiles + kTreeItemCost) > INT32_MAX ||
      tree_direct(items, units, resident, window > 0)) {
    pl.grid = static_cast<int>(items);
    return pl;
  }
  pl.W = static_cast<int>(std::max<int64_t>(1, std::min(resident, items * (tiles + kTreeItemCost) / tree_min_cost(slots))));
  pl.grid = pl.W;
  pl.meta_bytes = (8 * static_cast<size_t>(items) + 15) / 16 * 16;
  pl.bytes = pl.meta_bytes + sizeof(float) * 2 * static_cast<size_t>(pl.W) * (16 * wv.nb * wv.wr) * (head_dim + 2);
  return pl;
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
  if (!tree_shape_ok(batch, q_len, q_heads, kv_heads, head_dim, block_size, max_pages, has_mask, window, sinks, dtype))
    return 0;
  if (batch == 0) return 0;
  const size_t bytes = tree_plan(batch, q_len, q_heads, kv_heads, head_dim, block_size, max_pages, has_mask, window,
                                 sinks, dtype, flags)
                           .bytes;
  if (flags & QD_FLAG_FORCE_GENERIC) return bytes;
  // Unaligned tensors take the VALU kernel.
  return std::max(bytes, tree_plan(batch, q_len, q_heads, kv_heads, head_dim, block_size, max_pages, has_mask, window,
                                   sinks, dtype, flags | QD_FLAG_FORCE_GENERIC)
                             .bytes);
}

int qd_gqa_decode_tree_info(int batch, int q_len, int q_heads, int kv_heads, int head_dim, int block_size,
                            int max_pages, int has_mask, int window, int sinks, int dtype, int flags,
                            int* workgroups, int* rows) {
  if (!tree_shape_ok(batch, q_len, q_heads, kv_heads, head_dim, block_size, max_pages, has_mask, window, sinks, dtype))
    return -1;
  const TreePlan pl = tree_plan(batch, q_len, q_heads, kv_heads, head_dim, block_size, max_pages, has_mask, window,
                                sinks, dtype, flags);
  if (workgroups) *workgroups = pl.mfma ? pl.grid : batch * q_len * q_heads * pl.splits;
  if (rows) *rows = pl.mfma ? pl.chunk_rows : 1;
  return !pl.mfma ? QD_TREE_VALU : pl.W > 0 ? QD_TREE_MFMA_SPLIT : QD_TREE_MFMA;
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
  if (((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(k_cache) | reinterpret_cast<uintptr_t>(v_cache) |
        reinterpret_cast<uintptr_t>(out)) &
       15u) != 0)
    flags |= QD_FLAG_FORCE_GENERIC;
  const TreePlan pl = tree_plan(batch, q_len, q_heads, kv_heads, head_dim, block_size, max_pages, has_mask, window,
                                sinks, dtype, flags);
  if (pl.bytes > 0 && (!workspace || workspace_bytes < pl.bytes || (reinterpret_cast<uintptr_t>(workspace) & 15u)))
    return tree_fail(nullptr, 0, "workspace too small or not 16-byte aligned");
  TreeParams p;
  p.q = q;
  p.k = k_cache;
  p.v = v_cache;
  p.table = block_table;
  p.lens = context_lens;
  p.mask = tree_mask;
  p.out = out;
  p.meta = static_cast<int32_t*>(workspace);
  p.part = reinterpret_cast<float*>(static_cast<char*>(workspace) + pl.meta_bytes);
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
  p.splits = pl.splits;
  p.G = q_heads / kv_heads;
  p.R = q_len * p.G;
  p.chunks = pl.chunks;
  p.chunk_rows = pl.chunk_rows;
  p.W = pl.W;
  p.capacity = static_cast<int32_t>(std::min<int64_t>(static_cast<int64_t>(block_size) * max_pages, kTreeCapacity));
  p.last_block = static_cast<int32_t>(std::min<int64_t>(num_blocks - 1, INT32_MAX));
  p.pshift = (block_size & (block_size - 1)) == 0 ? __builtin_ctz(static_cast<unsigned>(block_size)) : -1;
  hipStream_t st = static_cast<hipStream_t>(stream);
  (void)hipGetLastError();
  hipError_t e = hipSuccess;
  if (pl.mfma) {
    const auto run = dtype == QD_DTYPE_F32   ? qd_tree_mfma_launch_f32
                     : dtype == QD_DTYPE_F16 ? qd_tree_mfma_launch_f16
                                             : qd_tree_mfma_launch_bf16;
    e = static_cast<hipError_t>(run(p, pl.dp, pl.grid, stream));
  } else {
    switch (dtype) {
      case QD_DTYPE_F32: launch_generic<QD_DTYPE_F32>(p, st); break;
      case QD_DTYPE_F16: launch_generic<QD_DTYPE_F16>(p, st); break;
      default: launch_generic<QD_DTYPE_BF16>(p, st); break;
    }
    e = hipGetLastError();
  }
  if (e != hipSuccess) {
    qd_set_last_error(static_cast<int>(e),
                      std::string("gqa_decode_tree kernel launch failed: ") + hipGetErrorString(e));
    return static_cast<int>(e);
  }
  return QD_OK;
}

}  // extern "C"
