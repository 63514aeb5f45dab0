// Compaction of a paged cache after drafted tokens were verified, for MI355X
// (gfx950): token len + accepted[i] moves to token len + i, in all caches of
// all layers at once.  C ABI in include/qd_attention.h.

#include <hip/hip_runtime.h>

#include <stdint.h>
#include <string.h>

#include <algorithm>
#include <new>
#include <string>
#include <vector>

#include "qd_attention.h"
#include "qd_device.h"

void qd_set_last_error(int status, const std::string& msg);

namespace {

// Caches of one launch: their pointers are kernel arguments (1 KB).
constexpr int kCompactCaches = 128;

struct CompactParams {
  char* caches[kCompactCaches];
  const int32_t* table;
  const int32_t* lens;
  const int32_t* accepted;
  int count, P, maxP;
  int64_t num_blocks, row_bytes;
};

// Pool row of token `tok` of sequence b, or -1 where there is none.
__device__ __forceinline__ int64_t pool_row(const CompactParams& p, int b, int64_t tok) {
  if (tok < 0 || tok >= static_cast<int64_t>(p.maxP) * p.P) return -1;
  const int64_t page = tok / p.P;
  const int32_t phys = p.table[static_cast<int64_t>(b) * p.maxP + page];
  if (phys < 0 || phys >= p.num_blocks) return -1;
  return static_cast<int64_t>(phys) * p.P + (tok - page * p.P);
}

// grid (sequences, caches, column blocks of 64 V), block 256: wave w holds
// rows w, w + 4, ... of a column block in registers; all rows of the block are
// read before any is written, so rows may move over each other without a copy
// of the cache.  Every row moved is read and written once: bound by HBM in large
// calls, by the launch and three dependent round trips (length, table, row) in
// small ones.  Measured: 72 caches, 32 sequences of 16 drafts, rows of 2 KB
// (57.5 MB in and out) 13.5 us, 4.3 TB/s, where a large copy makes 4.9; two
// caches, 4 sequences of 8 5.4 us.  ROWS rows per wave: registers for 16 rows in
// all where that is enough, or for 64 (16 drafts: 14.5 / 15.8 us).
template <typename V, int ROWS>
__global__ __launch_bounds__(256) void kv_compact_kernel(CompactParams p) {
  const int b = blockIdx.x;
  const int lane = threadIdx.x & 63;
  const int wv = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x >> 6));
  const int len = p.lens[b];
  // Lane i: where row i comes from and goes to.
  int64_t from = -1, to = -1;
  if (lane < p.count && len >= 0) {
    const int32_t a = p.accepted[static_cast<int64_t>(b) * p.count + lane];
    if (a >= 0 && a != lane) {
      from = pool_row(p, b, static_cast<int64_t>(len) + a);
      to = pool_row(p, b, static_cast<int64_t>(len) + lane);
      if (to < 0) from = -1;
    }
  }
  char* cache = p.caches[blockIdx.y];
  const int64_t col = (static_cast<int64_t>(blockIdx.z) * 64 + lane) * static_cast<int64_t>(sizeof(V));
  const bool inside = col < p.row_bytes;
  V held[ROWS];
#pragma unroll
  for (int i = 0; i < ROWS; ++i) {
    const int64_t row = readlane_i64(from, wv + 4 * i);
    if (row >= 0 && inside) held[i] = *reinterpret_cast<const V*>(cache + row * p.row_bytes + col);
  }
  // Every wave's rows have arrived before any wave writes.
  wait_memory_retired();
  __syncthreads();
#pragma unroll
  for (int i = 0; i < ROWS; ++i) {
    const int64_t row = readlane_i64(from, wv + 4 * i);
    const int64_t dst = readlane_i64(to, wv + 4 * i);
    if (row >= 0 && inside) *reinterpret_cast<V*>(cache + dst * p.row_bytes + col) = held[i];
  }
}

int compact_fail(char* msg, size_t cap, const char* text) {
  qd_set_last_error(QD_ERR_INVALID_VALUE, text);
  if (msg && cap) {
    size_t n = strlen(text);
    if (n >= cap) n = cap - 1;
    memcpy(msg, text, n);
    msg[n] = '\0';
  }
  return QD_ERR_INVALID_VALUE;
}

template <typename V>
void launch_compact(const CompactParams& p, int batch, int caches, hipStream_t st) {
  const int64_t blocks = (p.row_bytes + 64 * static_cast<int64_t>(sizeof(V)) - 1) / (64 * static_cast<int64_t>(sizeof(V)));
  const dim3 grid(static_cast<uint32_t>(batch), static_cast<uint32_t>(caches), static_cast<uint32_t>(blocks));
  if (p.count <= 16)
    hipLaunchKernelGGL((kv_compact_kernel<V, 4>), grid, dim3(256), 0, st, p);
  else
    hipLaunchKernelGGL((kv_compact_kernel<V, QD_TREE_MAX_DRAFTS / 4>), grid, dim3(256), 0, st, p);
}

}  // namespace

extern "C" {

int qd_kv_compact_validate(const qd_tensor_desc* cache, const qd_tensor_desc* block_table,
                           const qd_tensor_desc* context_lens, const qd_tensor_desc* accepted, char* msg,
                           size_t msg_cap) {
  const qd_tensor_desc* all[4] = {cache, block_table, context_lens, accepted};
  for (int i = 0; i < 4; ++i)
    if (!all[i]) return compact_fail(msg, msg_cap, "null tensor descriptor");
  for (int i = 0; i < 4; ++i) {
    if (!all[i]->defined || !all[i]->is_device || !all[i]->contiguous)
      return compact_fail(msg, msg_cap, "all tensors must be contiguous CUDA tensors");
    if (all[i]->device_index != cache->device_index)
      return compact_fail(msg, msg_cap, "all tensors must share a device");
  }
  if (cache->ndim < 3 || cache->ndim > 8) return compact_fail(msg, msg_cap, "cache must be [Nblocks, P, ...]");
  for (int i = 0; i < cache->ndim; ++i)
    if (cache->sizes[i] <= 0) return compact_fail(msg, msg_cap, "invalid dimensions");
  if (accepted->ndim != 2 || context_lens->ndim != 1 || block_table->ndim != 2 ||
      context_lens->sizes[0] != accepted->sizes[0] || block_table->sizes[0] != accepted->sizes[0] ||
      block_table->sizes[1] <= 0)
    return compact_fail(msg, msg_cap, "invalid metadata shape");
  if (block_table->dtype != QD_DTYPE_I32 || context_lens->dtype != QD_DTYPE_I32 || accepted->dtype != QD_DTYPE_I32)
    return compact_fail(msg, msg_cap, "metadata must be int32");
  if (accepted->sizes[1] > QD_TREE_MAX_DRAFTS)
    return compact_fail(msg, msg_cap, "at most 64 accepted tokens per sequence");
  if (cache->dtype != QD_DTYPE_F32 && cache->dtype != QD_DTYPE_F16 && cache->dtype != QD_DTYPE_BF16)
    return compact_fail(msg, msg_cap, "unsupported dtype");
  if (accepted->sizes[0] >= (1 << 24) || block_table->sizes[1] > 2147483647 || cache->sizes[1] > 2147483647)
    return compact_fail(msg, msg_cap, "tensor sizes exceed int32 CUDA launch limits");
  if (msg && msg_cap) msg[0] = '\0';
  return QD_OK;
}

int qd_kv_compact(void* const* caches, int num_caches, const int32_t* block_table, const int32_t* context_lens,
                  const int32_t* accepted, int batch, int count, int block_size, int max_pages, int64_t num_blocks,
                  int64_t row_bytes, void* stream) {
  if (num_caches < 0 || batch < 0 || batch >= (1 << 24))
    return compact_fail(nullptr, 0, "caches and batch must be >= 0, batch below 2^24");
  if (count < 0 || count > QD_TREE_MAX_DRAFTS)
    return compact_fail(nullptr, 0, "at most 64 accepted tokens per sequence");
  if (block_size <= 0 || max_pages <= 0 || num_blocks <= 0 || row_bytes <= 0 || row_bytes % 2 != 0 ||
      row_bytes > (int64_t{1} << 31) || num_blocks > (int64_t{1} << 62) / block_size / row_bytes)
    return compact_fail(nullptr, 0, "invalid dimensions");
  if (num_caches == 0 || batch == 0 || count == 0) return QD_OK;
  if (!caches || !block_table || !context_lens || !accepted) return compact_fail(nullptr, 0, "null tensor pointer");
  const uint64_t bytes = static_cast<uint64_t>(num_blocks) * block_size * row_bytes;
  uint64_t bits = static_cast<uint64_t>(row_bytes);
  try {
    std::vector<uint64_t> at(num_caches);
    for (int i = 0; i < num_caches; ++i) {
      if (!caches[i]) return compact_fail(nullptr, 0, "null tensor pointer");
      at[i] = static_cast<uint64_t>(reinterpret_cast<uintptr_t>(caches[i]));
      bits |= at[i];
    }
    std::sort(at.begin(), at.end());
    for (int i = 1; i < num_caches; ++i)
      if (at[i] - at[i - 1] < bytes) return compact_fail(nullptr, 0, "caches must not overlap");
  } catch (const std::bad_alloc&) {
    qd_set_last_error(static_cast<int>(hipErrorOutOfMemory), "out of host memory");
    return static_cast<int>(hipErrorOutOfMemory);
  }
  if (bits % 2 != 0) return compact_fail(nullptr, 0, "caches must be aligned to their elements");
  CompactParams p;
  p.table = block_table;
  p.lens = context_lens;
  p.accepted = accepted;
  p.count = count;
  p.P = block_size;
  p.maxP = max_pages;
  p.num_blocks = num_blocks;
  p.row_bytes = row_bytes;
  const int64_t unit = bits % 16 == 0 ? 16 : 2;
  if ((row_bytes + 64 * unit - 1) / (64 * unit) > 65535)
    return compact_fail(nullptr, 0, "tensor sizes exceed int32 CUDA launch limits");
  hipStream_t st = static_cast<hipStream_t>(stream);
  (void)hipGetLastError();
  for (int first = 0; first < num_caches; first += kCompactCaches) {
    const int n = std::min(kCompactCaches, num_caches - first);
    for (int i = 0; i < n; ++i) p.caches[i] = static_cast<char*>(caches[first + i]);
    if (unit == 16)
      launch_compact<u32x4>(p, batch, n, st);
    else
      launch_compact<uint16_t>(p, batch, n, st);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) {
      qd_set_last_error(static_cast<int>(e), std::string("kv_compact kernel launch failed: ") + hipGetErrorString(e));
      return static_cast<int>(e);
    }
  }
  return QD_OK;
}

}  // extern "C"
