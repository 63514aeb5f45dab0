/*
 * qd_attention.h — C ABI of the MI355X (gfx950) paged grouped-query decode
 * attention library `libqd_attention.so`.
 *
 * Everything here is plain C: pointers, sizes and integer codes.  No torch,
 * no C++ and no HIP types cross this boundary (a HIP stream is passed as an
 * opaque `void*`, NULL meaning the null stream).  The torch binding
 * (`attention_amd/csrc/torch_ops.cpp`) is one caller; a ctypes/cffi/cgo
 * binding is another.
 *
 * Reference interfaces replaced (paths relative to the reference tree):
 *   qd_gqa_decode_validate            csrc/cuda/dense/gqa_decode.cu:103-138
 *   qd_gqa_decode_validate_workspace  csrc/cuda/dense/gqa_decode.cu:148-152
 *   qd_gqa_decode_plan                attention/core.py:80-96 (gqa_decode_auto)
 *   qd_gqa_decode_workspace_bytes     csrc/cuda/dense/gqa_decode.cu:152-154
 *   qd_gqa_decode_launch              csrc/cuda/dense/gqa_decode.cu:140-183,
 *                                     kernels :18-87 (explicit splits)
 *   qd_gqa_decode_auto(+_stages, _workspace_bytes, _info)
 *                                     csrc/cuda/dense/gqa_decode.cu:186-188
 *                                     and attention/core.py:80-96
 *
 * Tensor layouts (all row-major, contiguous, on one device):
 *   q            [batch, q_heads, head_dim]                   dtype
 *   k/v cache    [num_blocks, block_size, kv_heads, head_dim] dtype
 *   block_table  [batch, max_pages]                           int32
 *   context_lens [batch]                                      int32
 *   out          [batch, q_heads, head_dim]                   dtype
 *   workspace    [batch, q_heads, splits, head_dim + 2]       float32
 *                per (b, h, s): {max scaled score, sum exp, acc[head_dim]}
 *
 * Metadata contents (page ids, lengths) are caller-owned and never checked
 * here: only table entries [0, ceil(len/block_size)) of each row are read,
 * and a length <= 0 yields an all-zero output row.
 */
#ifndef QD_ATTENTION_H
#define QD_ATTENTION_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define QD_ATTENTION_ABI_VERSION 2

/* Element type codes shared by every entry point. */
enum {
  QD_DTYPE_F32 = 0,
  QD_DTYPE_F16 = 1,
  QD_DTYPE_BF16 = 2,
  QD_DTYPE_I32 = 3,
  QD_DTYPE_I64 = 4,
  /* Elements of an 8-bit cache (kv_append_q8 and what reads it, only). */
  QD_DTYPE_E4M3 = 5,
  QD_DTYPE_I8 = 6,
  QD_DTYPE_OTHER = -1
};

/* Status codes.  0 is success; any other value is a hipError_t code
 * (hipErrorInvalidValue = 1 for argument errors).  qd_error_string() gives
 * the message of the last failure on the calling thread. */
enum { QD_OK = 0, QD_ERR_INVALID_VALUE = 1 };

/* Kernel-selection flags (qd_gqa_decode_launch, qd_mla_*). */
enum {
  /* Use the portable VALU kernel even where the MFMA kernel applies. */
  QD_FLAG_FORCE_GENERIC = 1,
  /* MLA attention: use the workgroup-staged MFMA kernel even where the
   * wave-streamed or the shared-tile kernel applies (testing and
   * comparison). */
  QD_FLAG_MLA_STAGED = 2,
  /* MLA attention: use the wave-streamed MFMA kernel even where the
   * shared-tile kernel applies (testing and comparison). */
  QD_FLAG_MLA_WAVE = 4
};

/* Shape/placement descriptor of one tensor, for validation only. */
typedef struct qd_tensor_desc {
  int32_t defined;      /* 0: argument absent (optional workspace)        */
  int32_t is_device;    /* 1: GPU tensor                                   */
  int32_t device_index; /* device ordinal (ignored when !is_device)        */
  int32_t contiguous;   /* 1: row-major contiguous                         */
  int32_t dtype;        /* QD_DTYPE_*                                      */
  int32_t ndim;         /* number of dimensions, <= 8                      */
  int64_t sizes[8];
} qd_tensor_desc;

/* ABI version of the loaded library (QD_ATTENTION_ABI_VERSION). */
int qd_abi_version(void);

/* Message for `status`: the detailed text of the calling thread's last
 * failure when it matches, else the HIP error name. Never NULL. */
const char* qd_error_string(int status);

/* Checks shapes, dtypes and placement in the reference's order
 * (gqa_decode.cu:103-138).  Returns 0, or QD_ERR_INVALID_VALUE with the
 * reference's message copied into msg (NUL-terminated, truncated to
 * msg_cap).  Reads no tensor contents. */
int qd_gqa_decode_validate(const qd_tensor_desc* q, const qd_tensor_desc* k_cache,
                           const qd_tensor_desc* v_cache, const qd_tensor_desc* block_table,
                           const qd_tensor_desc* context_lens, double scale, int64_t splits,
                           char* msg, size_t msg_cap);

/* Workspace checks of the split path (gqa_decode.cu:148-152); call after
 * qd_gqa_decode_validate succeeded and only when batch > 0. */
int qd_gqa_decode_validate_workspace(const qd_tensor_desc* q, const qd_tensor_desc* workspace,
                                     int64_t splits, char* msg, size_t msg_cap);

/* Launch plan for the automatic path: number of context splits and pages
 * per split, chosen from static shapes only (no device reads, no sync).
 * cu_count <= 0 means 256 (MI355X).  Writes *splits >= 1 and
 * *chunk_pages >= 1 (pages of block_size tokens per split). */
int qd_gqa_decode_plan(int batch, int q_heads, int kv_heads, int head_dim, int block_size,
                       int max_pages, int dtype, int cu_count, int* splits, int* chunk_pages);

/* Bytes of float32 workspace [batch, q_heads, splits, head_dim + 2]; 0 when
 * splits <= 1 (the single-split path needs none). */
size_t qd_gqa_decode_workspace_bytes(int batch, int q_heads, int head_dim, int splits);

/* Enqueues paged GQA decode on `stream` (a hipStream_t, NULL = null stream).
 *   splits      >= 1.  1: each (sequence, kv-head) in one pass, no
 *               workspace.  > 1: split-context partials into `workspace`
 *               and a log-sum-exp combine.
 *   chunk_pages 0: split s of a sequence with n pages covers pages
 *               [s*c, (s+1)*c), c = ceil(n/splits) (reference split API);
 *               > 0: fixed c = chunk_pages for every sequence (plan path;
 *               requires splits * chunk_pages >= max_pages).
 *   workspace   device float32 buffer of workspace_bytes >= the value of
 *               qd_gqa_decode_workspace_bytes(); may be NULL if splits == 1.
 * Does not allocate, does not synchronize and does not read metadata on
 * the host.  Returns 0 or a status code (argument errors are reported
 * before anything is enqueued). */
int qd_gqa_decode_launch(const void* q, const void* k_cache, const void* v_cache,
                         const int32_t* block_table, const int32_t* context_lens, void* out,
                         float* workspace, size_t workspace_bytes, int batch, int q_heads,
                         int kv_heads, int head_dim, int block_size, int max_pages,
                         int64_t num_blocks, int dtype, float scale, int splits,
                         int chunk_pages, int flags, void* stream);

/* Which kernel qd_gqa_decode_launch would run for these shapes:
 * 1 = the MFMA kernel for head_dim 64/96/128/256, whole 16-token groups per
 * page and groups of at most 16 q-heads, 0 = the others: the general MFMA
 * layout (head_dim a multiple of 8 up to 128 or of 16 up to 256, groups up to
 * 128, not with QD_FLAG_FORCE_GENERIC; fp32 above head_dim 96 only for at most
 * 512 workgroups) or the portable VALU kernel. */
int qd_gqa_decode_kernel_kind(int q_heads, int kv_heads, int head_dim, int block_size,
                              int dtype, int flags);

/* ---- Automatic path: the body of attention.gqa_decode ----------------
 * Replaces csrc/cuda/dense/gqa_decode.cu:186-188 (gqa_decode_cuda, always
 * one split) and the split heuristic of attention/core.py:80-96.  The
 * partition is chosen from static shapes and the device (CU count and
 * kernel occupancy), never from context_lens on the host:
 *   - 16-bit caches with head_dim 64/96/128/256, block_size a multiple of 16,
 *     group size <= 128 (a group above 16 is served as ceil(g/16) chunks of
 *     at most 16 q-heads, each like a kv-head of its own) and batch <= 4096,
 *     and fp32 caches with head_dim 64/128, block_size a multiple of 16,
 *     group size <= 16 and batch * max_pages * block_size >= 65536 (fp32
 *     matrix-core products):
 *     the (sequence, 16-token group)
 *     space is cut into cost-balanced ranges, one per resident workgroup;
 *     a sequence split across workgroups leaves one partial per workgroup,
 *     folded (log-sum-exp) either inside the same kernel by the last
 *     workgroup to finish a piece of it (the fused merge, when the merge is
 *     short: see qd_gqa_decode_auto_info) or by a second kernel on the same
 *     stream;
 *   - caches with any other block_size, or a head_dim that is another multiple
 *     of 8 up to 128 or of 16 up to 256 (same groups and batch, num_blocks *
 *     block_size < 2^31), and in fp32 any of these from 16384 tokens of
 *     capacity: the same partition with the general kernel (fp32 head_dim
 *     64/128 with its own), merged by a second kernel.  It serves whole calls only and is
 *     reported as kind 0 by qd_gqa_decode_auto_info; with a workspace that
 *     holds only the split layout's partials the split layout runs instead;
 *   - short contexts (wg_single_applies in gqa_decode.hip: by max_pages *
 *     block_size and the number of sequences and kv-heads) in one launch with
 *     one workgroup per (sequence, kv-head), no partials; QD_STAGE_DECODE is
 *     then the whole call and QD_STAGE_MERGE alone does nothing, and the
 *     QD_STAGE_UNFUSED / FUSED / VALU bodies stay selectable;
 *   - otherwise: the split layout of qd_gqa_decode_launch with the plan of
 *     qd_gqa_decode_plan.
 * The workspace is device memory, 16-byte aligned, of at least
 * qd_gqa_decode_auto_workspace_bytes() bytes.  Its first
 * qd_gqa_decode_auto_counter_bytes() bytes are the fused merge's arrival
 * counters: they must be zero before the workspace's first use (zero the
 * whole workspace once when allocating it), and every call leaves them
 * zero, so a workspace is reused as it is.  The rest needs no
 * initialization: every call writes what it reads.  Calls that may run
 * concurrently (different streams, or replays of captured graphs on
 * different streams) need different workspaces.  Workspace size and
 * partition depend on the current device (hipGetDevice), so query and
 * launch with the same device current.  Does not allocate or synchronize. */
size_t qd_gqa_decode_auto_workspace_bytes(int batch, int q_heads, int kv_heads, int head_dim,
                                          int block_size, int max_pages, int dtype);

/* Bytes of arrival counters at the start of every automatic-path workspace
 * (fixed: 256 KiB). */
size_t qd_gqa_decode_auto_counter_bytes(void);

int qd_gqa_decode_auto(const void* q, const void* k_cache, const void* v_cache,
                       const int32_t* block_table, const int32_t* context_lens, void* out,
                       void* workspace, size_t workspace_bytes, int batch, int q_heads,
                       int kv_heads, int head_dim, int block_size, int max_pages,
                       int64_t num_blocks, int dtype, float scale, void* stream);

/* The automatic path's kernels, for callers that time or schedule them
 * separately (the balanced MFMA path only; the split path needs
 * QD_STAGE_ALL).  With the fused merge, QD_STAGE_DECODE is the whole call
 * and QD_STAGE_MERGE alone does nothing.  Otherwise QD_STAGE_DECODE alone
 * leaves split sequences unmerged, and a following QD_STAGE_MERGE call with
 * the same arguments and workspace on the same stream completes the
 * output. */
enum { QD_STAGE_DECODE = 1, QD_STAGE_MERGE = 2, QD_STAGE_ALL = 3 };
/* OR'ed into `stages` for measurement only: run the balanced path's decode
 * kernel with VALU math (packed dot products and fp32 FMAs) in place of the
 * MFMA instructions, same loads and partition (never fused).  Head_dim 128,
 * group size <= 8, one kv-head per wave; other shapes are rejected. */
enum { QD_STAGE_VALU = 4 };
/* OR'ed into `stages` for measurement only: merge split sequences with the
 * separate merge kernel (QD_STAGE_UNFUSED) or inside the decode kernel
 * (QD_STAGE_FUSED; batch * kv_heads <= 65536 and the partial slots below
 * 2 GiB) whatever the plan chose. */
enum { QD_STAGE_UNFUSED = 8, QD_STAGE_FUSED = 16 };

int qd_gqa_decode_auto_stages(const void* q, const void* k_cache, const void* v_cache,
                              const int32_t* block_table, const int32_t* context_lens, void* out,
                              void* workspace, size_t workspace_bytes, int batch, int q_heads,
                              int kv_heads, int head_dim, int block_size, int max_pages,
                              int64_t num_blocks, int dtype, float scale, int stages, void* stream);

/* ---- Automatic path without allocation ------------------------------
 * No counterpart in the reference: for callers that cannot allocate device
 * memory (code under HIP graph capture, tight serving loops, harnesses that
 * forbid hipMalloc).  Same as qd_gqa_decode_auto, but its scratch is a
 * file-scope device array of qd_gqa_decode_noalloc_scratch_bytes() bytes
 * (16 MiB) per GPU, held until the process ends; shapes whose
 * qd_gqa_decode_auto_workspace_bytes() exceed it are rejected with
 * QD_ERR_INVALID_VALUE before anything is enqueued (shapes of the general
 * kernel, only where the split layout's partials exceed it too).  Nothing is allocated
 * (the array's address is looked up once per device).  Every call on a GPU
 * uses that GPU's one array: calls that may overlap on one GPU (different
 * streams, host threads) race and must be serialized by the caller. */
size_t qd_gqa_decode_noalloc_scratch_bytes(void);

int qd_gqa_decode_auto_noalloc(const void* q, const void* k_cache, const void* v_cache,
                               const int32_t* block_table, const int32_t* context_lens, void* out, int batch,
                               int q_heads, int kv_heads, int head_dim, int block_size, int max_pages,
                               int64_t num_blocks, int dtype, float scale, void* stream);

/* Describes the automatic path's choice (assuming aligned pointers):
 * returns 2 for the balanced MFMA path with the fused merge, 1 for it with
 * the separate merge kernel (*waves = its total wave count), 0 for the split
 * path (*splits, *chunk_pages), -1 for invalid shapes.  Whole calls whose
 * shape is reported as 0 may run the balanced kernels all the same (the
 * general layout, fp32 from 16384 tokens of capacity), and short contexts of
 * any kind run in one launch; what is reported is what stages, or a
 * workspace of the split layout's size, get (qd_gqa_decode_auto_path reports
 * whole calls).  Any output pointer may be NULL. */
int qd_gqa_decode_auto_info(int batch, int q_heads, int kv_heads, int head_dim, int block_size,
                            int max_pages, int dtype, int* waves, int* splits, int* chunk_pages);

/* What a whole qd_gqa_decode_auto call runs for these shapes and a pool of
 * num_blocks pages (aligned pointers, a workspace of
 * qd_gqa_decode_auto_workspace_bytes()): returns QD_PATH_* or -1 for invalid
 * shapes, with
 *   *layout      QD_LAYOUT_*: the per-wave kernel body
 *   *chunks      chunks that each kv-head's q-heads are served in (at most 16
 *                q-heads each, 8 on the VALU kernel)
 *   *workgroups  workgroups of the decode kernel
 *   *waves       waves per workgroup.
 * Any output pointer may be NULL. */
enum { QD_PATH_SPLIT = 0, QD_PATH_BALANCED = 1, QD_PATH_FUSED = 2, QD_PATH_ONE_LAUNCH = 3 };
enum { QD_LAYOUT_VALU = 0, QD_LAYOUT_EXACT = 1, QD_LAYOUT_GENERAL = 2 };
int qd_gqa_decode_auto_path(int batch, int q_heads, int kv_heads, int head_dim, int block_size, int max_pages,
                            int64_t num_blocks, int dtype, int* layout, int* chunks, int* workgroups, int* waves);

/* ---- Paged KV-cache append ------------------------------------------
 * Replaces csrc/cuda/cache/kv_append.cu:29-56 (kv_append_cuda) behind the
 * op kv_append (csrc/binding/torch_ops.cpp:52; attention/core.py:59-63).
 *   key, value   [batch, kv_heads, head_dim]                   dtype
 *   k/v cache    [num_blocks, block_size, kv_heads, head_dim]  dtype (written)
 *   block_table  [batch, max_pages] int32, positions [batch] int32
 * Sequence b's token goes to row (block_table[b][pos/block_size],
 * pos % block_size) of both caches.  Destinations are caller-owned and
 * must be distinct; a position outside [0, max_pages*block_size) or a page
 * id outside [0, num_blocks) is skipped (never written). */

/* The reference's checks in order (kv_append.cu:32-43), messages included. */
int qd_kv_append_validate(const qd_tensor_desc* key, const qd_tensor_desc* value,
                          const qd_tensor_desc* k_cache, const qd_tensor_desc* v_cache,
                          const qd_tensor_desc* block_table, const qd_tensor_desc* positions, char* msg,
                          size_t msg_cap);

/* Enqueues the append on `stream`; no allocation, no synchronization. */
int qd_kv_append_launch(const void* key, const void* value, void* k_cache, void* v_cache,
                        const int32_t* block_table, const int32_t* positions, int batch, int kv_heads,
                        int head_dim, int block_size, int max_pages, int64_t num_blocks, int dtype,
                        void* stream);

/* ---- Paged metadata validation --------------------------------------
 * Device-side body of attention.validation.validate_paged_metadata
 * (attention/validation.py:5-39).  Checks, per sequence b in order: the
 * length is in [0, max_pages*block_size]; every used page id
 * (ceil(len/block_size) of them) is in [0, num_blocks); and, when
 * `positions` is not NULL, the append position is in
 * [0, max_pages*block_size), its page id is in [0, num_blocks) and its
 * (page, slot) destination is not taken by an earlier sequence.
 * Writes to device memory `*result` the first failure in the reference's
 * order as (b << 35) | (check << 32) | page, or all ones when the metadata
 * is valid; `page` is the failing page index for QD_META_BAD_PAGE.
 * Enqueues two kernels on `stream`; the caller reads *result after them.
 * Requires batch < 2^28, max_pages > 0, block_size > 0, num_blocks > 0. */
enum {
  QD_META_BAD_LENGTH = 1,      /* "invalid length at batch {b}"          */
  QD_META_BAD_PAGE = 2,        /* "invalid block at batch {b}, page {p}" */
  QD_META_BAD_POSITION = 3,    /* "invalid append position at batch {b}" */
  QD_META_BAD_APPEND_PAGE = 4, /* "invalid append page at batch {b}"     */
  QD_META_CONFLICT = 5         /* "conflicting append destinations"      */
};

int qd_validate_paged_metadata(const int32_t* block_table, const int32_t* context_lens,
                               const int32_t* positions, int batch, int max_pages, int block_size,
                               int64_t num_blocks, unsigned long long* result, void* stream);

/* ---- Paged MLA (multi-head latent attention) decode -----------------
 * Replaces the reference's MLA decode operators (csrc/cuda/mla/mla.cu,
 * ops mla_project / latent_kv_write / mla_attend / mla_decode_fused,
 * csrc/binding/torch_ops.cpp:47-50; Python attention/mla.py:16-53).
 * Layouts (row-major, contiguous, one device, one dtype unless noted):
 *   cache        [num_blocks, block_size, latent_dim + rope_dim]
 *                (latent | rope key per token)
 *   block_table  [batch, max_pages] int32; lengths [batch] int32
 *   positions    [batch, q_len] int32 (absolute position of each query)
 *   indices      [batch, q_len, num_indices] int32 logical token ids;
 *                num_indices = -1 (indices unused, may be NULL) attends to
 *                all visible tokens; ids outside [0, end) are skipped
 *   q / q_nope   [batch, q_len, heads, latent_dim / nope_dim]
 *   q_rope       [batch, q_len, heads, rope_dim]
 *   w_uk [heads, nope_dim, latent_dim]; w_uv [heads, value_dim, latent_dim]
 * Query row (b, t) sees tokens [0, end) with end = min(len, max(0, pos+1))
 * when `causal`, else len (clamped to max_pages*block_size); a row with no
 * visible token is zero.  `splits` 0 picks the partition from static shapes
 * and the device; > 0 forces it: for the MFMA kernel (16-bit, latent and
 * rope widths multiples of 8, latent <= 512) the number of workgroups that
 * share the batch's (row, 32-token tile) space in equal ranges (stream-K),
 * (16-token tiles for the wave-streamed kernel, in cost units), for the
 * VALU kernel the number of context splits per row.
 * qd_mla_attend_info() reports the kernel and the partition.  flags:
 * QD_FLAG_FORCE_GENERIC selects the VALU kernels, QD_FLAG_MLA_STAGED the
 * workgroup-staged MFMA kernel where the wave-streamed or shared-tile kernel
 * would run, QD_FLAG_MLA_WAVE the wave-streamed kernel where the shared-tile
 * kernel would run.
 * Nothing here allocates or synchronizes. */

/* Reference checks in order, messages included (mla.cu:152-155). */
int qd_latent_kv_write_validate(const qd_tensor_desc* latent, const qd_tensor_desc* rope,
                                const qd_tensor_desc* cache, const qd_tensor_desc* slots, char* msg,
                                size_t msg_cap);

/* Writes [latent | rope] of token t to flat cache row slots[t] (int64) of
 * the [num_blocks*block_size, latent_dim+rope_dim] view (mla.cu:28-32,
 * :151-160).  Rows outside [0, cache_rows) are skipped. */
int qd_latent_kv_write(const void* latent, const void* rope, void* cache, const int64_t* slots, int64_t tokens,
                       int latent_dim, int rope_dim, int64_t cache_rows, int dtype, void* stream);

/* Reference checks in order, messages included (mla.cu:139-142). */
int qd_mla_project_validate(const qd_tensor_desc* x, const qd_tensor_desc* w, int absorb, char* msg,
                            size_t msg_cap);

/* Per-head projection over rows = batch*q_len (mla.cu:16-27, :138-150):
 *   absorb != 0: out[r,h,o] = sum_k x[r,h,k] * w[h,k,o]  (w [H, in, out])
 *   absorb == 0: out[r,h,o] = sum_k x[r,h,k] * w[h,o,k]  (w [H, out, in])
 * fp32 accumulation, output rounded to the dtype. */
int qd_mla_project(const void* x, const void* w, void* out, int64_t rows, int heads, int in_dim, int out_dim,
                   int absorb, int dtype, int flags, void* stream);

/* Reference checks of mla_attend in order, messages included
 * (mla.cu:162-171); `indices` may be NULL or undefined. */
int qd_mla_attend_validate(const qd_tensor_desc* q, const qd_tensor_desc* q_rope, const qd_tensor_desc* cache,
                           const qd_tensor_desc* table, const qd_tensor_desc* lengths,
                           const qd_tensor_desc* positions, const qd_tensor_desc* indices, double scale,
                           char* msg, size_t msg_cap);

/* Workspace bytes qd_mla_attend needs (partials of rows split across
 * workgroups or splits, and per-row spans); 0 when none is needed. */
size_t qd_mla_attend_workspace_bytes(int batch, int q_len, int heads, int latent_dim, int rope_dim,
                                     int block_size, int max_pages, int num_indices, int dtype, int splits,
                                     int flags);

/* The plan qd_mla_attend would use: returns 3 for the shared-tile MFMA
 * kernel (latent 512, rope 64: 64 heads or more on listed tokens, on pages of
 * a multiple of 32 tokens or of no multiple of 16; or fewer heads and several
 * queries on dense pages of a multiple of 32 tokens, folded into q_len * heads
 * heads, *head_groups = ceil(q_len * heads / 64): shared_fold_applies in
 * mla.hip), 2 for the
 * wave-streamed MFMA kernel (latent 512, rope 64, the other dense rows on
 * pages of a multiple of 16 tokens), 1 for the
 * workgroup-staged MFMA kernel (*out_splits = stream-K workgroups per head
 * group, *head_groups = head groups for both), 0 for the VALU kernel
 * (*out_splits = context splits per row, *head_groups = 0), -1 for invalid
 * shapes. */
int qd_mla_attend_info(int batch, int q_len, int heads, int latent_dim, int rope_dim, int block_size,
                       int max_pages, int num_indices, int dtype, int splits, int flags, int* out_splits,
                       int* head_groups);

/* Paged latent attention (mla.cu:34-82, :161-181): out [batch, q_len,
 * heads, latent_dim] = softmax((q . c + q_rope . k_rope) * scale) . c. */
int qd_mla_attend(const void* q, const void* q_rope, const void* cache, const int32_t* block_table,
                  const int32_t* lengths, const int32_t* positions, const int32_t* indices, void* out,
                  void* workspace, size_t workspace_bytes, int batch, int q_len, int heads, int latent_dim,
                  int rope_dim, int block_size, int max_pages, int64_t num_blocks, int num_indices, int causal,
                  int dtype, float scale, int splits, int flags, void* stream);

/* Reference checks of mla_decode_fused in order, messages included
 * (mla.cu:185-191). */
int qd_mla_decode_validate(const qd_tensor_desc* q_nope, const qd_tensor_desc* q_rope, const qd_tensor_desc* cache,
                           const qd_tensor_desc* table, const qd_tensor_desc* lengths,
                           const qd_tensor_desc* positions, const qd_tensor_desc* w_uk, const qd_tensor_desc* w_uv,
                           const qd_tensor_desc* indices, double scale, char* msg, size_t msg_cap);

/* Workspace bytes of qd_mla_decode (absorbed query, latent output and
 * split partials); 16-byte aligned device memory, no zeroing needed. */
size_t qd_mla_decode_workspace_bytes(int batch, int q_len, int heads, int latent_dim, int rope_dim,
                                     int block_size, int max_pages, int num_indices, int dtype, int splits,
                                     int flags);

/* Absorbed paged MLA decode (mla.cu:86-134, :184-198): query absorption,
 * latent attention and value projection, with the reference's rounding
 * points (absorbed query and latent output rounded to the dtype).
 * out [batch, q_len, heads, value_dim]. */
int qd_mla_decode(const void* q_nope, const void* q_rope, const void* cache, const int32_t* block_table,
                  const int32_t* lengths, const int32_t* positions, const void* w_uk, const void* w_uv,
                  const int32_t* indices, void* out, void* workspace, size_t workspace_bytes, int batch, int q_len,
                  int heads, int nope_dim, int latent_dim, int rope_dim, int value_dim, int block_size,
                  int max_pages, int64_t num_blocks, int num_indices, int causal, int dtype, float scale,
                  int splits, int flags, void* stream);

/* ---- Decoding with drafted tokens and sliding windows ----------------
 * No counterpart in the reference: the operators around gqa_decode that a
 * serving engine needs when it drafts several tokens per step or when a
 * layer keeps only the last tokens in sight.  One step is
 *   qd_qk_norm_rope_write   per-head norms, rotation, cache write
 *   qd_gqa_decode_tree      attention of the drafted tokens over the cache
 *                           (window and first tokens optional; q_len 1 and
 *                           no mask: one query per sequence)
 *   qd_kv_compact           the accepted drafted tokens' rows move next to
 *                           the context.
 * Caches, block_table and context_lens are those of gqa_decode.  Nothing
 * here allocates, synchronizes or reads metadata on the host. */

/* Largest number of drafted tokens per sequence (bits of a mask). */
enum { QD_TREE_MAX_DRAFTS = 64 };

/* Checks of qd_gqa_decode_tree in order.  tree_mask undefined or NULL: one
 * query per sequence, q [batch, q_heads, head_dim]; else q [batch, q_len,
 * q_heads, head_dim] and tree_mask [batch, q_len] int64, q_len in [1, 64].
 * window 0 means none; sinks needs a window. */
int qd_gqa_decode_tree_validate(const qd_tensor_desc* q, const qd_tensor_desc* k_cache,
                                const qd_tensor_desc* v_cache, const qd_tensor_desc* block_table,
                                const qd_tensor_desc* context_lens, const qd_tensor_desc* tree_mask, double scale,
                                int64_t window, int64_t sinks, char* msg, size_t msg_cap);

/* Workspace bytes of qd_gqa_decode_tree (fp32 partials of contexts split
 * over workgroups); 0 when none is needed.  16-byte aligned, no zeroing
 * needed: every call writes what it reads.  Calls that can overlap need
 * different workspaces.  Depends on the current device, like the launch. */
size_t qd_gqa_decode_tree_workspace_bytes(int batch, int q_len, int q_heads, int kv_heads, int head_dim,
                                          int block_size, int max_pages, int has_mask, int window, int sinks,
                                          int dtype, int flags);

/* What qd_gqa_decode_tree runs for these shapes on aligned tensors:
 * QD_TREE_* or -1 for invalid shapes, with *workgroups of the attention
 * kernel and *rows of one workgroup (queries x q-heads of a kv-head).
 * Output pointers may be NULL. */
enum { QD_TREE_VALU = 0, QD_TREE_MFMA = 1, QD_TREE_MFMA_SPLIT = 2 };
int qd_gqa_decode_tree_info(int batch, int q_len, int q_heads, int kv_heads, int head_dim, int block_size,
                            int max_pages, int has_mask, int window, int sinks, int dtype, int flags,
                            int* workgroups, int* rows);

/* out = softmax(q . k * scale) . v over the tokens that a query sees.
 * With a mask, len = context_lens[b] tokens precede the drafted ones and
 * drafted token j lies at token len + j of the cache.  Query t's mask m_t
 * (bits at and above q_len are ignored) holds the drafted tokens it sees,
 * itself among them, and puts it at position p_t = len + popcount(m_t) - 1.
 * m_t = 0 marks padding: a zero row.  Query t sees
 *   context token i < len    iff window == 0 or i > p_t - window or i < sinks
 *   drafted token j          iff bit j of m_t is set, and window == 0 or
 *                            p_j > p_t - window or p_j < sinks.
 * Without a mask, the query is the last of len = context_lens[b] tokens
 * (p = len - 1).  Lengths are clamped to [0, max_pages * block_size], tokens
 * past the table are not seen, page ids are clamped to the pool; table
 * entries of tokens that no query of the sequence can see by its length,
 * window and sinks are never read.  A query that sees nothing gets a zero
 * row.  Whatever a token holds that a query does not see (NaN included)
 * does not reach that query's row.
 * Without a window, max_pages * block_size stands for the longest context when
 * the work is cut: short contexts are up to twice as slow in a table much wider
 * than they need.
 * flags: QD_FLAG_FORCE_GENERIC selects the VALU kernel. */
int qd_gqa_decode_tree(const void* q, const void* k_cache, const void* v_cache, const int32_t* block_table,
                       const int32_t* context_lens, const int64_t* tree_mask, void* out, void* workspace,
                       size_t workspace_bytes, int batch, int q_len, int q_heads, int kv_heads, int head_dim,
                       int block_size, int max_pages, int64_t num_blocks, int dtype, float scale, int window,
                       int sinks, int flags, void* stream);

/* Checks of qd_qk_norm_rope_write in order.  `contiguous` of q, key and value
 * means that the rows of one token are ([heads, head_dim] row-major; tokens
 * may lie any stride apart).  q_weight and k_weight may be NULL or undefined
 * (no norm); weight dtype is q's or float32, the same for both. */
int qd_qk_norm_rope_write_validate(const qd_tensor_desc* q, const qd_tensor_desc* key, const qd_tensor_desc* value,
                                   const qd_tensor_desc* cos_sin, const qd_tensor_desc* positions,
                                   const qd_tensor_desc* k_cache, const qd_tensor_desc* v_cache,
                                   const qd_tensor_desc* slots, const qd_tensor_desc* q_weight,
                                   const qd_tensor_desc* k_weight, double eps, char* msg, size_t msg_cap);

/* For every token n: y = x * rsqrt(mean(x^2) + eps) * weight over each head of
 * q and key (weights NULL: y = x), then the first rotary_dim elements turned
 * by cos_sin[positions[n]] = {cos[rotary_dim / 2], sin[rotary_dim / 2]}
 * (float32 [max_positions, rotary_dim]): pairs (i, i + rotary_dim / 2), or
 * (2i, 2i + 1) when `interleaved`, (a, b) -> (a cos - b sin, b cos + a sin).
 * fp32 arithmetic, one rounding.  q goes to q_out [tokens, q_heads, head_dim]
 * (contiguous), key and value to flat row slots[n] of the caches [cache_rows,
 * kv_heads, head_dim].  q_stride, k_stride and v_stride are the elements from
 * one token to the next.  Outputs and inputs do not overlap, nor the caches
 * each other (checked).  Slots must be distinct; one outside [0, cache_rows)
 * is skipped.  A position outside the table gives a zero q row and writes
 * nothing to the caches. */
int qd_qk_norm_rope_write(const void* q, const void* key, const void* value, const float* cos_sin,
                          const int32_t* positions, void* k_cache, void* v_cache, const int64_t* slots,
                          const void* q_weight, const void* k_weight, void* q_out, int64_t tokens, int q_heads,
                          int kv_heads, int head_dim, int rotary_dim, int64_t q_stride, int64_t k_stride,
                          int64_t v_stride, int64_t max_positions, int64_t cache_rows, int dtype, int weight_dtype,
                          float eps, int interleaved, void* stream);

/* Checks of qd_kv_compact in order, on the first of the caches (all have one
 * shape) and the metadata. */
int qd_kv_compact_validate(const qd_tensor_desc* cache, const qd_tensor_desc* block_table,
                           const qd_tensor_desc* context_lens, const qd_tensor_desc* accepted, char* msg,
                           size_t msg_cap);

/* Moves, in every one of num_caches caches [num_blocks, block_size, row]
 * (row_bytes each row; K and V of any layers, or latent caches), token
 * context_lens[b] + accepted[b][i] to token context_lens[b] + i, for every i
 * in [0, count) with accepted[b][i] >= 0, as if all rows were read before any
 * is written.  count <= 64.  Tokens past the table, page ids outside the pool
 * and negative lengths are skipped (nothing is read or written).  `caches` is
 * a host array of device pointers, read during the call; the caches must not
 * overlap (checked).  Rows that move must be their sequence's own: a row that
 * one sequence writes is not read or written for another in the same call. */
int qd_kv_compact(void* const* caches, int num_caches, const int32_t* block_table, const int32_t* context_lens,
                  const int32_t* accepted, int batch, int count, int block_size, int max_pages, int64_t num_blocks,
                  int64_t row_bytes, void* stream);

/* ---- Prompts, and a cache held in 8 bits -----------------------------
 * No counterpart in the reference: attention over whole prompts, and a paged
 * cache of half the bytes.
 *   qd_gqa_prefill    packed prompts attend to their keys
 *   qd_kv_append_q8   writes prompts or single tokens to the 8-bit cache
 *   qd_gqa_decode_q8  attention of one token per sequence over it
 *   qd_kv_gather_q8   reads it back as packed rows: keys of a later chunk's
 *                     qd_gqa_prefill
 * An 8-bit cache is [num_blocks, block_size, kv_heads, head_dim] of
 * QD_DTYPE_E4M3 (OCP, finite, largest value 448) or QD_DTYPE_I8, with a
 * float32 scale per page and head, [num_blocks, kv_heads], for keys and
 * another for values: an element stands for itself times its scale.
 * Sequences are packed: cu[0] is 0 (and not read), sequence b has rows
 * [cu[b], cu[b + 1]) of q, key or value.  Metadata are caller-owned; values
 * outside their range are clamped, so that no access leaves a tensor.  Nothing
 * here allocates, synchronizes or reads metadata on the host. */

/* Checks of qd_gqa_prefill in order.  `contiguous` of q, key and value means
 * that the rows of one token are.  cu_k undefined or NULL: cu. */
int qd_gqa_prefill_validate(const qd_tensor_desc* q, const qd_tensor_desc* key, const qd_tensor_desc* value,
                            const qd_tensor_desc* cu, const qd_tensor_desc* cu_k, double scale, int64_t window,
                            int64_t sinks, char* msg, size_t msg_cap);

/* What qd_gqa_prefill runs for these sizes on aligned tensors: QD_PREFILL_*,
 * or -1 for invalid sizes, with *workgroups and *rows of one workgroup
 * (queries x q-heads of a kv-head).  Output pointers may be NULL. */
enum { QD_PREFILL_VALU = 0, QD_PREFILL_MFMA = 1 };
int qd_gqa_prefill_info(int batch, int64_t q_tokens, int64_t k_tokens, int q_heads, int kv_heads, int head_dim,
                        int dtype, int flags, int* workgroups, int* rows);

/* Workspace bytes of qd_gqa_prefill (fp32 partials of keys split over
 * workgroups); 0 when none is needed.  16-byte aligned, no zeroing needed.
 * Calls that can overlap need different workspaces.  Depends on the current
 * device, like the launch. */
size_t qd_gqa_prefill_workspace_bytes(int batch, int64_t q_tokens, int64_t k_tokens, int q_heads, int kv_heads,
                                      int head_dim, int dtype, int window, int sinks, int flags);

/* out = softmax(q . k * scale) . v over the keys that a query sees.  Query i of
 * the nq of a sequence with nk keys lies at position p = nk - nq + i and sees
 * key j iff j <= p and (window == 0 or j > p - window or j < sinks); one that
 * sees nothing, or nothing but scores of -inf, gets a zero row, and so do rows
 * behind the last sequence.
 * Whatever a key or value holds that a query does not see (NaN included)
 * does not reach that query's row.  q [q_tokens, q_heads, head_dim], key and
 * value [k_tokens, kv_heads, head_dim], their tokens q_stride, k_stride and
 * v_stride elements apart; out is contiguous.
 * Products and sums are float32; 16-bit types round each softmax weight to the
 * type once, and divide by the sum of the rounded ones.
 * Calls of 2^24 workgroups or more are refused: 2^24 rows (queries x q-heads) of
 * the VALU kernel, which takes unaligned tensors and rows of no whole 16 bytes, or
 * about 2^31 of the other.
 * flags: QD_FLAG_FORCE_GENERIC selects the VALU kernel. */
int qd_gqa_prefill(const void* q, const void* key, const void* value, const int32_t* cu, const int32_t* cu_k,
                   void* out, void* workspace, size_t workspace_bytes, int batch, int64_t q_tokens, int64_t k_tokens,
                   int q_heads, int kv_heads, int head_dim, int64_t q_stride, int64_t k_stride, int64_t v_stride,
                   int dtype, float scale, int window, int sinks, int flags, void* stream);

/* Checks of qd_kv_append_q8 in order.  `contiguous` of key and value means
 * that the rows of one token are.  cu undefined or NULL: one token per
 * sequence. */
int qd_kv_append_q8_validate(const qd_tensor_desc* key, const qd_tensor_desc* value, const qd_tensor_desc* k_cache,
                             const qd_tensor_desc* v_cache, const qd_tensor_desc* k_scales,
                             const qd_tensor_desc* v_scales, const qd_tensor_desc* block_table,
                             const qd_tensor_desc* positions, const qd_tensor_desc* cu, char* msg, size_t msg_cap);

/* Writes row cu[b] + i of key and value to token positions[b] + i of sequence
 * b's cache.  For each page and head that the call writes to, a is the largest
 * |x| of the new rows and s = 2^e the smallest power of two with a <= s * 448
 * (e4m3) or a <= s * 127 (int8), at least 2^-100.  If the call begins the page
 * (its first new row is the page's first), its scale becomes s; else the larger
 * in magnitude of s and the old one, and if that is s, the rows before are rounded
 * to it.
 * Elements are x / scale rounded to nearest, ties to even.  With an Inf or NaN
 * among the new rows, or if s would pass 2^100, the scale becomes NaN, and the
 * elements are unspecified.
 * Other rows keep their elements.  Sequences with a negative position write
 * nothing, nor do tokens past the table or in pages outside the pool.  Pages
 * that are written to must be their sequence's own.  Caches, scales and inputs
 * must not overlap (the caches and the scales are checked).  Calls that could
 * write 2^31 - 1023 tokens or more to one page are refused. */
int qd_kv_append_q8(const void* key, const void* value, void* k_cache, void* v_cache, float* k_scales,
                    float* v_scales, const int32_t* block_table, const int32_t* positions, const int32_t* cu,
                    int batch, int64_t tokens, int kv_heads, int head_dim, int block_size, int max_pages,
                    int64_t num_blocks, int64_t k_stride, int64_t v_stride, int dtype, int cache_dtype, void* stream);

/* Checks of qd_kv_gather_q8 in order, `contiguous` of key and value as above. */
int qd_kv_gather_q8_validate(const qd_tensor_desc* key, const qd_tensor_desc* value, const qd_tensor_desc* k_cache,
                             const qd_tensor_desc* v_cache, const qd_tensor_desc* k_scales,
                             const qd_tensor_desc* v_scales, const qd_tensor_desc* block_table,
                             const qd_tensor_desc* context_lens, const qd_tensor_desc* cu, char* msg, size_t msg_cap);

/* Row cu[b] + i of key and value becomes token i of sequence b's cache, for
 * every i < context_lens[b] inside the sequence's rows and its table; other
 * rows are left as they were.  Page ids are clamped to the pool.  Rows of key,
 * and of value, must not overlap. */
int qd_kv_gather_q8(void* key, void* value, const void* k_cache, const void* v_cache, const float* k_scales,
                    const float* v_scales, const int32_t* block_table, const int32_t* context_lens,
                    const int32_t* cu, int batch, int64_t tokens, int kv_heads, int head_dim, int block_size,
                    int max_pages, int64_t num_blocks, int64_t k_stride, int64_t v_stride, int dtype,
                    int cache_dtype, void* stream);

/* Checks of qd_gqa_decode_q8 in order. */
int qd_gqa_decode_q8_validate(const qd_tensor_desc* q, const qd_tensor_desc* k_cache, const qd_tensor_desc* v_cache,
                              const qd_tensor_desc* k_scales, const qd_tensor_desc* v_scales,
                              const qd_tensor_desc* block_table, const qd_tensor_desc* context_lens, double scale,
                              char* msg, size_t msg_cap);

/* Workspace bytes of qd_gqa_decode_q8 (partials of split contexts); 0 when
 * none is needed.  16-byte aligned, no zeroing needed: every call writes what it
 * reads.  Calls that can overlap need different workspaces.  Depends on the
 * current device, like the launch. */
size_t qd_gqa_decode_q8_workspace_bytes(int batch, int q_heads, int kv_heads, int head_dim, int block_size,
                                        int max_pages, int dtype, int flags);

/* What qd_gqa_decode_q8 runs for these shapes on aligned tensors: QD_Q8_*, or
 * -1 for invalid shapes, with *workgroups of the attention kernel. */
enum { QD_Q8_VALU = 0, QD_Q8_MFMA = 1, QD_Q8_MFMA_SPLIT = 2 };
int qd_gqa_decode_q8_info(int batch, int q_heads, int kv_heads, int head_dim, int block_size, int max_pages,
                          int dtype, int flags, int* workgroups);

/* qd_gqa_decode_auto over an 8-bit cache: out [batch, q_heads, head_dim] =
 * softmax(q . (s_k k) * scale) . (s_v v) over the context_lens[b] tokens of
 * each sequence; q and out are 16-bit.  Lengths are clamped to [0, max_pages *
 * block_size] (0: a zero row), page ids to the pool.  Scales may be any float32
 * of a magnitude in [2^-100, 2^100], or 0; a NaN one (qd_kv_append_q8) makes the
 * rows that see its page NaN.  Sums are float32; the matrix-core kernel rounds a
 * softmax weight times s_v to fp16 once, and holds bf16 queries exactly but for what
 * lies below 2^-38 of a head's largest element.  flags: QD_FLAG_FORCE_GENERIC selects the VALU kernel. */
int qd_gqa_decode_q8(const void* q, const void* k_cache, const void* v_cache, const float* k_scales,
                     const float* v_scales, const int32_t* block_table, const int32_t* context_lens, void* out,
                     void* workspace, size_t workspace_bytes, int batch, int q_heads, int kv_heads, int head_dim,
                     int block_size, int max_pages, int64_t num_blocks, int dtype, int cache_dtype, float scale,
                     int flags, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* QD_ATTENTION_H */
