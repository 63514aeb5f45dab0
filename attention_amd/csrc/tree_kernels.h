// Device code of windowed and tree decode shared by the VALU kernel
// (tree_decode.hip) and the matrix-core kernels (tree_mfma_*.hip): what a query
// sees, and the matrix-core kernel itself.  Everything lives in an anonymous
// namespace, so each translation unit keeps its own copy.
#ifndef QD_TREE_KERNELS_H
#define QD_TREE_KERNELS_H

#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include <atomic>

#include "qd_attention.h"
#include "qd_device.h"
#include "tile_device.h"

// Most tokens of a table row; the last 256 below 2^31 are left out, so that
// token numbers, the ends of their tiles and sums with 64 drafts fit 32 bits.
// Whatever reaches further ahead is compared as a distance.
constexpr int32_t kTreeCapacity = INT32_MAX - 255;

// Arguments of the matrix-core kernels, passed between translation units.
struct TreeParams {
  const void* q;
  const void* k;
  const void* v;
  const int32_t* table;
  const int32_t* lens;
  const int64_t* mask;  // null: one query per sequence, the last of its tokens
  void* out;
  float* part;          // partials of split contexts
  int32_t* meta;        // matrix-core kernel: {first workgroup, workgroups} per item
  int B, T, Hq, Hkv, D, P, maxP;
  int64_t num_blocks;
  int window, sinks;
  float sl2;  // scale * log2(e)
  int splits;    // VALU kernel: context splits
  int G, R;      // q-heads per kv-head, rows (queries x G) per (sequence, kv-head)
  int chunks;    // workgroups that share a (sequence, kv-head)'s rows
  int chunk_rows;
  int W;         // workgroups of a balanced launch; 0: one per item
  int pshift;    // log2(P), or -1
  int32_t last_block;  // largest page id that a table entry can hold
  int32_t capacity;    // tokens of a table row, at most kTreeCapacity
};

// Runs the matrix-core kernel for padded head_dim dp (tree_mfma_*.hip); grid
// workgroups.  Returns a hipError_t.
int qd_tree_mfma_launch_f32(const TreeParams& p, int dp, int grid, void* stream);
int qd_tree_mfma_launch_f16(const TreeParams& p, int dp, int grid, void* stream);
int qd_tree_mfma_launch_bf16(const TreeParams& p, int dp, int grid, void* stream);

namespace {

// Tokens of a sequence in its table.
__device__ __forceinline__ int clamp_len(const TreeParams& p, int32_t len) { return min(max(len, 0), p.capacity); }
__device__ __forceinline__ int context_len(const TreeParams& p, int b) { return clamp_len(p, p.lens[b]); }

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

// mask: draft_bits of the query (not read without masks); len: context_len.
__device__ __forceinline__ Row row_view(const TreeParams& p, int b, int len, uint64_t mask) {
  Row r;
  r.len = len;
  r.seen = 0;
  int depth = -1;
  if (p.mask) {
    const uint64_t m = mask;
    if (m == 0) {  // padding
      r.len = r.lo = r.sinks = 0;
      return r;
    }
    depth = __builtin_popcountll(m) - 1;
    // Drafted tokens past the table are not seen.
    const int room = p.capacity - r.len;
    r.seen = room >= 64 ? m : room > 0 ? m & ((uint64_t{1} << room) - 1) : 0;
    // The window hides drafted tokens only where it is shorter than a path.
    if (p.window > 0 && p.window <= depth + 1)
      for (uint64_t left = r.seen; left; left &= left - 1) {
        const int j = __builtin_ctzll(left);
        const int dj = __builtin_popcountll(draft_bits(p, b, j)) - 1;
        if (dj <= depth - p.window && r.len + dj >= p.sinks) r.seen &= ~(uint64_t{1} << j);
      }
  }
  const int lo = p.window > 0 ? r.len + depth - p.window + 1 : 0;
  r.lo = min(max(lo, 0), r.len);
  r.sinks = min(p.sinks, r.lo);
  return r;
}

// Pool row of token `tok`; page ids are clamped to the pool.
__device__ __forceinline__ int64_t pool_row(const TreeParams& p, int b, int tok) {
  const int page = p.pshift >= 0 ? tok >> p.pshift : tok / p.P;
  int64_t phys = p.table[static_cast<int64_t>(b) * p.maxP + page];
  phys = phys < 0 ? 0 : phys >= p.num_blocks ? p.num_blocks - 1 : phys;
  return phys * p.P + (tok - page * p.P);
}


// ----------------------------------------------------------------------------
// The matrix-core kernel
// ----------------------------------------------------------------------------
//
// An item is a (sequence, kv-head, chunk of its rows); a row is a (query,
// q-head of the kv-head's group).  A workgroup of NW waves goes through an
// item's virtual tokens in tiles of TT: K and V rows come straight into one of
// two LDS buffers (global_load_lds), one tile ahead, and wave (wr, wt) multiplies row blocks [16 NB wr, 16 NB (wr + 1)) with tokens [TT / WT
// wt, ...), at most 32 of them at a time:
//   scores   S^T = K Q^T, 16x16 blocks (A = K rows from LDS, B = Q from
//            registers): a lane holds one row and 4 tokens per block
//   softmax  per lane; the reference maximum of a row moves only when a score
//            exceeds it by 2^8 (fp16: by 2), so most tiles exchange nothing
//            between lanes
//   output   O^T += V^T P^T: the score layout is already the B operand, V^T
//            comes from transposing LDS reads.  16-bit weights go in as two
//            parts (split2): one rounding would add an error as large as the
//            output's own.
// Waves that share rows (WT > 1) merge at the end of an item through LDS.
//
// K and V are read once per chunk of rows, scores never leave registers.  With
// few rows HBM bounds the kernel, with many the issue of matrix and vector
// instructions: a 16x16 step of 32 tokens takes 3 matrix instructions of 16
// cycles per 16 columns (two parts of the weights) and about 50 cycles of vector
// instructions per score register, and two waves of a SIMD overlap them only
// in part.  Measured, bf16, heads of 128, pages of 16:
//   64 sequences, window 1024, 4 rows        48 us, 5.5 TB/s
//   16 sequences, window 32768, 8 rows       341 us, 6.3 TB/s
//   32 sequences, trees of 16, 64 rows       75 us, 4.2 TB/s
//   8 sequences, trees of 64, 512 rows       270 us, 474 TFLOP/s of QK^T and PV
//   fp32, 8 sequences, trees of 8, 32 rows   27 us
// Tried without gain: software pipelining of a wave's scores, softmax and values
// (302 to 340 us for trees of 64: the registers of two steps spill), barriers
// that make the two waves of a SIMD take turns at products and softmax (356 us),
// later K operands read under the last products of V (no change), 64-token
// tiles with eight waves, loads spread over a step.
//
// Balanced launches: an item costs its tiles and this many more (its queries,
// first round trips and stores take about as long; 2 instead of 4: trees of 16
// over 32 sequences 75 -> 81 us).
constexpr int kTreeItemCost = 4;
// Partials of an item, on average, from which the merge gives each row a whole
// workgroup (one sequence of 20000 tokens, 81 partials: 74.6 -> 38.2 us; 24
// items with 6 partials of 256 rows: 43.8 -> 50.2 us).
constexpr int kTreeManyPartials = 8;
// Sequences whose prefix of costs fits the kernel's LDS.
constexpr int kTreeMaxBalanced = 1024;
// Page ids that the kernel keeps in LDS at a time, one for each group of 16
// tokens (one for each token where pages do not hold whole groups).
constexpr int kTreePages = 1024;

// Padded head_dim of an instance; es: element size.
__host__ __device__ constexpr int tree_padded(int es, int d) {
  return d <= 64 ? 64 : d <= 96 ? 96 : d <= 128 ? 128 : d <= 192 && es == 2 ? 192 : 256;
}
// Tokens of a tile: a wave works on 16 to 128 of them, so that what it does
// once per tile stays small beside its products.
__host__ __device__ constexpr int tree_tile(int slots, int nw) {
  return slots == 64 ? 32 : slots <= 16 && nw == 8 ? 128 : 64;
}
// Least cost of a workgroup's range: shorter ones gain less than their
// partials cost (2 against 4: one sequence of 20000 tokens, rows of 512 bytes,
// 31.9 / 36.6 us, fp32 trees of 8 over 8 sequences 27.1 / 31.3 us; rows of 256
// bytes, 8 drafts over 8 sequences of 200 to 400 tokens, 20.6 / 18.8 us).
__host__ __device__ constexpr int tree_min_cost(int slots) { return slots >= 32 ? 2 : 4; }
// The most rows of a chunk: what the registers hold.
__host__ __device__ constexpr int tree_most_rows(int slots) { return slots <= 16 ? 256 : slots == 32 ? 128 : 32; }

// Row blocks per wave, waves along the rows and waves of a workgroup for a
// chunk of rows.  Two waves share a SIMD, of two workgroups or of one with eight
// waves, except where a row of LDS is 512 bytes or longer.  Eight waves on up to
// 64 rows took 123 us where four take 95 (trees of 16), four on 512 rows 619
// where eight take 335 (trees of 64); one row block of 16 per wave instead of
// two doubles the LDS reads per product.
struct TreeWaves {
  int nb, wr, nw;
};
__host__ __device__ constexpr TreeWaves tree_waves(int slots, int rows) {
  return slots == 64    ? TreeWaves{1, 2, 4}
         : rows <= 16   ? TreeWaves{1, 1, 4}
         : rows <= 32   ? TreeWaves{2, 1, 4}
         : slots == 32  ? (rows <= 64 ? TreeWaves{1, 4, 8} : TreeWaves{1, 8, 8})
         : rows <= 64   ? TreeWaves{2, 2, 4}
         : rows <= 128  ? TreeWaves{2, 4, 8}
                        : TreeWaves{2, 8, 8};
}
// Tiles in LDS, of K and V each.  Four where they fit (heads of 64, more than 64
// rows) made no call faster (64 drafts x 8 heads of 64: 115 us, 108 us with two).
constexpr int kTreeBufs = 2;
__host__ __device__ constexpr int tree_lds_bytes(int slots, int nw) {
  return kTreeBufs * 2 * tree_tile(slots, nw) * slots * 16 + 4 * kTreePages + 32;
}
// Resident workgroups per CU, which the launch bounds ask for (three of heads
// of 64 and up to 16 rows: 37.0 us, two 31.2 us, for 128 windows of 512).
__host__ __device__ constexpr int tree_occupancy(int slots, int nw) {
  const int by_lds = 160 * 1024 / (tree_lds_bytes(slots, nw) + 4 * kTreeMaxBalanced);
  const int by_regs = nw == 8 || slots >= 32 ? 1 : 2;
  return by_lds < by_regs ? by_lds : by_regs;
}

template <int DT, int DP, int NB, int WR, int NW>
struct TreeShape {
  static constexpr int kES = DT == QD_DTYPE_F32 ? 4 : 2;
  static constexpr int kSlots = tile_slots(kES, DP);
  static constexpr int TT = tree_tile(kSlots, NW);
  static constexpr int kWT = NW / WR;
  static constexpr int kRow = kSlots * 16;                   // bytes of an LDS row
  static constexpr int kTile = TT * kRow;                    // bytes of K or V
  static constexpr int kLoadRows = TT / NW;                  // rows that a wave loads
  static constexpr int kLoads = kLoadRows * kSlots / 64;     // its instructions, for K and for V
  static constexpr int kSteps = DP * kES / 64;
  static constexpr int kTW = TT / kWT;                       // tokens of a wave in a tile
  static constexpr int kTB = kTW >= 32 ? 2 : 1;              // 16-token blocks at a time
  static constexpr int kSub = kTW / (16 * kTB);
  static constexpr int kCols = DP / 16;
  // LDS reads ahead of their products, in steps of the scores and columns of
  // the output.
  static constexpr int kQkAhead = kSteps < 4 ? kSteps : 4;
  static constexpr int kPvAhead = kES == 2 ? 4 : 2;
  static constexpr int kRows = 16 * NB * WR;                 // rows of a workgroup
  static constexpr int kLds = tree_lds_bytes(kSlots, NW);
  static constexpr int kOcc = tree_occupancy(kSlots, NW);
  static_assert(kTW >= 16 && kLoadRows * kSlots % 64 == 0 && kOcc >= 1, "waves do not fit the tile");
};

__device__ __forceinline__ float tree_max_groups(float x) {
  const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  x = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
  const auto b = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}

__device__ __forceinline__ float tree_sum_groups(float x) {
  const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  x = __uint_as_float(a[0]) + __uint_as_float(a[1]);
  const auto b = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}

// Inclusive prefix sum over the wave's 64 lanes (the DPP scan of
// wave_incl_scan_small).
__device__ __forceinline__ int tree_wave_scan(int x) {
  x = dpp_add_i32<0x111, 0xF>(x);  // row_shr:1
  x = dpp_add_i32<0x112, 0xF>(x);  // row_shr:2
  x = dpp_add_i32<0x114, 0xF>(x);  // row_shr:4
  x = dpp_add_i32<0x118, 0xF>(x);  // row_shr:8
  x = dpp_add_i32<0x142, 0xA>(x);  // row_bcast:15
  return dpp_add_i32<0x143, 0xC>(x);  // row_bcast:31
}

// Or and maximum over the wave, in every lane: within rows of 16 lanes by DPP,
// across them by lane swaps (no LDS round trips).
template <int CTRL>
__device__ __forceinline__ uint32_t tree_dpp(uint32_t x) {
  return static_cast<uint32_t>(__builtin_amdgcn_update_dpp(static_cast<int>(x), static_cast<int>(x), CTRL, 0xF, 0xF, false));
}
template <typename F>
__device__ __forceinline__ uint32_t tree_wave_reduce(uint32_t x, F&& f) {
  x = f(x, tree_dpp<0xB1>(x));   // quad_perm [1,0,3,2]
  x = f(x, tree_dpp<0x4E>(x));   // quad_perm [2,3,0,1]
  x = f(x, tree_dpp<0x141>(x));  // row_half_mirror
  x = f(x, tree_dpp<0x140>(x));  // row_mirror
  const auto a = __builtin_amdgcn_permlane32_swap(x, x, false, false);
  x = f(a[0], a[1]);
  const auto b = __builtin_amdgcn_permlane16_swap(x, x, false, false);
  return f(b[0], b[1]);
}

template <int DT>
__device__ __forceinline__ uint32_t tree_pack(float x, float y) {
  if constexpr (DT == QD_DTYPE_F32)
    return 0;  // not called
  else
    return MfmaOps<DT>::pack2(x, y);
}

// Zeroes the elements of x that are Inf or NaN; returns whether there were any.
template <int DT>
__device__ __forceinline__ bool drop_not_finite(u32x4& x) {
  bool bad = false;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (DT == QD_DTYPE_F32) {
      if ((x[i] & 0x7F800000u) == 0x7F800000u) {
        x[i] = 0;
        bad = true;
      }
    } else {
      constexpr uint32_t e = DT == QD_DTYPE_F16 ? 0x7C00u : 0x7F80u;
      if ((x[i] & e) == e) {
        x[i] &= 0xFFFF0000u;
        bad = true;
      }
      if ((x[i] & (e << 16)) == e << 16) {
        x[i] &= 0x0000FFFFu;
        bad = true;
      }
    }
  }
  return bad;
}

// Tokens [0, sinks) and [lo, len) and nd drafted ones of an item: what its
// rows see at most (first tokens below `seen_sinks`, the others from `seen_lo`
// on), widened to whole groups of 16 tokens where pages hold whole groups: a
// wave then loads its rows from one page.
struct Span {
  int len, lo, sinks, nd, n;
  int seen_lo, seen_sinks;
};

__device__ __forceinline__ Span span_of(const TreeParams& p, int len) {
  Span s;
  s.len = len;
  s.nd = p.mask ? min(p.T, p.capacity - s.len) : 0;
  // The first query's window is the earliest: position len, or len - 1
  // without a mask.
  const int lo = p.window > 0 ? s.len + (p.mask ? 1 : 0) - p.window : 0;
  s.seen_lo = min(max(lo, 0), s.len);
  s.seen_sinks = min(p.sinks, s.seen_lo);
  s.lo = s.seen_lo;
  s.sinks = s.seen_sinks;
  if (p.P % 16 == 0) {
    s.lo &= ~15;
    s.sinks = min((s.sinks + 15) & ~15, s.lo);
  }
  s.n = s.sinks + s.len - s.lo + s.nd;
  return s;
}

__device__ __forceinline__ Span item_span(const TreeParams& p, int b) { return span_of(p, context_len(p, b)); }

template <int TT>
__device__ __forceinline__ int span_tiles(const Span& s) {
  return (s.n + TT - 1) / TT;
}

template <int DT, int DP, int NB, int WR, int NW>
__global__ __launch_bounds__(64 * NW, (TreeShape<DT, DP, NB, WR, NW>::kOcc * NW / 4)) void tree_mfma_kernel(TreeParams p) {
  using Sh = TreeShape<DT, DP, NB, WR, NW>;
  using E = Elem<DT>;
  using S = typename E::S;
  constexpr bool k16 = DT != QD_DTYPE_F32;
  constexpr int WT = Sh::kWT, TB = Sh::kTB, ES = Sh::kES;
  // A row's reference maximum moves when a score exceeds it by 2^kLazy; weights
  // are relative to it, times 2^kShift.  fp16 parts of a weight are multiples of
  // 2^-24, the low one at least that (split2), so what they add to a weight too
  // small for them is at most 2^-(24 + kShift) of the largest one; kShift + kLazy
  // = 15 keeps the largest inside fp16.  7 and 8 instead left 2^-31, 3e-5 of the
  // values of 65536 tokens without a weight (8 sequences, trees of 64, 64 heads
  // of 128, whose scores spread widely: 290 us, 299 us with 14 and 1; windows and
  // trees of 16 within 1%).
  constexpr float kShift = DT == QD_DTYPE_F16 ? 14.f : 0.f;
  constexpr float kLazy = DT == QD_DTYPE_F16 ? 1.f : 8.f;
  extern __shared__ __align__(16) char smem[];
  // Tokens with non-finite values that not all rows see: drafted ones, and
  // those at the window's edge (bit i: token seen_lo + i).
  unsigned long long* bad_words = reinterpret_cast<unsigned long long*>(smem + kTreeBufs * 2 * Sh::kTile);
  int32_t* pages = reinterpret_cast<int32_t*>(bad_words + 4);
  int32_t* incl = reinterpret_cast<int32_t*>(smem + Sh::kLds);
  const int tid = static_cast<int>(threadIdx.x);
  const int lane = tid & 63;
  const int wv = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wr = wv / WT, wt = wv % WT;
  const int per_seq = p.Hkv * p.chunks;
  auto process = [&](int b, int hc, const Span& sp, int t0, int t1, bool whole, int64_t slot) {
    // Opaque copies: what is derived from them (masks and offsets per column)
    // would otherwise be computed ahead of the first item and kept in registers
    // from item to item.
    int dim = p.D, lane = static_cast<int>(threadIdx.x) & 63;
    asm volatile("" : "+s"(dim), "+v"(lane));
    int r16 = lane & 15, g4 = lane >> 4;
    const int row_bytes = dim * ES;
    const int h = hc / p.chunks;
    const int row0 = (hc % p.chunks) * p.chunk_rows;
    const int rows = min(p.chunk_rows, p.R - row0);
    const int q0 = row0 / p.G, q1 = (row0 + rows - 1) / p.G;  // the chunk's queries
    const int context = sp.sinks + sp.len - sp.lo;
    auto token = [&](int v) { return v < sp.sinks ? v : sp.lo + (v - sp.sinks); };
    auto page_of = [&](int tok) { return p.pshift >= 0 ? tok >> p.pshift : tok / p.P; };
    const int last_page = sp.n > 0 ? page_of(token(sp.n - 1)) : 0;
    const int32_t* table = p.table + static_cast<int64_t>(b) * p.maxP;
    auto clamped = [&](int32_t phys) { return static_cast<uint32_t>(min(max(phys, 0), p.last_block)); };
    const uint32_t tok_bytes = static_cast<uint32_t>(p.Hkv) * row_bytes, page_bytes = tok_bytes * p.P;
    // Place of this lane's 16 bytes of load i in a group of rows of one page.
    // Slots past the head (head_dims below the row's power of two) are left
    // out; K's are cleared once, below, since its products run over them.
    const bool padded = row_bytes < Sh::kRow;
    uint32_t lane_off[Sh::kLoads];
#pragma unroll
    for (int i = 0; i < Sh::kLoads; ++i) {
      const int r = (64 * i + lane) / Sh::kSlots;
      lane_off[i] = r * tok_bytes + h * row_bytes +
                    16 * ((lane & (Sh::kSlots - 1)) ^ tile_swizzle(Sh::kSlots, Sh::kLoadRows * wv + r));
    }
    auto inside = [&](int i) {
      const int r = (64 * i + lane) / Sh::kSlots;
      return 16 * ((lane & (Sh::kSlots - 1)) ^ tile_swizzle(Sh::kSlots, Sh::kLoadRows * wv + r)) < row_bytes;
    };
    const uint32_t lds_wave = tile_lds_address(smem) + Sh::kLoadRows * wv * Sh::kRow;
    const bool grouped = p.P % 16 == 0;
    // The page list from a tile on: read, then put into LDS; it covers
    // list_tiles tiles.
    constexpr int kEach = kTreePages / (64 * NW);
    const int each = grouped ? 16 : 1, list_tiles = kTreePages * each / Sh::TT;
    struct Pages {
      int32_t id[kEach];
    };
    auto read_pages = [&](int tile) {
      // The list reaches up to 16 kTreePages tokens past the tile, which may pass
      // 2^31: only a place below `left` is added to the tile's first token.
      const int first = Sh::TT * tile, left = min(sp.n, Sh::TT * t1) - first;
      Pages x;
#pragma unroll
      for (int i = 0; i < kEach; ++i) {
        const int ahead = each * (64 * NW * i + tid);
        x.id[i] = 0;
        if (ahead < left) x.id[i] = table[page_of(token(first + ahead))];
      }
      return x;
    };
    auto put_pages = [&](const Pages& x) {
#pragma unroll
      for (int i = 0; i < kEach; ++i) pages[64 * NW * i + tid] = min(max(x.id[i], 0), p.last_block);
    };
    // Place of this wave's rows of a tile in the list that starts at tile
    // `base`.  Groups past the last token take its page.
    auto list_at = [&](int tile, int base) {
      const int at = Sh::TT * (tile - base) + Sh::kLoadRows * wv;
      return grouped ? min(at, sp.n - 1 - Sh::TT * base) / 16 : at;
    };
    // Loads of this wave's rows of a tile, from page `phys` (grouped) or from the
    // listed ones (`at`: this wave's first), piece by piece.  Rows past the last
    // token and drafted tokens that no row sees are loaded from some page of
    // the pool; they are cleared before they are used.
    struct TileLoad {
      const char* k;
      const char* v;
      int v0, at;
      uint32_t to;
    };
    auto tile_load = [&](int tile, int slot, int32_t phys, int at) {
      TileLoad x;
      x.v0 = Sh::TT * tile + Sh::kLoadRows * wv;
      x.at = at;
      x.to = __builtin_amdgcn_readfirstlane(lds_wave + slot * 2 * Sh::kTile);
      x.k = static_cast<const char*>(p.k);
      x.v = static_cast<const char*>(p.v);
      if (grouped) {
        const int tok0 = token(x.v0);
        const int64_t off = readlane_i64(  // the same in all lanes: scalar registers
            static_cast<int64_t>(static_cast<uint64_t>(static_cast<uint32_t>(phys)) * page_bytes +
                                 static_cast<uint32_t>(p.pshift >= 0 ? tok0 & (p.P - 1) : tok0 % p.P) * tok_bytes),
            0);
        x.k += off;
        x.v += off;
      }
      return x;
    };
    auto load_piece = [&](const TileLoad& x, int i) {
      const uint32_t to = x.to + 1024 * i;
      if (grouped && !padded) {
        // Not kept in the caches where no other chunk reads the rows (316 MB of
        // K and V 75 us, kept 82 us; 2.1 GB 341 / 381 us).
        if (p.chunks == 1) {
          tile_load_lds<true>(x.k, lane_off[i], to);
          tile_load_lds<true>(x.v, lane_off[i], to + Sh::kTile);
        } else {  // the other chunks read the same rows
          tile_load_lds<false>(x.k, lane_off[i], to);
          tile_load_lds<false>(x.v, lane_off[i], to + Sh::kTile);
        }
        return;
      }
      uint64_t off = lane_off[i];
      if (!grouped) {
        const int r = (64 * i + lane) / Sh::kSlots;
        const int v = min(x.v0 + r, sp.n - 1), tok = token(v);
        off += static_cast<uint64_t>(static_cast<uint32_t>(pages[x.at + v - x.v0])) * page_bytes +
               static_cast<uint32_t>(tok - page_of(tok) * p.P) * tok_bytes - r * tok_bytes;
      }
      // Padded heads and pages of no whole groups: never kept, also where other
      // chunks read the same rows (not measured against keeping them).
      if (inside(i)) {
        tile_load_lds<true>(x.k + off, to);
        tile_load_lds<true>(x.v + off, to + Sh::kTile);
      }
    };

    // This lane's rows: what they see is taken from lane (query - q0).
    int query[NB];
    bool real[NB];
    u32x4 qf[NB][Sh::kSteps];
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
      const int rr = 16 * (NB * wr + nb) + r16;
      real[nb] = rr < rows;
      const int row = row0 + (real[nb] ? rr : 0);
      query[nb] = row / p.G;
      const char* src =
          static_cast<const char*>(p.q) +
          ((static_cast<int64_t>(b) * p.T + query[nb]) * p.Hq + static_cast<int64_t>(h) * p.G + (row - query[nb] * p.G)) *
              row_bytes;
#pragma unroll
      for (int s = 0; s < Sh::kSteps; ++s) {
        const int at = 64 * s + 16 * g4;
        qf[nb][s] = real[nb] && at < row_bytes ? *reinterpret_cast<const u32x4*>(src + at) : u32x4{0u, 0u, 0u, 0u};
      }
    }
    // The first tile.  Its pages come through the scalar cache where one page
    // serves a wave's rows; the list takes a barrier.
    tile_barrier();  // the previous item's merge and the prefix are done with LDS
    if (tid < 2) bad_words[tid] = 0;
    if (padded) {
      for (int i = tid; i < kTreeBufs * Sh::kTile / 16; i += 64 * NW)
        *(reinterpret_cast<u32x4*>(smem + i / (Sh::kTile / 16) * 2 * Sh::kTile) + i % (Sh::kTile / 16)) = u32x4{0u, 0u, 0u, 0u};
    }
    int list_base = grouped ? t0 + 1 : t0;
    const Pages listed = read_pages(list_base);
    uint64_t my_mask = 0;
    if (p.mask && q0 + lane <= q1) my_mask = draft_bits(p, b, q0 + lane);
    if (!grouped) put_pages(listed);
    if (padded || !grouped) tile_barrier();
    if (t0 < t1) {
      int32_t phys = 0;
      if (grouped)
        phys = min(max(tile_scalar_load(table + min(page_of(token(Sh::TT * t0 + Sh::kLoadRows * wv)), last_page)), 0),
                   p.last_block);
      const TileLoad x = tile_load(t0, 0, phys, list_at(t0, t0));
#pragma unroll
      for (int j = 0; j < Sh::kLoads; ++j) load_piece(x, j);
    }
    if (grouped) put_pages(listed);
    // Lane t: what query q0 + t sees (at most 64 queries).
    Row mine;
    mine.len = mine.lo = mine.sinks = 0;
    mine.seen = 0;
    bool sees = false;
    if (q0 + lane <= q1) {
      sees = !p.mask || my_mask != 0;
      if (sees) mine = row_view(p, b, sp.len, my_mask);
    }
    auto bits_or = [](uint32_t x, uint32_t y) { return x | y; };
    const uint32_t seen_low = __builtin_amdgcn_readfirstlane(tree_wave_reduce(static_cast<uint32_t>(mine.seen), bits_or));
    const uint32_t seen_high = __builtin_amdgcn_readfirstlane(tree_wave_reduce(static_cast<uint32_t>(mine.seen >> 32), bits_or));
    const uint64_t any_seen = static_cast<uint64_t>(seen_high) << 32 | seen_low;
    const int lo_max = __builtin_amdgcn_readfirstlane(
        tree_wave_reduce(sees ? mine.lo : 0, [](uint32_t x, uint32_t y) { return x > y ? x : y; }));
    f32x4 acc[Sh::kCols][NB];
    float m[NB], l[NB];
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
      m[nb] = -INFINITY;
      l[nb] = 0.f;
#pragma unroll
      for (int c = 0; c < Sh::kCols; ++c) acc[c][nb] = f32x4{0.f, 0.f, 0.f, 0.f};
    }

    const int edge = sp.sinks + max(lo_max - sp.lo, 0);  // virtual tokens below: not in every row's window
    // Tokens between these: in no row's window.  The chunk's only query may be a
    // later one than the sequence's first.
    const int lo_all = q0 == q1 ? lo_max : sp.seen_lo, sinks_all = q0 == q1 ? min(p.sinks, lo_max) : sp.seen_sinks;
    // No register load is pending when the loop starts: the compiler would
    // wait for it, and so for the tiles in flight, in every turn.
    __builtin_amdgcn_s_waitcnt((0x7 << 4) | (0xF << 8));  // vmcnt(0)
    int slot_now = 0;
    for (int tile = t0; tile < t1; ++tile) {
      // The tile has arrived, and every wave is done with the one before it.
      tile_barrier_loads<0>();
      const int next = tile + 1;
      if (next < t1) {
        if (next >= list_base + list_tiles) {
          list_base = next;
          put_pages(read_pages(next));
          tile_barrier();
        }
        const int at = list_at(next, list_base);
        const TileLoad x = tile_load(next, slot_now ^ 1, grouped ? __builtin_amdgcn_readfirstlane(pages[at]) : 0, at);
#pragma unroll
        for (int j = 0; j < Sh::kLoads; ++j) load_piece(x, j);
      }
      char* buf = smem + slot_now * 2 * Sh::kTile;
      slot_now ^= 1;
      // Every row of the chunk sees all (existing) tokens of the tile.
      const int first = Sh::TT * tile, stop = first + Sh::TT;
      const bool whole_tile = stop <= sp.seen_sinks || (first >= edge && (stop <= context || (p.T == 1 && stop <= sp.n)));
      if (!whole_tile) {
        // Values of tokens that no row sees are cleared.  Where only some rows
        // see a token, a weight of 0 would not hide Inf and NaN from the
        // others: they are left out here and join the rows that do at the
        // item's end.  Slots past a padded head are looked at too: what LDS held
        // there may list a token in bad_words for nothing, which costs time at
        // the item's end (only values that are not finite are added).
        for (int i = tid; i < Sh::TT * Sh::kSlots; i += 64 * NW) {
          const int v = first + i / Sh::kSlots, tok = token(v);
          u32x4* at = reinterpret_cast<u32x4*>(buf + Sh::kTile) + i;
          if (v < context ? tok >= sinks_all && tok < lo_all : v >= sp.n || !((any_seen >> (v - context)) & 1)) {
            *at = u32x4{0u, 0u, 0u, 0u};
          } else if (q0 != q1 && (v >= context || (tok >= sp.seen_lo && tok < lo_max))) {
            u32x4 x = *at;
            if (drop_not_finite<DT>(x)) {
              *at = x;
              atomicOr(&bad_words[v >= context ? 0 : 1], 1ull << (v >= context ? v - context : tok - sp.seen_lo));
            }
          }
        }
        tile_barrier();
      }

#pragma unroll 1
      for (int sub = 0; sub < Sh::kSub; ++sub) {
        const int wave_tok = Sh::kTW * wt + 16 * TB * sub;
        const uint32_t at = tile_lds_address(buf) + wave_tok * Sh::kRow;
        const uint32_t kb = at + r16 * Sh::kRow + 16 * (g4 ^ tile_swizzle(Sh::kSlots, r16));
        f32x4 s[TB][NB];
#pragma unroll
        for (int tb = 0; tb < TB; ++tb)
#pragma unroll
          for (int nb = 0; nb < NB; ++nb) s[tb][nb] = f32x4{0.f, 0.f, 0.f, 0.f};
        // The matrix cores' phases go before another wave's softmax (trees of
        // 64: 277 -> 270 us).
        __builtin_amdgcn_s_setprio(1);
        // Operands are read ahead of their products: a product takes 16 cycles,
        // an LDS read here well over 100.  The scheduling barriers keep the
        // distance.
        u32x4 ka[Sh::kQkAhead][TB];
        auto read_k = [&](int st) {
#pragma unroll
          for (int tb = 0; tb < TB; ++tb)
            ka[st % Sh::kQkAhead][tb] = tile_lds_read<u32x4>((kb ^ (64 * st)) + 16 * tb * Sh::kRow);
        };
#pragma unroll
        for (int st = 0; st < Sh::kQkAhead; ++st) read_k(st);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int st = 0; st < Sh::kSteps; ++st) {
#pragma unroll
          for (int tb = 0; tb < TB; ++tb) {
            const u32x4 a = ka[st % Sh::kQkAhead][tb];
#pragma unroll
            for (int nb = 0; nb < NB; ++nb) {
              if constexpr (k16) {
                s[tb][nb] = MfmaOps<DT>::mma32(a, qf[nb][st], s[tb][nb]);
              } else {
#pragma unroll
                for (int j = 0; j < 4; ++j)
                  s[tb][nb] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(a[j]), __uint_as_float(qf[nb][st][j]),
                                                                   s[tb][nb], 0, 0, 0);
              }
            }
          }
          if (st + Sh::kQkAhead < Sh::kSteps) read_k(st + Sh::kQkAhead);
          __builtin_amdgcn_sched_barrier(0);
        }
        __builtin_amdgcn_s_setprio(0);
        // V^T of the first columns, in flight during the softmax.
        const uint32_t vb = at + Sh::kTile;
        const int vr = 4 * g4 + (k16 ? r16 >> 2 : 0);
        const uint32_t va =
            k16 ? vb + vr * Sh::kRow + 16 * (((r16 >> 1) & 1) ^ tile_swizzle(Sh::kSlots, vr)) + 8 * (r16 & 1) : vb;
        u32x2 vf[Sh::kPvAhead][2 * TB];  // fp32: 4 TB values
        auto read_v = [&](int c) {
#pragma unroll
          for (int tb = 0; tb < TB; ++tb) {
            if constexpr (k16) {
              vf[c % Sh::kPvAhead][tb] = tile_tr_read((va ^ (32 * c)) + 16 * tb * Sh::kRow);
            } else {
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                const int row = 4 * g4 + i;
                const uint32_t col = vb + row * Sh::kRow + 16 * ((r16 >> 2) ^ tile_swizzle(Sh::kSlots, row)) + 4 * (r16 & 3);
                vf[c % Sh::kPvAhead][2 * tb + i / 2][i % 2] =
                    tile_lds_read<uint32_t>((col ^ (64 * c)) + 16 * tb * Sh::kRow);
              }
            }
          }
        };
#pragma unroll
        for (int c = 0; c < Sh::kPvAhead; ++c) read_v(c);
        __builtin_amdgcn_sched_barrier(0);
        uint32_t vis[TB][NB];  // bits of this lane's 4 tokens of a block that its row sees
        if (!whole_tile) {
#pragma unroll
          for (int nb = 0; nb < NB; ++nb) {
            const int src = query[nb] - q0;
            const int sinks = __shfl(mine.sinks, src);
            const int lo = __shfl(mine.lo, src) - (sp.lo - sp.sinks);  // as a virtual token
            const uint64_t seen = static_cast<uint64_t>(__shfl(static_cast<long long>(mine.seen), src));
#pragma unroll
            for (int tb = 0; tb < TB; ++tb) {
              const int v = first + wave_tok + 16 * tb + 4 * g4;
              auto below = [&](int end) { return (1u << min(max(end - v, 0), 4)) - 1; };  // tokens before `end`
              const int j = v - context;
              const uint32_t drafts = j <= -4 || j >= 64 ? 0u
                                      : j < 0            ? static_cast<uint32_t>(seen) << -j
                                                         : static_cast<uint32_t>(seen >> j);
              vis[tb][nb] = below(sinks) | (below(context) & ~below(lo)) | drafts;
#pragma unroll
              for (int i = 0; i < 4; ++i) s[tb][nb][i] = (vis[tb][nb] >> i) & 1 ? s[tb][nb][i] : -INFINITY;
            }
          }
        }
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) {
          float mx = -INFINITY;
#pragma unroll
          for (int tb = 0; tb < TB; ++tb)
#pragma unroll
            for (int i = 0; i < 4; ++i) mx = fmaxf(mx, s[tb][nb][i]);
          if (__ballot(mx * p.sl2 > m[nb] + kLazy)) {
            const float mn = fmaxf(m[nb], tree_max_groups(mx) * p.sl2);
            const float alpha = mn == m[nb] ? 1.f : fast_exp2(m[nb] - mn);
            m[nb] = mn;
            l[nb] *= alpha;
#pragma unroll
            for (int c = 0; c < Sh::kCols; ++c) acc[c][nb] *= alpha;
          }
          const float ref = m[nb] == -INFINITY ? kShift : kShift - m[nb];
#pragma unroll
          for (int tb = 0; tb < TB; ++tb)
#pragma unroll
            for (int i = 0; i < 4; ++i) s[tb][nb][i] = fast_exp2(fmaf(s[tb][nb][i], p.sl2, ref));
        }
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
#pragma unroll
          for (int tb = 0; tb < TB; ++tb)
            l[nb] += (s[tb][nb][0] + s[tb][nb][1]) + (s[tb][nb][2] + s[tb][nb][3]);
        if constexpr (k16) {
          u32x2 hi[TB][NB], lw[TB][NB];
#pragma unroll
          for (int tb = 0; tb < TB; ++tb)
#pragma unroll
            for (int nb = 0; nb < NB; ++nb)
#pragma unroll
              for (int i = 0; i < 2; ++i) {
                uint32_t a, c;
                MfmaOps<DT>::split2(s[tb][nb][2 * i], s[tb][nb][2 * i + 1], a, c);
                hi[tb][nb][i] = a;
                lw[tb][nb][i] = c;
              }
          // split2's low part is never 0: cleared where the weight is a hidden
          // token's.
          if (!whole_tile) {
#pragma unroll
            for (int tb = 0; tb < TB; ++tb)
#pragma unroll
              for (int nb = 0; nb < NB; ++nb)
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                  const uint32_t two = vis[tb][nb] >> (2 * i);
                  lw[tb][nb][i] &= (two & 1 ? 0x0000FFFFu : 0u) | (two & 2 ? 0xFFFF0000u : 0u);
                }
          }
          __builtin_amdgcn_sched_barrier(0);
          __builtin_amdgcn_s_setprio(1);
#pragma unroll
          for (int c = 0; c < Sh::kCols; ++c) {
            const u32x2* f = vf[c % Sh::kPvAhead];
            if constexpr (TB == 1) {
#pragma unroll
              for (int nb = 0; nb < NB; ++nb) acc[c][nb] = MfmaOps<DT>::pv(f[0], hi[0][nb], acc[c][nb]);
#pragma unroll
              for (int nb = 0; nb < NB; ++nb) acc[c][nb] = MfmaOps<DT>::pv(f[0], lw[0][nb], acc[c][nb]);
            } else {
              const u32x4 a = {f[0][0], f[0][1], f[1][0], f[1][1]};
#pragma unroll
              for (int nb = 0; nb < NB; ++nb)
                acc[c][nb] =
                    MfmaOps<DT>::mma32(a, u32x4{hi[0][nb][0], hi[0][nb][1], hi[1][nb][0], hi[1][nb][1]}, acc[c][nb]);
#pragma unroll
              for (int nb = 0; nb < NB; ++nb)
                acc[c][nb] =
                    MfmaOps<DT>::mma32(a, u32x4{lw[0][nb][0], lw[0][nb][1], lw[1][nb][0], lw[1][nb][1]}, acc[c][nb]);
            }
            if (c + Sh::kPvAhead < Sh::kCols) {
              read_v(c + Sh::kPvAhead);
              __builtin_amdgcn_sched_barrier(0);
            }
          }
        } else {
#pragma unroll
          for (int c = 0; c < Sh::kCols; ++c) {
#pragma unroll
            for (int tb = 0; tb < TB; ++tb)
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                const float a = __uint_as_float(vf[c % Sh::kPvAhead][2 * tb + i / 2][i % 2]);
#pragma unroll
                for (int nb = 0; nb < NB; ++nb)
                  acc[c][nb] = __builtin_amdgcn_mfma_f32_16x16x4f32(a, s[tb][nb][i], acc[c][nb], 0, 0, 0);
              }
            if (c + Sh::kPvAhead < Sh::kCols) {
              read_v(c + Sh::kPvAhead);
              __builtin_amdgcn_sched_barrier(0);
            }
          }
        }
        __builtin_amdgcn_s_setprio(0);
      }
    }

    // The item's end: its rows' sums, and the output or a partial.
    asm volatile("" : "+s"(dim), "+v"(lane), "+v"(r16), "+v"(g4));
    tile_barrier();
    float sum[NB], scale[NB];
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) sum[nb] = tree_sum_groups(l[nb]);
    float share[NB][WT];  // factors of the waves' parts of the same rows
    if constexpr (WT > 1) {
      // Every wave leaves its part in LDS, {m, l} of its rows where the page
      // list was, and takes up a share of the columns.
      static_assert(NW * NB * Sh::kCols * 1024 <= kTreeBufs * 2 * Sh::kTile && NW * NB * 128 <= 4 * kTreePages,
                    "the waves' parts fit the tile buffers and the page list");
      f32x2* stats = reinterpret_cast<f32x2*>(pages);
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) {
#pragma unroll
        for (int c = 0; c < Sh::kCols; ++c)
          *reinterpret_cast<f32x4*>(smem + ((wv * NB + nb) * Sh::kCols + c) * 1024 + 16 * lane) = acc[c][nb];
        if (g4 == 0) stats[(wv * NB + nb) * 16 + r16] = f32x2{m[nb], sum[nb]};
      }
      tile_barrier();
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) {
        f32x2 ml[WT];
        float mx = -INFINITY;
#pragma unroll
        for (int w = 0; w < WT; ++w) {
          ml[w] = stats[((wr * WT + w) * NB + nb) * 16 + r16];
          mx = fmaxf(mx, ml[w][0]);
        }
        const float ref = mx == -INFINITY ? 0.f : mx;
        sum[nb] = 0.f;
#pragma unroll
        for (int w = 0; w < WT; ++w) {
          share[nb][w] = ml[w][0] == mx && mx != -INFINITY ? 1.f : fast_exp2(ml[w][0] - ref);
          sum[nb] += share[nb][w] * ml[w][1];
        }
        m[nb] = mx;
      }
    }
    bool has[NB];
    char* to[NB];  // the row of the output or of the partial
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
      has[nb] = __shfl(static_cast<int>(sees), query[nb] - q0) != 0 && (sum[nb] > 0.f || sum[nb] != sum[nb]);
      scale[nb] = has[nb] ? (whole ? 1.f / sum[nb] : 1.f) : 0.f;
      const int rr = 16 * (NB * wr + nb) + r16;
      if (whole) {
        to[nb] = static_cast<char*>(p.out) +
                 ((static_cast<int64_t>(b) * p.T + query[nb]) * p.Hq + static_cast<int64_t>(h) * p.G +
                  (row0 + rr - query[nb] * p.G)) *
                     row_bytes;
      } else {
        float* part = p.part + slot * (static_cast<int64_t>(Sh::kRows) * (dim + 2));
        to[nb] = reinterpret_cast<char*>(part + static_cast<int64_t>(rr) * dim);
        if (wt == 0 && g4 == 0 && real[nb])
          *reinterpret_cast<f32x2*>(part + static_cast<int64_t>(Sh::kRows) * dim + 2 * rr) =
              has[nb] ? f32x2{m[nb], sum[nb]} : f32x2{-INFINITY, 0.f};
      }
    }
    const uint64_t bad_drafts = static_cast<uint64_t>(readlane_i64(static_cast<int64_t>(bad_words[0]), 0));
    const uint64_t bad_edge = static_cast<uint64_t>(readlane_i64(static_cast<int64_t>(bad_words[1]), 0));
    auto finish = [&](int c, f32x4 (&y)[NB]) {
      const int d = 16 * c + 4 * g4;
      if (bad_drafts | bad_edge) {
        // Inf and NaN that only some rows see: whatever their weight, the sum
        // is no longer finite.
#pragma unroll 1
        for (int kind = 0; kind < 2; ++kind) {
          uint64_t bad = kind == 0 ? bad_drafts : bad_edge;
#pragma unroll 1
          while (bad) {
            const int x = __builtin_ctzll(bad);
            bad &= bad - 1;
            const int tok = kind == 0 ? sp.len + x : sp.seen_lo + x;
            const S* src = reinterpret_cast<const S*>(static_cast<const char*>(p.v) +
                                                      (pool_row(p, b, tok) * p.Hkv + h) * row_bytes);
#pragma unroll
            for (int nb = 0; nb < NB; ++nb) {
              const int from = query[nb] - q0;
              const int lo = __shfl(mine.lo, from), sinks = __shfl(mine.sinks, from);
              const uint64_t seen = static_cast<uint64_t>(__shfl(static_cast<long long>(mine.seen), from));
              if (d < dim && (kind == 0 ? ((seen >> x) & 1) != 0 : tok < sinks || tok >= lo))
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                  const float val = E::to_f(src[d + i]);
                  if (!(fabsf(val) < INFINITY)) y[nb][i] += val;
                }
            }
          }
        }
      }
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) {
        if (!real[nb] || d >= dim) continue;
        const f32x4 z = has[nb] ? y[nb] * scale[nb] : f32x4{0.f, 0.f, 0.f, 0.f};
        if (k16 && whole)
          *reinterpret_cast<u32x2*>(to[nb] + d * 2) = u32x2{tree_pack<DT>(z[0], z[1]), tree_pack<DT>(z[2], z[3])};
        else
          *reinterpret_cast<f32x4*>(to[nb] + d * 4) = z;
      }
    };
    if constexpr (WT > 1) {
#pragma unroll 2
      for (int c = wt * Sh::kCols / WT; c < (wt + 1) * Sh::kCols / WT; ++c) {
        f32x4 y[NB];
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) {
          y[nb] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int w = 0; w < WT; ++w)
            y[nb] += share[nb][w] * *reinterpret_cast<const f32x4*>(
                                        smem + (((wr * WT + w) * NB + nb) * Sh::kCols + c) * 1024 + 16 * lane);
        }
        finish(c, y);
      }
    } else {
#pragma unroll
      for (int c = 0; c < Sh::kCols; ++c) finish(c, acc[c]);
    }
  };

  // Balanced: the costs of all items in a row (below 2^31: the host sees to
  // it), cut into equal ranges.  Up to 64 sequences, every wave keeps the prefix
  // of the costs in its lanes.
  int total = 0, used = 1, pos = 0, end = 1, mine_incl = 0, mine_len = 0;
  const int w = static_cast<int>(blockIdx.x);
  int b = 0;
  const bool in_lanes = p.B <= 64;
  auto prefix = [&](int i) {
    return in_lanes ? __builtin_amdgcn_readlane(mine_incl, i) : __builtin_amdgcn_readfirstlane(incl[i]);
  };
  // a n / d below 2^31; a n is below 2^42, so that the rounded quotient of
  // doubles is never on the wrong side of an integer.
  auto part_of = [](int a, int n, int d) {
    return __builtin_amdgcn_readfirstlane(static_cast<int>(static_cast<double>(a) * n / d));
  };
  if (p.W > 0) {
    auto cost_of = [&](int len) {
      const int tiles = span_tiles<Sh::TT>(span_of(p, len));
      return tiles > 0 ? (tiles + kTreeItemCost) * per_seq : 0;
    };
    if (in_lanes) {
      if (lane < p.B) mine_len = context_len(p, lane);
      mine_incl = tree_wave_scan(lane < p.B ? cost_of(mine_len) : 0);
    } else {
      for (int i = tid; i < p.B; i += 64 * NW) incl[i] = cost_of(context_len(p, i));
      __syncthreads();
      if (wv == 0) {
        int carry = 0;
        for (int base = 0; base < p.B; base += 64) {
          const int i = base + lane;
          const int v = carry + tree_wave_scan(i < p.B ? incl[i] : 0);
          if (i < p.B) incl[i] = v;
          carry = __builtin_amdgcn_readlane(v, 63);
        }
      }
      __syncthreads();
    }
    total = prefix(p.B - 1);
    used = min(p.W, max(1, total / tree_min_cost(Sh::kSlots)));
    if (w >= used) return;
    pos = part_of(w, total, used);
    end = part_of(w + 1, total, used);
    if (in_lanes) {
      b = __builtin_popcountll(__ballot(lane < p.B && mine_incl <= pos));
    } else {
      int lo = 0, hi = p.B - 1;
      while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (incl[mid] > pos) hi = mid; else lo = mid + 1;
      }
      b = __builtin_amdgcn_readfirstlane(lo);
    }
  } else {
    b = static_cast<int>(blockIdx.x) / per_seq;
  }
  while (pos < end) {
    int hc, t0 = 0, t1, tiles, step = 1;
    Span sp;
    if (p.W > 0) {
      while (prefix(b) <= pos) ++b;
      const int before = b > 0 ? prefix(b - 1) : 0;
      const int cost = static_cast<int>(static_cast<uint32_t>(prefix(b) - before) / static_cast<uint32_t>(per_seq));
      hc = static_cast<int>(static_cast<uint32_t>(pos - before) / static_cast<uint32_t>(cost));
      const int off = pos - before - hc * cost;
      const int stop = min(cost, off + (end - pos));
      t0 = max(0, off - kTreeItemCost);
      t1 = max(0, stop - kTreeItemCost);
      tiles = cost - kTreeItemCost;
      step = stop - off;
      if (t1 > t0 && t0 == 0 && tid == 0) {
        // The workgroup w that holds a place x: w total / used <= x.
        const int x = before + hc * cost + cost - 1;  // the item's last tile
        int last = part_of(x, used, total);
        while (last + 1 < used && part_of(last + 1, total, used) <= x) ++last;
        int32_t* meta = p.meta + 2 * (static_cast<int64_t>(b) * per_seq + hc);
        meta[0] = w;
        meta[1] = last - w + 1;
      }
      sp = span_of(p, in_lanes ? __builtin_amdgcn_readlane(mine_len, b) : clamp_len(p, tile_scalar_load(p.lens + b)));
    } else {
      hc = static_cast<int>(blockIdx.x) % per_seq;
      sp = span_of(p, clamp_len(p, tile_scalar_load(p.lens + b)));
      t1 = tiles = span_tiles<Sh::TT>(sp);
    }
    if (t1 > t0 || p.W == 0) process(b, hc, sp, t0, t1, t0 == 0 && t1 == tiles, 2 * static_cast<int64_t>(w) + (t0 == 0 ? 1 : 0));
    pos += step;
  }
}

// Log-sum-exp merge of the items that a balanced launch split, and the rows of
// sequences without any token.  A workgroup of 4 waves serves 16 / LANES rows of
// an item: LANES x 16 lanes per row, 16 of them stride its columns, LANES its
// partials.
// grid (items, row blocks), block 256.
template <int DT, int KROWS, int LANES>
__global__ __launch_bounds__(256) void tree_merge_kernel(TreeParams p) {
  using E = Elem<DT>;
  const int per_seq = p.Hkv * p.chunks;
  const int item = blockIdx.x;
  const int b = item / per_seq, hc = item % per_seq;
  const bool empty = item_span(p, b).n == 0;
  const int first = empty ? 0 : p.meta[2 * static_cast<int64_t>(item)];
  const int count = empty ? 0 : p.meta[2 * static_cast<int64_t>(item) + 1];
  if (count == 1) return;
  const int h = hc / p.chunks, row0 = (hc % p.chunks) * p.chunk_rows;
  const int rows = min(p.chunk_rows, p.R - row0);
  const int l16 = threadIdx.x & 15, group = threadIdx.x >> 4;
  const int rr = 16 / LANES * static_cast<int>(blockIdx.y) + group / LANES, lane = group % LANES;
  if (rr >= rows) return;  // LANES > 1: the whole workgroup
  const int t = (row0 + rr) / p.G, g = (row0 + rr) % p.G;
  typename E::S* out = static_cast<typename E::S*>(p.out) +
                       ((static_cast<int64_t>(b) * p.T + t) * p.Hq + static_cast<int64_t>(h) * p.G + g) * p.D;
  const int64_t slot_floats = static_cast<int64_t>(KROWS) * (p.D + 2);
  auto part = [&](int s) { return p.part + (2 * static_cast<int64_t>(first + s) + (s == 0 ? 1 : 0)) * slot_floats; };
  auto stat = [&](int s) { return *reinterpret_cast<const f32x2*>(part(s) + static_cast<int64_t>(KROWS) * p.D + 2 * rr); };
  static_assert(LANES == 1 || LANES == 16, "a row per group of 16 lanes or per workgroup");
  __shared__ f32x4 values[LANES > 1 ? 16 : 1][16];
  __shared__ f32x2 stats[16];
  for (int d0 = 0; d0 < p.D; d0 += 64) {
    const int d = d0 + 4 * l16;
    f32x4 a = {0.f, 0.f, 0.f, 0.f};
    float mx = -INFINITY, sum = 0.f;
    // Four partials at a time, statistics and values in flight together.
    if (d < p.D) {
      for (int s0 = 4 * lane; s0 < count; s0 += 4 * LANES) {
        f32x2 ml[4];
        f32x4 x[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int s = min(s0 + i, count - 1);
          ml[i] = stat(s);
          x[i] = *reinterpret_cast<const f32x4*>(part(s) + static_cast<int64_t>(rr) * p.D + d);
        }
        float most = mx;
#pragma unroll
        for (int i = 0; i < 4; ++i) most = fmaxf(most, ml[i][0]);
        const float ref = most == -INFINITY ? 0.f : most;
        const float old = fast_exp2(mx - ref);
        sum *= old;
        a *= old;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if (s0 + i >= count) continue;
          const float f = fast_exp2(ml[i][0] - ref);
          sum += f * ml[i][1];
          a += f * x[i];
        }
        mx = most;
      }
    }
    if constexpr (LANES > 1) {
      if (d0 > 0) __syncthreads();
      values[group][l16] = a;
      if (l16 == 0) stats[group] = f32x2{mx, sum};
      __syncthreads();
      if (lane > 0) continue;
      float most = -INFINITY;
#pragma unroll
      for (int i = 0; i < LANES; ++i) most = fmaxf(most, stats[i][0]);
      const float ref = most == -INFINITY ? 0.f : most;
      a = f32x4{0.f, 0.f, 0.f, 0.f};
      sum = 0.f;
#pragma unroll
      for (int i = 0; i < LANES; ++i) {
        const float f = fast_exp2(stats[i][0] - ref);
        sum += f * stats[i][1];
        a += f * values[i][l16];
      }
    }
    if (d >= p.D) continue;
    const float inv = sum > 0.f || sum != sum ? 1.f / sum : 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) out[d + i] = E::from_f(sum > 0.f || sum != sum ? a[i] * inv : 0.f);
  }
}

// One launch (and the merge of a balanced one).
template <int DT, int DP, int NB, int WR, int NW>
hipError_t tree_launch(const TreeParams& p, int grid, hipStream_t st) {
  using Sh = TreeShape<DT, DP, NB, WR, NW>;
  const size_t lds = Sh::kLds + (p.W > 0 ? sizeof(int32_t) * static_cast<size_t>(p.B) : 0);
  void (*fn)(TreeParams) = tree_mfma_kernel<DT, DP, NB, WR, NW>;
  static std::atomic<uint64_t> allowed{0};  // devices on which more than 64 KB of LDS were asked for
  int dev = 0;
  if (hipGetDevice(&dev) != hipSuccess) dev = 0;
  const uint64_t bit = uint64_t{1} << (dev & 63);
  if (!(allowed.load(std::memory_order_relaxed) & bit)) {
    const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(fn), hipFuncAttributeMaxDynamicSharedMemorySize,
                                             Sh::kLds + 4 * kTreeMaxBalanced);
    if (e != hipSuccess) return e;
    allowed.fetch_or(bit, std::memory_order_relaxed);
  }
  hipLaunchKernelGGL(fn, dim3(static_cast<uint32_t>(grid)), dim3(64 * NW), lds, st, p);
  if (p.W > 0) {
    const int64_t items = static_cast<int64_t>(p.B) * p.Hkv * p.chunks;
    const bool many = p.W >= kTreeManyPartials * items;
    void (*merge)(TreeParams) = many ? tree_merge_kernel<DT, Sh::kRows, 16> : tree_merge_kernel<DT, Sh::kRows, 1>;
    hipLaunchKernelGGL(merge, dim3(static_cast<uint32_t>(items), static_cast<uint32_t>(many ? p.chunk_rows : (p.chunk_rows + 15) / 16)),
                       dim3(256), 0, st, p);
  }
  return hipGetLastError();
}

template <int DT, int DP, int ROWS>
hipError_t tree_launch_rows(const TreeParams& p, int grid, hipStream_t st) {
  constexpr int kSlots = tile_slots(DT == QD_DTYPE_F32 ? 4 : 2, DP);
  if constexpr (ROWS <= tree_most_rows(kSlots)) {
    if (p.chunk_rows <= ROWS) {
      constexpr TreeWaves w = tree_waves(kSlots, ROWS);
      return tree_launch<DT, DP, w.nb, w.wr, w.nw>(p, grid, st);
    }
    return tree_launch_rows<DT, DP, 2 * ROWS>(p, grid, st);
  }
  return hipErrorInvalidValue;
}

}  // namespace

#endif  // QD_TREE_KERNELS_H
