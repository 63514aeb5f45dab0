// Device code of prompt attention shared by the VALU kernel (prefill.hip) and
// the matrix-core kernels (prefill_mfma_*.hip).
#ifndef QD_PREFILL_KERNELS_H
#define QD_PREFILL_KERNELS_H

#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include <atomic>
#include <type_traits>

#include "packed.h"
#include "qd_attention.h"
#include "qd_device.h"
#include "tile_device.h"

// Arguments of the kernels, passed between translation units.
struct PrefillParams {
  const void* q;
  const void* k;
  const void* v;
  const int32_t* cu;
  const int32_t* cu_k;
  void* out;
  int64_t q_stride, k_stride, v_stride;  // elements from token to token
  int B, Tq, Tk, Hq, Hkv, D, G;          // G q-heads per kv-head
  int window, sinks;
  float sl2;    // scale * log2(e)
  float inv_g;  // 1 / G
  PackedDivide by_g, by_hkv, by_splits;
  int groups;   // items per kv-head
  int splits;   // workgroups that share an item's tiles; more than 1: partials in `part`
  float* part;  // [splits][Tq Hq][D + 4]: {m, l, -, -, acc[D]}
};

// Runs the matrix-core kernel for padded head_dim dp with workgroups of `rows`
// rows (prefill_mfma_*.hip).  Returns a hipError_t.
int qd_prefill_mfma_launch_f32(const PrefillParams& p, int dp, int rows, uint32_t grid, void* stream);
int qd_prefill_mfma_launch_f16(const PrefillParams& p, int dp, int rows, uint32_t grid, void* stream);
int qd_prefill_mfma_launch_bf16(const PrefillParams& p, int dp, int rows, uint32_t grid, void* stream);

namespace {

typedef float f32x16 __attribute__((ext_vector_type(16)));

// Tokens of a tile.
__host__ __device__ constexpr int prefill_tile(int slots) { return slots == 64 ? 32 : 64; }

template <int DT, int DP, int NB, int NW>
struct PrefillShape {
  static constexpr int kES = DT == QD_DTYPE_F32 ? 4 : 2;
  static constexpr int kSlots = tile_slots(kES, DP);
  static constexpr int TT = prefill_tile(kSlots);
  static constexpr int kRow = kSlots * 16;                // bytes of an LDS row
  static constexpr int kTile = TT * kRow;                 // bytes of K or V
  static constexpr int kLoadRows = TT / NW;               // rows that a wave loads
  static constexpr int kLoads = kLoadRows * kSlots / 64;  // its instructions, for K and for V
  static constexpr int kSteps = DP * kES / 32;            // 32 bytes of a row per step of the scores
  static constexpr int kTB = TT / 32;                     // blocks of 32 tokens
  static constexpr int kCols = DP / 32;
  static constexpr int kRows = 32 * NB * NW;
  // A wave's rows (its queries, later its output) in LDS: over K's and V's second
  // buffers where both halves of the workgroup fit, else behind all four.
  static constexpr bool kOver = kRows * kRow == 2 * kTile;
  __host__ __device__ static constexpr int rows_at(int wv) {
    return 32 * NB * kRow * wv + (!kOver ? 4 * kTile : 2 * wv < NW ? kTile : 2 * kTile);
  }
  static constexpr int kWord = kES == 2 && !kOver ? 4 * kTile + kRows * kRow : 4 * kTile;
  static constexpr int kLds = kWord + 16;
  static_assert(kLoadRows * kSlots % 64 == 0 && DP % 32 == 0, "waves do not fit the tile");
};

// As tile_swizzle, for operands of 32 rows: a transposing V read takes 4 rows of 64
// neighbouring bytes for each half of the wave, which have to be 4 different 64
// bytes of the 64 banks (with tile_swizzle they were the same 128: a third of the
// LDS cycles in conflicts).
__device__ __forceinline__ int prefill_swizzle(int slots, int row) {
  return slots == 8 ? 4 * ((row >> 1) & 1) + 2 * ((row >> 2) & 1) + ((row >> 3) & 1)
                    : 4 * (row & 3) + 2 * ((row >> 2) & 1) + ((row >> 3) & 1);
}

__device__ __forceinline__ float prefill_max_halves(float x) {
  const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
}
__device__ __forceinline__ float prefill_sum_halves(float x) {
  const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(a[0]) + __uint_as_float(a[1]);
}

template <int DT>
struct PrefillMma {
  // 32 x 32 block += A 16 bytes per lane . B 16 bytes per lane, whose elements
  // pair up by their place.
  __device__ static f32x16 mma(u32x4 a, u32x4 b, f32x16 c) {
    if constexpr (DT == QD_DTYPE_BF16) {
      return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
    } else if constexpr (DT == QD_DTYPE_F16) {
      return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        c = __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(a[j]), __uint_as_float(b[j]), c, 0, 0, 0);
      return c;
    }
  }
};

// What a value that is not finite counts as in the products that tell which rows
// see one: sums over a tile of up to 64 tokens keep the three apart.
constexpr float kPrefillPlusInf = 1.f, kPrefillMinusInf = 256.f, kPrefillNan = 32768.f;

// Scaled scores (of base 2) from which a row's weights come of differences.
constexpr float kPrefillFar = 0x1p20f;

template <int DT>
__device__ __forceinline__ float prefill_flag(typename Elem<DT>::S x) {
  const float f = Elem<DT>::to_f(x);
  return f != f ? kPrefillNan : f == INFINITY ? kPrefillPlusInf : f == -INFINITY ? kPrefillMinusInf : 0.f;
}

template <int DT>
__device__ __forceinline__ bool prefill_finite(u32x4 x) {
  bool ok = true;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (DT == QD_DTYPE_F32) {
      ok &= (x[i] & 0x7F800000u) != 0x7F800000u;
    } else {
      constexpr uint32_t e = DT == QD_DTYPE_F16 ? 0x7C00u : 0x7F80u;
      ok &= (x[i] & e) != e && (x[i] & (e << 16)) != e << 16;
    }
  }
  return ok;
}

// An item is a (sequence, kv-head, kRows of its rows); a row is a (query, q-head
// of the kv-head's group), numbered query by query, so that the heads that share
// K and V share a workgroup's reads of them and the rows of a workgroup span few
// positions.  Positions below 0 (more queries than keys) see nothing: -1.
struct PrefillItem {
  int h, q0, rows;         // rows of the workgroup: from q-head `rest` of query q0 on
  int rest;
  int k0, nk, at0;         // keys, position of query q0
  int p_min, p_max;        // positions of the first and the last row
  // Tiles [0, sink_tiles), then from lo_tile on; the workgroup's are `tiles` from
  // the place `skip` of that list on.
  int lo_tile, sink_tiles, skip, tiles;
  int split;
};

// Query (counted from q0) and q-head of the group of a row.
struct PrefillRow {
  int query, g;
};
__device__ __forceinline__ PrefillRow prefill_row(const PrefillParams& p, const PrefillItem& x, int row) {
  const int y = x.rest + row;  // below G + 256
  PrefillRow r;
  // y + 1/2 is at least 1/2 away from multiples of G: exact in fp32.
  r.query = p.G > 4096 ? static_cast<int>(y >= p.G) : static_cast<int>((static_cast<float>(y) + 0.5f) * p.inv_g);
  r.g = y - r.query * p.G;
  return r;
}
// Bytes of a row from query q0's first head on, where queries lie `pitch` and heads
// `head` bytes apart: query pitch + (y - query G) head, in products of 24 bits
// (heads and strides within 2^21 elements).
struct PrefillRowAt {
  const PrefillParams& p;
  int rest, rest_pitch, head;
  __device__ __forceinline__ PrefillRowAt(const PrefillParams& p, const PrefillItem& x, int pitch, int head)
      : p(p), rest(x.rest), rest_pitch(pitch - p.G * head), head(head) {}
  __device__ __forceinline__ uint32_t operator()(int row) const {
    const int y = rest + row;
    const int query = p.G > 4096 ? static_cast<int>(y >= p.G) : static_cast<int>((static_cast<float>(y) + 0.5f) * p.inv_g);
    return static_cast<uint32_t>(__mul24(query, rest_pitch) + __mul24(y, head));
  }
};
// Position of a row of the workgroup, or of its last one.
__device__ __forceinline__ int prefill_place(const PrefillParams& p, const PrefillItem& x, int row) {
  return max(x.at0 + prefill_row(p, x, min(row, x.rows - 1)).query, -1);
}

template <int ROWS, int TT>
__device__ __forceinline__ bool prefill_item(const PrefillParams& p, PrefillItem& x) {
  // What comes from the vector units goes back to scalar registers, or all that
  // follows from it stays with those too.
  auto scalar = [](int y) { return __builtin_amdgcn_readfirstlane(y); };
  // Parts of one item run on different XCDs: as evenly as there are parts, and no
  // XCD has all of a head's keys to fetch.
  const int item = packed_divide(blockIdx.x, p.by_splits);
  x.split = static_cast<int>(blockIdx.x) - item * p.splits;
  const int group = packed_divide(static_cast<uint32_t>(item), p.by_hkv);
  x.h = item - group * p.Hkv;
  // The last rows of a sequence see most: first.
  const int64_t u = p.groups - 1 - group;
  int b, q1, k1;
  const int lane = static_cast<int>(threadIdx.x) & 63;
  if (p.B < 64) {
    // Lane b holds sequence b's starts: one round trip.
    const int at = min(lane, p.B);
    const int qs = packed_start(p.cu, at, p.Tq), ks = packed_start(p.cu_k, at, p.Tk);
    const int64_t base = static_cast<int64_t>(qs) * p.G / ROWS + lane;
    b = 63 - __builtin_clzll(__ballot(lane == 0 || (lane <= p.B && base <= u)));
    const int next = min(b + 1, p.B);
    x.q0 = __builtin_amdgcn_readlane(qs, b);
    q1 = __builtin_amdgcn_readlane(qs, next);
    x.k0 = __builtin_amdgcn_readlane(ks, b);
    k1 = __builtin_amdgcn_readlane(ks, next);
  } else {
    b = packed_find(p.cu, p.B + 1, p.Tq, p.G, ROWS, 1, u);
    const int next = min(b + 1, p.B);
    x.q0 = packed_start(p.cu, b, p.Tq);
    q1 = packed_start(p.cu, next, p.Tq);
    x.k0 = packed_start(p.cu_k, b, p.Tk);
    k1 = packed_start(p.cu_k, next, p.Tk);
  }
  const bool tail = b == p.B;  // rows behind the last sequence
  if (tail) q1 = p.Tq;
  const int rows_all = max(q1 - x.q0, 0) * p.G;  // below 2^31: Tq Hq is
  const int64_t row0 = (u - static_cast<int64_t>(x.q0) * p.G / ROWS - b) * ROWS;
  if (row0 >= rows_all) return false;
  x.rows = min(ROWS, rows_all - static_cast<int>(row0));
  const int query0 = packed_divide(static_cast<uint32_t>(row0), p.by_g);
  x.rest = static_cast<int>(row0) - query0 * p.G;
  x.nk = tail ? 0 : max(k1 - x.k0, 0);
  x.at0 = x.nk - (q1 - x.q0) + query0;
  x.q0 += query0;
  x.p_min = max(x.at0, -1);
  x.p_max = scalar(prefill_place(p, x, ROWS));
  const int end = x.p_max + 1;  // at most nk
  const int lo = p.window > 0 ? max(x.p_min - p.window + 1, 0) : 0;
  x.lo_tile = lo / TT;
  x.sink_tiles = min((min(p.sinks, lo) + TT - 1) / TT, x.lo_tile);
  const int all = end > 0 ? x.sink_tiles + (end + TT - 1) / TT - x.lo_tile : 0;
  x.skip = 0;
  x.tiles = all;
  if (p.splits > 1) {
    const uint32_t n = all;  // below 2^26, and at most 32 parts
    x.skip = packed_divide(n * x.split, p.by_splits);
    x.tiles = packed_divide(n * (x.split + 1), p.by_splits) - x.skip;
  }
  for (int* y : {&x.q0, &x.rows, &x.rest, &x.k0, &x.nk, &x.at0, &x.p_min, &x.p_max, &x.lo_tile, &x.sink_tiles, &x.skip, &x.tiles})
    *y = scalar(*y);
  return true;
}

template <int TT>
__device__ __forceinline__ int prefill_first(const PrefillItem& x, int i) {
  i += x.skip;
  return TT * (i < x.sink_tiles ? i : i - x.sink_tiles + x.lo_tile);
}

// The places in the list of tiles whose tokens rows at positions lowest .. highest
// all see: from, .. from + count - 1.  Tiles of the first tokens are not among
// them.
struct PrefillWhole {
  int from;
  uint32_t count;
  __device__ __forceinline__ bool operator()(int i) const { return static_cast<uint32_t>(i - from) < count; }
};
template <int TT>
__device__ __forceinline__ PrefillWhole prefill_whole(const PrefillParams& p, const PrefillItem& x, int lowest, int highest) {
  const int shift = x.sink_tiles - x.lo_tile - x.skip;
  const int lo = p.window > 0 && highest >= p.window ? (highest - p.window) / TT + 1 : 0;
  PrefillWhole w;
  w.from = __builtin_amdgcn_readfirstlane(max(max(lo, x.lo_tile) + shift, 0));
  w.count = __builtin_amdgcn_readfirstlane(max((lowest + 1) / TT + shift - w.from, 0));
  return w;
}

// Whether rows at positions lowest .. highest all see tokens first .. last.
__device__ __forceinline__ bool prefill_sees_all(const PrefillParams& p, int first, int last, int lowest, int highest) {
  return last <= lowest && (p.window == 0 || first > highest - p.window || last < p.sinks);
}

// The tokens from `token` on that a row at `place` sees: o <= hi with o > lo or o <
// sinks, o counted from `token`.
struct PrefillView {
  int hi, lo, sinks;
  __device__ __forceinline__ bool operator()(int o) const {
    return static_cast<bool>(static_cast<int>(o <= hi) & (static_cast<int>(o > lo) | static_cast<int>(o < sinks)));
  }
};
__device__ __forceinline__ PrefillView prefill_view(const PrefillParams& p, int place, int token) {
  PrefillView v;
  v.hi = place - token;
  v.lo = p.window > 0 ? max(place - p.window, token - 1) - token : -1;
  v.sinks = p.sinks - token;
  return v;
}

// A wave-uniform pointer, in scalar registers.
__device__ __forceinline__ const char* prefill_scalar(const char* x) {
  return reinterpret_cast<const char*>(readlane_i64(static_cast<int64_t>(reinterpret_cast<uintptr_t>(x)), 0));
}

// Loads of K and V rows into LDS: a wave's rows of a tile, one instruction at a
// time.  What lies past the last key is taken from the end of its row instead:
// no query sees it.
template <typename Sh>
struct PrefillLoads {
  const char* base[2];  // K, V
  uint32_t bytes[2];
  int row_bytes, nk;
  uint32_t off[2][Sh::kLoads], lds_wave;
  bool inside[Sh::kLoads];
  __device__ __forceinline__ PrefillLoads(const PrefillParams& p, const PrefillItem& x, uint32_t lds, int wv, int lane) {
    row_bytes = p.D * Sh::kES;
    nk = x.nk;
    base[0] = prefill_scalar(static_cast<const char*>(p.k) + (x.k0 * p.k_stride + static_cast<int64_t>(x.h) * p.D) * Sh::kES);
    base[1] = prefill_scalar(static_cast<const char*>(p.v) + (x.k0 * p.v_stride + static_cast<int64_t>(x.h) * p.D) * Sh::kES);
    bytes[0] = static_cast<uint32_t>(p.k_stride * Sh::kES);
    bytes[1] = static_cast<uint32_t>(p.v_stride * Sh::kES);
#pragma unroll
    for (int i = 0; i < Sh::kLoads; ++i) {
      const int row = Sh::kLoadRows * wv + (64 * i + lane) / Sh::kSlots;
      const int col = 16 * ((lane & (Sh::kSlots - 1)) ^ prefill_swizzle(Sh::kSlots, row));
      inside[i] = col < row_bytes;  // false only in padded rows
      off[0][i] = row * bytes[0] + col;
      off[1][i] = row * bytes[1] + col;
    }
    lds_wave = __builtin_amdgcn_readfirstlane(lds + Sh::kLoadRows * wv * Sh::kRow);
  }
  // K (which 0) or V (1) of the tile at token `first`, to the buffer at `to` in
  // LDS.
  struct Tile {
    const char* src;
    uint32_t most, to;
  };
  __device__ __forceinline__ Tile tile(int which, int first, uint32_t to) const {
    return {base[which] + static_cast<int64_t>(first) * bytes[which],
            static_cast<uint32_t>(min(nk - 1 - first, Sh::TT - 1)) * bytes[which] + row_bytes - 16, lds_wave + to};
  }
  __device__ __forceinline__ void one(int which, int i, const Tile& x) const {
    const uint32_t at = min(off[which][i], x.most);
    if (row_bytes == Sh::kRow) {
      tile_load_lds<false>(x.src, at, x.to + 1024 * i);
    } else if (inside[i]) {
      asm volatile("; padded rows");  // keeps the two apart: no mask for whole rows
      tile_load_lds<false>(x.src, at, x.to + 1024 * i);
    }
  }
  __device__ __forceinline__ void operator()(int which, int first, uint32_t to) const {
    const Tile x = tile(which, first, to);
#pragma unroll
    for (int i = 0; i < Sh::kLoads; ++i) one(which, i, x);
  }
};

// Puts zeros in place of values that are not finite; whether this thread found
// any.
template <int DT, int PIECES, int STEP>
__device__ __forceinline__ bool prefill_drop_bad(char* v, int tid) {
  using S = typename Elem<DT>::S;
  constexpr int kEach = 16 / static_cast<int>(sizeof(S));
  bool found = false;
#pragma unroll 4
  for (int i = tid; i < PIECES; i += STEP) {
    u32x4* at = reinterpret_cast<u32x4*>(v) + i;
    if (prefill_finite<DT>(*at)) continue;
    found = true;
    S* val = reinterpret_cast<S*>(at);
#pragma unroll
    for (int e = 0; e < kEach; ++e)
      if (prefill_flag<DT>(val[e]) != 0.f) val[e] = Elem<DT>::from_f(0.f);
  }
  return found;
}

// Flags in place of all values.
template <int DT, int PIECES, int STEP>
__device__ __forceinline__ void prefill_to_flags(char* v, int tid) {
  using S = typename Elem<DT>::S;
  constexpr int kEach = 16 / static_cast<int>(sizeof(S));
  for (int i = tid; i < PIECES; i += STEP) {
    S* val = reinterpret_cast<S*>(v) + i * kEach;
#pragma unroll
    for (int e = 0; e < kEach; ++e) val[e] = Elem<DT>::from_f(prefill_flag<DT>(val[e]));
  }
}

// y plus the values that a sum of flags stands for.
__device__ __forceinline__ float prefill_add_bad(float y, float seen) {
  const float negative = __builtin_amdgcn_fractf(seen / kPrefillMinusInf) == 0.f && seen < kPrefillNan ? -INFINITY : NAN;
  return y + (seen >= kPrefillMinusInf ? negative : seen > 0.f ? INFINITY : 0.f);
}

// out rows of a lane, or their partials: acc of column block c, element e is
// column 32 c + 8 (e / 4) + 4 half + e % 4 of row wave_row + 32 nb + lane % 32, m a
// score that the row's weights count from.  16-bit rows: partials only, whole ones go
// through prefill_store_rows.
template <int DT, int DP, int NB>
__device__ __forceinline__ void prefill_store(const PrefillParams& p, const PrefillItem& x, int wave_row,
                                              const f32x16 (&acc)[DP / 32][NB], const float (&m)[NB], const float (&l)[NB]) {
  const int lane = static_cast<int>(threadIdx.x) & 63, half = lane >> 5;
#pragma unroll
  for (int nb = 0; nb < NB; ++nb) {
    const float sum = prefill_sum_halves(l[nb]);
    const bool has = sum > 0.f || sum != sum;
    const int rr = wave_row + 32 * nb + (lane & 31);
    if (rr >= x.rows) continue;
    const PrefillRow row = prefill_row(p, x, rr);
    const int64_t at = static_cast<int64_t>(x.q0 + row.query) * p.Hq + static_cast<int64_t>(x.h) * p.G + row.g;
    if (DT != QD_DTYPE_F32 || p.splits > 1) {
      float* to = p.part + (x.split * (static_cast<int64_t>(p.Tq) * p.Hq) + at) * (p.D + 4);
      if (half == 0) *reinterpret_cast<f32x2*>(to) = has ? f32x2{m[nb] * p.sl2, sum} : f32x2{-INFINITY, 0.f};
#pragma unroll
      for (int c = 0; c < DP / 32; ++c)
#pragma unroll
        for (int e = 0; e < 16; e += 4) {
          const int d = 32 * c + 2 * e + 4 * half;
          if (d < p.D)
            *reinterpret_cast<f32x4*>(to + 4 + d) =
                f32x4{acc[c][nb][e], acc[c][nb][e + 1], acc[c][nb][e + 2], acc[c][nb][e + 3]};
        }
      continue;
    }
    const float scale = has ? 1.f / sum : 0.f;
    float* to = static_cast<float*>(p.out) + at * p.D;
#pragma unroll
    for (int c = 0; c < DP / 32; ++c)
#pragma unroll
      for (int e = 0; e < 16; e += 4) {
        const int d = 32 * c + 2 * e + 4 * half;
        if (d >= p.D) continue;
        f32x4 y;
#pragma unroll
        for (int j = 0; j < 4; ++j) y[j] = has ? acc[c][nb][e + j] * scale : 0.f;
        *reinterpret_cast<f32x4*>(to + d) = y;
      }
  }
}

// 16-bit rows: through the wave's place in LDS, so that whole rows are stored (as
// they lie in registers, a store reaches 16 bytes of 32 rows).
template <typename Sh, int DT, int DP, int NB>
__device__ __forceinline__ void prefill_store_rows(const PrefillParams& p, const PrefillItem& x, int wave_row, char* place,
                                                   f32x16 (&acc)[DP / 32][NB], const float (&l)[NB]) {
  const int lane = static_cast<int>(threadIdx.x) & 63, half = lane >> 5, n32 = lane & 31;
#pragma unroll
  for (int nb = 0; nb < NB; ++nb) {
    const float sum = prefill_sum_halves(l[nb]);
    const bool has = sum > 0.f || sum != sum;
    const float scale = has ? 1.f / sum : 0.f;
    // Without weights the output is 0, whatever values scores of -inf belong to.
    if (__ballot(!has)) {
#pragma unroll
      for (int c = 0; c < DP / 32; ++c)
#pragma unroll
        for (int e = 0; e < 16; ++e) acc[c][nb][e] = has ? acc[c][nb][e] : 0.f;
    }
    char* row = place + (32 * nb + n32) * Sh::kRow;
    const int swizzle = 16 * prefill_swizzle(Sh::kSlots, n32);
#pragma unroll
    for (int c = 0; c < DP / 32; ++c)
#pragma unroll
      for (int e = 0; e < 16; e += 4) {
        f32x4 y;
#pragma unroll
        for (int j = 0; j < 4; ++j) y[j] = acc[c][nb][e + j] * scale;
        // Column 32 c + 2 e + 4 half.
        *reinterpret_cast<u32x2*>(row + ((64 * c + 4 * e) ^ swizzle) + 8 * half) =
            u32x2{MfmaOps<DT>::pack2(y[0], y[1]), MfmaOps<DT>::pack2(y[2], y[3])};
      }
  }
  const int row_bytes = 2 * p.D;
  char* base = const_cast<char*>(prefill_scalar(static_cast<const char*>(p.out) +
                                                (static_cast<int64_t>(x.q0) * p.Hq + static_cast<int64_t>(x.h) * p.G) * row_bytes));
  const PrefillRowAt at(p, x, p.Hq * row_bytes, row_bytes);
#pragma unroll
  for (int i = 0; i < NB * Sh::kSlots / 2; ++i) {
    const int r = (64 * i + lane) / Sh::kSlots;
    const int slot = lane & (Sh::kSlots - 1), col = 16 * (slot ^ prefill_swizzle(Sh::kSlots, r));
    const u32x4 y = *reinterpret_cast<const u32x4*>(place + r * Sh::kRow + 16 * slot);
    if (wave_row + r >= x.rows || col >= row_bytes) continue;
    *reinterpret_cast<u32x4*>(base + (at(wave_row + r) + col)) = y;
  }
}

// Log-sum-exp merge of split items: a wave per row, LANES lanes stride its columns
// four at a time, the others its partials.
// grid ceil(Tq Hq / 4), block 256.
template <int DT, int LANES>
__global__ __launch_bounds__(256) void prefill_merge_kernel(PrefillParams p) {
  constexpr int TEAMS = 64 / LANES, kAhead = 8;  // partials in flight
  const int64_t rows = static_cast<int64_t>(p.Tq) * p.Hq;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 6);
  if (row >= rows) return;
  const int lane = static_cast<int>(threadIdx.x) & 63, team = lane / LANES, l = lane % LANES;
  auto part = [&](int s) { return p.part + (s * rows + row) * (p.D + 4); };
  for (int d = 4 * l; d < p.D + 4 * l; d += 4 * LANES) {
    const bool in = d < p.D;
    float mx = -INFINITY, sum = 0.f;
    f32x4 a = {0.f, 0.f, 0.f, 0.f};
    for (int s0 = kAhead * team; s0 < p.splits; s0 += kAhead * TEAMS) {
      f32x2 ml[kAhead];
      f32x4 x[kAhead];
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
        const float* src = part(min(s0 + i, p.splits - 1));
        ml[i] = *reinterpret_cast<const f32x2*>(src);
        x[i] = in ? *reinterpret_cast<const f32x4*>(src + 4 + d) : f32x4{0.f, 0.f, 0.f, 0.f};
      }
      float most = mx;
#pragma unroll
      for (int i = 0; i < kAhead; ++i) most = fmaxf(most, ml[i][0]);
      const float ref = most == -INFINITY ? 0.f : most;
      const float old = fast_exp2(mx - ref);
      sum *= old;
      a *= old;
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
        // A part without weight has no say, whatever it holds.  One whose scores are
        // all NaN has a NaN for its sum, which goes on to the row.
        if (s0 + i >= p.splits || (ml[i][0] == -INFINITY && ml[i][1] == 0.f)) continue;
        const float f = fast_exp2(ml[i][0] - ref);
        sum += f * ml[i][1];
        a += f * x[i];
      }
      mx = most;
    }
#pragma unroll
    for (int off = LANES; off < 64; off <<= 1) {
      const float om = __shfl_xor(mx, off), os = __shfl_xor(sum, off);
      f32x4 oa;
#pragma unroll
      for (int i = 0; i < 4; ++i) oa[i] = __shfl_xor(a[i], off);
      const float most = fmaxf(mx, om), ref = most == -INFINITY ? 0.f : most;
      const float f = fast_exp2(mx - ref), g = fast_exp2(om - ref);
      sum = f * sum + g * os;
      a = f * a + g * oa;
      mx = most;
    }
    if (team == 0 && in) {
      const bool has = sum > 0.f || sum != sum;
      const float inv = has ? 1.f / sum : 0.f;
      if (!has) a = f32x4{0.f, 0.f, 0.f, 0.f};
      if constexpr (DT == QD_DTYPE_F32)
        *reinterpret_cast<f32x4*>(static_cast<float*>(p.out) + row * p.D + d) = a * inv;
      else
        *reinterpret_cast<u32x2*>(static_cast<char*>(p.out) + (row * p.D + d) * 2) =
            u32x2{MfmaOps<DT>::pack2(a[0] * inv, a[1] * inv), MfmaOps<DT>::pack2(a[2] * inv, a[3] * inv)};
    }
  }
}

// The workgroup goes through the tokens that its rows see in tiles of TT: K and V
// rows come straight into LDS, a tile ahead, and each wave multiplies its 32 NB
// rows with them, 32 tokens at a time:
//   scores   S^T = K Q^T, 32x32 blocks (A = K rows from LDS, B = Q from
//            registers): a lane holds one row and 16 of 32 tokens
//   softmax  per lane, weights 2^(s - m) with a reference m of the row that
//            was one of its scores.  m moves only when a lane's weights of a
//            step sum to more than 2^kLazy (which every weight beyond that
//            does): the maximum is not computed otherwise, and lanes exchange
//            nothing.  A weight is 2^(s c + r), r = -m c rounded once, and where |m c|
//            passes 2^20 that rounding would show (past 2^27 it takes weights out of
//            fp16's range): such rows find m in every step, and subtract before they
//            multiply.
//   output   O^T += V^T P^T: the score layout is already the B operand (the
//            products sum over tokens in the order that the lanes hold them in),
//            V^T comes from transposing LDS reads.
// 16-bit weights are rounded to nearest once: half a step of the output's type,
// which a sum over many values averages out; their sum is that of the rounded
// ones.
//
// Three steps are in work at once, in one stream of instructions: the scores of
// the next 32 tokens, the softmax of these, the values of the ones before.  A
// 32x32x16 product takes 32 cycles of the matrix cores; for heads of 128 there are
// two elements' worth of softmax beside it (two multiply-adds, two exponentials at 8
// cycles, a conversion and a sum of two), for heads of 64 four.  What bounds it:
// products of random data alone run at 1709 TFLOP/s (the card's power takes the
// clock to 1.7 GHz), with that much softmax beside them and nothing else at 1267;
// one prompt of 12001 tokens, 32 heads of 128, takes 1060 to 1125 us, 1050 to 1110
// TFLOP/s: 2.0 million cycles, of which the matrix cores are busy for 57%, at a clock
// that the card moves with its load (1.82 GHz in dispatches of 1100 us; 1.43 and 1376 us
// at times under counters).  16x16x32 products need
// twice the issue slots and ran at 1116 beside the same softmax.  Heads of 64 (16 and
// 32 of 1000 to 8192 tokens) reach 650 to 720 TFLOP/s, bound by vector instructions.
//
// A workgroup's start and end (which rows, operands' first trip, output) take 17000
// cycles, of which the other workgroup of its CU can use most: 16 prompts of 65 to
// 2000 tokens run at 750 TFLOP/s.  128 rows per workgroup and two workgroups per CU:
// eight waves of one (986 TFLOP/s then, against 1120) wait for each other, one wave
// of 64 rows per SIMD (972) issues an instruction every five cycles at most.
template <int DT, int DP, int NB, int NW>
__global__ __launch_bounds__(64 * NW, (NB * DP <= 128 ? 2 : 1)) void prefill_pipe_kernel(PrefillParams p) {
  using Sh = PrefillShape<DT, DP, NB, NW>;
  static_assert(DT != QD_DTYPE_F32 && Sh::TT == 64, "16-bit types");
  // fp16 weights are multiples of 2^-24 and the largest of a row is at least
  // 2^kShift: what that grid adds is at most 2^-32 of it.
  constexpr float kShift = DT == QD_DTYPE_F16 ? 7.f : 0.f;
  constexpr float kMost = DT == QD_DTYPE_F16 ? 32768.f : 256.f;  // 2^(kShift + kLazy)
  constexpr int kN = Sh::kSteps;      // steps of the scores, and (token 16, column 32) pairs of the output
  constexpr int kCols = Sh::kCols;
  constexpr int kRing = NB == 2 ? 2 : kN % 4 == 0 ? 4 : 3;  // operands in registers, read ahead
  constexpr int kPairs = 8 * NB;      // packed pairs of weights
  constexpr int kSlots = kN * NB;     // slots of one product each of scores and output
  extern __shared__ __align__(16) char smem[];
  // K in two buffers, V in two, queries and output over or behind them, a word.
  int* word = reinterpret_cast<int*>(smem + Sh::kWord);
  const int tid = static_cast<int>(threadIdx.x), lane = tid & 63;
  const int wv = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int n32 = lane & 31, half = lane >> 5, r16 = lane & 15;
  PrefillItem x;
  if (!prefill_item<Sh::kRows, Sh::TT>(p, x)) return;
  const int wave_row = 32 * NB * wv;
  const uint32_t lds0 = tile_lds_address(smem);
  const PrefillLoads<Sh> load(p, x, lds0, wv, lane);
  auto k_buf = [](int t) { return static_cast<uint32_t>((t & 1) * Sh::kTile); };
  auto v_buf = [](int t) { return static_cast<uint32_t>((2 + (t & 1)) * Sh::kTile); };
  if (load.row_bytes < Sh::kRow) {  // products run over the slots past the head
    for (int i = tid; i < Sh::kWord / 16; i += 64 * NW) reinterpret_cast<u32x4*>(smem)[i] = u32x4{0u, 0u, 0u, 0u};
    tile_barrier();
  }
  if (tid == 0) *word = 0;
  f32x16 acc[kCols][NB];
  float m[NB], l[NB], ref[NB];
  auto clear = [&]() {
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
      m[nb] = -INFINITY;
      ref[nb] = INFINITY;  // the first step finds its maximum
      l[nb] = 0.f;
#pragma unroll
      for (int c = 0; c < kCols; ++c) acc[c][nb] = f32x16{};
    }
  };
  // Wide heads' accumulators lie in both register files and are cleared ahead of the
  // loop (4 x 2048 tokens, 16 heads of 256: 192 us, 219 in it); others in it, where
  // they are not copied (64 prompts of 200 tokens, heads of 128: 82 us for 84).
  constexpr bool kClearAhead = DP > 128;
  if (kClearAhead || x.tiles == 0) clear();
  if (x.tiles == 0) {  // the same for all waves
    if (p.splits > 1)
      prefill_store<DT, DP, NB>(p, x, wave_row, acc, m, l);
    else
      prefill_store_rows<Sh, DT, DP, NB>(p, x, wave_row, smem + Sh::rows_at(wv), acc, l);
    return;
  }
  // Each wave's queries go through LDS too: as operands straight from memory they
  // would come in pieces of 32 bytes.
  {
    const char* base = prefill_scalar(static_cast<const char*>(p.q) +
                                      (x.q0 * p.q_stride + static_cast<int64_t>(x.h) * p.G * p.D) * Sh::kES);
    const PrefillRowAt at(p, x, static_cast<int>(p.q_stride) * Sh::kES, load.row_bytes);
    const uint32_t to = __builtin_amdgcn_readfirstlane(lds0 + Sh::rows_at(wv));
#pragma unroll
    for (int i = 0; i < NB * Sh::kSlots / 2; ++i) {
      const int r = (64 * i + lane) / Sh::kSlots;
      const uint32_t col = 16 * ((lane & (Sh::kSlots - 1)) ^ prefill_swizzle(Sh::kSlots, r));
      if (static_cast<int>(col) < load.row_bytes)
        tile_load_lds<false>(base, at(min(wave_row + r, x.rows - 1)) + col, to + 1024 * i);
    }
  }
  load(0, prefill_first<64>(x, 0), k_buf(0));
  load(1, prefill_first<64>(x, 0), v_buf(0));  // needed last
  int place[NB];
#pragma unroll
  for (int nb = 0; nb < NB; ++nb) place[nb] = prefill_place(p, x, wave_row + 32 * nb + n32);
  const int w_min = __builtin_amdgcn_readfirstlane(prefill_place(p, x, wave_row));
  const int w_max = __builtin_amdgcn_readfirstlane(prefill_place(p, x, wave_row + 32 * NB - 1));
  const PrefillWhole whole = prefill_whole<64>(p, x, x.p_min, x.p_max), wave_whole = prefill_whole<64>(p, x, w_min, w_max);
  // Operands' places in LDS, in the buffers that the next step reads: step st of
  // a K row, columns 32 c.. of V's token rows 4 half.. and 8 further.
  uint32_t k_at[kN], v_at[kCols][2];
#pragma unroll
  for (int st = 0; st < kN; ++st)
    k_at[st] = lds0 + n32 * Sh::kRow + (16 * (half ^ prefill_swizzle(Sh::kSlots, n32)) ^ (32 * st));
  const int vr = 4 * half + (r16 >> 2);
#pragma unroll
  for (int c = 0; c < kCols; ++c)
#pragma unroll
    for (int i = 0; i < 2; ++i)
      v_at[c][i] = lds0 + v_buf(1) + (vr + 8 * i) * Sh::kRow +
                   ((16 * ((2 * ((lane >> 4) & 1) + ((r16 >> 1) & 1)) ^ prefill_swizzle(Sh::kSlots, vr)) + 8 * (r16 & 1)) ^
                    (64 * c) ^ (16 * i));
  auto read_k = [&](int token, int st) { return tile_lds_read<u32x4>(k_at[st] + token * Sh::kRow); };
  // V^T of 16 tokens from `token` on, columns 32 c..
  auto read_v = [&](int token, int c) {
    const u32x2 a = tile_tr_read(v_at[c][0] + token * Sh::kRow), b = tile_tr_read(v_at[c][1] + token * Sh::kRow);
    return u32x4{a[0], a[1], b[0], b[1]};
  };
  auto next_buffers = [&]() {
#pragma unroll
    for (int st = 0; st < kN; ++st) k_at[st] ^= Sh::kTile;
#pragma unroll
    for (int c = 0; c < kCols; ++c) {
      v_at[c][0] ^= Sh::kTile;
      v_at[c][1] ^= Sh::kTile;
    }
  };
  auto sum2 = [](uint32_t w, float c) {
    if constexpr (DT == QD_DTYPE_BF16)
      return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2, w), __builtin_bit_cast(bf16x2, 0x3F803F80u), c, false);
    else
      return __builtin_amdgcn_fdot2(__builtin_bit_cast(f16x2, w), __builtin_bit_cast(f16x2, 0x3C003C00u), c, false);
  };
  struct Weights {
    u32x4 w[2][NB];  // 16 tokens each
  };
  u32x4 qf[NB][kN];
  tile_wait_loads<2 * Sh::kLoads>();
#pragma unroll
  for (int nb = 0; nb < NB; ++nb)
#pragma unroll
    for (int st = 0; st < kN; ++st)
      qf[nb][st] = tile_lds_read<u32x4>(k_at[st] + Sh::rows_at(wv) + 32 * nb * Sh::kRow);

  // The largest score of a row, or m.
  auto largest = [&](const f32x16& s, float m) {
    float mx = -INFINITY;
#pragma unroll
    for (int e = 0; e < 16; ++e) mx = fmaxf(mx, s[e]);
    return fmaxf(m, prefill_max_halves(mx));
  };
  // What to add to scaled scores that count from m; Inf: m has to be found anew.
  auto reference = [&](float m) {
    const float x = m * p.sl2;
    return fabsf(x) < kPrefillFar ? kShift - x : INFINITY;
  };

  u32x4 ka[kRing], va[kRing];  // operands read ahead of their products
  // The scores of the 32 tokens from `at` on in K's buffer, the weights of `cur`,
  // the products of the weights `prev` with those from `at` on in V's.  `midway`
  // runs when the last operands of the step are on their way, and the next step's
  // first ones, from 32 - `at` on, follow; `aside` runs beside every slot's products.
  auto step = [&](f32x16 (&cur)[NB], f32x16 (&next)[NB], const Weights& prev, Weights& now, auto at, auto&& midway,
                  auto&& aside) {
    float arg[kPairs][2], val[kPairs][2], sum[NB];
    uint64_t move = 0;  // lanes whose weights outgrow their reference
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) sum[nb] = 0.f;
    // Pair j: elements 2 (j / NB), + 1 of row block j % NB.  The empty statements
    // keep each stage in its slot.
    auto scale2 = [&](int j) {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        arg[j][e] = fmaf(cur[j % NB][2 * (j / NB) + e], p.sl2, ref[j % NB]);
        asm volatile("" : "+v"(arg[j][e]));
      }
    };
    auto exp2 = [&](int j) {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        val[j][e] = fast_exp2(arg[j][e]);
        asm volatile("" : "+v"(val[j][e]));
      }
    };
    auto pack = [&](int j) {
      uint32_t w = MfmaOps<DT>::pack2(val[j][0], val[j][1]);
      asm volatile("" : "+v"(w));
      now.w[(j / NB) >> 2][j % NB][(j / NB) & 3] = w;
      sum[j % NB] = sum2(w, sum[j % NB]);
    };
    // Stages of a pair, a slot apart; the last one is done before the last slot, so
    // that the sums are there at the end.
    auto from = [](int slot) { return slot < 0 ? 0 : slot >= kSlots - 1 ? kPairs : slot * kPairs / (kSlots - 1); };
    auto score = [&](int i, int nb) {
      next[nb] = PrefillMma<DT>::mma(ka[i % kRing], qf[nb][i], i == 0 ? f32x16{} : next[nb]);
    };
    // Scores go a slot ahead of the values: what the next step needs first is not
    // what this one does last.
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) score(0, nb);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int j = 0; j < from(2); ++j) scale2(j);
#pragma unroll
    for (int j = 0; j < from(1); ++j) exp2(j);
#pragma unroll
    for (int slot = 0; slot < kSlots; ++slot) {
      const int i = slot / NB, nb = slot % NB;
      if (nb == 0) {
        // The places of K's operand i and V's i - 1 are free.
        const int v = i + kRing - 1, k = i + kRing;
        va[v % kRing] = read_v((v < kN ? at : 32 - at) + 16 * (v % kN / kCols), v % kCols);
        if (k == kN) midway();
        ka[k % kRing] = read_k(k < kN ? at : 32 - at, k % kN);
      }
      if (i + 1 < kN) score(i + 1, nb);
      if (slot == kSlots - 1) {  // NaN sums too
        bool over = false;
#pragma unroll
        for (int x = 0; x < NB; ++x) over |= !(sum[x] <= kMost);
        move = __ballot(over);
        asm volatile("" : "+s"(move));
      }
      acc[i % kCols][nb] = PrefillMma<DT>::mma(va[i % kRing], prev.w[i / kCols][nb], acc[i % kCols][nb]);
#pragma unroll
      for (int j = from(slot + 2); j < from(slot + 3); ++j) scale2(j);
#pragma unroll
      for (int j = from(slot + 1); j < from(slot + 2); ++j) exp2(j);
#pragma unroll
      for (int j = from(slot); j < from(slot + 1); ++j) pack(j);
      aside(slot);
      __builtin_amdgcn_sched_barrier(0);
    }
    if (__builtin_expect(move != 0, 0)) {
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) {
        asm volatile("" : "+v"(cur[nb]));  // nothing of this is computed ahead of the branch
        const float mn = largest(cur[nb], m[nb]);
        const float alpha = mn == m[nb] ? 1.f : fast_exp2((m[nb] - mn) * p.sl2);
        m[nb] = mn;
        ref[nb] = reference(mn);
        const bool far = ref[nb] == INFINITY;
        const float from = far && mn != -INFINITY ? mn : 0.f;
        if (far) ref[nb] = kShift;
#pragma unroll
        for (int e = 0; e < 16; ++e) cur[nb][e] -= from;
        l[nb] *= alpha;
#pragma unroll
        for (int c = 0; c < kCols; ++c) acc[c][nb] *= alpha;
        sum[nb] = 0.f;
      }
#pragma unroll
      for (int j = 0; j < kPairs; ++j) {
        scale2(j);
        exp2(j);
        pack(j);
        if (j % 4 == 3) __builtin_amdgcn_sched_barrier(0);
      }
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) ref[nb] = reference(m[nb]);
    }
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) l[nb] += sum[nb];
  };
  // An opaque copy: what is derived from it is not computed ahead of the loops and
  // kept in registers.
  auto apart = [](int y) {
    asm volatile("" : "+v"(y));
    return y;
  };
  // Hides the scores of 32 tokens from `first` on that rows do not see.
  auto hide = [&](f32x16 (&s)[NB], int first) {
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
      const PrefillView sees = prefill_view(p, apart(place[nb]), apart(first + 4 * half));
#pragma unroll
      for (int e = 0; e < 16; ++e) s[nb][e] = sees(8 * (e / 4) + e % 4) ? s[nb][e] : -INFINITY;
    }
  };

  // A value that is not finite reaches rows that do not see it as 0 x NaN.  What
  // comes out not finite is computed again, with care: where only some rows see a
  // token, such values are left out (zeros) and joined to the rows that do see
  // them at the end.
#pragma unroll 1
  for (bool careful = false;; careful = true) {
    if constexpr (!kClearAhead) clear();
    f32x16 s0[NB], s1[NB];
    Weights w0, w1;
    // The first K has arrived, and every wave has its queries.
    tile_barrier_loads<Sh::kLoads>();
    if (x.tiles > 1) load(0, prefill_first<64>(x, 1), k_buf(1));
    // The first step has no tokens before it: no weights, and values of 0.
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) w1.w[0][nb] = w1.w[1][nb] = u32x4{0u, 0u, 0u, 0u};
    for (int i = apart(tid); i < Sh::kTile / 32; i += 64 * NW)
      reinterpret_cast<u32x4*>(smem + v_buf(1) + Sh::kTile / 2)[i] = u32x4{0u, 0u, 0u, 0u};
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) s0[nb] = f32x16{};
    {
      u32x4 a[kN < 8 ? kN : 8];
      constexpr int kFirst = kN < 8 ? kN : 8;  // reads ahead of the first product
#pragma unroll
      for (int st = 0; st < kFirst; ++st) a[st] = read_k(0, st);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int st = 0; st < kN; ++st) {
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) s0[nb] = PrefillMma<DT>::mma(a[st % kFirst], qf[nb][st], s0[nb]);
        if (st + kFirst < kN) a[st % kFirst] = read_k(0, st + kFirst);
      }
    }
    if (!wave_whole(0)) hide(s0, prefill_first<64>(x, 0));
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
      m[nb] = largest(s0[nb], -INFINITY);
      ref[nb] = reference(m[nb]);
    }
    tile_barrier();  // the zeros are there
#pragma unroll
    for (int i = 0; i < kRing; ++i) {
      ka[i] = read_k(32, i);
      if (i < kRing - 1) va[i] = read_v(32 + 16 * (i / kCols), i % kCols);
    }
    using Lower = std::integral_constant<int, 0>;
    using Upper = std::integral_constant<int, 32>;
#pragma unroll 1
    for (int t = 0; t < x.tiles; ++t) {
      step(
          s0, s1, w1, w0, Upper{},
          [&]() {
            // This V and the next K have arrived, and every wave has read what it
            // needs of this K and the V before.
            tile_barrier_loads<0>();
            next_buffers();
            if (__builtin_expect(careful && !whole(t), 0)) {
              prefill_drop_bad<DT, Sh::kTile / 16, 64 * NW>(smem + v_buf(t), apart(tid));
              tile_barrier();
            }
          },
          [](int) {});
      if (__builtin_expect(!wave_whole(t), 0)) hide(s1, prefill_first<64>(x, t) + 32);
      // After the last tile: scores of no use.
      const bool more_v = t + 1 < x.tiles, more_k = t + 2 < x.tiles;
      const auto k_next = load.tile(0, prefill_first<64>(x, more_k ? t + 2 : t), k_buf(t));
      const auto v_next = load.tile(1, prefill_first<64>(x, more_v ? t + 1 : t), v_buf(t + 1));
      step(
          s1, s0, w0, w1, Lower{}, []() {},
          [&](int slot) {
            // Where there are two slots per load, every other wave takes the second:
            // the loads of all at once would wait for each other.
            constexpr int kAll = 2 * Sh::kLoads;
            const int begin = slot * kAll / kSlots, end = (slot + 1) * kAll / kSlots;
            auto issue = [&](int j) {
              if (j < Sh::kLoads) {
                if (more_k) load.one(0, j, k_next);
              } else {
                if (more_v) load.one(1, j - Sh::kLoads, v_next);
              }
            };
            if constexpr (kSlots % (2 * kAll) == 0) {
              constexpr int kEvery = kSlots / kAll;
              if (slot % kEvery < 2 && (wv & 1) == slot % kEvery) issue(slot / kEvery);
            } else {
#pragma unroll
              for (int j = begin; j < end; ++j) issue(j);
            }
          });
      if (__builtin_expect(!wave_whole(t + 1), 0)) hide(s0, prefill_first<64>(x, t + 1));
    }
#pragma unroll
    for (int i = 0; i < kN; ++i) {
      const u32x4 a = i < kRing - 1 ? va[i] : read_v(32 + 16 * (i / kCols), i % kCols);
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) acc[i % kCols][nb] = PrefillMma<DT>::mma(a, w1.w[i / kCols][nb], acc[i % kCols][nb]);
    }
    if (!careful) {
      float test[4] = {0.f, 0.f, 0.f, 0.f};  // NaN if anything is not finite
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) {
        test[0] = fmaf(l[nb], 0.f, test[0]);
#pragma unroll
        for (int c = 0; c < kCols; ++c)
#pragma unroll
          for (int e = 0; e < 16; ++e) test[e % 4] = fmaf(acc[c][nb][e], 0.f, test[e % 4]);
      }
      const float all = (test[0] + test[1]) + (test[2] + test[3]);
      if (all != all) *word = 1;
      tile_barrier();
      if (__builtin_amdgcn_readfirstlane(*word) == 0) break;
      if constexpr (kClearAhead) clear();
      if (x.tiles & 1) next_buffers();  // as at the start: K's first, V's second
      load(0, prefill_first<64>(x, 0), k_buf(0));
      load(1, prefill_first<64>(x, 0), v_buf(0));
      continue;
    }
    if (x.tiles & 1) next_buffers();
    // A product of what is visible with the flags of values that are not finite.
#pragma unroll 1
    for (int t = 0; t < x.tiles; ++t) {
      if (whole(t)) continue;
      const int first = prefill_first<64>(x, t);
      tile_barrier();
      load(1, first, v_buf(1));
      tile_barrier_loads<0>();
      prefill_to_flags<DT, Sh::kTile / 16, 64 * NW>(smem + v_buf(1), apart(tid));
      tile_barrier();
#pragma unroll 1
      for (int ks = 0; ks < 4; ++ks)
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) {
          const PrefillView sees = prefill_view(p, place[nb], first + 16 * ks + 4 * half);
          u32x4 one;
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int o = 8 * (j >> 1) + 2 * (j & 1);
            one[j] = MfmaOps<DT>::pack2(sees(o) ? 1.f : 0.f, sees(o + 1) ? 1.f : 0.f);
          }
#pragma unroll
          for (int c = 0; c < kCols; ++c) {
            const f32x16 seen = PrefillMma<DT>::mma(read_v(16 * ks, c), one, f32x16{});
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[c][nb][e] = prefill_add_bad(acc[c][nb][e], seen[e]);
          }
        }
    }
    break;
  }
  if (p.splits > 1) {
    prefill_store<DT, DP, NB>(p, x, wave_row, acc, m, l);
    return;
  }
  tile_barrier_loads<0>();  // nothing reads or writes LDS any more
  prefill_store_rows<Sh, DT, DP, NB>(p, x, wave_row, smem + Sh::rows_at(wv), acc, l);
}

// fp32: the same products on the fp32 matrix cores, tile by tile, without the
// overlap: they take eight times as long as the 16-bit ones.  Scores, softmax and values
// follow each other, and a barrier each tile, with one workgroup per CU: 2 prompts of
// 2048 tokens, 16 heads of 128, take 378 us, 91 TFLOP/s of the 137 that a large product
// reaches.
template <int DP, int NW>
__global__ __launch_bounds__(64 * NW, 1) void prefill_f32_kernel(PrefillParams p) {
  using Sh = PrefillShape<QD_DTYPE_F32, DP, 1, NW>;
  constexpr int TT = Sh::TT, TB = Sh::kTB;
  constexpr float kLazy = 8.f;
  extern __shared__ __align__(16) char smem[];
  int* word = reinterpret_cast<int*>(smem + Sh::kWord);
  const int tid = static_cast<int>(threadIdx.x), lane = tid & 63;
  const int wv = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int n32 = lane & 31, half = lane >> 5;
  PrefillItem x;
  if (!prefill_item<Sh::kRows, TT>(p, x)) return;
  const int wave_row = 32 * wv;
  const int w_min = __builtin_amdgcn_readfirstlane(prefill_place(p, x, wave_row));
  const int w_max = __builtin_amdgcn_readfirstlane(prefill_place(p, x, wave_row + 31));
  const uint32_t lds0 = tile_lds_address(smem);
  const PrefillLoads<Sh> load(p, x, lds0, wv, lane);
  if (load.row_bytes < Sh::kRow) {  // products run over the slots past the head
    for (int i = tid; i < 4 * Sh::kTile / 16; i += 64 * NW) reinterpret_cast<u32x4*>(smem)[i] = u32x4{0u, 0u, 0u, 0u};
    tile_barrier();
  }
  auto load_tile = [&](int i) {
    const uint32_t to = (i & 1) * 2 * Sh::kTile;
    load(0, prefill_first<TT>(x, i), to);
    load(1, prefill_first<TT>(x, i), to + Sh::kTile);
  };
  if (x.tiles > 0) load_tile(0);
  const int place = prefill_place(p, x, wave_row + n32);
  u32x4 qf[Sh::kSteps];
  {
    const PrefillRow row = prefill_row(p, x, min(wave_row + n32, x.rows - 1));
    const char* src = static_cast<const char*>(p.q) +
                      ((x.q0 + row.query) * p.q_stride + (static_cast<int64_t>(x.h) * p.G + row.g) * p.D) * Sh::kES;
#pragma unroll
    for (int st = 0; st < Sh::kSteps; ++st) {
      const int at = 32 * st + 16 * half;
      qf[st] = at < load.row_bytes ? *reinterpret_cast<const u32x4*>(src + at) : u32x4{0u, 0u, 0u, 0u};
    }
  }
  f32x16 acc[Sh::kCols][1];
  float m[1] = {-INFINITY}, l[1] = {0.f};
#pragma unroll
  for (int c = 0; c < Sh::kCols; ++c) acc[c][0] = f32x16{};
  const uint32_t k_at = n32 * Sh::kRow + 16 * (half ^ prefill_swizzle(Sh::kSlots, n32));
  const uint32_t v_at = (4 * half * Sh::kRow + 16 * (n32 >> 2) + 4 * (n32 & 3)) ^ (32 * half);
  // V[token 32 tb + 8 (e / 4) + 4 half + e % 4][32 c + n32].
  auto read_v = [&](uint32_t at, int tb, int e, int c) {
    const int row = 32 * tb + 8 * (e / 4) + e % 4;
    return tile_lds_read<float>((at + v_at + row * Sh::kRow) ^ (128 * c) ^ (16 * (4 * (e % 4) + ((e / 4) & 1))));
  };
  __builtin_amdgcn_s_waitcnt((0x7 << 4) | (0xF << 8));  // vmcnt(0): no register load is pending in the loop
  bool found = false;
#pragma unroll 1
  for (int i = 0; i < x.tiles; ++i) {
    // The tile has arrived, and every wave is done with the one before it.
    tile_barrier_loads<0>();
    const int first = prefill_first<TT>(x, i), last = first + TT - 1;
    if (i + 1 < x.tiles) load_tile(i + 1);
    char* tile = smem + (i & 1) * 2 * Sh::kTile;
    const uint32_t at = lds0 + (i & 1) * 2 * Sh::kTile, vt = at + Sh::kTile;
    // Where only some rows see a token, a weight of 0 would not hide Inf and NaN
    // from the others: they are left out here and added at the end.
    if (!prefill_sees_all(p, first, last, x.p_min, x.p_max)) {
      found |= prefill_drop_bad<QD_DTYPE_F32, Sh::kTile / 16, 64 * NW>(tile + Sh::kTile, tid);
      tile_barrier();
    }
    const bool none = wave_row >= x.rows || first > w_max || (p.window > 0 && last <= w_min - p.window && first >= p.sinks);
    if (none) continue;
    f32x16 s[TB];
#pragma unroll
    for (int tb = 0; tb < TB; ++tb) s[tb] = f32x16{};
#pragma unroll
    for (int st = 0; st < Sh::kSteps; ++st)
#pragma unroll
      for (int tb = 0; tb < TB; ++tb)
        s[tb] = PrefillMma<QD_DTYPE_F32>::mma(tile_lds_read<u32x4>((at + k_at + 32 * tb * Sh::kRow) ^ (32 * st)), qf[st], s[tb]);
    if (!prefill_sees_all(p, first, last, w_min, w_max)) {
#pragma unroll
      for (int tb = 0; tb < TB; ++tb) {
        const PrefillView sees = prefill_view(p, place, first + 32 * tb + 4 * half);
#pragma unroll
        for (int e = 0; e < 16; ++e) s[tb][e] = sees(8 * (e / 4) + e % 4) ? s[tb][e] : -INFINITY;
      }
    }
    float mx = -INFINITY;
#pragma unroll
    for (int tb = 0; tb < TB; ++tb)
#pragma unroll
      for (int e = 0; e < 16; ++e) mx = fmaxf(mx, s[tb][e]);
    // The reference maximum moves when a weight would exceed 2^kLazy.
    if (__ballot((mx - m[0]) * p.sl2 > kLazy)) {
      const float mn = fmaxf(m[0], prefill_max_halves(mx));
      const float alpha = mn == m[0] ? 1.f : fast_exp2((m[0] - mn) * p.sl2);
      m[0] = mn;
      l[0] *= alpha;
#pragma unroll
      for (int c = 0; c < Sh::kCols; ++c) acc[c][0] *= alpha;
    }
    // As above, large scores are subtracted before they are multiplied.
    const float from = m[0] != -INFINITY && fabsf(m[0] * p.sl2) >= kPrefillFar ? m[0] : 0.f;
    if (__ballot(from != 0.f)) {
#pragma unroll
      for (int tb = 0; tb < TB; ++tb)
#pragma unroll
        for (int e = 0; e < 16; ++e) s[tb][e] -= from;
    }
    const float ref = from != 0.f || m[0] == -INFINITY ? 0.f : -m[0] * p.sl2;
#pragma unroll
    for (int tb = 0; tb < TB; ++tb)
#pragma unroll
      for (int e = 0; e < 16; ++e) s[tb][e] = fast_exp2(fmaf(s[tb][e], p.sl2, ref));
#pragma unroll
    for (int tb = 0; tb < TB; ++tb)
#pragma unroll
      for (int e = 0; e < 16; e += 4) l[0] += (s[tb][e] + s[tb][e + 1]) + (s[tb][e + 2] + s[tb][e + 3]);
#pragma unroll
    for (int tb = 0; tb < TB; ++tb)
#pragma unroll
      for (int e = 0; e < 16; ++e)
#pragma unroll
        for (int c = 0; c < Sh::kCols; ++c)
          acc[c][0] = __builtin_amdgcn_mfma_f32_32x32x2f32(read_v(vt, tb, e, c), s[tb][e], acc[c][0], 0, 0, 0);
  }
  tile_barrier();
  if (tid == 0) *word = 0;
  tile_barrier();
  if (found) *word = 1;
  tile_barrier();
  if (__builtin_amdgcn_readfirstlane(*word) != 0) {
#pragma unroll 1
    for (int i = 0; i < x.tiles; ++i) {
      const int first = prefill_first<TT>(x, i);
      if (prefill_sees_all(p, first, first + TT - 1, x.p_min, x.p_max)) continue;
      tile_barrier();
      load(1, first, 0);
      tile_barrier_loads<0>();
      prefill_to_flags<QD_DTYPE_F32, Sh::kTile / 16, 64 * NW>(smem, tid);
      tile_barrier();
#pragma unroll 1
      for (int tb = 0; tb < TB; ++tb) {
        const PrefillView sees = prefill_view(p, place, first + 32 * tb + 4 * half);
#pragma unroll
        for (int c = 0; c < Sh::kCols; ++c) {
          f32x16 seen = f32x16{};
#pragma unroll
          for (int e = 0; e < 16; ++e)
            seen = __builtin_amdgcn_mfma_f32_32x32x2f32(read_v(lds0 + 32 * tb * Sh::kRow, 0, e, c),
                                                        sees(8 * (e / 4) + e % 4) ? 1.f : 0.f, seen, 0, 0, 0);
#pragma unroll
          for (int e = 0; e < 16; ++e) acc[c][0][e] = prefill_add_bad(acc[c][0][e], seen[e]);
        }
      }
    }
  }
  prefill_store<QD_DTYPE_F32, DP, 1>(p, x, wave_row, acc, m, l);
}

template <int DT, int DP, int NB, int NW>
hipError_t prefill_launch(const PrefillParams& p, uint32_t grid, hipStream_t st) {
  using Sh = PrefillShape<DT, DP, NB, NW>;
  void (*fn)(PrefillParams);
  if constexpr (DT == QD_DTYPE_F32)
    fn = prefill_f32_kernel<DP, NW>;
  else
    fn = prefill_pipe_kernel<DT, DP, NB, NW>;
  static std::atomic<uint64_t> allowed{0};  // devices on which more than 64 KB of LDS were asked for
  int dev = 0;
  if (hipGetDevice(&dev) != hipSuccess) dev = 0;
  const uint64_t bit = uint64_t{1} << (dev & 63);
  if (!(allowed.load(std::memory_order_relaxed) & bit)) {
    const hipError_t e =
        hipFuncSetAttribute(reinterpret_cast<const void*>(fn), hipFuncAttributeMaxDynamicSharedMemorySize, Sh::kLds);
    if (e != hipSuccess) return e;
    allowed.fetch_or(bit, std::memory_order_relaxed);
  }
  hipLaunchKernelGGL(fn, dim3(grid), dim3(64 * NW), Sh::kLds, st, p);
  if (p.splits > 1)
    hipLaunchKernelGGL((prefill_merge_kernel<DT, (DP <= 64 ? 16 : 32)>),
                       dim3(static_cast<uint32_t>((static_cast<int64_t>(p.Tq) * p.Hq + 3) / 4)), dim3(256), 0, st, p);
  return hipGetLastError();
}

}  // namespace

#endif  // QD_PREFILL_KERNELS_H
