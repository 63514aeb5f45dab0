// A paged K/V cache in 8 bits with a scale per page and kv-head, for MI355X
// (gfx950): writing tokens to it (kv_append_q8) and reading it back as packed
// rows (kv_gather_q8).  C ABI in include/qd_attention.h.
//
// An element stands for itself times the scale of its page and head.  The
// writer's scales are powers of two, 2^e with the largest |x| of the page's
// rows in (2^(e-1), 2^e] times the type's largest value (448 or 127): x / 2^e is
// exact, so an element is off by its one rounding, and every element is
// determined.  For e4m3 that costs no precision (its steps are relative); int8
// gives away up to one of its seven bits against a scale of max / 127.  In
// return a page that goes on growing is rounded again only where its scale
// doubles, and the errors of all roundings add up to at most one step of the
// last scale (1/2 + 1/4 + ...), where scales that follow the maximum would add
// half a step for each of the page's tokens.

#include <hip/hip_runtime.h>

#include <stdint.h>
#include <string.h>

#include <algorithm>
#include <string>
#include <type_traits>

#include "packed.h"
#include "qd_device.h"

void qd_set_last_error(int status, const std::string& msg);

namespace {

typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));

struct CacheParams {
  void* key;  // append: read; gather: written
  void* value;
  void* kc;
  void* vc;
  float* ks;
  float* vs;
  const int32_t* table;
  const int32_t* at;  // append: positions; gather: context lengths
  const int32_t* cu;  // append: may be null
  int64_t k_stride, v_stride, num_blocks;
  int64_t parts;      // append: runs of tokens of one page
  int B, tokens, Hkv, D, P, maxP;
  PackedDivide by_page;
  PackedDivide by_hkv, by_row;  // append; by_row: pieces of a row
  int row_step, col_step;                // append: from a piece to the 64th after it
};

// VEC elements of a row, as loaded.
template <int DT, int VEC>
struct Piece {
  using S = typename Elem<DT>::S;
  typedef S Vec __attribute__((ext_vector_type(VEC)));
  Vec x;
  __device__ __forceinline__ void load(const S* p) { x = *reinterpret_cast<const Vec*>(p); }
  __device__ __forceinline__ float get(int i) const { return Elem<DT>::to_f(x[i]); }
};
template <int DT>
struct Piece<DT, 1> {
  using S = typename Elem<DT>::S;
  S x;
  __device__ __forceinline__ void load(const S* p) { x = *p; }
  __device__ __forceinline__ float get(int) const { return Elem<DT>::to_f(x); }
};

// Largest |x| seen, as the bits of |x| in x's own type: they order like the
// values, Inf and NaN above all finite ones.
template <int DT, int VEC>
struct Largest {
  uint32_t bits = 0;
  __device__ __forceinline__ void add(const Piece<DT, VEC>& p) {
    if constexpr (DT == QD_DTYPE_F32) {
#pragma unroll
      for (int i = 0; i < VEC; ++i) bits = max(bits, __float_as_uint(p.get(i)) & 0x7FFFFFFFu);
    } else if constexpr (VEC == 1) {
      bits = max(bits, static_cast<uint32_t>(__builtin_bit_cast(uint16_t, p.x) & 0x7FFF));
    } else {
      const u32x4 w = __builtin_bit_cast(u32x4, p.x);
#pragma unroll
      for (int i = 0; i < 4; ++i)
        bits = __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(u16x2, bits),
                                                                      __builtin_bit_cast(u16x2, w[i] & 0x7FFF7FFFu)));
    }
  }
  // The bits of the largest as a float32.
  __device__ __forceinline__ uint32_t f32_bits() const {
    if constexpr (DT == QD_DTYPE_F32) return bits;
    const uint32_t m = max(bits & 0xFFFFu, bits >> 16);
    if constexpr (DT == QD_DTYPE_BF16) return m << 16;
    return __float_as_uint(static_cast<float>(__builtin_bit_cast(_Float16, static_cast<uint16_t>(m))));
  }
};

__device__ __forceinline__ uint32_t q8_dpp_max(uint32_t x) {
  auto step = [](uint32_t a, uint32_t b) { return a > b ? a : b; };
  auto dpp = [](uint32_t y, auto ctrl) {
    return static_cast<uint32_t>(
        __builtin_amdgcn_update_dpp(static_cast<int>(y), static_cast<int>(y), decltype(ctrl)::value, 0xF, 0xF, false));
  };
  x = step(x, dpp(x, std::integral_constant<int, 0xB1>{}));   // quad_perm [1,0,3,2]
  x = step(x, dpp(x, std::integral_constant<int, 0x4E>{}));   // quad_perm [2,3,0,1]
  x = step(x, dpp(x, std::integral_constant<int, 0x141>{}));  // row_half_mirror
  x = step(x, dpp(x, std::integral_constant<int, 0x140>{}));  // row_mirror
  const auto a = __builtin_amdgcn_permlane32_swap(x, x, false, false);
  x = step(a[0], a[1]);
  const auto b = __builtin_amdgcn_permlane16_swap(x, x, false, false);
  return step(b[0], b[1]);
}

// The smallest power of two that keeps a finite |x| of these bits within the
// type, at least 2^-100; NaN for Inf, NaN and what would take more than 2^100.
template <int KIND>
__device__ __forceinline__ float power_scale(uint32_t bits) {
  if (bits >= 0x7F800000u) return __uint_as_float(0x7FC00000u);
  // bits = 2^(e - 1) times a fraction in [1, 2) (subnormal: below the floor).
  const int e = static_cast<int>(bits >> 23) - 126;
  const uint32_t top = KIND == QD_DTYPE_E4M3 ? 0x600000u : 0x7E0000u;  // of 448 = 1.75 * 2^8, of 127 = 127/64 * 2^6
  const int s = e - (KIND == QD_DTYPE_E4M3 ? 9 : 7) + ((bits & 0x7FFFFFu) > top ? 1 : 0);
  return __uint_as_float(s > 100 ? 0x7FC00000u : static_cast<uint32_t>(max(s, -100) + 127) << 23);
}

// Two and four elements of the cache from scaled values: one rounding, to
// nearest even.
template <int KIND>
__device__ __forceinline__ uint32_t pack4(float a, float b, float c, float d) {
  if constexpr (KIND == QD_DTYPE_E4M3) {
    const int w = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
    return static_cast<uint32_t>(__builtin_amdgcn_cvt_pk_fp8_f32(c, d, w, true));
  } else {
    const auto i8 = [](float x) { return static_cast<uint32_t>(static_cast<int>(__builtin_rintf(x))) & 0xFFu; };
    return i8(a) | i8(b) << 8 | i8(c) << 16 | i8(d) << 24;
  }
}

// Element i (0 to 3) of a word of the cache.
template <int KIND>
__device__ __forceinline__ f32x4 unpack4(uint32_t w) {
  if constexpr (KIND == QD_DTYPE_E4M3) {
    const auto a = __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(w), false);
    const auto b = __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(w), true);
    return f32x4{a[0], a[1], b[0], b[1]};
  } else {
    const int x = static_cast<int>(w);
    return f32x4{static_cast<float>(x << 24 >> 24), static_cast<float>(x << 16 >> 24), static_cast<float>(x << 8 >> 24),
                 static_cast<float>(x >> 24)};
  }
}

// The sequence that part u of `per` tokens lies in (base: its first part), its rows
// and its entry of `at`; for fewer than 64 sequences all in one round trip.
struct Packed {
  int b, start, count, at;
};
template <typename Base>
__device__ __forceinline__ Packed packed_at(const CacheParams& p, int per, int spare, Base&& base, int64_t u) {
  Packed x;
  if (p.B < 64) {
    const int lane = static_cast<int>(threadIdx.x) & 63;
    const int start = packed_start(p.cu, min(lane, p.B), p.tokens), at = p.at[min(lane, p.B - 1)];
    x.b = 63 - __builtin_clzll(__ballot(lane == 0 || (lane < p.B && base(start, lane) <= u)));
    x.start = __builtin_amdgcn_readlane(start, x.b);
    x.count = __builtin_amdgcn_readlane(start, x.b + 1) - x.start;
    x.at = __builtin_amdgcn_readlane(at, x.b);
  } else {
    x.b = packed_find(p.cu, p.B, p.tokens, 1, per, spare, u);
    x.start = __builtin_amdgcn_readfirstlane(packed_start(p.cu, x.b, p.tokens));
    x.count = __builtin_amdgcn_readfirstlane(packed_start(p.cu, x.b + 1, p.tokens)) - x.start;
    x.at = __builtin_amdgcn_readfirstlane(p.at[x.b]);
  }
  return x;
}

// A wave writes a run (the new tokens of one page) of one head's keys or values:
// largest value, scale, elements, with the rows in registers in between where
// they fit (HOLD pieces of 16 bytes per lane: 16 are 64 tokens of 128 16-bit
// elements, 32 twice that); longer runs are read again, from L2.  What it moves is 2
// T rows in and half as many bytes out: HBM bounds it for prompts, the round trips
// position -> page -> scale for single tokens (HOLD 0: a row per sequence, read
// beside the position).  24 prompts of up to 6000 tokens, 8 heads of 128, bf16 to
// e4m3, pages of 64: 93 us, 5.0 TB/s (streaming two bytes in for one out reaches 6.2
// over 4 GB); with the pieces' addresses kept from reading to writing it was 138 (160 registers, three waves per SIMD
// instead of four).  Up to 4000 tokens, pages of 128: 72 us, 101 with the runs read
// twice.  512 single tokens: 4.2 us, of 3 that an empty trip takes.
// grid ceil(2 parts Hkv / 4), block 256; a workgroup's waves have neighbouring
// heads, whose rows are neighbours in memory.
template <int DT, int KIND, int VEC, int HOLD>
__global__ __launch_bounds__(256, HOLD == 32 ? 2 : 4) void append_q8_kernel(CacheParams p) {
  using S = typename Elem<DT>::S;
  constexpr bool TOKENS = HOLD == 0;
  constexpr int kHold = !TOKENS ? HOLD : VEC == 1 ? 4 : 1;
  const int lane = static_cast<int>(threadIdx.x) & 63;
  const int64_t item = static_cast<int64_t>(blockIdx.x) * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (item >= 2 * p.parts * p.Hkv) return;
  const int pair = packed_divide(static_cast<uint32_t>(item), p.by_hkv);
  const int h = static_cast<int>(item) - pair * p.Hkv;
  const bool is_v = pair & 1;
  const int u = pair >> 1;
  const int64_t stride = is_v ? p.v_stride : p.k_stride;
  const S* rows_in = static_cast<const S*>(is_v ? p.value : p.key) + static_cast<int64_t>(h) * p.D;
  // Pieces of a run are numbered row by row; a lane takes every 64th.
  const int per_row = p.D / VEC;
  const int lane_row = packed_divide(static_cast<uint32_t>(lane), p.by_row), lane_col = lane - lane_row * per_row;
  struct Walk {
    int row, col;
  };
  // An opaque copy for each pass over the pieces: their places are computed again,
  // not kept in registers beside them.
  auto begin = [&]() {
    Walk w{lane_row, lane_col};
    asm volatile("" : "+v"(w.row), "+v"(w.col));
    return w;
  };
  auto next = [&](Walk& w) {
    w.row += p.row_step;
    w.col += p.col_step;
    if (w.col >= per_row) {
      w.col -= per_row;
      ++w.row;
    }
  };
  // Loads every piece of `held` that lies within `rows` rows.
  auto read = [&](auto& held, Walk& w, const S* src, int rows) {
#pragma unroll
    for (auto& x : held) {
      if (w.row < rows) x.load(src + w.row * stride + w.col * VEC);
      next(w);
    }
  };
  Piece<DT, VEC> held[kHold];
  int b = u, row0 = u, count = 1, page_at = 0, pos;
  if constexpr (TOKENS) {
    pos = p.at[b];
    Walk w = begin();
    read(held, w, rows_in + row0 * stride, 1);
  } else {
    // Parts of P tokens, with a spare one for a run begun at either end.
    auto base = [&](int start, int seq) { return packed_divide(static_cast<uint32_t>(start), p.by_page) + int64_t{2} * seq; };
    const Packed x = packed_at(p, p.P, 2, base, u);
    b = x.b;
    row0 = x.start;
    count = x.count;
    pos = x.at;
    page_at = static_cast<int>(u - base(row0, b));
  }
  if (pos < 0 || count <= 0) return;
  const int64_t page = packed_divide(static_cast<uint32_t>(pos), p.by_page) + static_cast<int64_t>(page_at);
  // Tokens [first, last) of the sequence's rows lie in the page.
  const int64_t first = max(page * p.P - pos, int64_t{0});
  const int64_t last = min((page + 1) * p.P - pos, static_cast<int64_t>(count));
  if (first >= last || page >= p.maxP) return;
  const int32_t phys = p.table[static_cast<int64_t>(b) * p.maxP + page];
  const int slot0 = static_cast<int>(pos + first - page * p.P);
  const int rows = static_cast<int>(last - first);
  const S* src = rows_in + (row0 + first) * stride;
  const int64_t total = static_cast<int64_t>(rows) * per_row;
  const bool held_all = TOKENS || total <= 64 * kHold;
  if (!TOKENS && held_all) {
    Walk w = begin();
    read(held, w, src, rows);
  }
  if (phys < 0 || phys >= p.num_blocks) return;
  float* scale_at = (is_v ? p.vs : p.ks) + static_cast<int64_t>(phys) * p.Hkv + h;
  uint8_t* page_base = static_cast<uint8_t*>(is_v ? p.vc : p.kc) +
                       (static_cast<int64_t>(phys) * p.P * p.Hkv + h) * p.D;
  const int64_t row_bytes = static_cast<int64_t>(p.Hkv) * p.D;
  const float old = slot0 > 0 ? *scale_at : 0.f;
  Largest<DT, VEC> most;
  auto weigh = [&](auto& held, Walk& w) {
#pragma unroll
    for (auto& x : held) {
      if (w.row < rows) most.add(x);
      next(w);
    }
  };
  constexpr int kSome = 8;  // pieces in flight of a longer run
  Walk all = begin();
  if (held_all) {
    weigh(held, all);
  } else {
    for (Walk w = all; __ballot(all.row < rows);) {
      Piece<DT, VEC> some[kSome];
      read(some, w, src, rows);
      weigh(some, all);
    }
  }
  const float fresh = power_scale<KIND>(q8_dpp_max(most.f32_bits()));
  // A NaN on either side stays; a caller's own scale may be negative.
  const float scale = slot0 == 0 || !(fabsf(old) >= fresh) ? (old != old ? old : fresh) : old;
  if (slot0 > 0 && !(scale == old)) {
    // The page's earlier rows, on the new scale (a power of two, so the factor
    // is exact).
    const float by = old / scale;
    const int64_t before = static_cast<int64_t>(slot0) * p.D;
    if constexpr (VEC > 1) {
      for (int64_t x = lane; x < before / 4; x += 64) {
        const int64_t r = div_nonneg(x, p.D / 4);
        uint32_t* at = reinterpret_cast<uint32_t*>(page_base + r * row_bytes) + (x - r * (p.D / 4));
        const f32x4 y = unpack4<KIND>(*at) * by;
        *at = pack4<KIND>(y[0], y[1], y[2], y[3]);
      }
    } else {
      for (int64_t x = lane; x < before; x += 64) {
        const int64_t r = div_nonneg(x, p.D);
        uint8_t* at = page_base + r * row_bytes + (x - r * p.D);
        *at = static_cast<uint8_t>(pack4<KIND>(unpack4<KIND>(*at)[0] * by, 0.f, 0.f, 0.f));
      }
    }
  }
  if (lane == 0) *scale_at = scale;
  // x / scale: a product where the scale is a power of two, as this kernel's
  // are; a caller's own may be anything.
  uint8_t* to = page_base + slot0 * row_bytes;
  auto write = [&](auto& held, Walk& w, auto&& scaled) {
#pragma unroll
    for (auto& x : held) {
      if (w.row < rows) {
        auto at = [&](int e) { return scaled(x.get(e)); };
        uint8_t* y = to + w.row * row_bytes + w.col * VEC;
        if constexpr (VEC == 8)
          *reinterpret_cast<u32x2*>(y) = u32x2{pack4<KIND>(at(0), at(1), at(2), at(3)), pack4<KIND>(at(4), at(5), at(6), at(7))};
        else if constexpr (VEC == 4)
          *reinterpret_cast<uint32_t*>(y) = pack4<KIND>(at(0), at(1), at(2), at(3));
        else
          *y = static_cast<uint8_t>(pack4<KIND>(at(0), 0.f, 0.f, 0.f));
      }
      next(w);
    }
  };
  auto write_all = [&](auto&& scaled) {
    Walk w = begin();
    if (held_all) {
      write(held, w, scaled);
    } else {
      for (Walk r = w; __ballot(w.row < rows);) {
        Piece<DT, VEC> some[kSome];
        read(some, r, src, rows);
        write(some, w, scaled);
      }
    }
  };
  if (__builtin_amdgcn_readfirstlane(__float_as_uint(scale) & 0x007FFFFFu) == 0) {
    const float inv = 1.f / scale;
    write_all([&](float x) { return x * inv; });
  } else {
    write_all([&](float x) { return x / scale; });
  }
}

// Tokens of a gather workgroup.
constexpr int kGatherRows = 32;

// A workgroup reads kGatherRows tokens of one sequence, keys or values, VEC
// elements per lane at a time; a lane keeps its column, and so its head.  Bound by
// HBM: one byte in and an element out.  Lanes write 16 neighbouring bytes each (16
// elements per lane, written in two halves: 111 us instead of 104 for 16 contexts
// of 1000 to 9000 tokens, 8 heads of 128), past the caches (104 -> 100 us, 5.3 TB/s; streaming one byte in for two out reaches 5.9):
// what reads the rows next mostly runs behind another L2.
// grid (tokens / kGatherRows + B, 2), block 256.
template <int DT, int KIND, int VEC>
__global__ __launch_bounds__(256) void gather_q8_kernel(CacheParams p) {
  using E = Elem<DT>;
  using S = typename E::S;
  __shared__ int64_t from[kGatherRows];  // pool row of a token
  __shared__ int32_t pages[kGatherRows];
  const int tid = static_cast<int>(threadIdx.x);
  const bool is_v = blockIdx.y != 0;
  const int64_t u = blockIdx.x;
  auto base = [](int start, int seq) { return int64_t{start / kGatherRows} + seq; };
  const Packed x = packed_at(p, kGatherRows, 1, base, u);
  const int64_t first = (u - base(x.start, x.b)) * kGatherRows;
  const int64_t have = min(static_cast<int64_t>(max(x.at, 0)), static_cast<int64_t>(p.maxP) * p.P);
  const int rows = static_cast<int>(min(min(have, static_cast<int64_t>(x.count)) - first, int64_t{kGatherRows}));
  if (rows <= 0) return;
  if (tid < rows) {
    const int tok = static_cast<int>(first) + tid, page = packed_divide(static_cast<uint32_t>(tok), p.by_page);
    const int32_t id = p.table[static_cast<int64_t>(x.b) * p.maxP + page];
    const int64_t phys = min(max(static_cast<int64_t>(id), int64_t{0}), p.num_blocks - 1);
    pages[tid] = static_cast<int32_t>(phys);
    from[tid] = phys * p.P + (tok - page * p.P);
  }
  __syncthreads();
  const int per_row = p.Hkv * (p.D / VEC);
  const int width = min(per_row, 256), teams = 256 / width;
  const int team = tid / width;
  if (team >= teams) return;
  const uint8_t* cache = static_cast<const uint8_t*>(is_v ? p.vc : p.kc);
  const float* scales = is_v ? p.vs : p.ks;
  const int64_t stride = is_v ? p.v_stride : p.k_stride, row_bytes = static_cast<int64_t>(p.Hkv) * p.D;
  S* out = static_cast<S*>(is_v ? p.value : p.key) + (x.start + first) * stride;
  constexpr int kAhead = 8;  // rows in flight
  constexpr int kWords = VEC >= 4 ? VEC / 4 : 1;
  for (int c = tid - team * width; c < per_row; c += width) {
    const int h = c / (p.D / VEC);
    for (int r0 = team; r0 < rows; r0 += kAhead * teams) {
      uint32_t w[kAhead][kWords];
      float scale[kAhead];
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
        const int r = min(r0 + i * teams, rows - 1);
        const uint8_t* src = cache + from[r] * row_bytes + static_cast<int64_t>(c) * VEC;
        if constexpr (VEC == 8) {
          const u32x2 x = stream_load8(reinterpret_cast<const char*>(src));
          w[i][0] = x[0];
          w[i][1] = x[1];
        } else if constexpr (VEC == 4) {
          w[i][0] = stream_load4(reinterpret_cast<const char*>(src));
        } else {
          w[i][0] = *src;
        }
        scale[i] = scales[static_cast<int64_t>(pages[r]) * p.Hkv + h];
      }
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
        const int r = r0 + i * teams;
        if (r >= rows) continue;
        S* to = out + r * stride + static_cast<int64_t>(c) * VEC;
        if constexpr (VEC == 1) {
          *to = E::from_f(unpack4<KIND>(w[i][0])[0] * scale[i]);
        } else if constexpr (VEC == 4) {
          __builtin_nontemporal_store(unpack4<KIND>(w[i][0]) * scale[i], reinterpret_cast<f32x4*>(to));
        } else {
          const f32x4 y = unpack4<KIND>(w[i][0]) * scale[i], z = unpack4<KIND>(w[i][1]) * scale[i];
          __builtin_nontemporal_store(u32x4{MfmaOps<DT>::pack2(y[0], y[1]), MfmaOps<DT>::pack2(y[2], y[3]),
                                            MfmaOps<DT>::pack2(z[0], z[1]), MfmaOps<DT>::pack2(z[2], z[3])},
                                      reinterpret_cast<u32x4*>(to));
        }
      }
    }
  }
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

// Workgroups of 256 threads, which are counted in 32 bits.
constexpr int64_t kMaxGrid = (1 << 24) - 1;

bool float_dtype(int dt) { return dt == QD_DTYPE_F32 || dt == QD_DTYPE_F16 || dt == QD_DTYPE_BF16; }
bool cache_dtype_ok(int dt) { return dt == QD_DTYPE_E4M3 || dt == QD_DTYPE_I8; }
uintptr_t bits_of(const void* p) { return reinterpret_cast<uintptr_t>(p); }

// Checks that kv_append_q8 and kv_gather_q8 share; `at` and its name: positions
// or context_lens.
int validate_rows(const qd_tensor_desc* key, const qd_tensor_desc* value, const qd_tensor_desc* k_cache,
                  const qd_tensor_desc* v_cache, const qd_tensor_desc* k_scales, const qd_tensor_desc* v_scales,
                  const qd_tensor_desc* table, const qd_tensor_desc* at, const qd_tensor_desc* cu, bool need_cu,
                  char* msg, size_t cap) {
  const qd_tensor_desc* all[9] = {key, value, k_cache, v_cache, k_scales, v_scales, table, at, cu};
  const bool has_cu = cu && cu->defined;
  for (int i = 0; i < 8; ++i)
    if (!all[i]) return q8_fail(msg, cap, "null tensor descriptor");
  if (need_cu && !has_cu) return q8_fail(msg, cap, "cu_seqlens must be int32 [B + 1]");
  for (int i = 0; i < (has_cu ? 9 : 8); ++i) {
    if (!all[i]->defined || !all[i]->is_device) return q8_fail(msg, cap, "all tensors must be CUDA tensors");
    if (all[i]->device_index != key->device_index) return q8_fail(msg, cap, "all tensors must share a device");
    if (!all[i]->contiguous)
      return q8_fail(msg, cap,
                     i < 2 ? "the heads of a token must be contiguous in key and value"
                           : "caches, scales and metadata must be contiguous");
  }
  if (key->ndim != 3) return q8_fail(msg, cap, "key/value must be [T, Hkv, D]");
  for (int i = 0; i < 3; ++i)
    if (value->ndim != 3 || value->sizes[i] != key->sizes[i]) return q8_fail(msg, cap, "key/value must be [T, Hkv, D]");
  if (k_cache->ndim != 4 || v_cache->ndim != 4) return q8_fail(msg, cap, "cache must be [Nblocks, P, Hkv, D]");
  for (int i = 0; i < 4; ++i)
    if (k_cache->sizes[i] != v_cache->sizes[i]) return q8_fail(msg, cap, "cache must be [Nblocks, P, Hkv, D]");
  if (k_cache->sizes[2] != key->sizes[1] || k_cache->sizes[3] != key->sizes[2])
    return q8_fail(msg, cap, "cache head shape mismatch");
  if (!(key->sizes[1] > 0 && key->sizes[2] > 0 && k_cache->sizes[0] > 0 && k_cache->sizes[1] > 0))
    return q8_fail(msg, cap, "invalid dimensions");
  if (key->sizes[2] > 256) return q8_fail(msg, cap, "supported head_dim is [1, 256]");
  for (const qd_tensor_desc* s : {k_scales, v_scales})
    if (s->ndim != 2 || s->dtype != QD_DTYPE_F32 || s->sizes[0] != k_cache->sizes[0] || s->sizes[1] != k_cache->sizes[2])
      return q8_fail(msg, cap, "scales must be float32 [Nblocks, Hkv]");
  if (!(at->ndim == 1 && table->ndim == 2 && table->sizes[0] == at->sizes[0] && table->sizes[1] > 0))
    return q8_fail(msg, cap, "invalid metadata shape");
  if (table->dtype != QD_DTYPE_I32 || at->dtype != QD_DTYPE_I32) return q8_fail(msg, cap, "metadata must be int32");
  if (has_cu && (cu->ndim != 1 || cu->dtype != QD_DTYPE_I32 || cu->sizes[0] != at->sizes[0] + 1))
    return q8_fail(msg, cap, "cu_seqlens must be int32 [B + 1]");
  if (!has_cu && key->sizes[0] != at->sizes[0])
    return q8_fail(msg, cap, "without cu_seqlens there must be one token per sequence");
  if (!float_dtype(key->dtype)) return q8_fail(msg, cap, "unsupported dtype");
  if (value->dtype != key->dtype) return q8_fail(msg, cap, "dtype mismatch");
  if (!cache_dtype_ok(k_cache->dtype) || v_cache->dtype != k_cache->dtype)
    return q8_fail(msg, cap, "caches must both be float8_e4m3fn or int8");
  if (key->sizes[0] > INT32_MAX || at->sizes[0] >= (1 << 24) || key->sizes[1] > 65535 ||
      k_cache->sizes[0] > INT32_MAX || k_cache->sizes[1] > INT32_MAX || table->sizes[1] > INT32_MAX)
    return q8_fail(msg, cap, "tensor sizes exceed int32 CUDA launch limits");
  if (msg && cap) msg[0] = '\0';
  return QD_OK;
}

// Argument checks of a launch; QD_OK with p filled.
int fill(CacheParams& p, void* key, void* value, void* kc, void* vc, float* ks, float* vs, const int32_t* table,
         const int32_t* at, const int32_t* cu, int batch, int64_t tokens, int kv_heads, int head_dim, int block_size,
         int max_pages, int64_t num_blocks, int64_t k_stride, int64_t v_stride, int dtype, int cache_dtype) {
  if (batch < 0 || batch >= (1 << 24) || tokens < 0 || tokens > INT32_MAX)
    return q8_fail(nullptr, 0, "batch and tokens must be >= 0, batch below 2^24");
  if (kv_heads <= 0 || kv_heads > 65535 || block_size <= 0 || max_pages <= 0 || num_blocks <= 0 ||
      num_blocks > INT32_MAX || k_stride < 0 || v_stride < 0)
    return q8_fail(nullptr, 0, "invalid dimensions");
  if (head_dim < 1 || head_dim > 256) return q8_fail(nullptr, 0, "supported head_dim is [1, 256]");
  if (!float_dtype(dtype) || !cache_dtype_ok(cache_dtype)) return q8_fail(nullptr, 0, "unsupported dtype");
  if (!cu && tokens != batch) return q8_fail(nullptr, 0, "without cu_seqlens there must be one token per sequence");
  if (batch > 0 && tokens > 0 && (!key || !value || !kc || !vc || !ks || !vs || !table || !at))
    return q8_fail(nullptr, 0, "null tensor pointer");
  p.key = key;
  p.value = value;
  p.kc = kc;
  p.vc = vc;
  p.ks = ks;
  p.vs = vs;
  p.table = table;
  p.at = at;
  p.cu = cu;
  p.k_stride = k_stride;
  p.v_stride = v_stride;
  p.num_blocks = num_blocks;
  p.B = batch;
  p.tokens = static_cast<int>(tokens);
  p.Hkv = kv_heads;
  p.D = head_dim;
  p.P = block_size;
  p.maxP = max_pages;
  return QD_OK;
}

template <typename F>
void by_types(int dtype, int cache_dtype, F&& run) {
  auto kind = [&](auto dt) {
    if (cache_dtype == QD_DTYPE_E4M3)
      run(dt, std::integral_constant<int, QD_DTYPE_E4M3>{});
    else
      run(dt, std::integral_constant<int, QD_DTYPE_I8>{});
  };
  if (dtype == QD_DTYPE_F32)
    kind(std::integral_constant<int, QD_DTYPE_F32>{});
  else if (dtype == QD_DTYPE_F16)
    kind(std::integral_constant<int, QD_DTYPE_F16>{});
  else
    kind(std::integral_constant<int, QD_DTYPE_BF16>{});
}

int launched(const char* what) {
  const hipError_t e = hipGetLastError();
  if (e == hipSuccess) return QD_OK;
  qd_set_last_error(static_cast<int>(e), std::string(what) + " kernel launch failed: " + hipGetErrorString(e));
  return static_cast<int>(e);
}

}  // namespace

extern "C" {

int qd_kv_append_q8_validate(const qd_tensor_desc* key, const qd_tensor_desc* value, const qd_tensor_desc* k_cache,
                             const qd_tensor_desc* v_cache, const qd_tensor_desc* k_scales,
                             const qd_tensor_desc* v_scales, const qd_tensor_desc* block_table,
                             const qd_tensor_desc* positions, const qd_tensor_desc* cu, char* msg, size_t msg_cap) {
  return validate_rows(key, value, k_cache, v_cache, k_scales, v_scales, block_table, positions, cu, false, msg,
                       msg_cap);
}

int qd_kv_append_q8(const void* key, const void* value, void* k_cache, void* v_cache, float* k_scales,
                    float* v_scales, const int32_t* block_table, const int32_t* positions, const int32_t* cu,
                    int batch, int64_t tokens, int kv_heads, int head_dim, int block_size, int max_pages,
                    int64_t num_blocks, int64_t k_stride, int64_t v_stride, int dtype, int cache_dtype, void* stream) {
  CacheParams p;
  const int bad = fill(p, const_cast<void*>(key), const_cast<void*>(value), k_cache, v_cache, k_scales, v_scales,
                       block_table, positions, cu, batch, tokens, kv_heads, head_dim, block_size, max_pages, num_blocks,
                       k_stride, v_stride, dtype, cache_dtype);
  if (bad != QD_OK) return bad;
  if (batch == 0 || tokens == 0) return QD_OK;
  const auto apart = [&](const void* a, const void* b, uint64_t unit) {
    return (std::max(bits_of(a), bits_of(b)) - std::min(bits_of(a), bits_of(b))) / unit >= static_cast<uint64_t>(num_blocks);
  };
  // Rows are bounded first, so that the pool's unit fits 64 bits.
  if (!apart(k_cache, v_cache, static_cast<uint64_t>(block_size) * kv_heads * head_dim))
    return q8_fail(nullptr, 0, "k_cache and v_cache must not overlap");
  if (!apart(k_scales, v_scales, 4 * static_cast<uint64_t>(kv_heads)))
    return q8_fail(nullptr, 0, "k_scales and v_scales must not overlap");
  p.parts = cu ? tokens / block_size + 2 * static_cast<int64_t>(batch) : batch;
  // Rows and items are counted in 32 bits, past their ends: a lane's pieces of a run
  // are up to 64 rows apart, and go on eight at a time.
  if (tokens > INT32_MAX - 255 || std::min<int64_t>(tokens, block_size) > INT32_MAX - 1023 ||
      2 * p.parts * kv_heads > 4 * kMaxGrid)
    return q8_fail(nullptr, 0, "tensor sizes exceed int32 CUDA launch limits");
  const int es = dtype == QD_DTYPE_F32 ? 4 : 2;
  const bool vec = (bits_of(key) | bits_of(value) | static_cast<uintptr_t>(head_dim * es) |
                    static_cast<uintptr_t>(k_stride * es) | static_cast<uintptr_t>(v_stride * es)) % 16 == 0 &&
                   (bits_of(k_cache) | bits_of(v_cache)) % 8 == 0;
  const int per_row = head_dim / (!vec ? 1 : dtype == QD_DTYPE_F32 ? 4 : 8);
  p.by_hkv = packed_divide_by(static_cast<uint32_t>(kv_heads));
  p.by_page = packed_divide_by(static_cast<uint32_t>(block_size));
  p.by_row = packed_divide_by(static_cast<uint32_t>(per_row));
  p.row_step = 64 / per_row;
  p.col_step = 64 % per_row;
  hipStream_t st = static_cast<hipStream_t>(stream);
  (void)hipGetLastError();
  by_types(dtype, cache_dtype, [&](auto dt, auto kind) {
    constexpr int DT = decltype(dt)::value, KIND = decltype(kind)::value, VEC = DT == QD_DTYPE_F32 ? 4 : 8;
    const dim3 grid(static_cast<uint32_t>((2 * p.parts * kv_heads + 3) / 4));
    // A page's pieces that 32 per lane hold and 16 do not.
    const int64_t pieces = static_cast<int64_t>(block_size) * per_row;
    if (vec && cu && pieces > 64 * 16 && pieces <= 64 * 32)
      hipLaunchKernelGGL((append_q8_kernel<DT, KIND, VEC, 32>), grid, dim3(256), 0, st, p);
    else if (vec && cu)
      hipLaunchKernelGGL((append_q8_kernel<DT, KIND, VEC, 16>), grid, dim3(256), 0, st, p);
    else if (vec)
      hipLaunchKernelGGL((append_q8_kernel<DT, KIND, VEC, 0>), grid, dim3(256), 0, st, p);
    else if (cu)
      hipLaunchKernelGGL((append_q8_kernel<DT, KIND, 1, 16>), grid, dim3(256), 0, st, p);
    else
      hipLaunchKernelGGL((append_q8_kernel<DT, KIND, 1, 0>), grid, dim3(256), 0, st, p);
  });
  return launched("kv_append_q8");
}

int qd_kv_gather_q8_validate(const qd_tensor_desc* key, const qd_tensor_desc* value, const qd_tensor_desc* k_cache,
                             const qd_tensor_desc* v_cache, const qd_tensor_desc* k_scales,
                             const qd_tensor_desc* v_scales, const qd_tensor_desc* block_table,
                             const qd_tensor_desc* context_lens, const qd_tensor_desc* cu, char* msg, size_t msg_cap) {
  return validate_rows(key, value, k_cache, v_cache, k_scales, v_scales, block_table, context_lens, cu, true, msg,
                       msg_cap);
}

int qd_kv_gather_q8(void* key, void* value, const void* k_cache, const void* v_cache, const float* k_scales,
                    const float* v_scales, const int32_t* block_table, const int32_t* context_lens,
                    const int32_t* cu, int batch, int64_t tokens, int kv_heads, int head_dim, int block_size,
                    int max_pages, int64_t num_blocks, int64_t k_stride, int64_t v_stride, int dtype,
                    int cache_dtype, void* stream) {
  CacheParams p;
  if (batch > 0 && tokens > 0 && !cu) return q8_fail(nullptr, 0, "null tensor pointer");
  const int bad = fill(p, key, value, const_cast<void*>(k_cache), const_cast<void*>(v_cache),
                       const_cast<float*>(k_scales), const_cast<float*>(v_scales), block_table, context_lens, cu, batch,
                       tokens, kv_heads, head_dim, block_size, max_pages, num_blocks, k_stride, v_stride, dtype,
                       cache_dtype);
  if (bad != QD_OK) return bad;
  if (batch == 0 || tokens == 0) return QD_OK;
  if (tokens > 1 && std::min(k_stride, v_stride) < static_cast<int64_t>(kv_heads) * head_dim)
    return q8_fail(nullptr, 0, "rows of key and value must not overlap");
  p.parts = tokens / kGatherRows + batch;
  if (p.parts > kMaxGrid) return q8_fail(nullptr, 0, "tensor sizes exceed int32 CUDA launch limits");
  p.by_page = packed_divide_by(static_cast<uint32_t>(block_size));
  const int es = dtype == QD_DTYPE_F32 ? 4 : 2;
  const bool out16 = (bits_of(key) | bits_of(value) | static_cast<uintptr_t>(k_stride * es) |
                      static_cast<uintptr_t>(v_stride * es)) % 16 == 0;
  const uintptr_t in = bits_of(k_cache) | bits_of(v_cache) | static_cast<uintptr_t>(head_dim);
  hipStream_t st = static_cast<hipStream_t>(stream);
  (void)hipGetLastError();
  const dim3 grid(static_cast<uint32_t>(p.parts), 2);
  by_types(dtype, cache_dtype, [&](auto dt, auto kind) {
    constexpr int DT = decltype(dt)::value, KIND = decltype(kind)::value;
    constexpr int VEC = DT == QD_DTYPE_F32 ? 4 : 8;
    if (out16 && in % VEC == 0)
      hipLaunchKernelGGL((gather_q8_kernel<DT, KIND, VEC>), grid, dim3(256), 0, st, p);
    else
      hipLaunchKernelGGL((gather_q8_kernel<DT, KIND, 1>), grid, dim3(256), 0, st, p);
  });
  return launched("kv_gather_q8");
}

}  // extern "C"
