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

#include "packed.h"
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
  int splits;                    // VALU kernel
  float sl2;                     // scale * log2(e)
  // Matrix-core kernel.
  int32_t* meta;                 // {first workgroup, last workgroup} per item
  int chunks, per;               // virtual kv-heads per kv-head and their q-heads (16 at most)
  int hw, groups;                // virtual heads of a workgroup, workgroups that share a sequence's tokens
  int W;                         // workgroups of a balanced launch; 0: one per item
  PackedDivide by_page, by_groups, by_chunks;
  int last_page;                 // num_blocks - 1
  int64_t page_bytes;
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

// ----------------------------------------------------------------------------
// The matrix-core kernel
// ----------------------------------------------------------------------------
//
// A wave serves up to 16 q-heads of a kv-head (a virtual kv-head) over 32 tokens
// at a time, straight from registers:
//   scores   S^T = K Q^T, 16x16x32 in fp16: a lane's 16 bytes of a K row become
//            operands of two products as they lie (the order of the head's
//            elements is the queries' too)
//   softmax  per lane; a token's weight is p = 2^(s - m) and goes into the values'
//            product as p s_v, whose running reference m is that of s + log2 |s_v|
//            (in two parts, a score and the rest, so that neither is lost beside
//            scores past 2^24):
//            whatever the pages' scales, the largest p s_v of a row is near 2^kShift
//            and fp16 holds the rest as far below it as fp16 goes.  p itself is up to
//            2^115 where scales are 2^-100 (a page of zeros): its sum is kept times
//            2^-12, so that 2^24 such terms fit, and one of scales of 2^100 (p down to
//            2^-93) loses nothing.
//   output   O^T += V^T (p s_v)^T, 16x16x32 in fp16: a lane reads E = DP / 16
//            neighbouring elements of 8 tokens' V rows and exchanges bytes
//            between token pairs in registers.
// Elements of both types are exact in fp16 (4 and 8 significant bits within 2^-9
// .. 448), and so are 16-bit queries, bf16 ones times a power of two that puts the
// largest of a head just inside fp16's range: 2^-24 of 2^14 is the least that
// they keep.  Weights are rounded to nearest once, 2^-12 on average.
//
// Half the bytes of 16-bit caches come in, and HBM bounds the kernel still: 48
// sequences of 2000 to 30000 tokens, 64 heads over 8 of 128, fp16 over int8, take 260 us, 5.9
// TB/s (reading alone reaches 6.9).  Per 32 tokens x 128 a wave moves 8 KB and
// issues about 200 (e4m3) or 300 (int8) vector instructions, where the SIMD has
// 2500 cycles.  Two tiles in registers, two waves per SIMD; three waves in 168
// registers spill (312 us).  Small batches are bound by their start: length,
// ranges, page and rows follow each other (5.8 us of 28 for 32 sequences of 512 to
// 4096 tokens, 32 heads), and by the merge's launch (4.6 us).
//
// Up to four waves of a workgroup take neighbouring virtual heads at the same
// tokens (whole rows of memory), or, with fewer heads, neighbouring 32 tokens.

constexpr float kQ8Shift = 7.f, kQ8Lazy = 8.f, kQ8Sum = 0x1p-12f;
// Balanced launches: what an item's start costs, in tiles, and the least cost of a
// workgroup's range.  Starts of 1 or 4 tiles: 256 sequences of 50 to 200 tokens 28.0
// us for 26.7; ranges of 4: one sequence of 1500 tokens 12.2 for 11.5, 16 sequences
// of up to 2000 with one kv-head 15.8 for 12.2.
constexpr int kQ8ItemCost = 2;
constexpr int kQ8MinCost = 2;
// Ranges per item from which a workgroup merges each row: one sequence of 30000
// tokens 37.6 -> 23.9 us, of 1500 11.1 -> 10.1, 16 of 2000 (16 ranges each) 22.2 ->
// 21.4, 20 of 2000 (12 each) 24.0 for 24.1.
constexpr int kQ8WideMerge = 12;
// Sequences whose prefix of costs fits the kernel's LDS.
constexpr int kQ8MaxBalanced = 1024;

__host__ __device__ constexpr int q8_padded(int d) { return d <= 64 ? 64 : d <= 128 ? 128 : 256; }

__device__ __forceinline__ float q8_max_groups(float x) {
  const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  x = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
  const auto b = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
__device__ __forceinline__ float q8_sum_groups(float x) {
  const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  x = __uint_as_float(a[0]) + __uint_as_float(a[1]);
  const auto b = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}

// fp16 pairs (0, 1) and (2, 3) of a word's elements.
template <int KIND>
__device__ __forceinline__ u32x2 q8_unpack(uint32_t w) {
  if constexpr (KIND == QD_DTYPE_E4M3) {
    return u32x2{__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.f, false)),
                 __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.f, true))};
  } else {
    // x + 128 as the low byte of 0x6400 is 1024 + 128 + x in fp16.
    const uint32_t y = w ^ 0x80808080u;
    const f16x2 off = {static_cast<_Float16>(-1152.f), static_cast<_Float16>(-1152.f)};
    const f16x2 a = __builtin_bit_cast(f16x2, __builtin_amdgcn_perm(0x64646464u, y, 0x04010400u)) + off,
                b = __builtin_bit_cast(f16x2, __builtin_amdgcn_perm(0x64646464u, y, 0x04030402u)) + off;
    return u32x2{__builtin_bit_cast(uint32_t, a), __builtin_bit_cast(uint32_t, b)};
  }
}

// Element e of words a and b as an fp16 pair, for e = 0 .. 3.
template <int KIND>
__device__ __forceinline__ void q8_pairs(uint32_t a, uint32_t b, uint32_t (&out)[4]) {
  if constexpr (KIND == QD_DTYPE_E4M3) {
    const uint32_t lo = __builtin_amdgcn_perm(b, a, 0x05010400u), hi = __builtin_amdgcn_perm(b, a, 0x07030602u);
    const u32x2 x = q8_unpack<KIND>(lo), y = q8_unpack<KIND>(hi);
    out[0] = x[0];
    out[1] = x[1];
    out[2] = y[0];
    out[3] = y[1];
  } else {
    const f16x2 off = {static_cast<_Float16>(-1152.f), static_cast<_Float16>(-1152.f)};
    const uint32_t w[4] = {__builtin_amdgcn_perm(b, a, 0x0C040C00u), __builtin_amdgcn_perm(b, a, 0x0C050C01u),
                           __builtin_amdgcn_perm(b, a, 0x0C060C02u), __builtin_amdgcn_perm(b, a, 0x0C070C03u)};
#pragma unroll
    for (int e = 0; e < 4; ++e)
      out[e] = __builtin_bit_cast(uint32_t, static_cast<f16x2>(__builtin_bit_cast(f16x2, w[e] ^ 0x64806480u) + off));
  }
}

// a b, rounded by itself: the same score is the same number whatever follows.
__device__ __forceinline__ float q8_rounded(float a, float b) {
#pragma clang fp contract(off)
  return a * b;
}

// What a row's weights count from: a score, and what to add to it.  -Inf: nothing yet.
struct Q8Ref {
  float score = -INFINITY, rest = -INFINITY;
  __device__ __forceinline__ Q8Ref() {}
  // Statistics of a part: score, sum of weights, rest.
  __device__ __forceinline__ explicit Q8Ref(f32x4 x) : score(x[0]), rest(x[2]) {}
  __device__ __forceinline__ f32x4 with(float sum) const { return f32x4{score, sum, rest, 0.f}; }
  __device__ __forceinline__ float from() const { return score == -INFINITY ? 0.f : score; }
  // The same with the score of n, which is not smaller.
  __device__ __forceinline__ float rest_from(const Q8Ref& n) const { return (score - n.from()) + rest; }
  // 2^(this - n).
  __device__ __forceinline__ float weight(const Q8Ref& n) const {
    return fast_exp2(rest_from(n) - (n.rest == -INFINITY ? 0.f : n.rest));
  }
  // The larger of both.
  __device__ __forceinline__ Q8Ref joined(const Q8Ref& o) const {
    Q8Ref n;
    n.score = fmaxf(score, o.score);
    n.rest = fmaxf(rest_from(n), o.rest_from(n));
    return n;
  }
};

template <int DP>
struct Q8Shape {
  static constexpr int E = DP / 16;       // V elements of a lane per token
  static constexpr int kPieces = DP / 64; // 16-byte pieces of a K row per lane
  static constexpr int kFrags = DP / 32;  // operands of the queries
  static constexpr int kLds = 4 * E * 1024 + 4 * 16 * 16;  // parts of waves that share heads, their rows' statistics
};

template <int DT, int KIND, int DP>
__global__ __launch_bounds__(256, DP == 256 ? 1 : 2) void q8_mfma_kernel(Q8Params p) {
  using Sh = Q8Shape<DP>;
  using Ops = MfmaOps<QD_DTYPE_F16>;
  constexpr int E = Sh::E;
  extern __shared__ __align__(16) char smem[];
  const int tid = static_cast<int>(threadIdx.x);
  const int lane = tid & 63, r16 = lane & 15, g4 = lane >> 4;
  const int wv = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int hw_log = p.hw >> 1;               // of 1, 2, 4
  const int tw_count = 4 >> hw_log;           // waves along the tokens
  const int wh = wv & (p.hw - 1), tw = wv >> hw_log;
  const int vheads = p.Hkv * p.chunks;
  const int row_bytes = p.Hkv * p.D;  // below 2^26

  auto process = [&](int b, int hg, int len, int t0, int t1, bool whole, int64_t slot) {
    const int v = hg * p.hw + wh;  // below vheads: hw divides it
    const int h = packed_divide(static_cast<uint32_t>(v), p.by_chunks), g0 = (v - h * p.chunks) * p.per;
    const int heads = min(p.per, p.G - g0);
    const bool real = r16 < heads;
    const int64_t q_row = static_cast<int64_t>(b) * p.Hq + static_cast<int64_t>(h) * p.G + g0 + (real ? r16 : 0);
    // Blocks of 16 tokens of this wave's tiles, 64 at a time (a window): lane i holds
    // block 2 (tile of pair i / 2) + i % 2, its page's scales, and ahead of need the
    // page of the next window's.
    const int32_t* table = p.table + static_cast<int64_t>(b) * p.maxP;
    const int last_block = (len - 1) >> 4;  // len > 0
    int64_t at_lane = 0;                    // byte of the block's first row in the pool
    float ks_lane = 0.f, vs_lane = 0.f;
    int32_t id_lane = 0;
    auto token_of = [&](int tile) {  // blocks are below 2^27
      return 16 * min(2 * ((tile + (lane >> 1)) * tw_count + tw) + (lane & 1), last_block);
    };
    auto find = [&](int tile) { id_lane = table[packed_divide(static_cast<uint32_t>(token_of(tile)), p.by_page)]; };
    // The window that find() was called for.
    auto window = [&](int tile, float& ks, float& vs) {
      const int tok = token_of(tile), page = packed_divide(static_cast<uint32_t>(tok), p.by_page);
      const int phys = min(max(id_lane, 0), p.last_page);
      at_lane = phys * p.page_bytes + (static_cast<int64_t>(tok - page * p.P) * row_bytes + h * p.D);
      const int64_t scale_at = static_cast<int64_t>(phys) * p.Hkv + h;
      ks = p.ks[scale_at];
      vs = p.vs[scale_at];
    };
    find(t0);
    window(t0, ks_lane, vs_lane);

    struct Raw {
      u32x4 k[2][Sh::kPieces];
      uint32_t v[2][4][E / 4];
    };
    // Columns past the head are read from its first ones: the queries are zero
    // there, and such columns of the output go nowhere.
    uint32_t k_off[Sh::kPieces];
#pragma unroll
    for (int j = 0; j < Sh::kPieces; ++j) k_off[j] = r16 * row_bytes + (64 * j + 16 * g4 < p.D ? 64 * j + 16 * g4 : 0);
    const uint32_t v_off = 4 * g4 * row_bytes + (E * r16 < p.D ? E * r16 : 0);
    auto load = [&](Raw& x, int i) {  // tile i of the window
#pragma unroll
      for (int tb = 0; tb < 2; ++tb) {
        const int64_t at = readlane_i64(at_lane, 2 * i + tb);
        const char* k = reinterpret_cast<const char*>(p.k) + at;
        const char* v = reinterpret_cast<const char*>(p.v) + at;
#pragma unroll
        for (int j = 0; j < Sh::kPieces; ++j) x.k[tb][j] = stream_load16(k + k_off[j]);
#pragma unroll
        for (int i2 = 0; i2 < 4; ++i2) {
          const char* src = v + v_off + i2 * row_bytes;
          if constexpr (E == 4) {
            x.v[tb][i2][0] = stream_load4(src);
          } else if constexpr (E == 8) {
            const u32x2 y = stream_load8(src);
            x.v[tb][i2][0] = y[0];
            x.v[tb][i2][1] = y[1];
          } else {
            const u32x4 y = stream_load16(src);
#pragma unroll
            for (int e = 0; e < 4; ++e) x.v[tb][i2][e] = y[e];
          }
        }
      }
    };
    Raw raw[2];
    int base = t0;  // the window's first tile
    if (t0 < t1) load(raw[0], 0);
    if (t0 + 32 < t1) find(t0 + 32);

    // Queries: operand 2 j + u holds elements 64 j + 16 g4 + 8 u .. of this
    // lane's head.
    u32x4 qf[Sh::kFrags];
    float q_inv = 1.f;
    {
      const char* src = static_cast<const char*>(p.q) + q_row * p.D * 2;
#pragma unroll
      for (int f = 0; f < Sh::kFrags; ++f) {
        const int d = 64 * (f >> 1) + 16 * g4 + 8 * (f & 1);
        qf[f] = real && d < p.D ? *reinterpret_cast<const u32x4*>(src + 2 * d) : u32x4{0u, 0u, 0u, 0u};
      }
      if constexpr (DT == QD_DTYPE_BF16) {
        float mx = 0.f;
#pragma unroll
        for (int f = 0; f < Sh::kFrags; ++f)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const f32x2 x = MfmaOps<QD_DTYPE_BF16>::unpack2(qf[f][i]);
            mx = fmaxf(mx, fmaxf(fabsf(x[0]), fabsf(x[1])));
          }
        mx = q8_max_groups(mx);
        const int e = static_cast<int>(__float_as_uint(mx) >> 23);  // 2^(e - 127) <= mx
        const int up = mx > 0.f && e < 255 ? min(max(14 - (e - 127), -120), 120) : 0;
        const float mul = __uint_as_float(static_cast<uint32_t>(127 + up) << 23);
        q_inv = __uint_as_float(static_cast<uint32_t>(127 - up) << 23);
#pragma unroll
        for (int f = 0; f < Sh::kFrags; ++f)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const f32x2 x = MfmaOps<QD_DTYPE_BF16>::unpack2(qf[f][i]);
            qf[f][i] = Ops::pack2(x[0] * mul, x[1] * mul);
          }
      }
    }
    f32x4 acc[E];
#pragma unroll
    for (int e = 0; e < E; ++e) acc[e] = f32x4{0.f, 0.f, 0.f, 0.f};
    Q8Ref m;
    float l = 0.f;

    auto compute = [&](Raw& x, int i, int tile) {
      const int first = (tile * tw_count + tw) * 32;
      f32x4 s[2];
      float high[2], lv[2], vs[2], ksc[2];
      const bool cut = first + 32 > len;
#pragma unroll
      for (int tb = 0; tb < 2; ++tb) {
        s[tb] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int j = 0; j < Sh::kPieces; ++j)
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            const u32x2 a = q8_unpack<KIND>(x.k[tb][j][2 * u]), c = q8_unpack<KIND>(x.k[tb][j][2 * u + 1]);
            s[tb] = Ops::mma32(u32x4{a[0], a[1], c[0], c[1]}, qf[2 * j + u], s[tb]);
          }
        vs[tb] = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(vs_lane), 2 * i + tb));
        ksc[tb] = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(ks_lane), 2 * i + tb)) * (p.sl2 * q_inv);
        lv[tb] = __builtin_amdgcn_logf(fmaxf(fabsf(vs[tb]), 0x1p-100f));
#pragma unroll
        for (int e = 0; e < 4; ++e) s[tb][e] = q8_rounded(s[tb][e], ksc[tb]);
        if (cut) {
          // Behind the last token: no weight, and no value (a NaN x 0).
          const int left = len - first - 16 * tb - 4 * g4;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            s[tb][e] = e < left ? s[tb][e] : -INFINITY;
#pragma unroll
            for (int w = 0; w < E / 4; ++w) x.v[tb][e][w] = e < left ? x.v[tb][e][w] : 0u;
          }
        }
        high[tb] = fmaxf(fmaxf(s[tb][0], s[tb][1]), fmaxf(s[tb][2], s[tb][3]));
      }
      auto rest = [&](float from) { return fmaxf((high[0] - from) + lv[0], (high[1] - from) + lv[1]); };
      if (__ballot(rest(m.from()) > m.rest + kQ8Lazy)) {
        Q8Ref n;
        n.score = fmaxf(m.score, q8_max_groups(fmaxf(high[0], high[1])));
        n.rest = fmaxf(m.rest_from(n), q8_max_groups(rest(n.from())));
        const float alpha = m.weight(n);
        m = n;
        l *= alpha;
#pragma unroll
        for (int e = 0; e < E; ++e) acc[e] *= alpha;
      }
      const float from = m.from(), ref = m.rest == -INFINITY ? kQ8Shift : kQ8Shift - m.rest;
      u32x4 w;
#pragma unroll
      for (int tb = 0; tb < 2; ++tb) {
#pragma unroll
        for (int e = 0; e < 4; ++e) s[tb][e] = fast_exp2((s[tb][e] - from) + ref);
        l = fmaf((s[tb][0] + s[tb][1]) + (s[tb][2] + s[tb][3]), kQ8Sum, l);
        w[2 * tb] = Ops::pack2(s[tb][0] * vs[tb], s[tb][1] * vs[tb]);
        w[2 * tb + 1] = Ops::pack2(s[tb][2] * vs[tb], s[tb][3] * vs[tb]);
      }
#pragma unroll
      for (int word = 0; word < E / 4; ++word) {
        uint32_t a[4][4];  // token pair, element
#pragma unroll
        for (int pair = 0; pair < 4; ++pair)
          q8_pairs<KIND>(x.v[pair >> 1][2 * (pair & 1)][word], x.v[pair >> 1][2 * (pair & 1) + 1][word], a[pair]);
#pragma unroll
        for (int e = 0; e < 4; ++e)
          acc[4 * word + e] = Ops::mma32(u32x4{a[0][e], a[1][e], a[2][e], a[3][e]}, w, acc[4 * word + e]);
      }
    };
    for (int tile = t0; tile < t1; tile += 2) {
      // 32 tiles of a window: both halves of the loop stay within it (its first
      // tile is a multiple of two from t0).
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const int now = tile + half;
        if (now >= t1) break;
        const int i = now - base;
        const bool more = now + 1 < t1, over = i == 31;
        float ks = 0.f, vs = 0.f;
        if (more) {
          if (over) window(now + 1, ks, vs);
          load(raw[half ^ 1], over ? 0 : i + 1);
        }
        __builtin_amdgcn_sched_barrier(0);
        compute(raw[half], i, now);
        if (more && over) {
          base = now + 1;
          ks_lane = ks;
          vs_lane = vs;
          if (base + 32 < t1) find(base + 32);
        }
      }
    }

    float sum = q8_sum_groups(l);
    if (tw_count > 1) {
      // Waves of the same heads: each leaves its part in LDS, the first of them
      // takes them up.
      __syncthreads();
      f32x4* stats = reinterpret_cast<f32x4*>(smem + 4 * E * 1024);
      f32x4* parts = reinterpret_cast<f32x4*>(smem);
#pragma unroll
      for (int e = 0; e < E; ++e) parts[(wv * E + e) * 64 + lane] = acc[e];
      if (g4 == 0) stats[wv * 16 + r16] = m.with(sum);
      __syncthreads();
      if (tw == 0) {
        Q8Ref most;
        for (int w = 0; w < tw_count; ++w) most = most.joined(Q8Ref(stats[(w * p.hw + wh) * 16 + r16]));
        sum = 0.f;
#pragma unroll
        for (int e = 0; e < E; ++e) acc[e] = f32x4{0.f, 0.f, 0.f, 0.f};
        for (int w = 0; w < tw_count; ++w) {
          const f32x4 x = stats[(w * p.hw + wh) * 16 + r16];
          const float f = Q8Ref(x).weight(most);
          sum += f * x[1];
#pragma unroll
          for (int e = 0; e < E; ++e) acc[e] += f * parts[((w * p.hw + wh) * E + e) * 64 + lane];
        }
        m = most;
      }
      __syncthreads();
      if (tw != 0) return;
    }
    if (!real) return;
    const bool has = sum > 0.f || sum != sum;
    if (whole) {
      const float inv = has ? kQ8Sum / sum : 0.f;
      char* to = static_cast<char*>(p.out) + q_row * p.D * 2;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int d = E * (4 * g4 + i);
        if (d >= p.D) continue;
        float y[E];
#pragma unroll
        for (int e = 0; e < E; ++e) y[e] = has ? acc[e][i] * inv : 0.f;
#pragma unroll
        for (int e = 0; e < E; e += 4)
          *reinterpret_cast<u32x2*>(to + 2 * (d + e)) =
              u32x2{MfmaOps<DT>::pack2(y[e], y[e + 1]), MfmaOps<DT>::pack2(y[e + 2], y[e + 3])};
      }
    } else {
      float* part = p.part + (slot * p.hw * 16 + wh * 16 + r16) * (p.D + 4);
      if (g4 == 0) *reinterpret_cast<f32x4*>(part) = has ? m.with(sum) : Q8Ref().with(0.f);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int d = E * (4 * g4 + i);
        if (d >= p.D) continue;
#pragma unroll
        for (int e = 0; e < E; e += 4)
          *reinterpret_cast<f32x4*>(part + 4 + d + e) =
              has ? f32x4{acc[e][i], acc[e + 1][i], acc[e + 2][i], acc[e + 3][i]} : f32x4{0.f, 0.f, 0.f, 0.f};
      }
    }
  };

  const int tile_tokens = 32 * tw_count;
  auto zero_rows = [&](int b, int hg) {  // a sequence without tokens
    const int first = hg * p.hw;
    for (int i = tid; i < p.hw * p.per * p.D; i += 256) {
      const int v = first + i / (p.per * p.D), x = i % (p.per * p.D);
      const int h = v / p.chunks, g = (v % p.chunks) * p.per + x / p.D;
      if (v < vheads && g < p.G)
        static_cast<uint16_t*>(p.out)[(static_cast<int64_t>(b) * p.Hq + h * p.G + g) * p.D + x % p.D] = 0;
    }
  };
  // Balanced: the costs of all items in a row (below 2^31: the host sees to it),
  // cut into equal ranges.  A lane holds a sequence's sum of costs up to its end;
  // more than 64 of them are in LDS.
  auto cost_of = [&](int len) { return len > 0 ? (((len + tile_tokens - 1) >> (7 - hw_log)) + kQ8ItemCost) * p.groups : 0; };
  auto scan = [](int x) {
    x = dpp_add_i32<0x111, 0xF>(x);     // row_shr:1
    x = dpp_add_i32<0x112, 0xF>(x);     // row_shr:2
    x = dpp_add_i32<0x114, 0xF>(x);     // row_shr:4
    x = dpp_add_i32<0x118, 0xF>(x);     // row_shr:8
    x = dpp_add_i32<0x142, 0xA>(x);     // row_bcast:15
    return dpp_add_i32<0x143, 0xC>(x);  // row_bcast:31
  };
  int32_t* incl = reinterpret_cast<int32_t*>(smem + (tw_count > 1 ? Sh::kLds : 0));
  const bool in_lanes = p.B <= 64;
  const int w = static_cast<int>(blockIdx.x);
  int len_lane = 0, incl_lane = 0, b = 0, pos = 0, end = 1;
  if (p.W > 0) {
    int total;
    if (in_lanes) {
      if (lane < p.B) len_lane = q8_len(p, lane);
      incl_lane = scan(cost_of(len_lane));
      total = __builtin_amdgcn_readlane(incl_lane, 63);
    } else {
      for (int i = tid; i < p.B; i += 256) incl[i] = cost_of(q8_len(p, i));
      __syncthreads();
      if (wv == 0) {
        int carry = 0;
        for (int from = 0; from < p.B; from += 64) {
          const int i = from + lane;
          const int x = scan(i < p.B ? incl[i] : 0) + carry;
          if (i < p.B) incl[i] = x;
          carry = __builtin_amdgcn_readlane(x, 63);
        }
      }
      __syncthreads();
      total = __builtin_amdgcn_readfirstlane(incl[p.B - 1]);
    }
    const int used = min(p.W, max(1, total / kQ8MinCost));
    if (w >= used) return;
    // The first `rem` ranges have a cost of `each` + 1.
    const int each = __builtin_amdgcn_readfirstlane(static_cast<int>(static_cast<uint32_t>(total) / static_cast<uint32_t>(used)));
    const int rem = total - each * used;
    pos = w * each + min(w, rem);
    end = pos + each + (w < rem ? 1 : 0);
    if (!in_lanes) {
      int lo = 0, hi = p.B - 1;
      while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (incl[mid] > pos) hi = mid; else lo = mid + 1;
      }
      b = __builtin_amdgcn_readfirstlane(lo);
    }
  }
  while (pos < end) {
    int len, hg, t0, t1, tiles;
    if (p.W == 0) {
      b = packed_divide(blockIdx.x, p.by_groups);
      hg = w - b * p.groups;
      len = __builtin_amdgcn_readfirstlane(q8_len(p, b));
      if (len == 0) zero_rows(b, hg);
      t0 = 0;
      tiles = t1 = (len + tile_tokens - 1) >> (7 - hw_log);
      pos = end;
    } else {
      // The first sequence that ends behind pos (pos < total: there is one).
      int upto, before;
      if (in_lanes) {
        b = __builtin_popcountll(__ballot(incl_lane <= pos));
        upto = __builtin_amdgcn_readlane(incl_lane, b);
        before = b > 0 ? __builtin_amdgcn_readlane(incl_lane, b - 1) : 0;
        len = __builtin_amdgcn_readlane(len_lane, b);
      } else {
        while (__builtin_amdgcn_readfirstlane(incl[b]) <= pos) ++b;
        upto = __builtin_amdgcn_readfirstlane(incl[b]);
        before = b > 0 ? __builtin_amdgcn_readfirstlane(incl[b - 1]) : 0;
        len = __builtin_amdgcn_readfirstlane(q8_len(p, b));
      }
      const uint32_t cost = packed_divide(static_cast<uint32_t>(upto - before), p.by_groups);
      hg = p.groups == 1 ? 0 : __builtin_amdgcn_readfirstlane(static_cast<int>(static_cast<uint32_t>(pos - before) / cost));
      const int off = pos - before - hg * static_cast<int>(cost);
      const int stop = min(static_cast<int>(cost), off + (end - pos));
      t0 = max(0, off - kQ8ItemCost);
      t1 = max(0, stop - kQ8ItemCost);
      tiles = static_cast<int>(cost) - kQ8ItemCost;
      pos += stop - off;
      if (t1 > t0 && tid == 0) {
        int32_t* meta = p.meta + 2 * (static_cast<int64_t>(b) * p.groups + hg);
        if (t0 == 0) meta[0] = w;
        if (t1 == tiles) meta[1] = w;
      }
    }
    if (t1 > t0)
      process(b, hg, len, t0, t1, t0 == 0 && t1 == tiles, 2 * static_cast<int64_t>(w) + (t0 == 0 ? 1 : 0));
  }
}

// Log-sum-exp merge of the items that a balanced launch split, and the rows of
// sequences without tokens: a wave per row, LANES lanes stride its columns four at
// a time, the others its partials; or, where items have many, a workgroup.
// grid (items, ceil(hw per / 4) or hw per), block 256.
template <int DT, int DP, int WAVES>
__global__ __launch_bounds__(256) void q8_merge_kernel(Q8Params p) {
  constexpr int LANES = DP / 4 < 32 ? DP / 4 : 32, TEAMS = 64 / LANES * WAVES, STEP = 4 * LANES;
  __shared__ f32x4 stats[4];
  __shared__ f32x4 joined[4][LANES];
  const int item = static_cast<int>(blockIdx.x), b = packed_divide(blockIdx.x, p.by_groups), hg = item - b * p.groups;
  const int lane = static_cast<int>(threadIdx.x) & 63;
  const int wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int row = WAVES == 4 ? static_cast<int>(blockIdx.y) : 4 * static_cast<int>(blockIdx.y) + wv;
  if (row >= p.hw * p.per) return;
  const int wh = row / p.per, n = row - wh * p.per;
  const int v = hg * p.hw + wh, h = v / p.chunks, g = (v - h * p.chunks) * p.per + n;
  if (g >= p.G) return;
  // One round trip (an empty sequence's entry was not written: not used).
  const int32_t first_of = p.meta[2 * static_cast<int64_t>(item)], last_of = p.meta[2 * static_cast<int64_t>(item) + 1];
  const bool empty = q8_len(p, b) == 0;
  const int first = empty ? 0 : first_of, count = empty ? 0 : last_of - first_of + 1;
  if (count == 1) return;
  const int team = lane / LANES + (WAVES == 4 ? 64 / LANES * wv : 0), l = lane % LANES;
  const int64_t slot_floats = static_cast<int64_t>(p.hw) * 16 * (p.D + 4);
  auto part = [&](int s) {
    return p.part + (2 * static_cast<int64_t>(first + s) + (s == 0 ? 1 : 0)) * slot_floats + (wh * 16 + n) * (p.D + 4);
  };
  char* out = static_cast<char*>(p.out) + (static_cast<int64_t>(b) * p.Hq + static_cast<int64_t>(h) * p.G + g) * p.D * 2;
  for (int d0 = 0; d0 < p.D; d0 += STEP) {
    const int d = d0 + 4 * l;
    Q8Ref m;
    float sum = 0.f;
    f32x4 a = {0.f, 0.f, 0.f, 0.f};
    // Eight partials at a time, statistics and values in flight together.
    constexpr int kAhead = 8;
    for (int s0 = kAhead * team; s0 < count; s0 += kAhead * TEAMS) {
      f32x2 ml[kAhead];
      float rest[kAhead];
      f32x4 x[kAhead];
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
        const float* src = part(min(s0 + i, count - 1));
        ml[i] = *reinterpret_cast<const f32x2*>(src);
        rest[i] = src[2];
        x[i] = d < p.D ? *reinterpret_cast<const f32x4*>(src + 4 + d) : f32x4{0.f, 0.f, 0.f, 0.f};
      }
      Q8Ref most = m;
#pragma unroll
      for (int i = 0; i < kAhead; ++i) most.score = fmaxf(most.score, ml[i][0]);
      const float from = most.from(), mine = (m.score - from) + m.rest;
      most.rest = mine;
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
        rest[i] += ml[i][0] - from;
        most.rest = fmaxf(most.rest, rest[i]);
      }
      const float ref = most.rest == -INFINITY ? 0.f : most.rest, old = fast_exp2(mine - ref);
      sum *= old;
      a *= old;
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
        if (s0 + i >= count) continue;
        const float f = fast_exp2(rest[i] - ref);
        sum += f * ml[i][1];
        a += f * x[i];
      }
      m = most;
    }
#pragma unroll
    for (int off = LANES; off < 64; off <<= 1) {
      Q8Ref o;
      o.score = __shfl_xor(m.score, off);
      o.rest = __shfl_xor(m.rest, off);
      const float os = __shfl_xor(sum, off);
      f32x4 oa;
#pragma unroll
      for (int i = 0; i < 4; ++i) oa[i] = __shfl_xor(a[i], off);
      const Q8Ref most = m.joined(o);
      const float f = m.weight(most), of = o.weight(most);
      sum = f * sum + of * os;
      a = f * a + of * oa;
      m = most;
    }
    if constexpr (WAVES == 4) {
      if (lane < LANES) joined[wv][lane] = a;
      if (lane == 0) stats[wv] = m.with(sum);
      __syncthreads();
      Q8Ref most;
#pragma unroll
      for (int w = 0; w < 4; ++w) most = most.joined(Q8Ref(stats[w]));
      sum = 0.f;
      a = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const float f = Q8Ref(stats[w]).weight(most);
        sum += f * stats[w][1];
        a += f * joined[w][l];
      }
      __syncthreads();
    }
    if (team == 0 && d < p.D) {
      const bool has = sum > 0.f || sum != sum;
      const float inv = has ? kQ8Sum / sum : 0.f;
      if (!has) a = f32x4{0.f, 0.f, 0.f, 0.f};
      *reinterpret_cast<u32x2*>(out + 2 * d) =
          u32x2{MfmaOps<DT>::pack2(a[0] * inv, a[1] * inv), MfmaOps<DT>::pack2(a[2] * inv, a[3] * inv)};
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

int q8_cu_count() {
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

// How a call runs.  All from static shapes and the device: the table's width
// stands for the longest context.
struct Q8Plan {
  bool mfma;
  int splits;                            // VALU kernel
  int chunks, per, hw, groups, W, grid;  // matrix-core kernel
  size_t meta_bytes, bytes;
};

Q8Plan q8_plan(int batch, int q_heads, int kv_heads, int head_dim, int block_size, int max_pages, int flags) {
  Q8Plan pl{};
  const int64_t cap = q8_capacity(block_size, max_pages);
  // Rows of a block at 32-bit offsets.
  pl.mfma = head_dim % 16 == 0 && block_size % 16 == 0 && !(flags & QD_FLAG_FORCE_GENERIC) &&
            static_cast<int64_t>(kv_heads) * head_dim <= INT32_MAX / 32;
  if (!pl.mfma) {
    pl.splits = generic_splits(batch, q_heads, cap);
    if (pl.splits > 1) pl.bytes = sizeof(float) * static_cast<size_t>(batch) * q_heads * pl.splits * (head_dim + 2);
    return pl;
  }
  const int group = q_heads / kv_heads;
  pl.chunks = (group + 15) / 16;
  pl.per = (group + pl.chunks - 1) / pl.chunks;
  pl.chunks = (group + pl.per - 1) / pl.per;
  const int vheads = kv_heads * pl.chunks;
  pl.hw = vheads % 4 == 0 ? 4 : vheads % 2 == 0 ? 2 : 1;
  pl.groups = vheads / pl.hw;
  const int64_t items = static_cast<int64_t>(batch) * pl.groups;
  const int tile = 32 * (4 / pl.hw);
  const int64_t tiles = (cap + tile - 1) / tile;
  const int64_t resident = static_cast<int64_t>(q8_cu_count()) * (q8_padded(head_dim) == 256 ? 1 : 2);
  pl.grid = static_cast<int>(items);
  // One workgroup per item, without a merge, where contexts are short (up to 8 tiles,
  // or 16 with items for every workgroup that the card holds), and where the items'
  // costs do not fit the kernel's LDS or 31 bits.  us, ranges / items, 32 heads over 8
  // of 128: 256 sequences of 50 to 200 tokens 27.2 / 19.6, of 100 to 500 44.2 / 40.0,
  // of 100 to 1000 67.4 / 71.5; 64 of 100 to 250 15.2 / 13.0, of 100 to 500 17.8 /
  // 20.9; 4 of 100 11.5 / 8.9.
  if (batch > kQ8MaxBalanced || items * (tiles + kQ8ItemCost) > INT32_MAX || tiles <= (items >= resident ? 16 : 8))
    return pl;
  pl.W = static_cast<int>(std::max<int64_t>(1, std::min(resident, items * (tiles + kQ8ItemCost) / kQ8MinCost)));
  pl.grid = pl.W;
  pl.meta_bytes = (8 * static_cast<size_t>(items) + 15) / 16 * 16;
  pl.bytes = pl.meta_bytes + sizeof(float) * 2 * static_cast<size_t>(pl.W) * pl.hw * 16 * (head_dim + 4);
  return pl;
}

template <int DT, int KIND, int DP>
hipError_t launch_mfma(const Q8Params& p, int grid, hipStream_t st) {
  const size_t lds = (p.hw < 4 ? Q8Shape<DP>::kLds : 0) + (p.W > 0 ? sizeof(int32_t) * static_cast<size_t>(p.B) : 0);
  void (*fn)(Q8Params) = q8_mfma_kernel<DT, KIND, DP>;
  static std::atomic<uint64_t> allowed{0};  // devices on which more than 64 KB of LDS were asked for
  int dev = 0;
  if (hipGetDevice(&dev) != hipSuccess) dev = 0;
  const uint64_t bit = uint64_t{1} << (dev & 63);
  if (!(allowed.load(std::memory_order_relaxed) & bit)) {
    const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(fn), hipFuncAttributeMaxDynamicSharedMemorySize,
                                             Q8Shape<DP>::kLds + 4 * kQ8MaxBalanced);
    if (e != hipSuccess) return e;
    allowed.fetch_or(bit, std::memory_order_relaxed);
  }
  hipLaunchKernelGGL(fn, dim3(static_cast<uint32_t>(grid)), dim3(256), lds, st, p);
  if (p.W == 0) return hipGetLastError();
  const uint32_t items = static_cast<uint32_t>(p.B * p.groups), rows = static_cast<uint32_t>(p.hw * p.per);
  if (p.W >= kQ8WideMerge * p.B * p.groups)
    hipLaunchKernelGGL((q8_merge_kernel<DT, DP, 4>), dim3(items, rows), dim3(256), 0, st, p);
  else
    hipLaunchKernelGGL((q8_merge_kernel<DT, DP, 1>), dim3(items, (rows + 3) / 4), dim3(256), 0, st, p);
  return hipGetLastError();
}

template <int DT, int KIND>
hipError_t launch_padded(const Q8Params& p, int grid, hipStream_t st) {
  switch (q8_padded(p.D)) {
    case 64: return launch_mfma<DT, KIND, 64>(p, grid, st);
    case 128: return launch_mfma<DT, KIND, 128>(p, grid, st);
    default: return launch_mfma<DT, KIND, 256>(p, grid, st);
  }
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
  if (!q8_shape_ok(batch, q_heads, kv_heads, head_dim, block_size, max_pages, dtype) || batch == 0) return 0;
  // Unaligned tensors take the VALU kernel.
  return std::max(q8_plan(batch, q_heads, kv_heads, head_dim, block_size, max_pages, flags).bytes,
                  q8_plan(batch, q_heads, kv_heads, head_dim, block_size, max_pages, QD_FLAG_FORCE_GENERIC).bytes);
}

int qd_gqa_decode_q8_info(int batch, int q_heads, int kv_heads, int head_dim, int block_size, int max_pages,
                          int dtype, int flags, int* workgroups) {
  if (!q8_shape_ok(batch, q_heads, kv_heads, head_dim, block_size, max_pages, dtype)) return -1;
  const Q8Plan pl = q8_plan(batch, q_heads, kv_heads, head_dim, block_size, max_pages, flags);
  if (workgroups) *workgroups = pl.mfma ? pl.grid : batch * q_heads * pl.splits;
  return !pl.mfma ? QD_Q8_VALU : pl.W > 0 ? QD_Q8_MFMA_SPLIT : QD_Q8_MFMA;
}

int qd_gqa_decode_q8(const void* q, const void* k_cache, const void* v_cache, const float* k_scales,
                     const float* v_scales, const int32_t* block_table, const int32_t* context_lens, void* out,
                     void* workspace, size_t workspace_bytes, int batch, int q_heads, int kv_heads, int head_dim,
                     int block_size, int max_pages, int64_t num_blocks, int dtype, int cache_dtype, float scale,
                     int flags, void* stream) {
  if (!q8_shape_ok(batch, q_heads, kv_heads, head_dim, block_size, max_pages, dtype) || num_blocks <= 0 ||
      num_blocks > INT32_MAX || (cache_dtype != QD_DTYPE_E4M3 && cache_dtype != QD_DTYPE_I8))
    return q8_fail(nullptr, 0, "invalid dimensions");
  if (!(scale > 0.f) || !isfinite(scale)) return q8_fail(nullptr, 0, "scale must be positive and finite");
  if (batch == 0) return QD_OK;
  if (!q || !k_cache || !v_cache || !k_scales || !v_scales || !block_table || !context_lens || !out)
    return q8_fail(nullptr, 0, "null tensor pointer");
  if (((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(k_cache) | reinterpret_cast<uintptr_t>(v_cache) |
        reinterpret_cast<uintptr_t>(out)) &
       15u) != 0)
    flags |= QD_FLAG_FORCE_GENERIC;
  const Q8Plan pl = q8_plan(batch, q_heads, kv_heads, head_dim, block_size, max_pages, flags);
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
  p.part = reinterpret_cast<float*>(static_cast<char*>(workspace) + pl.meta_bytes);
  p.meta = static_cast<int32_t*>(workspace);
  p.chunks = pl.chunks;
  p.per = pl.per;
  p.hw = pl.hw;
  p.groups = pl.groups;
  p.W = pl.W;
  p.last_page = static_cast<int>(num_blocks - 1);
  p.page_bytes = static_cast<int64_t>(block_size) * kv_heads * head_dim;
  p.by_page = packed_divide_by(static_cast<uint32_t>(block_size));
  p.by_groups = packed_divide_by(static_cast<uint32_t>(std::max(pl.groups, 1)));
  p.by_chunks = packed_divide_by(static_cast<uint32_t>(std::max(pl.chunks, 1)));
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
  hipError_t e = hipSuccess;
  if (pl.mfma) {
    const bool e4m3 = cache_dtype == QD_DTYPE_E4M3;
    if (dtype == QD_DTYPE_F16)
      e = e4m3 ? launch_padded<QD_DTYPE_F16, QD_DTYPE_E4M3>(p, pl.grid, st)
               : launch_padded<QD_DTYPE_F16, QD_DTYPE_I8>(p, pl.grid, st);
    else
      e = e4m3 ? launch_padded<QD_DTYPE_BF16, QD_DTYPE_E4M3>(p, pl.grid, st)
               : launch_padded<QD_DTYPE_BF16, QD_DTYPE_I8>(p, pl.grid, st);
  } else {
    if (dtype == QD_DTYPE_F16)
      launch_generic<QD_DTYPE_F16>(p, cache_dtype, st);
    else
      launch_generic<QD_DTYPE_BF16>(p, cache_dtype, st);
    e = hipGetLastError();
  }
  if (e != hipSuccess) {
    qd_set_last_error(static_cast<int>(e), std::string("gqa_decode_q8 kernel launch failed: ") + hipGetErrorString(e));
    return static_cast<int>(e);
  }
  return QD_OK;
}

}  // extern "C"
