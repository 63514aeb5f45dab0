// Device code of prompt attention shared by the VALU kernel (prefill.hip) and
// the matrix-core kernels (prefill_mfma_*.hip).
#ifndef QD_PREFILL_KERNELS_H
#define QD_PREFILL_KERNELS_H

#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include <atomic>

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
  float sl2;  // scale * log2(e)
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
  static constexpr int kLds = 4 * kTile + 16;
  static_assert(kLoadRows * kSlots % 64 == 0 && DP % 32 == 0, "waves do not fit the tile");
};

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
// positions.  The workgroup goes through the tokens that its rows see in tiles of
// TT: K and V rows come straight into one of two LDS buffers, one tile ahead, and
// each wave multiplies its 32 NB rows with them:
//   scores   S^T = K Q^T, 32x32 blocks (A = K rows from LDS, B = Q from
//            registers): a lane holds one row and 16 of 32 tokens
//   softmax  per lane; the reference maximum of a row moves only when a score
//            exceeds it by 2^kLazy, so most tiles exchange nothing between lanes
//   output   O^T += V^T P^T: the score layout is already the B operand (the
//            products sum over tokens in the order that the lanes hold them in),
//            V^T comes from transposing LDS reads.
// 16-bit weights are rounded to nearest once: half a step of the output's type,
// which a sum over many values averages out.
template <int DT, int DP, int NB, int NW>
__global__ __launch_bounds__(64 * NW, (NB == 1 && DP <= 128 && DT != QD_DTYPE_F32 ? 2 : 1)) void prefill_mfma_kernel(PrefillParams p) {
  using Sh = PrefillShape<DT, DP, NB, NW>;
  using E = Elem<DT>;
  using S = typename E::S;
  constexpr bool k16 = DT != QD_DTYPE_F32;
  constexpr int ES = Sh::kES, TT = Sh::TT, TB = Sh::kTB;
  // fp16 weights are multiples of 2^-24 and the largest of a row is at least
  // 2^kShift: what that grid adds is at most 2^-32 of it.
  constexpr float kShift = DT == QD_DTYPE_F16 ? 7.f : 0.f;
  constexpr float kLazy = 8.f;
  extern __shared__ __align__(16) char smem[];
  int* bad_word = reinterpret_cast<int*>(smem + 4 * Sh::kTile);
  const int tid = static_cast<int>(threadIdx.x), lane = tid & 63;
  const int wv = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int n32 = lane & 31, half = lane >> 5;
  const int h = static_cast<int>(blockIdx.x % static_cast<uint32_t>(p.Hkv));
  // The last rows of a sequence see most: first.
  const int64_t u = gridDim.x / static_cast<uint32_t>(p.Hkv) - 1 - blockIdx.x / static_cast<uint32_t>(p.Hkv);
  const int b = packed_find(p.cu, p.B + 1, p.Tq, p.G, Sh::kRows, 1, u);
  const bool tail = b == p.B;  // rows behind the last sequence
  const int q0 = packed_start(p.cu, b, p.Tq), q1 = tail ? p.Tq : packed_start(p.cu, b + 1, p.Tq);
  const int rows_all = max(q1 - q0, 0) * p.G;  // below 2^31: Tq Hq is
  const int64_t row0_64 = (u - packed_base(p.cu, b, p.Tq, p.G, Sh::kRows, 1)) * Sh::kRows;
  if (row0_64 >= rows_all) return;
  const int row0 = static_cast<int>(row0_64);
  const int rows = min(Sh::kRows, rows_all - row0);
  const int k0 = tail ? 0 : packed_start(p.cu_k, b, p.Tk);
  const int nk = tail ? 0 : max(packed_start(p.cu_k, b + 1, p.Tk) - k0, 0);
  const int before = nk - (q1 - q0);  // position of query 0
  const int row_bytes = p.D * ES;
  // Positions of the workgroup's rows, and of this wave's.
  const int p_min = before + row0 / p.G, p_max = before + (row0 + rows - 1) / p.G;
  const int wave_row = 32 * NB * wv;
  const int w_min = before + min(row0 + wave_row, row0 + rows - 1) / p.G;
  const int w_max = before + min(row0 + wave_row + 32 * NB - 1, row0 + rows - 1) / p.G;
  const bool wave_real = wave_row < rows;
  // Tiles [0, sink_tiles) and from lo_tile on.
  const int end = min(p_max + 1, nk);
  const int lo = p.window > 0 ? max(p_min - p.window + 1, 0) : 0;
  const int lo_tile = lo / TT;
  const int sink_tiles = min((min(p.sinks, lo) + TT - 1) / TT, lo_tile);
  const int tiles = end > 0 ? sink_tiles + (end + TT - 1) / TT - lo_tile : 0;
  auto first_of = [&](int i) { return TT * (i < sink_tiles ? i : i - sink_tiles + lo_tile); };

  const char* k_base = static_cast<const char*>(p.k) + (k0 * p.k_stride + static_cast<int64_t>(h) * p.D) * ES;
  const char* v_base = static_cast<const char*>(p.v) + (k0 * p.v_stride + static_cast<int64_t>(h) * p.D) * ES;
  const uint32_t k_bytes = static_cast<uint32_t>(p.k_stride * ES), v_bytes = static_cast<uint32_t>(p.v_stride * ES);
  const bool padded = row_bytes < Sh::kRow;
  uint32_t col[Sh::kLoads];
  int load_row[Sh::kLoads];
#pragma unroll
  for (int i = 0; i < Sh::kLoads; ++i) {
    load_row[i] = Sh::kLoadRows * wv + (64 * i + lane) / Sh::kSlots;
    col[i] = 16 * ((lane & (Sh::kSlots - 1)) ^ tile_swizzle(Sh::kSlots, load_row[i]));
  }
  const uint32_t lds0 = tile_lds_address(smem);
  const uint32_t lds_wave = __builtin_amdgcn_readfirstlane(lds0 + Sh::kLoadRows * wv * Sh::kRow);
  // Rows past the last key repeat it: they are hidden from every query.
  auto load_tile = [&](int first, int slot) {
    const char* k = k_base + static_cast<int64_t>(first) * k_bytes;
    const char* v = v_base + static_cast<int64_t>(first) * v_bytes;
    const uint32_t to = lds_wave + slot * 2 * Sh::kTile;
    const int last = nk - 1 - first;
#pragma unroll
    for (int i = 0; i < Sh::kLoads; ++i) {
      const uint32_t r = min(load_row[i], last);
      if (!padded || static_cast<int>(col[i]) < row_bytes) {
        tile_load_lds<false>(k, r * k_bytes + col[i], to + 1024 * i);
        tile_load_lds<false>(v, r * v_bytes + col[i], to + Sh::kTile + 1024 * i);
      }
    }
  };

  if (padded) {  // products run over the slots past the head
    for (int i = tid; i < 4 * Sh::kTile / 16; i += 64 * NW) reinterpret_cast<u32x4*>(smem)[i] = u32x4{0u, 0u, 0u, 0u};
    tile_barrier();
  }
  if (tiles > 0) load_tile(first_of(0), 0);

  // This lane's rows.
  int place[NB];  // position of its query
  u32x4 qf[NB][Sh::kSteps];
#pragma unroll
  for (int nb = 0; nb < NB; ++nb) {
    const int row = row0 + min(wave_row + 32 * nb + n32, rows - 1);
    const int query = row / p.G;
    place[nb] = before + query;
    const char* src = static_cast<const char*>(p.q) +
                      ((q0 + query) * p.q_stride + (static_cast<int64_t>(h) * p.G + (row - query * p.G)) * p.D) * ES;
#pragma unroll
    for (int st = 0; st < Sh::kSteps; ++st) {
      const int at = 32 * st + 16 * half;
      qf[nb][st] = at < row_bytes ? *reinterpret_cast<const u32x4*>(src + at) : u32x4{0u, 0u, 0u, 0u};
    }
  }
  f32x16 acc[Sh::kCols][NB];
  float m[NB], l[NB];
#pragma unroll
  for (int nb = 0; nb < NB; ++nb) {
    m[nb] = -INFINITY;
    l[nb] = 0.f;
#pragma unroll
    for (int c = 0; c < Sh::kCols; ++c) acc[c][nb] = f32x16{};
  }
  // Addresses of operands within a tile (bytes).
  const uint32_t k_at = n32 * Sh::kRow + 16 * (half ^ tile_swizzle(Sh::kSlots, n32));
  const int r16 = lane & 15;
  const int vr = 4 * half + (k16 ? r16 >> 2 : 0);
  const uint32_t v_at = k16 ? vr * Sh::kRow + 16 * ((2 * ((lane >> 4) & 1) + ((r16 >> 1) & 1)) ^ tile_swizzle(Sh::kSlots, vr)) + 8 * (r16 & 1)
                            : 4 * half * Sh::kRow + 16 * (n32 >> 2) + 4 * (n32 & 3);
  __builtin_amdgcn_s_waitcnt((0x7 << 4) | (0xF << 8));  // vmcnt(0): no register load is pending in the loop

  auto visible = [&](int nb, int token) {
    return token <= place[nb] && (p.window == 0 || token > place[nb] - p.window || token < p.sinks);
  };
  // V^T operand of 16 tokens (16-bit) for columns 32 c..
  auto read_v16 = [&](uint32_t at, int ks, int c) {
    const uint32_t a = at + v_at + 16 * ks * Sh::kRow;
    const u32x2 x = tile_tr_read(a ^ (64 * c)), y = tile_tr_read((a + 8 * Sh::kRow) ^ (64 * c) ^ 16);
    return u32x4{x[0], x[1], y[0], y[1]};
  };
  // V[token 32 tb + 8 (i / 4) + 4 half + i % 4][32 c + n32] (fp32).
  auto read_v32 = [&](uint32_t at, int tb, int i, int c) {
    const int row = 32 * tb + 8 * (i / 4) + i % 4;
    return tile_lds_read<float>((at + v_at + row * Sh::kRow) ^ (128 * c) ^ (16 * (8 * half)) ^ (16 * (2 * (i % 4) + ((i / 4) & 1))));
  };

  for (int i = 0; i < tiles; ++i) {
    // The tile has arrived, and every wave is done with the one before it.
    tile_barrier_loads<0>();
    const int first = first_of(i), slot = i & 1;
    if (i + 1 < tiles) load_tile(first_of(i + 1), slot ^ 1);
    const uint32_t at = lds0 + slot * 2 * Sh::kTile, vt = at + Sh::kTile;
    char* tile = smem + slot * 2 * Sh::kTile;
    const int last = first + TT - 1;
    // Every row of the workgroup (of the wave) sees all of the tile.
    auto sees_all = [&](int lowest, int highest) {
      return last <= lowest && (p.window == 0 || first > highest - p.window || last < p.sinks);
    };
    const bool whole = sees_all(p_min, p_max);
    bool bad = false;
    if (!whole) {
      // Where only some rows see a token, a weight of 0 would not hide Inf and
      // NaN from the others.
      if (tid == 0) *bad_word = 0;
      tile_barrier();
      bool found = false;
      for (int x = tid; x < Sh::kTile / 16; x += 64 * NW)
        found |= !prefill_finite<DT>(reinterpret_cast<const u32x4*>(tile + Sh::kTile)[x]);
      if (found) *bad_word = 1;
      tile_barrier();
      bad = __builtin_amdgcn_readfirstlane(*bad_word) != 0;
    }
    const bool none = !wave_real || first > w_max || (p.window > 0 && last <= w_min - p.window && first >= p.sinks);
    if (none && !bad) continue;
    const bool masked = !sees_all(w_min, w_max);

    f32x16 s[TB][NB];
#pragma unroll
    for (int tb = 0; tb < TB; ++tb)
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) s[tb][nb] = f32x16{};
#pragma unroll
    for (int st = 0; st < Sh::kSteps; ++st)
#pragma unroll
      for (int tb = 0; tb < TB; ++tb) {
        const u32x4 a = tile_lds_read<u32x4>((at + k_at + 32 * tb * Sh::kRow) ^ (32 * st));
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) s[tb][nb] = PrefillMma<DT>::mma(a, qf[nb][st], s[tb][nb]);
      }
    if (masked) {
#pragma unroll
      for (int nb = 0; nb < NB; ++nb)
#pragma unroll
        for (int tb = 0; tb < TB; ++tb)
#pragma unroll
          for (int e = 0; e < 16; ++e)
            s[tb][nb][e] = visible(nb, first + 32 * tb + 8 * (e / 4) + 4 * half + e % 4) ? s[tb][nb][e] : -INFINITY;
    }
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
      float mx = -INFINITY;
#pragma unroll
      for (int tb = 0; tb < TB; ++tb)
#pragma unroll
        for (int e = 0; e < 16; ++e) mx = fmaxf(mx, s[tb][nb][e]);
      if (__ballot(mx * p.sl2 > m[nb] + kLazy)) {
        const float mn = fmaxf(m[nb], prefill_max_halves(mx) * p.sl2);
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
        for (int e = 0; e < 16; ++e) s[tb][nb][e] = fast_exp2(fmaf(s[tb][nb][e], p.sl2, ref));
#pragma unroll
      for (int tb = 0; tb < TB; ++tb)
#pragma unroll
        for (int e = 0; e < 16; e += 4)
          l[nb] += (s[tb][nb][e] + s[tb][nb][e + 1]) + (s[tb][nb][e + 2] + s[tb][nb][e + 3]);
    }
    if (bad) {
      // Values that are not finite: which rows see which of them by a product of
      // what is visible with their flags (in K's place, which is done with),
      // and zeros in their place.
      tile_barrier();
      for (int x = tid; x < Sh::kTile / 16; x += 64 * NW) {
        constexpr int kEach = 16 / ES;
        S* val = reinterpret_cast<S*>(tile + Sh::kTile) + x * kEach;
        S* flag = reinterpret_cast<S*>(tile) + x * kEach;
#pragma unroll
        for (int e = 0; e < kEach; ++e) {
          const float f = prefill_flag<DT>(val[e]);
          flag[e] = E::from_f(f);
          if (f != 0.f) val[e] = E::from_f(0.f);
        }
      }
      tile_barrier();
#pragma unroll 1
      for (int nb_at = 0; nb_at < NB; ++nb_at)
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) {
          if (nb != nb_at || !wave_real) continue;
#pragma unroll
          for (int c = 0; c < Sh::kCols; ++c) {
            f32x16 seen = f32x16{};
#pragma unroll
            for (int tb = 0; tb < TB; ++tb)
#pragma unroll
              for (int ks = 0; ks < 2; ++ks) {
                auto one = [&](int e) {
                  return visible(nb, first + 32 * tb + 8 * (e / 4) + 4 * half + e % 4) ? 1.f : 0.f;
                };
                if constexpr (k16) {
                  u32x4 w;
#pragma unroll
                  for (int j = 0; j < 4; ++j) w[j] = MfmaOps<DT>::pack2(one(8 * ks + 2 * j), one(8 * ks + 2 * j + 1));
                  seen = PrefillMma<DT>::mma(read_v16(at, 2 * tb + ks, c), w, seen);
                } else {
#pragma unroll
                  for (int e = 8 * ks; e < 8 * ks + 8; ++e)
                    seen = __builtin_amdgcn_mfma_f32_32x32x2f32(read_v32(at, tb, e, c), one(e), seen, 0, 0, 0);
                }
              }
#pragma unroll
            for (int e = 0; e < 16; ++e) {
              const float minus = floorf(seen[e] / kPrefillMinusInf), plus = seen[e] - minus * kPrefillMinusInf;
              if (seen[e] >= kPrefillNan) {
                acc[c][nb][e] = NAN;
              } else {
                if (plus > 0.f) acc[c][nb][e] += INFINITY;
                if (minus > 0.f) acc[c][nb][e] -= INFINITY;
              }
            }
          }
        }
    }
    if constexpr (k16) {
#pragma unroll
      for (int ks = 0; ks < TT / 16; ++ks) {
        u32x4 w[NB];
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
#pragma unroll
          for (int j = 0; j < 4; ++j)
            w[nb][j] = MfmaOps<DT>::pack2(s[ks / 2][nb][8 * (ks & 1) + 2 * j], s[ks / 2][nb][8 * (ks & 1) + 2 * j + 1]);
#pragma unroll
        for (int c = 0; c < Sh::kCols; ++c) {
          const u32x4 a = read_v16(vt, ks, c);
#pragma unroll
          for (int nb = 0; nb < NB; ++nb) acc[c][nb] = PrefillMma<DT>::mma(a, w[nb], acc[c][nb]);
        }
      }
    } else {
#pragma unroll
      for (int tb = 0; tb < TB; ++tb)
#pragma unroll
        for (int e = 0; e < 16; ++e)
#pragma unroll
          for (int c = 0; c < Sh::kCols; ++c) {
            const float a = read_v32(vt, tb, e, c);
#pragma unroll
            for (int nb = 0; nb < NB; ++nb)
              acc[c][nb] = __builtin_amdgcn_mfma_f32_32x32x2f32(a, s[tb][nb][e], acc[c][nb], 0, 0, 0);
          }
    }
  }

#pragma unroll
  for (int nb = 0; nb < NB; ++nb) {
    const float sum = prefill_sum_halves(l[nb]);
    const bool has = sum > 0.f || sum != sum;
    const float scale = has ? 1.f / sum : 0.f;
    const int rr = wave_row + 32 * nb + n32;
    if (rr >= rows) continue;
    const int row = row0 + rr, query = row / p.G;
    char* to = static_cast<char*>(p.out) +
               ((static_cast<int64_t>(q0 + query) * p.Hq + static_cast<int64_t>(h) * p.G + (row - query * p.G)) * p.D) * ES;
#pragma unroll
    for (int c = 0; c < Sh::kCols; ++c)
#pragma unroll
      for (int e = 0; e < 16; e += 4) {
        const int d = 32 * c + 2 * e + 4 * half;
        if (d >= p.D) continue;
        f32x4 y;
#pragma unroll
        for (int j = 0; j < 4; ++j) y[j] = has ? acc[c][nb][e + j] * scale : 0.f;
        if constexpr (k16)
          *reinterpret_cast<u32x2*>(to + d * ES) = u32x2{MfmaOps<DT>::pack2(y[0], y[1]), MfmaOps<DT>::pack2(y[2], y[3])};
        else
          *reinterpret_cast<f32x4*>(to + d * ES) = y;
      }
  }
}

template <int DT, int DP, int NB, int NW>
hipError_t prefill_launch(const PrefillParams& p, uint32_t grid, hipStream_t st) {
  using Sh = PrefillShape<DT, DP, NB, NW>;
  void (*fn)(PrefillParams) = prefill_mfma_kernel<DT, DP, NB, NW>;
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
  return hipGetLastError();
}

}  // namespace

#endif  // QD_PREFILL_KERNELS_H
