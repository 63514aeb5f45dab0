// Per-head norm of queries and keys, position rotation and paged cache write
// in one pass for MI355X (gfx950).  C ABI in include/qd_attention.h.
//
// y = x rsqrt(mean(x^2) + eps) w over the head, pairs (a, b) of the first
// rotary_dim elements -> (a cos - b sin, b cos + a sin), in fp32 with one
// rounding at the end; values are copied.

#include <hip/hip_runtime.h>

#include <math.h>
#include <stdint.h>
#include <string.h>

#include <algorithm>
#include <string>
#include <type_traits>

#include "qd_attention.h"
#include "qd_device.h"

void qd_set_last_error(int status, const std::string& msg);

namespace {

struct RopeParams {
  const void* q;
  const void* key;
  const void* value;
  const float* cos_sin;
  const int32_t* pos;
  void* kc;
  void* vc;
  const int64_t* slots;
  const void* qw;  // null: no norm
  const void* kw;
  void* out;
  int64_t q_stride, k_stride, v_stride;  // elements from one token to the next
  int64_t max_positions, cache_rows;
  int Hq, Hkv, D, rot;
  int interleaved;
  float eps;
};

// Any head_dim and alignment: one wave per (token, head), element by element;
// an element's rotation partner is read again rather than exchanged.  16384
// tokens of 32 + 8 heads of 128 (411 MB): 450 us, against 79 us of the vector
// kernel.
// grid (tokens, ceil(heads / 4)), block 256.
template <int DT, int WDT>
__global__ __launch_bounds__(256) void rope_generic_kernel(RopeParams p) {
  using E = Elem<DT>;
  using S = typename E::S;
  using W = Elem<WDT>;
  const int64_t n = blockIdx.x;
  const int h = static_cast<int>(blockIdx.y) * 4 + static_cast<int>(threadIdx.x >> 6);
  const int lane = threadIdx.x & 63;
  if (h >= p.Hq + 2 * p.Hkv) return;
  const int64_t at = p.pos[n], slot = p.slots[n];
  const bool turned = at >= 0 && at < p.max_positions;
  const bool kept = turned && slot >= 0 && slot < p.cache_rows;
  const bool is_q = h < p.Hq, is_k = !is_q && h < p.Hq + p.Hkv;
  if (!is_q && !kept) return;
  const int hh = is_q ? h : is_k ? h - p.Hq : h - p.Hq - p.Hkv;
  const S* x = is_q   ? static_cast<const S*>(p.q) + n * p.q_stride
               : is_k ? static_cast<const S*>(p.key) + n * p.k_stride
                      : static_cast<const S*>(p.value) + n * p.v_stride;
  x += static_cast<int64_t>(hh) * p.D;
  S* y = is_q ? static_cast<S*>(p.out) + (n * p.Hq + hh) * p.D
              : static_cast<S*>(is_k ? p.kc : p.vc) + (slot * p.Hkv + hh) * p.D;
  if (!is_q && !is_k) {
    for (int d = lane; d < p.D; d += 64) y[d] = x[d];
    return;
  }
  if (!turned) {
    for (int d = lane; d < p.D; d += 64) y[d] = E::from_f(0.f);
    return;
  }
  const typename W::S* w = static_cast<const typename W::S*>(is_q ? p.qw : p.kw);
  float r = 1.f;
  if (w) {
    float sum = 0.f;
    for (int d = lane; d < p.D; d += 64) sum += E::to_f(x[d]) * E::to_f(x[d]);
    r = 1.f / sqrtf(wave_sum(sum) / static_cast<float>(p.D) + p.eps);
  }
  auto normed = [&](int d) { return w ? E::to_f(x[d]) * r * W::to_f(w[d]) : E::to_f(x[d]); };
  const float* cs = p.cos_sin + at * p.rot;
  const int half = p.rot / 2;
  for (int d = lane; d < p.D; d += 64) {
    float v = normed(d);
    if (d < p.rot) {
      const int i = p.interleaved ? d / 2 : d < half ? d : d - half;
      const bool first = p.interleaved ? (d & 1) == 0 : d < half;
      const float other = normed(p.interleaved ? d ^ 1 : first ? d + half : d - half);
      v = first ? v * cs[i] - other * cs[half + i] : v * cs[i] + other * cs[half + i];
    }
    y[d] = E::from_f(v);
  }
}

// Lanes of one head: four pairs (eight elements) per lane.
__host__ __device__ constexpr int rope_lanes(int head_dim) { return head_dim <= 64 ? 8 : head_dim <= 128 ? 16 : 32; }

// Four elements as loaded.
template <int DT>
struct RopeRaw {
  using V = u32x2;
};
template <>
struct RopeRaw<QD_DTYPE_F32> {
  using V = u32x4;
};

template <int DT>
__device__ __forceinline__ f32x4 rope_floats(typename RopeRaw<DT>::V v) {
  if constexpr (DT == QD_DTYPE_F32) {
    return __builtin_bit_cast(f32x4, v);
  } else {
    const f32x2 a = MfmaOps<DT>::unpack2(v[0]), b = MfmaOps<DT>::unpack2(v[1]);
    return f32x4{a[0], a[1], b[0], b[1]};
  }
}

template <int DT>
__device__ __forceinline__ typename RopeRaw<DT>::V rope_raw(f32x4 y) {
  if constexpr (DT == QD_DTYPE_F32)
    return __builtin_bit_cast(u32x4, y);
  else
    return u32x2{MfmaOps<DT>::pack2(y[0], y[1]), MfmaOps<DT>::pack2(y[2], y[3])};
}

// Sum over the LANES lanes of a head.
template <int LANES>
__device__ __forceinline__ float head_sum(float x) {
  x += dpp_f<0xB1>(x);   // quad_perm [1,0,3,2]
  x += dpp_f<0x4E>(x);   // quad_perm [2,3,0,1]
  x += dpp_f<0x141>(x);  // row_half_mirror
  if (LANES >= 16) x += dpp_f<0x140>(x);  // row_mirror
  if (LANES >= 32) x += __shfl_xor(x, 16);
  return x;
}

// head_dim a multiple of 8, tensors aligned to four elements: a workgroup per
// token, LANES lanes per head, each with two groups of four elements.  In the
// half-split rotation lane i < R / 8 holds pairs 4i.. as the groups at 4i and
// R / 2 + 4i, the other lanes neighbouring groups past R; interleaved, and
// for values, a lane's groups are neighbours.  So no element has its partner
// in another lane, and a token's angles are loaded once for all its heads.
// Nothing passes through LDS: a head's sum of squares takes 3 to 5 lane
// exchanges.  A lane has the loads of 4 heads in flight before it needs a
// position or a weight.  Bound by HBM in large calls: 16384 tokens of 32 + 8
// heads of 128, bf16 (411 MB in and out) 79 us, 5.2 TB/s, where a large copy
// makes 4.9; 512 tokens 7.3 us and 4 tokens 7.2 us, the launch and the call.
// grid tokens, block a multiple of LANES.
template <int DT, int WDT, int LANES, bool INTER>
__global__ __launch_bounds__(256) void rope_vec_kernel(RopeParams p) {
  using E = Elem<DT>;
  using S = typename E::S;
  using V = typename RopeRaw<DT>::V;
  constexpr int kAhead = 4;  // heads whose loads a lane has in flight
  const int64_t n = blockIdx.x;
  const int lane = static_cast<int>(threadIdx.x) % LANES;
  const int team = static_cast<int>(threadIdx.x) / LANES, teams = static_cast<int>(blockDim.x) / LANES;
  const int heads = p.Hq + 2 * p.Hkv;
  const bool live = 8 * lane < p.D;
  const int half = p.rot / 2;
  // Element offsets of the lane's two groups.
  const bool split = !INTER && 8 * lane < p.rot;
  const int a_at = split ? 4 * lane : 8 * lane, b_at = split ? half + 4 * lane : 8 * lane + 4;
  const int64_t at = p.pos[n], slot = p.slots[n];
  auto source = [&](int h) -> const S* {
    return h < p.Hq           ? static_cast<const S*>(p.q) + n * p.q_stride + static_cast<int64_t>(h) * p.D
           : h < p.Hq + p.Hkv ? static_cast<const S*>(p.key) + n * p.k_stride + static_cast<int64_t>(h - p.Hq) * p.D
                              : static_cast<const S*>(p.value) + n * p.v_stride +
                                    static_cast<int64_t>(h - p.Hq - p.Hkv) * p.D;
  };
  V xa[kAhead], xb[kAhead];
  auto load = [&](int first) {
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      const int h = first + i * teams;
      if (h >= heads || !live) continue;
      const S* x = source(h);
      xa[i] = __builtin_nontemporal_load(reinterpret_cast<const V*>(x + a_at));
      xb[i] = __builtin_nontemporal_load(reinterpret_cast<const V*>(x + b_at));
    }
  };
  load(team);
  const bool turned = at >= 0 && at < p.max_positions;
  const bool kept = turned && slot >= 0 && slot < p.cache_rows;
  // The lane's angles: of pairs 4 lane.. (half-split), 4 lane.. as well
  // (interleaved: group a holds pairs 4 lane and 4 lane + 1, b the next two).
  f32x4 c = {1.f, 1.f, 1.f, 1.f}, s = {0.f, 0.f, 0.f, 0.f};
  if (turned) {
    const float* cs = p.cos_sin + at * p.rot;
    if constexpr (INTER) {
#pragma unroll
      for (int g = 0; g < 2; ++g)
        if (8 * lane + 4 * g < p.rot) {
          const f32x2 cg = *reinterpret_cast<const f32x2*>(cs + 4 * lane + 2 * g);
          const f32x2 sg = *reinterpret_cast<const f32x2*>(cs + half + 4 * lane + 2 * g);
          c[2 * g] = cg[0];
          c[2 * g + 1] = cg[1];
          s[2 * g] = sg[0];
          s[2 * g + 1] = sg[1];
        }
    } else if (split) {
      c = *reinterpret_cast<const f32x4*>(cs + 4 * lane);
      s = *reinterpret_cast<const f32x4*>(cs + half + 4 * lane);
    }
  }
  auto weights = [&](const void* w, f32x4& wa, f32x4& wb) {
    wa = wb = f32x4{1.f, 1.f, 1.f, 1.f};
    if (w && live) {
      using W = typename Elem<WDT>::S;
      using WV = typename RopeRaw<WDT>::V;
      wa = rope_floats<WDT>(*reinterpret_cast<const WV*>(static_cast<const W*>(w) + a_at));
      wb = rope_floats<WDT>(*reinterpret_cast<const WV*>(static_cast<const W*>(w) + b_at));
    }
  };
  f32x4 qa, qb, ka, kb;
  weights(p.qw, qa, qb);
  weights(p.kw, ka, kb);
  const float inv_d = 1.f / static_cast<float>(p.D);
  for (int first = team; first < heads; first += kAhead * teams) {
    if (first != team) load(first);
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      const int h = first + i * teams;
      if (h >= heads) break;  // the whole head's lanes
      const bool is_q = h < p.Hq, is_k = !is_q && h < p.Hq + p.Hkv;
      V ya = xa[i], yb = xb[i];
      if (is_q || is_k) {
        f32x4 a = {0.f, 0.f, 0.f, 0.f}, b = a;
        if (live) {
          a = rope_floats<DT>(xa[i]);
          b = rope_floats<DT>(xb[i]);
        }
        if (is_q ? p.qw != nullptr : p.kw != nullptr) {
          float sum = 0.f;
#pragma unroll
          for (int j = 0; j < 4; ++j) sum = fmaf(a[j], a[j], fmaf(b[j], b[j], sum));
          const float r = 1.f / sqrtf(fmaf(head_sum<LANES>(sum), inv_d, p.eps));
          a = a * r * (is_q ? qa : ka);
          b = b * r * (is_q ? qb : kb);
        }
        if constexpr (INTER) {
          const f32x4 u = a, w = b;
          a = f32x4{u[0] * c[0] - u[1] * s[0], u[1] * c[0] + u[0] * s[0], u[2] * c[1] - u[3] * s[1],
                    u[3] * c[1] + u[2] * s[1]};
          b = f32x4{w[0] * c[2] - w[1] * s[2], w[1] * c[2] + w[0] * s[2], w[2] * c[3] - w[3] * s[3],
                    w[3] * c[3] + w[2] * s[3]};
        } else if (split) {
          const f32x4 u = a;
          a = u * c - b * s;
          b = b * c + u * s;
        }
        if (is_q && !turned) a = b = f32x4{0.f, 0.f, 0.f, 0.f};
        ya = rope_raw<DT>(a);
        yb = rope_raw<DT>(b);
      }
      if (!live || (!is_q && !kept)) continue;
      S* y = is_q   ? static_cast<S*>(p.out) + (n * p.Hq + h) * p.D
             : is_k ? static_cast<S*>(p.kc) + (slot * p.Hkv + (h - p.Hq)) * p.D
                    : static_cast<S*>(p.vc) + (slot * p.Hkv + (h - p.Hq - p.Hkv)) * p.D;
      *reinterpret_cast<V*>(y + a_at) = ya;
      *reinterpret_cast<V*>(y + b_at) = yb;
    }
  }
}

int rope_fail(char* msg, size_t cap, const char* text) {
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

template <int DT>
void launch_rope(const RopeParams& p, int64_t tokens, int wdt, hipStream_t st) {
  // The vector kernel's groups of four elements must not cross the end of the
  // rotated part, and every row starts at a group.
  constexpr uintptr_t kGroup = DT == QD_DTYPE_F32 ? 16 : 8;
  const uintptr_t bits = reinterpret_cast<uintptr_t>(p.q) | reinterpret_cast<uintptr_t>(p.key) |
                         reinterpret_cast<uintptr_t>(p.value) | reinterpret_cast<uintptr_t>(p.kc) |
                         reinterpret_cast<uintptr_t>(p.vc) | reinterpret_cast<uintptr_t>(p.out);
  const uintptr_t weights = reinterpret_cast<uintptr_t>(p.qw) | reinterpret_cast<uintptr_t>(p.kw);
  if (p.D % 8 == 0 && p.rot % (p.interleaved ? 4 : 8) == 0 && bits % kGroup == 0 &&
      (p.q_stride | p.k_stride | p.v_stride) % 4 == 0 && weights % (wdt == QD_DTYPE_F32 ? 16 : 8) == 0 &&
      reinterpret_cast<uintptr_t>(p.cos_sin) % 16 == 0) {
    const int lanes = rope_lanes(p.D);
    const int teams = std::min(p.Hq + 2 * p.Hkv, 256 / lanes);
    const dim3 block(static_cast<uint32_t>((teams * lanes + 63) / 64 * 64));
    const dim3 grid(static_cast<uint32_t>(tokens));
    auto run = [&](auto wtype, auto inter) {
      constexpr int W = decltype(wtype)::value;
      constexpr bool I = decltype(inter)::value;
      if (lanes == 8)
        hipLaunchKernelGGL((rope_vec_kernel<DT, W, 8, I>), grid, block, 0, st, p);
      else if (lanes == 16)
        hipLaunchKernelGGL((rope_vec_kernel<DT, W, 16, I>), grid, block, 0, st, p);
      else
        hipLaunchKernelGGL((rope_vec_kernel<DT, W, 32, I>), grid, block, 0, st, p);
    };
    using F = std::integral_constant<int, QD_DTYPE_F32>;
    using T = std::integral_constant<int, DT>;
    if (wdt == QD_DTYPE_F32)
      p.interleaved ? run(F{}, std::true_type{}) : run(F{}, std::false_type{});
    else
      p.interleaved ? run(T{}, std::true_type{}) : run(T{}, std::false_type{});
    return;
  }
  const dim3 grid(static_cast<uint32_t>(tokens), static_cast<uint32_t>((p.Hq + 2 * p.Hkv + 3) / 4));
  if (wdt == QD_DTYPE_F32)
    hipLaunchKernelGGL((rope_generic_kernel<DT, QD_DTYPE_F32>), grid, dim3(256), 0, st, p);
  else
    hipLaunchKernelGGL((rope_generic_kernel<DT, DT>), grid, dim3(256), 0, st, p);
}

}  // namespace

extern "C" {

int qd_qk_norm_rope_write_validate(const qd_tensor_desc* q, const qd_tensor_desc* key, const qd_tensor_desc* value,
                                   const qd_tensor_desc* cos_sin, const qd_tensor_desc* positions,
                                   const qd_tensor_desc* k_cache, const qd_tensor_desc* v_cache,
                                   const qd_tensor_desc* slots, const qd_tensor_desc* q_weight,
                                   const qd_tensor_desc* k_weight, double eps, char* msg, size_t msg_cap) {
  const qd_tensor_desc* all[8] = {q, key, value, cos_sin, positions, k_cache, v_cache, slots};
  for (int i = 0; i < 8; ++i)
    if (!all[i]) return rope_fail(msg, msg_cap, "null tensor descriptor");
  const bool has_qw = q_weight && q_weight->defined, has_kw = k_weight && k_weight->defined;
  for (int i = 0; i < 10; ++i) {
    const qd_tensor_desc* t = i < 8 ? all[i] : i == 8 ? q_weight : k_weight;
    if (i >= 8 && !(i == 8 ? has_qw : has_kw)) continue;
    if (!t->defined || !t->is_device) return rope_fail(msg, msg_cap, "all tensors must be CUDA tensors");
    if (t->device_index != q->device_index) return rope_fail(msg, msg_cap, "all tensors must share a device");
    if (!t->contiguous)
      return rope_fail(msg, msg_cap,
                       i < 3 ? "the heads of a token must be contiguous in q, key and value"
                             : "cos_sin, positions, caches, slots and weights must be contiguous");
  }
  if (q->ndim != 3) return rope_fail(msg, msg_cap, "q must be [N, Hq, D]");
  if (key->ndim != 3 || value->ndim != 3 || key->sizes[0] != q->sizes[0] || value->sizes[0] != q->sizes[0] ||
      key->sizes[2] != q->sizes[2] || value->sizes[2] != q->sizes[2] || value->sizes[1] != key->sizes[1])
    return rope_fail(msg, msg_cap, "key/value must be [N, Hkv, D]");
  if (k_cache->ndim != 4 || v_cache->ndim != 4) return rope_fail(msg, msg_cap, "cache must be [Nblocks, P, Hkv, D]");
  for (int i = 0; i < 4; ++i)
    if (k_cache->sizes[i] != v_cache->sizes[i]) return rope_fail(msg, msg_cap, "cache must be [Nblocks, P, Hkv, D]");
  if (k_cache->sizes[2] != key->sizes[1] || k_cache->sizes[3] != key->sizes[2])
    return rope_fail(msg, msg_cap, "cache head shape mismatch");
  if (!(q->sizes[1] > 0 && key->sizes[1] > 0 && k_cache->sizes[0] > 0 && k_cache->sizes[1] > 0))
    return rope_fail(msg, msg_cap, "invalid dimensions");
  if (!(q->sizes[2] >= 1 && q->sizes[2] <= 256)) return rope_fail(msg, msg_cap, "supported head_dim is [1, 256]");
  if (cos_sin->ndim != 2 || cos_sin->dtype != QD_DTYPE_F32)
    return rope_fail(msg, msg_cap, "cos_sin must be float32 [MaxPositions, R]");
  if (!(cos_sin->sizes[1] >= 0 && cos_sin->sizes[1] % 2 == 0 && cos_sin->sizes[1] <= q->sizes[2]))
    return rope_fail(msg, msg_cap, "the rotary dim must be even and at most head_dim");
  if (positions->ndim != 1 || positions->dtype != QD_DTYPE_I32 || positions->sizes[0] != q->sizes[0])
    return rope_fail(msg, msg_cap, "positions must be int32 [N]");
  if (slots->ndim != 1 || slots->dtype != QD_DTYPE_I64 || slots->sizes[0] != q->sizes[0])
    return rope_fail(msg, msg_cap, "slots must be int64 [N]");
  if (!float_dtype(q->dtype)) return rope_fail(msg, msg_cap, "unsupported dtype");
  if (key->dtype != q->dtype || value->dtype != q->dtype || k_cache->dtype != q->dtype || v_cache->dtype != q->dtype)
    return rope_fail(msg, msg_cap, "dtype mismatch");
  const qd_tensor_desc* ws[2] = {has_qw ? q_weight : nullptr, has_kw ? k_weight : nullptr};
  for (const qd_tensor_desc* w : ws) {
    if (!w) continue;
    if (w->ndim != 1 || w->sizes[0] != q->sizes[2]) return rope_fail(msg, msg_cap, "weights must be [D]");
    if (w->dtype != q->dtype && w->dtype != QD_DTYPE_F32)
      return rope_fail(msg, msg_cap, "weights must have q's dtype or be float32");
  }
  if (ws[0] && ws[1] && ws[0]->dtype != ws[1]->dtype)
    return rope_fail(msg, msg_cap, "q_weight and k_weight must have one dtype");
  if (!(eps >= 0.0 && eps <= 3.0e38)) return rope_fail(msg, msg_cap, "eps must be finite and not negative");
  if (!(q->sizes[0] < (1 << 24) && q->sizes[1] + 2 * key->sizes[1] <= 65535 * 4))
    return rope_fail(msg, msg_cap, "tensor sizes exceed int32 CUDA launch limits");
  if (msg && msg_cap) msg[0] = '\0';
  return QD_OK;
}

int qd_qk_norm_rope_write(const void* q, const void* key, const void* value, const float* cos_sin,
                          const int32_t* positions, void* k_cache, void* v_cache, const int64_t* slots,
                          const void* q_weight, const void* k_weight, void* q_out, int64_t tokens, int q_heads,
                          int kv_heads, int head_dim, int rotary_dim, int64_t q_stride, int64_t k_stride,
                          int64_t v_stride, int64_t max_positions, int64_t cache_rows, int dtype, int weight_dtype,
                          float eps, int interleaved, void* stream) {
  if (tokens < 0 || tokens >= (1 << 24)) return rope_fail(nullptr, 0, "tokens must be in [0, 2^24)");
  if (q_heads <= 0 || kv_heads <= 0 || cache_rows <= 0 || max_positions < 0 ||
      static_cast<int64_t>(q_heads) + 2 * static_cast<int64_t>(kv_heads) > 65535 * 4 || q_stride < 0 ||
      k_stride < 0 || v_stride < 0)
    return rope_fail(nullptr, 0, "invalid dimensions");
  if (head_dim < 1 || head_dim > 256) return rope_fail(nullptr, 0, "supported head_dim is [1, 256]");
  if (rotary_dim < 0 || rotary_dim % 2 != 0 || rotary_dim > head_dim)
    return rope_fail(nullptr, 0, "the rotary dim must be even and at most head_dim");
  if (!float_dtype(dtype)) return rope_fail(nullptr, 0, "unsupported dtype");
  if ((q_weight || k_weight) && weight_dtype != dtype && weight_dtype != QD_DTYPE_F32)
    return rope_fail(nullptr, 0, "weights must have q's dtype or be float32");
  if (!(eps >= 0.f) || !isfinite(eps)) return rope_fail(nullptr, 0, "eps must be finite and not negative");
  if (tokens == 0) return QD_OK;
  if (!q || !key || !value || !positions || !k_cache || !v_cache || !slots || !q_out ||
      (!cos_sin && rotary_dim > 0 && max_positions > 0))
    return rope_fail(nullptr, 0, "null tensor pointer");
  // A token's key and value would be written to one place by different lanes.
  const uintptr_t kc = reinterpret_cast<uintptr_t>(k_cache), vc = reinterpret_cast<uintptr_t>(v_cache);
  const uint64_t row_bytes = static_cast<uint64_t>(kv_heads) * head_dim * (dtype == QD_DTYPE_F32 ? 4 : 2);
  if ((std::max(kc, vc) - std::min(kc, vc)) / row_bytes < static_cast<uint64_t>(cache_rows))
    return rope_fail(nullptr, 0, "k_cache and v_cache must not overlap");
  RopeParams p;
  p.q = q;
  p.key = key;
  p.value = value;
  p.cos_sin = cos_sin;
  p.pos = positions;
  p.kc = k_cache;
  p.vc = v_cache;
  p.slots = slots;
  p.qw = q_weight;
  p.kw = k_weight;
  p.out = q_out;
  p.q_stride = q_stride;
  p.k_stride = k_stride;
  p.v_stride = v_stride;
  p.max_positions = max_positions;
  p.cache_rows = cache_rows;
  p.Hq = q_heads;
  p.Hkv = kv_heads;
  p.D = head_dim;
  p.rot = rotary_dim;
  p.interleaved = interleaved;
  p.eps = eps;
  hipStream_t st = static_cast<hipStream_t>(stream);
  const int wdt = q_weight || k_weight ? weight_dtype : dtype;
  (void)hipGetLastError();
  switch (dtype) {
    case QD_DTYPE_F32: launch_rope<QD_DTYPE_F32>(p, tokens, wdt, st); break;
    case QD_DTYPE_F16: launch_rope<QD_DTYPE_F16>(p, tokens, wdt, st); break;
    default: launch_rope<QD_DTYPE_BF16>(p, tokens, wdt, st); break;
  }
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) {
    qd_set_last_error(static_cast<int>(e),
                      std::string("qk_norm_rope_write kernel launch failed: ") + hipGetErrorString(e));
    return static_cast<int>(e);
  }
  return QD_OK;
}

}  // extern "C"
