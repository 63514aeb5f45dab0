// Packed sequences: which sequence and which part of it a workgroup serves.
// cu[b] .. cu[b + 1] are the rows of sequence b; cu[0] counts as 0, every other
// entry is clamped to [0, total], so that no row leaves the tensors whatever
// cu holds.  Included by the .hip sources only.
#ifndef QD_PACKED_H
#define QD_PACKED_H

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace {

// n / d for n < 2^31 as (n m) >> s, on the scalar units: m = ceil(2^s / d) with s =
// 31 + ceil(log2 d) exceeds 2^s / d by less than 1, and so n m / 2^s exceeds n / d
// by less than n / 2^s < 1 / d.
struct PackedDivide {
  uint32_t m;
  int s;
};
inline PackedDivide packed_divide_by(uint32_t d) {
  int bits = 0;
  while ((uint64_t{1} << bits) < d) ++bits;
  return {static_cast<uint32_t>(((uint64_t{1} << (31 + bits)) + d - 1) / d), 31 + bits};
}
__device__ __forceinline__ int packed_divide(uint32_t n, PackedDivide d) {
  return static_cast<int>((static_cast<uint64_t>(n) * d.m) >> d.s);
}

__device__ __forceinline__ int packed_start(const int32_t* cu, int b, int total) {
  return b == 0 ? 0 : min(max(cu[b], 0), total);
}

// Parts of `per` rows each are numbered through: sequence b's first is
// start(b) * mult / per + spare * b, which leaves room for a part begun at either
// end.  Returns the sequence that part u lies in, of `batch` (wave-uniform): 64
// candidates per round trip, one round for up to 64 sequences.
__device__ __forceinline__ int64_t packed_base(const int32_t* cu, int b, int total, int mult, int per, int spare) {
  return static_cast<int64_t>(packed_start(cu, b, total)) * mult / per + static_cast<int64_t>(spare) * b;
}

__device__ __forceinline__ int packed_find(const int32_t* cu, int batch, int total, int mult, int per, int spare,
                                           int64_t u) {
  const int lane = static_cast<int>(threadIdx.x) & 63;
  int lo = 0, hi = batch;
  while (hi - lo > 1) {
    const int step = (hi - lo + 63) / 64;
    const int64_t at = lo + static_cast<int64_t>(lane) * step;
    const bool before = lane == 0 || (at < hi && packed_base(cu, static_cast<int>(at), total, mult, per, spare) <= u);
    const uint64_t all = __ballot(before);
    lo += step * (63 - __builtin_clzll(all));
    hi = min(hi, lo + step);
  }
  return __builtin_amdgcn_readfirstlane(lo);
}

}  // namespace

#endif  // QD_PACKED_H
