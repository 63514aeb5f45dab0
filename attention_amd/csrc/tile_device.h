// Tiles of K and V rows in LDS, shared by the matrix-core attention kernels
// (tree_kernels.h, prefill_kernels.h): layout, loads past the registers, waits and
// operand reads.  Included by the .hip sources only.
#ifndef QD_TILE_DEVICE_H
#define QD_TILE_DEVICE_H

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "qd_device.h"

namespace {

// LDS rows are a power of two of 16-byte slots; chunk c of row r lies in slot
// c ^ tile_swizzle(r), which spreads both the 16 rows of a K operand read and
// the 32-byte pieces of a transposing V read over the 64 banks.
// 16-byte slots of an LDS row.
__host__ __device__ constexpr int tile_slots(int es, int dp) {
  return dp * es <= 128 ? 8 : dp * es <= 256 ? 16 : dp * es <= 512 ? 32 : 64;
}
__device__ __forceinline__ int tile_swizzle(int slots, int row) {
  return slots == 8 ? 2 * ((row >> 1) & 3) + ((row >> 3) & 1) : 2 * (row & 7) + ((row >> 3) & 1);
}

// Workgroup barrier for LDS traffic: waits for this wave's LDS operations and
// for all but the last kLeft of its loads into LDS.
template <int kLeft>
__device__ __forceinline__ void tile_barrier_loads() {
  static_assert(kLeft >= 0 && kLeft < 64, "vmcnt is 6 bits");
  constexpr int imm = (kLeft & 0xF) | ((kLeft >> 4) << 14) | (0x7 << 4) | (0x0 << 8);  // lgkmcnt(0)
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt(imm);
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}
// This wave's part of it only.
template <int kLeft>
__device__ __forceinline__ void tile_wait_loads() {
  static_assert(kLeft >= 0 && kLeft < 64, "vmcnt is 6 bits");
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt((kLeft & 0xF) | ((kLeft >> 4) << 14) | (0x7 << 4) | (0xF << 8));
  asm volatile("" ::: "memory");
}
__device__ __forceinline__ void tile_barrier() { tile_barrier_loads<63>(); }

// 16 bytes per lane from `src` to LDS bytes lds + 16 lane.  Written in assembly
// so that the compiler does not wait for it before LDS reads of other buffers:
// tile_barrier_loads does.  M0 (the LDS side) is written and used within one
// statement; the compiler keeps nothing in it from one statement to another (a
// reserved register, which a clobber list may not name), and nothing else in
// these kernels uses it.  At least one lane is active (the loads of a tile are counted).
// STREAM: not kept in the caches.
template <bool STREAM>
__device__ __forceinline__ void tile_load_lds(const char* src, uint32_t lds) {
  if constexpr (STREAM)
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off nt" ::"s"(lds), "v"(src) : "memory");
  else
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(lds), "v"(src) : "memory");
}

// The same from base + off, base wave-uniform.
template <bool STREAM>
__device__ __forceinline__ void tile_load_lds(const char* base, uint32_t off, uint32_t lds) {
  if constexpr (STREAM)
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2 nt" ::"s"(lds), "v"(off), "s"(base)
                 : "memory");
  else
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(lds), "v"(off), "s"(base)
                 : "memory");
}

__device__ __forceinline__ uint32_t tile_lds_address(const char* p) {
  return static_cast<uint32_t>(reinterpret_cast<uintptr_t>((const __attribute__((address_space(3))) char*)p));
}

// A table entry at a wave-uniform place, through the scalar cache: a vector
// load would complete only after the tiles in flight.
__device__ __forceinline__ int32_t tile_scalar_load(const int32_t* p) {
  return *reinterpret_cast<const __attribute__((address_space(4))) int32_t*>(reinterpret_cast<uintptr_t>(p));
}

// Reads by LDS byte address: slots of a row are exchanged by an exclusive or of
// its bits, without a step from address to pointer.
template <typename X>
__device__ __forceinline__ X tile_lds_read(uint32_t at) {
  return *reinterpret_cast<const __attribute__((address_space(3))) X*>(at);
}

// Four transposed 16-bit elements: lane (g4, r16) of the wave gets column r16
// of the 4 x 16 block whose row r16 / 4, columns 4 (r16 % 4).. this lane
// addresses.
__device__ __forceinline__ u32x2 tile_tr_read(uint32_t at) {
  typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
  return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(reinterpret_cast<lds_s16x4*>(at)));
}

}  // namespace

#endif  // QD_TILE_DEVICE_H
