// LDS tiles and lane exchanges shared by the matrix-core attention kernels.
#pragma once
#include "lv_common.h"
#include "lv_mfma.h"

namespace lv {

// LDS tile of K or V: 16 W key rows of D elements, unpadded; 16-byte chunk j
// of row r holds the row's chunk j ^ swz(r % 16).  The XOR swizzle keeps
// both read patterns free of bank conflicts on 64 banks of 4 bytes: the K
// reads (16 consecutive rows at one chunk per LDS cycle) need swz to be a
// permutation of 0..15, and the V transpose reads (32 lanes per cycle:
// rows 4i..4i+3 at four consecutive chunks) need bits 2-3 of swz distinct
// over rows 4i..4i+3 -- and bits 1-2 as well, for the 16-lane, 32-bank
// grouping.  swz = 0 6 10 12 1 7 11 13 2 4 8 14 3 5 9 15 meets all three;
// plain r % 16 makes rows 4i..4i+3 share banks.  (D = 64 takes swz % 8.)
template <int D, int W> struct ChunkLds {
  static constexpr int CPR = D / 8;                 // 16-byte chunks per row
  static constexpr int TILE = 16 * W * D;           // elements per K or V tile
  __device__ __forceinline__ static int swz(int row) {
    return (int)((0xF953E842DB71CA60ull >> (4 * (row & 15))) & (CPR - 1));
  }
  __device__ __forceinline__ static int at(int row, int chunk) {
    return row * D + 8 * (chunk ^ swz(row));
  }
};

// max / sum of x over lanes l and l ^ 32 (v_permlane32_swap: lanes 0-31 of
// one copy trade places with lanes 32-63 of the other, so each lane holds
// its own value and its partner's), no LDS round trip.
__device__ __forceinline__ float xor32_max(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false,
                                                  false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float xor32_sum(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false,
                                                  false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

__device__ __forceinline__ i16x4_t lds_read_tr16(const uint16_t* p) {
  return __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) i16x4_t*)p);
}

}  // namespace lv
