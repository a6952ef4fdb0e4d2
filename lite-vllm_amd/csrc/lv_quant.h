// 8-bit codes of the quantised K/V cache: rows of D codes with one fp32 scale.
//
//   scale = fl32(max|x| / top),  code = nearest(fl32(x / scale)),  top = 127 or 448
//   value = code * scale
// with LV_INT8 codes whole numbers in [-127, 127] and LV_E4M3 codes OCP e4m3
// values (3 fraction bits, no infinities), both rounded to nearest, ties to
// even.  A row of zeros (or so small that its scale rounds to zero) has scale
// 0 and codes 0; a row that holds a value that is not finite has scale NaN
// and codes 0, so it reads back as NaN.
#pragma once
#include "lv_common.h"

namespace lv {

struct int8_code {};
struct e4m3_code {};

template <typename C> struct code;
template <> struct code<int8_code> {
  static constexpr float kTop = 127.0f;
  // Four values, already divided by the scale, as four codes.  (Only a scale
  // among the subnormals, which holds few bits, puts a value past the top.)
  __device__ __forceinline__ static uint32_t pack4(const float* y) {
    uint32_t w = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int c = (int)rintf(fminf(fmaxf(y[i], -kTop), kTop));
      w |= (uint32_t)(c & 0xff) << (8 * i);
    }
    return w;
  }
  __device__ __forceinline__ static void unpack4(uint32_t w, float* out) {
#pragma unroll
    for (int i = 0; i < 4; ++i) out[i] = (float)(int8_t)(w >> (8 * i));
  }
};
template <> struct code<e4m3_code> {
  static constexpr float kTop = 448.0f;
  __device__ __forceinline__ static uint32_t pack4(const float* y) {
    float z[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) z[i] = fminf(fmaxf(y[i], -kTop), kTop);
    int w = __builtin_amdgcn_cvt_pk_fp8_f32(z[0], z[1], 0, false);
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(z[2], z[3], w, true);
  }
  __device__ __forceinline__ static void unpack4(uint32_t w, float* out) {
    const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false);
    const auto hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true);
    out[0] = lo[0]; out[1] = lo[1]; out[2] = hi[0]; out[3] = hi[1];
  }
};

// Largest of x over aligned groups of W lanes (W a power of two up to 64).
template <int CTRL>
__device__ __forceinline__ uint32_t dpp_u32(uint32_t x) {
  return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, CTRL, 0xf, 0xf, false);
}
template <int W>
__device__ __forceinline__ uint32_t group_umax(uint32_t x) {
  if constexpr (W >= 2) x = max(x, dpp_u32<0xB1>(x));
  if constexpr (W >= 4) x = max(x, dpp_u32<0x4E>(x));
  if constexpr (W >= 8) x = max(x, dpp_u32<0x141>(x));
  if constexpr (W >= 16) x = max(x, dpp_u32<0x140>(x));
  if constexpr (W >= 32) x = max(x, (uint32_t)__shfl_xor((int)x, 16));
  if constexpr (W >= 64) x = max(x, (uint32_t)__shfl_xor((int)x, 32));
  return x;
}

// Scale of a row and its N values x of this lane divided by it (zeros where
// the scale is 0 or NaN), the row spread over W lanes.  Magnitudes are
// compared as bits, which keeps NaN the largest of all.
// The quotients are the correctly rounded ones: x r, r the correctly rounded
// reciprocal, corrected once by its exact remainder (Markstein's division; the
// scales outside the range where no step of it underflows are divided).  Three
// instructions instead of ten for each value, which bounded the writers: 7872
// tokens of 8 heads of 128 bf16 dims 17.7 -> 15.8 us.
template <typename C, int W, int N>
__device__ __forceinline__ float row_scale(float* x) {
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < N; ++i) top = max(top, __float_as_uint(x[i]) & 0x7fffffffu);
  top = group_umax<W>(top);
  const float scale = top >= 0x7f800000u ? __builtin_nanf("")
                                         : __uint_as_float(top) / code<C>::kTop;
  if (scale >= 0x1p-80f && scale <= 0x1p100f) {
    const float r = 1.0f / scale;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const float q = x[i] * r;
      x[i] = fmaf(fmaf(-q, scale, x[i]), r, q);
    }
  } else {
    const bool live = scale > 0.0f;
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = live ? x[i] / scale : 0.0f;
  }
  return scale;
}

}  // namespace lv
