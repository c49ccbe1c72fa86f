// Rounding to e4m3 with a scale for a block: shared by quant_fp8 and by the
// experts' layers, which round their hidden rows on the way out.
#pragma once
#include <hip/hip_runtime.h>

#include <cstdint>

namespace tile {

// The largest |v| as the bits of a float: on bits the order is that of the
// numbers, and NaN lies above infinity, so that it isn't lost.
template <int R>
__device__ __forceinline__ uint32_t amax_bits(const float (&v)[R]) {
  uint32_t top = 0;
#pragma unroll
  for (int e = 0; e < R; ++e)
    top = max(top, __builtin_bit_cast(uint32_t, v[e]) & 0x7fffffffu);
  return top;
}

// amax / 448, and no less than the smallest normal number, so that a block of
// zeros needs no case of its own and no quotient passes 448 by more than its
// own rounding
__device__ __forceinline__ float scale_of(uint32_t top) {
  const float s = __builtin_bit_cast(float, top) / 448.f;
  return s < 0x1p-126f ? 0x1p-126f : s;
}

// R values over their scale, each quotient rounded to f32 as by a division
// and then to the nearest e4m3 value, the even one of two. Values of bf16
// meet such ties often, so the quotient has to be the exact one: two
// corrections from the reciprocal of the whole block give it in 5 operations
// where a division takes twice as many. They need their remainders exact:
// scales near the ends of the range take the division.
template <int R>
__device__ __forceinline__ void to_fp8(const float (&v)[R], float s,
                                       uint32_t (&out)[R / 4]) {
  float q[R];
  if (s > 0x1p-90f && s < 0x1p120f) {
    const float r = 1.f / s;
#pragma unroll
    for (int e = 0; e < R; ++e) {
      float y = v[e] * r;
      y = __builtin_fmaf(__builtin_fmaf(-y, s, v[e]), r, y);
      q[e] = __builtin_fmaf(__builtin_fmaf(-y, s, v[e]), r, y);
    }
  } else {
#pragma unroll
    for (int e = 0; e < R; ++e) q[e] = v[e] / s;
  }
#pragma unroll
  for (int e = 0; e < R; e += 4) {
    const int lo = __builtin_amdgcn_cvt_pk_fp8_f32(q[e], q[e + 1], 0, false);
    out[e / 4] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(q[e + 2], q[e + 3],
                                                           lo, true);
  }
}

}  // namespace tile
