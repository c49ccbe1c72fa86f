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

// 8 values from p on, the ones from `have` on as 0. The copy needs no
// alignment: rows of an odd width start anywhere.
template <typename T>
__device__ __forceinline__ void load8(const T* p, int have, float (&v)[8]) {
  if (have >= 8) {
    T t[8];
    __builtin_memcpy(t, p, sizeof(t));
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = (float)t[e];
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = e < have ? (float)p[e] : 0.f;
  }
}

__device__ __forceinline__ void store_fp8(uint8_t* to, const float (&v)[8],
                                          float s) {
  uint32_t q[2];
  to_fp8(v, s, q);
  *(uint2*)to = make_uint2(q[0], q[1]);
}

// Rows to round, 16 a workgroup and `per` blocks of 128 each: 16 lanes take a
// block of a row, 8 values each. Bound by the bytes it moves.
template <typename T>
struct QuantRows {
  const T* X;
  int64_t ldx, M;
  int K;
  uint8_t* Q;
  int Kp;
  float* S;  // [Kp / 128][M]
  int per;

  // Whole rows, unless so few that the workgroups don't fill the chip: 64 x
  // 25088 would take 115 us, cut up it takes 3.6; 12544 x 1536 12.8 cut up into
  // 2048 workgroups, 14.7 in whole rows.
  static QuantRows of(const T* X, int64_t ldx, int64_t M, int K, void* Q,
                      int Kp, float* S) {
    const int64_t rows = (M + 15) / 16, kb = Kp / 128;
    const int64_t cuts =
        rows >= 2048 ? 1 : kb < 2048 / rows ? kb : 2048 / rows;
    return {X, ldx, M, K, (uint8_t*)Q, Kp, S, (int)((kb + cuts - 1) / cuts)};
  }
  __host__ __device__ int64_t across() const {
    return (Kp / 128 + per - 1) / per;
  }
  int64_t workgroups() const { return (M + 15) / 16 * across(); }

  __device__ __forceinline__ void run(int64_t block) const {
    const int64_t rows = block / across();
    const int kb0 = (int)(block - rows * across()) * per;
    const int l = threadIdx.x & 15;
    const int64_t m = rows * 16 + (threadIdx.x >> 4);
    if (m >= M) return;
    const int end = min(kb0 + per, Kp / 128);
    for (int kb = kb0; kb < end; ++kb) {
      const int k = kb * 128 + l * 8;
      float v[8];
      load8(X + m * ldx + k, K - k, v);
      uint32_t top = amax_bits(v);
#pragma unroll
      for (int d = 8; d; d >>= 1)
        top = max(top, (uint32_t)__shfl_xor((int)top, d));
      const float s = scale_of(top);
      store_fp8(Q + m * Kp + k, v, s);
      if (l == 0) S[kb * M + m] = s;
    }
  }
};

}  // namespace tile
