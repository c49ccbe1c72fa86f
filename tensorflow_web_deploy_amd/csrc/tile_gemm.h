// The tile of a matrix product that the fp8 dense layers (gemm_fp8.hip) and
// the experts' layers (moe.hip) share:  acc[m][n] = sum_k A[m][k] B[n][k].
//
// A and B are rows of K contiguous values. One K step is 128 bytes of a row,
// 128 e4m3 or 64 bf16 values, so both types move through the same staging
// and the same LDS image; only the matrix instruction differs:
//   bf16  2 x v_mfma_f32_16x16x32_bf16, accumulated in place
//   e4m3  1 x v_mfma_f32_16x16x128_f8f6f4 into a fresh register, then
//         acc += product * (row scale * column scale): the scales are any
//         f32 numbers, so each block of 128 along K is scaled by the VALU.
// The K index of a lane's bytes may be permuted at will as long as A and B
// agree: a lane takes the 16-byte chunks g and g+4 of its row (g = lane/16),
// for both types.
//
// The operands are swapped (B is the instruction's first operand), so a lane
// holds one row m and, over its tiles, 4*NT consecutive columns n: the row
// scale is one value a lane, and the stores are 16 bytes wide without a
// detour over LDS. The column that row i of tile t stands for is
//   n = (i / 4) * 4 * NT + t * 4 + i % 4.
#pragma once
#include <hip/hip_runtime.h>

#include <cstdint>

namespace tile {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x8 __attribute__((ext_vector_type(8)));

constexpr int STEP = 128;                 // bytes of a row in one K step
constexpr uint32_t NOWHERE = 0xfffffff0u;  // past every buffer: reads as 0

// BM x BN outputs by WM x WN waves; DEPTH stages in LDS, DEPTH-1 in flight
template <bool FP8_, int BM_, int BN_, int WM_, int WN_, int DEPTH_>
struct Shape {
  static constexpr bool FP8 = FP8_;
  static constexpr int BM = BM_, BN = BN_, WM = WM_, WN = WN_, DEPTH = DEPTH_;
  static constexpr int WAVES = WM * WN, THREADS = WAVES * 64;
  static constexpr int MT = BM / WM / 16, NT = BN / WN / 16;  // a wave's tiles
  static constexpr int CA = BM / 8 / WAVES, CB = BN / 8 / WAVES;
  static_assert(CA * 8 * WAVES == BM && CB * 8 * WAVES == BN, "whole loads");
  static_assert(128 % (NT * 16) == 0, "a wave's columns share a scale");
  // the last wave's load of row scales writes past BM: 64 floats of slack
  static constexpr int SCALES = FP8 ? (BM + 64) * 4 : 0;
  static constexpr int STAGE = (BM + BN) * STEP + SCALES;
  static constexpr int LDS = DEPTH * STAGE;
  static constexpr int LOADS = CA + CB + (FP8 ? 1 : 0);  // a wave and stage
};

__device__ __forceinline__ __amdgpu_buffer_rsrc_t buffer(const void* p,
                                                         uint32_t bytes) {
  return __builtin_amdgcn_make_buffer_rsrc((void*)p, 0, (int)bytes,
                                           0x00020000);
}

template <int BYTES>
__device__ __forceinline__ void load_lds(__amdgpu_buffer_rsrc_t r, char* to,
                                         uint32_t at) {
  const auto lds = (__attribute__((address_space(3))) void*)to;
  if constexpr (BYTES == 16)
    __builtin_amdgcn_raw_ptr_buffer_load_lds(r, lds, 16, (int)at, 0, 0, 0);
  else
    __builtin_amdgcn_raw_ptr_buffer_load_lds(r, lds, 4, (int)at, 0, 0, 0);
}

// The rows that this lane stages: byte offsets of their first value, NOWHERE
// for a row that isn't there
template <class S>
struct Rows {
  uint32_t a[S::CA], b[S::CB], s;
};

// 8 rows of 128 bytes a load: lane / 8 is the row, lane % 8 the LDS slot.
// Chunk c of row r lies in slot c ^ key(r), so that the 16 rows of a fragment
// spread over all banks. key: r % 8 for A; for B the same of the fragment's
// row i, which the column order above puts at bits 0, 1 and log2(4*NT).
template <class S>
__device__ __forceinline__ int key_b(int n) {
  return (n & 3) | ((n / (4 * S::NT) & 1) << 2);
}

template <class S>
__device__ __forceinline__ int staged_row(int wave, int count, int i,
                                          int lane) {
  return (wave * count + i) * 8 + (lane >> 3);
}

template <class S>
__device__ __forceinline__ void stage(char* lds, __amdgpu_buffer_rsrc_t ra,
                                      __amdgpu_buffer_rsrc_t rb,
                                      __amdgpu_buffer_rsrc_t rs,
                                      const Rows<S>& at, int step,
                                      uint32_t s_stride,
                                      int wave, int lane) {
  const int slot = lane & 7;
#pragma unroll
  for (int i = 0; i < S::CA; ++i) {
    const int r = staged_row<S>(wave, S::CA, i, lane);
    const uint32_t k = (uint32_t)step * STEP + ((slot ^ (r & 7)) << 4);
    load_lds<16>(ra, lds + (wave * S::CA + i) * 1024,
                 at.a[i] == NOWHERE ? NOWHERE : at.a[i] + k);
  }
  char* ldsb = lds + S::BM * STEP;
#pragma unroll
  for (int i = 0; i < S::CB; ++i) {
    const int r = staged_row<S>(wave, S::CB, i, lane);
    const uint32_t k = (uint32_t)step * STEP + ((slot ^ key_b<S>(r)) << 4);
    load_lds<16>(rb, ldsb + (wave * S::CB + i) * 1024, at.b[i] + k);
  }
  if (S::FP8) {
    // wave w brings the rows from w*BM/WAVES on, 64 of them: where two waves
    // overlap they write the same values
    load_lds<4>(rs, lds + (S::BM + S::BN) * STEP + wave * (S::BM / S::WAVES) * 4,
                at.s == NOWHERE ? NOWHERE : at.s + (uint32_t)step * s_stride);
  }
}

template <class S>
__device__ __forceinline__ void compute(const char* lds, float sb, int wm,
                                        int wn, int lane,
                                        f32x4 (&acc)[S::MT][S::NT]) {
  const int i16 = lane & 15, g = lane >> 4;
  const char* ldsb = lds + S::BM * STEP;
  i32x4 b[S::NT][2];
#pragma unroll
  for (int t = 0; t < S::NT; ++t) {
    const int n = wn * S::NT * 16 + (i16 >> 2) * 4 * S::NT + t * 4 + (i16 & 3);
    const char* row = ldsb + n * STEP;
    const int key = key_b<S>(n);
    b[t][0] = *(const i32x4*)(row + ((g ^ key) << 4));
    b[t][1] = *(const i32x4*)(row + (((g + 4) ^ key) << 4));
  }
#pragma unroll
  for (int i = 0; i < S::MT; ++i) {
    const int m = wm * S::MT * 16 + i * 16 + i16;
    const char* row = lds + m * STEP;
    i32x4 a[2];
    a[0] = *(const i32x4*)(row + ((g ^ (m & 7)) << 4));
    a[1] = *(const i32x4*)(row + (((g + 4) ^ (m & 7)) << 4));
    if constexpr (S::FP8) {
      const float f =
          *(const float*)(lds + (S::BM + S::BN) * STEP + m * 4) * sb;
      const i32x8 a8 = __builtin_shufflevector(a[0], a[1], 0, 1, 2, 3, 4, 5,
                                               6, 7);
#pragma unroll
      for (int t = 0; t < S::NT; ++t) {
        const i32x8 b8 = __builtin_shufflevector(b[t][0], b[t][1], 0, 1, 2, 3,
                                                 4, 5, 6, 7);
        const f32x4 p = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(
            b8, a8, f32x4{0.f, 0.f, 0.f, 0.f}, 0, 0, 0, 0, 0, 0);
#pragma unroll
        for (int r = 0; r < 4; ++r)
          acc[i][t][r] = __builtin_fmaf(p[r], f, acc[i][t][r]);
      }
    } else {
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int t = 0; t < S::NT; ++t)
          acc[i][t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
              __builtin_bit_cast(bf16x8, b[t][h]),
              __builtin_bit_cast(bf16x8, a[h]), acc[i][t], 0, 0, 0);
    }
  }
}

// Steps [first, first + count) of the product. sb: the scales of the wave's
// columns, one a step.
template <class S>
__device__ __forceinline__ void product(char* smem, __amdgpu_buffer_rsrc_t ra,
                                        __amdgpu_buffer_rsrc_t rb,
                                        __amdgpu_buffer_rsrc_t rs,
                                        const Rows<S>& at, int first,
                                        int count, uint32_t s_stride,
                                        const float* sb,
                                        int wave, int lane,
                                        f32x4 (&acc)[S::MT][S::NT]) {
  const int wm = wave / S::WN, wn = wave % S::WN;
#pragma unroll
  for (int i = 0; i < S::MT; ++i)
#pragma unroll
    for (int t = 0; t < S::NT; ++t) acc[i][t] = f32x4{0.f, 0.f, 0.f, 0.f};
  constexpr int AHEAD = S::DEPTH - 1;
#pragma unroll
  for (int j = 0; j < AHEAD; ++j)
    if (j < count)
      stage<S>(smem + j * S::STAGE, ra, rb, rs, at, first + j,
                     s_stride, wave, lane);
  int now = 0, next = AHEAD % S::DEPTH;
  for (int j = 0; j < count; ++j) {
    // step j has landed once only the later ones are still on their way
    const int later = min(count - 1 - j, AHEAD - 1);
    if (later >= 2)
      asm volatile("s_waitcnt vmcnt(%0)" ::"i"(2 * S::LOADS) : "memory");
    else if (later == 1)
      asm volatile("s_waitcnt vmcnt(%0)" ::"i"(S::LOADS) : "memory");
    else
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    if (j + AHEAD < count)
      stage<S>(smem + next * S::STAGE, ra, rb, rs, at, first + j + AHEAD,
                     s_stride, wave, lane);
    compute<S>(smem + now * S::STAGE, S::FP8 ? sb[first + j] : 0.f, wm, wn,
               lane, acc);
    // the stage is free for the load behind the next barrier
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    now = now + 1 == S::DEPTH ? 0 : now + 1;
    next = next + 1 == S::DEPTH ? 0 : next + 1;
  }
}

// 0 none, 1 relu, 2 relu6, 5 erf-GELU: the codes of the bf16 GEMM
template <int ACT>
__device__ __forceinline__ float activate(float v) {
  if (ACT == 1) return v < 0.f ? 0.f : v;
  if (ACT == 2) return v < 0.f ? 0.f : v > 6.f ? 6.f : v;
  if (ACT == 5) return 0.5f * v * (1.f + erff(v * 0.70710678f));
  return v;
}

template <int ACT, int R>
__device__ __forceinline__ void activate_all(float (&v)[R]) {
#pragma unroll
  for (int e = 0; e < R; ++e) v[e] = activate<ACT>(v[e]);
}

template <int R>
__device__ __forceinline__ void activate_by(float (&v)[R], int act) {
  if (act == 1)
    activate_all<1>(v);
  else if (act == 2)
    activate_all<2>(v);
  else if (act == 5)
    activate_all<5>(v);
}

// Workgroups go round the 8 XCDs in turn. Give each XCD a contiguous run of
// tiles, so that neighbours share their rows of A and B in its L2.
__device__ __forceinline__ int by_xcd(int bid, int n) {
  const int q = n >> 3, r = n & 7, xcd = bid & 7, off = bid >> 3;
  return (xcd < r ? xcd * (q + 1) : r * (q + 1) + (xcd - r) * q) + off;
}

}  // namespace tile
