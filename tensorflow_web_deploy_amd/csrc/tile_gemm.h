// The tile of a matrix product that the fp8 dense layers (gemm_fp8.hip) and
// the experts' layers (moe.hip) share:  acc[m][n] = sum_k A[m][k] B[n][k].
//
// A and B are rows of K contiguous values. One K step is 128 bytes of a row,
// 128 e4m3 or 64 bf16 values, so both types move through the same staging
// and the same LDS image; only the matrix instruction differs:
//   bf16  2 x v_mfma_f32_16x16x32_bf16, accumulated in place
//   e4m3  1 x v_mfma_f32_16x16x128_f8f6f4 into a fresh register, then
//         acc += product * (row scale * column scale): the scales are any
//         f32 numbers, so each block of 128 along K is scaled by the VALU
//         (or, EXACT, 4 x v_mfma_f32_16x16x32_f16 on what e4m3 converts to).
// The K index of a lane's bytes may be permuted at will as long as A and B
// agree: a lane takes the 16-byte chunks g and g+4 of its row (g = lane/16),
// for both types.
//
// The operands are swapped (B is the instruction's first operand), so a lane
// holds one row m: the row scale is one value a lane. Which columns the rows
// i of the NT tiles stand for is free. They are dealt so that a lane ends up
// with runs of W neighbouring columns, 16 bytes of the result's type (W = 16
// for e4m3, 8 for bf16, 4 for f32), and 4 lanes with 64 bytes of a row: the
// stores are wide and fill whole segments without a detour over LDS.
//   n = t / (W/4) * 4W + (i / 4) * W + t % (W/4) * 4 + i % 4
#pragma once
#include <hip/hip_runtime.h>

#include <cstdint>

namespace tile {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x8 __attribute__((ext_vector_type(8)));

constexpr int STEP = 128;  // bytes of a row in one K step

// BM x BN outputs by WM x WN waves; DEPTH stages in LDS, DEPTH-1 in flight;
// W neighbouring columns a lane
template <bool FP8_, int BM_, int BN_, int WM_, int WN_, int DEPTH_, int W_>
struct Shape {
  static constexpr bool FP8 = FP8_;
  static constexpr int W = W_;
  static constexpr int BM = BM_, BN = BN_, WM = WM_, WN = WN_, DEPTH = DEPTH_;
  static constexpr int WAVES = WM * WN, THREADS = WAVES * 64;
  static constexpr int MT = BM / WM / 16, NT = BN / WN / 16;  // a wave's tiles
  static constexpr int CA = BM / 8 / WAVES, CB = BN / 8 / WAVES;
  static_assert(CA * 8 * WAVES == BM && CB * 8 * WAVES == BN, "whole loads");
  static_assert(128 % (NT * 16) == 0, "a wave's columns share a scale");
  static_assert(NT * 4 % W == 0, "whole runs");
  static constexpr int RUNS = NT * 4 / W;  // of W columns a lane and row
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
                                         uint32_t at, uint32_t step_at) {
  const auto lds = (__attribute__((address_space(3))) void*)to;
  if constexpr (BYTES == 16)
    __builtin_amdgcn_raw_ptr_buffer_load_lds(r, lds, 16, (int)at,
                                             (int)step_at, 0, 0);
  else
    __builtin_amdgcn_raw_ptr_buffer_load_lds(r, lds, 4, (int)at, (int)step_at,
                                             0, 0);
}

// What this lane stages, as byte offsets at step 0: 16 bytes of a row of A or
// B a load, and one row scale. A row past the tile's end is another, existing
// row: its products are never stored, so every load stays inside its buffer.
template <class S>
struct Rows {
  uint32_t a[S::CA], b[S::CB], s;
};

// 8 rows of 128 bytes a load: lane / 8 is the row, lane % 8 the LDS slot.
// Chunk c of row r lies in slot c ^ key(r), so that the 16 rows of a fragment
// spread over all banks. key: r % 8 for A; for B the same of the fragment's
// row i, which the column order above puts at bits 0, 1 and log2(W).
template <class S>
__device__ __forceinline__ int key_b(int n) {
  return (n & 3) | ((n / S::W & 1) << 2);
}

__device__ __forceinline__ int staged_row(int wave, int count, int i,
                                          int lane) {
  return (wave * count + i) * 8 + (lane >> 3);
}

__device__ __forceinline__ uint32_t chunk_a(int wave, int count, int i,
                                            int lane) {
  const int r = staged_row(wave, count, i, lane);
  return ((lane & 7) ^ (r & 7)) << 4;
}

// row(r): byte offset of row r of the tile, for r below its BM or BN
template <class S, class A>
__device__ __forceinline__ void rows_of_a(Rows<S>& at, int wave, int lane,
                                          A row) {
#pragma unroll
  for (int i = 0; i < S::CA; ++i) {
    const int r = staged_row(wave, S::CA, i, lane);
    at.a[i] = row(r) + chunk_a(wave, S::CA, i, lane);
  }
}

template <class S, class B>
__device__ __forceinline__ void rows_of_b(Rows<S>& at, int wave, int lane,
                                          B row) {
#pragma unroll
  for (int i = 0; i < S::CB; ++i) {
    const int r = staged_row(wave, S::CB, i, lane);
    at.b[i] = row(r) + (((lane & 7) ^ key_b<S>(r)) << 4);
  }
}

// wave w brings the scales from row w*BM/WAVES on, 64 of them: where two waves
// overlap they write the same values, and what lies behind BM isn't read
template <class S>
__device__ __forceinline__ int scale_row(int wave, int lane) {
  return min(wave * (S::BM / S::WAVES) + lane, S::BM - 1);
}

// a step's rows of A and their scales
template <class S>
__device__ __forceinline__ void stage_a(char* lds, __amdgpu_buffer_rsrc_t ra,
                                        __amdgpu_buffer_rsrc_t rs,
                                        const Rows<S>& at, int step,
                                        uint32_t s_stride, int wave) {
#pragma unroll
  for (int i = 0; i < S::CA; ++i)
    load_lds<16>(ra, lds + (wave * S::CA + i) * 1024, at.a[i], step * STEP);
  if (S::FP8)
    load_lds<4>(rs,
                lds + (S::BM + S::BN) * STEP + wave * (S::BM / S::WAVES) * 4,
                at.s, step * s_stride);
}

template <class S>
__device__ __forceinline__ void stage_b(char* lds, __amdgpu_buffer_rsrc_t rb,
                                        const Rows<S>& at, int step,
                                        int wave) {
#pragma unroll
  for (int i = 0; i < S::CB; ++i)
    load_lds<16>(rb, lds + S::BM * STEP + (wave * S::CB + i) * 1024, at.b[i],
                 step * STEP);
}

// B's part of the steps that are on their way before the first is multiplied,
// for a caller that still waits to learn which rows of A it needs. Always as
// many, of a step that is there, so that the wait for something older needn't
// be one for these too.
template <class S>
__device__ __forceinline__ void send_b(char* smem, __amdgpu_buffer_rsrc_t rb,
                                       const Rows<S>& at, int first, int count,
                                       int wave) {
#pragma unroll
  for (int j = 0; j < S::DEPTH - 1; ++j)
    stage_b<S>(smem + j * S::STAGE, rb, at, first + min(j, count - 1), wave);
  asm volatile("" ::: "memory");  // the waits count on this order
}

// The product of two e4m3 tiles by the f16 instruction, whose sums keep what
// f32 holds, where the 8-bit one drops what lies 2^13 under the largest of 8
// neighbours. Half as fast, and 16 conversions a fragment.
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

__device__ __forceinline__ f16x8 wider(int lo, int hi) {
  typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
  const f16x2 a = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 1.f, false);
  const f16x2 b = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 1.f, true);
  const f16x2 c = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 1.f, false);
  const f16x2 d = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 1.f, true);
  return f16x8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

// of NT tiles of B with one of A: a chain of 4 instructions each, in turn
template <int NT>
__device__ __forceinline__ void exact_products(const i32x4 (&b)[NT][2],
                                               const i32x4 (&a)[2],
                                               f32x4 (&p)[NT]) {
#pragma unroll
  for (int t = 0; t < NT; ++t) p[t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int h = 0; h < 2; ++h)
#pragma unroll
    for (int i = 0; i < 4; i += 2) {
      const f16x8 wide = wider(a[h][i], a[h][i + 1]);
#pragma unroll
      for (int t = 0; t < NT; ++t)
        p[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(
            wider(b[t][h][i], b[t][h][i + 1]), wide, p[t], 0, 0, 0);
    }
}

template <class S>
struct FragA {
  i32x4 v[2];
  float f;
};

template <class S>
__device__ __forceinline__ FragA<S> read_a(const char* lds, int wm, int i,
                                           int lane) {
  const int m = wm * S::MT * 16 + i * 16 + (lane & 15), g = lane >> 4;
  const char* row = lds + m * STEP;
  FragA<S> a;
  a.v[0] = *(const i32x4*)(row + ((g ^ (m & 7)) << 4));
  a.v[1] = *(const i32x4*)(row + (((g + 4) ^ (m & 7)) << 4));
  a.f = S::FP8 ? *(const float*)(lds + (S::BM + S::BN) * STEP + m * 4) : 0.f;
  return a;
}

__device__ __forceinline__ i32x8 both(const i32x4 (&v)[2]) {
  return __builtin_shufflevector(v[0], v[1], 0, 1, 2, 3, 4, 5, 6, 7);
}

// the column, counted from the tile's first, that row i16 of a wave's tile t of
// B stands for
template <class S>
__device__ __forceinline__ int column_of(int wn, int t, int i16) {
  constexpr int Q = S::W / 4;
  return wn * S::NT * 16 + t / Q * 4 * S::W + (i16 >> 2) * S::W + t % Q * 4 +
         (i16 & 3);
}

// Blocks are scaled by the product of their two scales, which may leave the
// range of f32 where the scaled block doesn't: by an infinite one a block of 0
// becomes NaN, a subnormal one has lost bits. Both are factors above 1, or
// below, then, and one after the other they lose nothing.
struct Factors {
  float most = 0.f, least = 1.f;

  __device__ __forceinline__ void see(float f) {
    most = fmaxf(most, fabsf(f));
    least = fminf(least, fabsf(f));
  }
  __device__ __forceinline__ bool odd() const {
    return !(most < INFINITY && least >= 0x1p-126f);
  }
};

__device__ __forceinline__ float add_scaled(float sum, float p, float sa,
                                            float sb) {
  const float f = sa * sb;
  return __builtin_amdgcn_classf(f, 0x108)  // normal
             ? __builtin_fmaf(p, f, sum)
             : sum + p * sa * sb;
}

template <class S, bool EXACT>
__device__ __forceinline__ void compute(const char* lds, float sb, int wm,
                                        int wn, int lane, Factors& seen,
                                        f32x4 (&acc)[S::MT][S::NT]) {
  const int i16 = lane & 15, g = lane >> 4;
  const char* ldsb = lds + S::BM * STEP;
  i32x4 b[S::NT][2];
#pragma unroll
  for (int t = 0; t < S::NT; ++t) {
    const int n = column_of<S>(wn, t, i16);
    const char* row = ldsb + n * STEP;
    const int key = key_b<S>(n);
    b[t][0] = *(const i32x4*)(row + ((g ^ key) << 4));
    b[t][1] = *(const i32x4*)(row + (((g + 4) ^ key) << 4));
  }
  if constexpr (EXACT) {
#pragma unroll
    for (int i = 0; i < S::MT; ++i) {
      const FragA<S> a = read_a<S>(lds, wm, i, lane);
      const float f = a.f * sb;
      seen.see(f);
      f32x4 p[S::NT];
      exact_products(b, a.v, p);
#pragma unroll
      for (int t = 0; t < S::NT; ++t)
#pragma unroll
        for (int r = 0; r < 4; ++r)
          acc[i][t][r] = __builtin_fmaf(p[t][r], f, acc[i][t][r]);
    }
  } else if constexpr (S::FP8) {
    // Three things at a time: rows i + 2 are read, rows i multiplied, and the
    // products of rows i - 1 scaled and added, 4 additions behind each
    // matrix instruction, which takes 8 times the time of one. The order is
    // held, as the compiler's own puts the additions of a step together.
    FragA<S> a[3];
    a[0] = read_a<S>(lds, wm, 0, lane);
    if (S::MT > 1) a[1] = read_a<S>(lds, wm, 1, lane);
    __builtin_amdgcn_sched_barrier(0);
    f32x4 p[2][S::NT];
    float f[2];
#pragma unroll
    for (int i = 0; i <= S::MT; ++i) {
      if (i + 2 < S::MT) a[(i + 2) % 3] = read_a<S>(lds, wm, i + 2, lane);
      if (i < S::MT) f[i & 1] = a[i % 3].f * sb;
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int t = 0; t < S::NT; ++t) {
        if (i < S::MT)
          p[i & 1][t] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(
              both(b[t]), both(a[i % 3].v), f32x4{0.f, 0.f, 0.f, 0.f}, 0, 0, 0,
              0, 0, 0);
        if (i > 0)
#pragma unroll
          for (int r = 0; r < 4; ++r)
            acc[i - 1][t][r] = __builtin_fmaf(p[(i - 1) & 1][t][r],
                                              f[(i - 1) & 1],
                                              acc[i - 1][t][r]);
        if (t == S::NT - 1 && i < S::MT && (i & 1 || i == S::MT - 1)) {
          if (i & 1) seen.see(f[0]);
          seen.see(f[i & 1]);
        }
        __builtin_amdgcn_sched_barrier(0);
      }
    }
  } else {
    // rows i + 2 are read while rows i are multiplied
    FragA<S> a[3];
    a[0] = read_a<S>(lds, wm, 0, lane);
    if (S::MT > 1) a[1] = read_a<S>(lds, wm, 1, lane);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int i = 0; i < S::MT; ++i) {
      if (i + 2 < S::MT) a[(i + 2) % 3] = read_a<S>(lds, wm, i + 2, lane);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int t = 0; t < S::NT; ++t)
          acc[i][t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
              __builtin_bit_cast(bf16x8, b[t][h]),
              __builtin_bit_cast(bf16x8, a[i % 3].v[h]), acc[i][t], 0, 0, 0);
      __builtin_amdgcn_sched_barrier(0);
    }
  }
}

// Steps [first, first + count) of the product. sb: the scales of the wave's
// columns, one a step. B_SENT: send_b has been called. EXACT: e4m3 by the f16
// instruction. The answer: whether one of this lane's factors was odd.
template <class S, bool B_SENT, bool EXACT>
__device__ __forceinline__ bool product(char* smem, __amdgpu_buffer_rsrc_t ra,
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
    if (j < count) {
      if (!B_SENT) stage_b<S>(smem + j * S::STAGE, rb, at, first + j, wave);
      stage_a<S>(smem + j * S::STAGE, ra, rs, at, first + j, s_stride, wave);
      asm volatile("" ::: "memory");  // the waits count on this order
    }
  // constant memory, so that the scale comes by a scalar load: a vector load
  // here would wait for every stage that is on its way
  const auto sbc =
      (const __attribute__((address_space(4))) float*)(uintptr_t)sb;
  float fb = S::FP8 && count > 0 ? sbc[first] : 0.f;
  Factors seen;
  int now = 0, next = AHEAD % S::DEPTH;
  for (int j = 0; j < count; ++j) {
    // step j has landed once only the later ones are still on their way
    const int later = min(count - 1 - j, AHEAD - 1);
    // of those that send_b began, A's part alone is behind this one's
    constexpr int PART = S::LOADS - S::CB;
    if (B_SENT && j < AHEAD - 1 && later >= 2)
      asm volatile("s_waitcnt vmcnt(%0)" ::"i"(2 * PART) : "memory");
    else if (B_SENT && j < AHEAD - 1 && later == 1)
      asm volatile("s_waitcnt vmcnt(%0)" ::"i"(PART) : "memory");
    else if (later >= 2)
      asm volatile("s_waitcnt vmcnt(%0)" ::"i"(2 * S::LOADS) : "memory");
    else if (later == 1)
      asm volatile("s_waitcnt vmcnt(%0)" ::"i"(S::LOADS) : "memory");
    else
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::"s"(fb) : "memory");  // here, not among the LDS reads
    if (j + AHEAD < count) {
      char* to = smem + next * S::STAGE;
      stage_a<S>(to, ra, rs, at, first + j + AHEAD, s_stride, wave);
      stage_b<S>(to, rb, at, first + j + AHEAD, wave);
    }
    compute<S, EXACT>(smem + now * S::STAGE, fb, wm, wn, lane, seen,
                      acc);
    // the stage is free for the load behind the next barrier
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    if (S::FP8) fb = sbc[first + min(j + 1, count - 1)];
    now = now + 1 == S::DEPTH ? 0 : now + 1;
    next = next + 1 == S::DEPTH ? 0 : next + 1;
  }
  return seen.odd();
}

// The sums that a product with an odd factor has left, again and carefully, if
// it shows in them: some aren't finite, or lie between 2^-126 and 2^-103,
// where blocks with a subnormal factor end up (2^25 of 2^-126 and of 2^-149).
// Each wave for itself, from memory to registers, with the rows that row_a,
// row_b and row_s (a scale's offset) give. The largest and the least of the
// factors cost the steps 0 to 1%; a class test of each and an OR 2% (16200 x
// 4096 x 8192 540 / 544 / 552 us), a test of each sum behind the steps up to
// 9% (12544 x 768 x 2304 32.6 / 35.6).
template <class S, bool EXACT, class A, class B, class C>
__device__ __forceinline__ void mend_sums(
    __amdgpu_buffer_rsrc_t ra, __amdgpu_buffer_rsrc_t rb,
    __amdgpu_buffer_rsrc_t rs, A row_a, B row_b, C row_s, int first, int count,
    uint32_t s_stride, const float* sb, int wave, int lane, bool odd,
    f32x4 (&acc)[S::MT][S::NT]) {
  if (!__any(odd)) return;
  odd = false;
#pragma unroll
  for (int i = 0; i < S::MT; ++i)
#pragma unroll
    for (int t = 0; t < S::NT; ++t)
#pragma unroll
      for (int r = 0; r < 4; ++r)
        // NaN, infinite or subnormal
        odd |= __builtin_amdgcn_classf(acc[i][t][r] * 0x1p-23f, 0x297);
  if (!__any(odd)) return;
  // nothing of this is to be computed ahead, where it would take registers
  asm volatile("" : "+v"(lane), "+s"(wave));
  const int wm = wave / S::WN, wn = wave % S::WN, g = lane >> 4;
  auto load16 = [](__amdgpu_buffer_rsrc_t r, uint32_t at, int step) {
    return __builtin_bit_cast(i32x4, __builtin_amdgcn_raw_buffer_load_b128(
                                         r, (int)at, step * STEP, 0));
  };
#pragma unroll
  for (int i = 0; i < S::MT; ++i) {
    const int m = wm * S::MT * 16 + i * 16 + (lane & 15);
    const uint32_t at_a = row_a(m) + g * 16, at_s = row_s(m);
#pragma unroll
    for (int t = 0; t < S::NT; ++t) acc[i][t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll 1
    for (int j = first; j < first + count; ++j) {
      const i32x4 a[2] = {load16(ra, at_a, j), load16(ra, at_a + 64, j)};
      const float sa = __builtin_bit_cast(
          float, __builtin_amdgcn_raw_buffer_load_b32(
                     rs, (int)at_s, (int)(j * s_stride), 0));
#pragma unroll
      for (int t = 0; t < S::NT; ++t) {
        const uint32_t at_b =
            row_b(column_of<S>(wn, t, lane & 15)) + g * 16;
        const i32x4 b[1][2] = {
            {load16(rb, at_b, j), load16(rb, at_b + 64, j)}};
        f32x4 p[1];
        if constexpr (EXACT)
          exact_products(b, a, p);
        else
          p[0] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(
              both(b[0]), both(a), f32x4{0.f, 0.f, 0.f, 0.f}, 0, 0, 0, 0, 0,
              0);
#pragma unroll
        for (int r = 0; r < 4; ++r)
          acc[i][t][r] = add_scaled(acc[i][t][r], p[0][r], sa, sb[j]);
      }
    }
  }
}

// The product of up to 16 RT rows with 16 columns by one wave, for calls that
// read their weights for a few rows: bound by the time that the weights take
// to come, so they go from memory to registers at once, a step ahead: more of
// them was slower at every size (1 x 2048 x 16384, 1 / 2 / 3 / 4: 7.7 / 8.4 /
// 10.0 / 10.3 us), as fewer waves find room, and a step too many, loaded in
// vain, cost 0.3 us of 3.5.
// a[i], b, sa[i]: this lane's row of A, in each row tile, and of B (16 bytes
// from their start a quarter of the wave) and its row's scale at step 0. As in
// a tile, a lane ends up with row lane % 16 of each row tile and the columns
// lane / 16 * 4 + 0..3.
template <bool FP8, int RT>
struct FewStep {
  i32x4 a[RT][2], b[1][2];
  float sa[RT], sb;
};

template <bool FP8, int RT>
__device__ __forceinline__ FewStep<FP8, RT> few_step(
    const uint8_t* const (&a)[RT], const uint8_t* b,
    const float* const (&sa)[RT], int64_t s_rows, const float* sb, int step) {
  FewStep<FP8, RT> r;
  const int64_t k = (int64_t)step * STEP;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    r.b[0][h] = *(const i32x4*)(b + k + h * 64);
#pragma unroll
    for (int i = 0; i < RT; ++i) r.a[i][h] = *(const i32x4*)(a[i] + k + h * 64);
  }
#pragma unroll
  for (int i = 0; i < RT; ++i) r.sa[i] = FP8 ? sa[i][step * s_rows] : 0.f;
  r.sb = FP8 ? sb[step] : 0.f;
  return r;
}

template <bool FP8, bool EXACT, int RT>
__device__ __forceinline__ void few_multiply(const FewStep<FP8, RT>& s,
                                             f32x4 (&acc)[RT]) {
#pragma unroll
  for (int i = 0; i < RT; ++i) {
    if constexpr (FP8) {
      f32x4 q[1];
      f32x4& p = q[0];
      if constexpr (EXACT)
        exact_products(s.b, s.a[i], q);
      else
        p = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(
            both(s.b[0]), both(s.a[i]), f32x4{0.f, 0.f, 0.f, 0.f}, 0, 0, 0, 0,
            0, 0);
#pragma unroll
      for (int r = 0; r < 4; ++r)
        acc[i][r] = add_scaled(acc[i][r], p[r], s.sa[i], s.sb);
    } else {
#pragma unroll
      for (int h = 0; h < 2; ++h)
        acc[i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
            __builtin_bit_cast(bf16x8, s.b[0][h]),
            __builtin_bit_cast(bf16x8, s.a[i][h]), acc[i], 0, 0, 0);
    }
  }
}

template <bool FP8, bool EXACT, int RT>
__device__ __forceinline__ void few_product(
    const uint8_t* const (&a)[RT], const uint8_t* b,
    const float* const (&sa)[RT], int64_t s_rows, const float* sb, int first,
    int last, f32x4 (&acc)[RT]) {
#pragma unroll
  for (int i = 0; i < RT; ++i) acc[i] = f32x4{0.f, 0.f, 0.f, 0.f};
  if (first >= last) return;
  auto now = few_step<FP8, RT>(a, b, sa, s_rows, sb, first);
  for (int s = first; s < last; ++s) {
    FewStep<FP8, RT> next;
    if (s + 1 < last) next = few_step<FP8, RT>(a, b, sa, s_rows, sb, s + 1);
    few_multiply<FP8, EXACT>(now, acc);
    now = next;
  }
}

// one row tile
template <bool FP8, bool EXACT>
__device__ __forceinline__ f32x4 few_product(const uint8_t* a,
                                             const uint8_t* b, const float* sa,
                                             int64_t s_rows, const float* sb,
                                             int first, int last) {
  const uint8_t* const as[1] = {a};
  const float* const sas[1] = {sa};
  f32x4 acc[1];
  few_product<FP8, EXACT>(as, b, sas, s_rows, sb, first, last, acc);
  return acc[0];
}

// What KS waves have of the same 16 x 16 results, added up in their order;
// part: 1 KB of LDS a wave. The sum is for the waves with ks = 0.
template <int KS>
__device__ __forceinline__ f32x4 few_join(f32x4 acc, float* part, int group,
                                          int ks, int lane) {
  if constexpr (KS == 1) return acc;
  f32x4* at = (f32x4*)part + group * KS * 64 + lane;
  at[ks * 64] = acc;
  __syncthreads();
  f32x4 sum = at[0];
#pragma unroll
  for (int k = 1; k < KS; ++k) sum += at[k * 64];
  return sum;
}

// Run q of a lane's columns in row tile i: v[c] is column
//   run_column(q) + c,  counted from the wave's first one.
template <class S>
__device__ __forceinline__ int run_column(int q, int lane) {
  return q * 4 * S::W + (lane >> 4) * S::W;
}

template <class S>
__device__ __forceinline__ void run_of(const f32x4 (&acc)[S::NT], int q,
                                       float (&v)[S::W]) {
#pragma unroll
  for (int c = 0; c < S::W; ++c) v[c] = acc[q * (S::W / 4) + c / 4][c % 4];
}

// R numbers from p on that the caller knows to be there, or those below
// `have` and 0 for the rest
template <int R>
__device__ __forceinline__ void load_run(const float* p, int have,
                                         float (&v)[R]) {
  if (have >= R) {
    __builtin_memcpy(v, p, sizeof(v));
  } else {
#pragma unroll
    for (int c = 0; c < R; ++c) v[c] = c < have ? p[c] : 0.f;
  }
}

template <int R>
__device__ __forceinline__ void store_run(float* p, int have,
                                          const float (&v)[R]) {
  if (have >= R) {
    __builtin_memcpy(p, v, sizeof(v));
  } else {
#pragma unroll
    for (int c = 0; c < R; ++c)
      if (c < have) p[c] = v[c];
  }
}

// v Phi(v), the erf-GELU. The normal distribution's tail beyond |v| is
// Abramowitz and Stegun's 7.1.26, 1/2 t (a1 + .. + a5 t^4) exp(-v^2 / 2) with
// t = 1 / (1 + p |v| / sqrt 2): off by less than 1e-7, as 1 + erf in f32 is, in
// 13 operations. With erff the activation alone took a quarter of a large
// product's time; with erfcf 12544 x 768 x 768 into f32 took 45 us, not 38.
__device__ __forceinline__ float gelu(float v) {
  const float t = __builtin_amdgcn_rcpf(
      __builtin_fmaf(0.3275911f * 0.70710678f, fabsf(v), 1.f));
  float h = __builtin_fmaf(0.5f * 1.061405429f, t, 0.5f * -1.453152027f);
  h = __builtin_fmaf(h, t, 0.5f * 1.421413741f);
  h = __builtin_fmaf(h, t, 0.5f * -0.284496736f);
  h = __builtin_fmaf(h, t, 0.5f * 0.254829592f);
  h *= t * __builtin_amdgcn_exp2f(v * v * -0.72134752f);  // log2(e) / 2
  return v * (v < 0.f ? h : 1.f - h);
}

// What an activation's code comes to: nothing, a clamp, GELU. Kernels of many
// rows are made for one of them.
enum { PLAIN, CLAMP, GELU };

inline int kind_of(int act) {
  return act == 0 ? PLAIN : act == 5 ? GELU : CLAMP;
}

template <int KIND, int R>
__device__ __forceinline__ void activate_kind(float (&v)[R], int act) {
  if constexpr (KIND == CLAMP) {
    const float high = act == 2 ? 6.f : INFINITY;
#pragma unroll
    for (int e = 0; e < R; ++e)  // NaN stays
      v[e] = v[e] < 0.f ? 0.f : v[e] > high ? high : v[e];
  } else if constexpr (KIND == GELU) {
#pragma unroll
    for (int e = 0; e < R; ++e) v[e] = gelu(v[e]);
  }
}

// act: 0 none, 1 relu, 2 relu6, 5 erf-GELU, the codes of the bf16 GEMM
template <int R>
__device__ __forceinline__ void activate(float (&v)[R], int act) {
  if (act == 5)
    activate_kind<GELU>(v, act);
  else if (act)
    activate_kind<CLAMP>(v, act);
}

// Workgroups go round the 8 XCDs in turn. Give each XCD a contiguous run of
// tiles, and let the run go down HIGH rows of tiles before it moves a column
// on: what an XCD holds at once then shares both its rows and its columns in
// the XCD's L2.
struct Place {
  int m, n;
};

constexpr int HIGH = 8;  // 2, 4 and 16 were up to 1% slower

__device__ __forceinline__ Place place_of(int bid, int tiles_m, int tiles_n) {
  const int n = tiles_m * tiles_n;
  const int q = n >> 3, r = n & 7, xcd = bid & 7, off = bid >> 3;
  const int i = (xcd < r ? xcd * (q + 1) : r * (q + 1) + (xcd - r) * q) + off;
  const int band = i / (HIGH * tiles_n), in = i - band * HIGH * tiles_n;
  const int rows = min(HIGH, tiles_m - band * HIGH);
  return {band * HIGH + in % rows, in / rows};
}

}  // namespace tile
