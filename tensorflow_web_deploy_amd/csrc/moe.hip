// Mixture-of-experts layers.
//   moe_route  scores = softmax(logits) | sigmoid(logits); the k experts with
//              the largest score + bias, out of the groups that are kept;
//              their scores, renormalised and scaled, are the weights
//   moe_mlp    Y[t] = sum_j w[t][j] (act(x W1_e^T + b1_e) W2_e^T + b2_e)
//              + residual[t],  e = ids[t][j]
// An assignment a = t * k + j is one row of the experts' products. The rows
// are put in the order of their experts (plan), two grouped products run over
// tiles of one expert's rows each, and every token adds up its k rows.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstdint>

#include "kernels.h"
#include "quant_fp8.h"
#include "tile_gemm.h"

namespace {

using namespace tile;

int up(int64_t a, int64_t b) { return (int)((a + b - 1) / b); }

// ------------------------------------------------------------ moe_route

struct Route {
  const void* x;
  const float* bias;
  int* ids;
  float* weights;
  int64_t ldx;
  int T, E, k, groups, kept, best;
  bool sigmoid, renorm;
  float scale;
};

__device__ __forceinline__ float exp_of(float v) { return expf(v); }
__device__ __forceinline__ double exp_of(double v) { return exp(v); }

template <typename R>
__device__ __forceinline__ R wave_max(R v) {
#pragma unroll
  for (int d = 32; d; d >>= 1) {
    const R o = __shfl_xor(v, d);
    v = o > v ? o : v;
  }
  return v;
}

template <typename R>
__device__ __forceinline__ R wave_sum(R v) {
#pragma unroll
  for (int d = 32; d; d >>= 1) v += __shfl_xor(v, d);
  return v;
}

// How far the f32 score p and key = p + bias may be off: exp's argument is at
// most 104 wide where p isn't 0, its rounding and those of exp, sum, division
// and addition stay within 128 * 2^-24 of p and 2^-23 of the key.
__device__ __forceinline__ float error_of(float p, float key) {
  return 0x1p-17f * p + 0x1p-23f * fabsf(key) + 1e-37f;
}

// One row by one wave, lane l with the experts l + 64 v. With R = float it
// answers whether every decision is safe from rounding; if not, nothing has
// been written and the row is done again with R = double. Which experts are
// chosen, and their order, is so that of the scores in 64 bits, the lower
// index first among equals.
template <typename R, int V>
__device__ bool route_row(const Route& p, int64_t t, const float (&x)[V],
                          const float (&b)[V], R* lds, int lane) {
  constexpr bool FAST = sizeof(R) == 4;
  const R NONE = -(R)INFINITY;
  R s[V], key[V];
  if (p.sigmoid) {
#pragma unroll
    for (int v = 0; v < V; ++v)
      s[v] = x[v] > -INFINITY ? 1 / (1 + exp_of(-(R)x[v])) : 0;
  } else {
    float top = x[0];
#pragma unroll
    for (int v = 1; v < V; ++v) top = fmaxf(top, x[v]);
    top = wave_max(top);
    R sum = 0;
#pragma unroll
    for (int v = 0; v < V; ++v) {
      // an infinite logit leaves nothing to the finite ones
      s[v] = x[v] == top ? (R)1 : exp_of((R)x[v] - (R)top);
      if (!(x[v] > -INFINITY)) s[v] = 0;
      sum += s[v];
    }
    sum = wave_sum(sum);
#pragma unroll
    for (int v = 0; v < V; ++v) s[v] = sum > 0 ? s[v] / sum : 0;
  }
#pragma unroll
  for (int v = 0; v < V; ++v) {
    key[v] = s[v] + (R)b[v];
    if (!(x[v] > -INFINITY) || !(key[v] > NONE)) key[v] = NONE;
  }
  bool safe = true;

  if (p.groups > 1) {
    const int size = p.E / p.groups;
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int v = 0; v < V; ++v)
      if (v * 64 + lane < p.E) {
        lds[v * 64 + lane] = key[v];
        if (FAST) lds[p.E + v * 64 + lane] = error_of(s[v], key[v]);
      }
    __builtin_amdgcn_wave_barrier();
    R first = NONE, second = NONE;
    float e1 = 0, e2 = 0;
    if (lane < p.groups)
      for (int i = 0; i < size; ++i) {
        const R y = lds[lane * size + i];
        const float e = FAST ? (float)lds[p.E + lane * size + i] : 0.f;
        if (y > first) {
          second = first, e2 = e1;
          first = y, e1 = e;
        } else if (y > second) {
          second = y, e2 = e;
        }
      }
    R total = first;
    if (p.best == 2 && second > NONE) total += second, e1 += e2;
    e1 += 0x1p-23f * fabsf((float)total);
    int rank = 0;
    for (int g = 0; g < p.groups; ++g) {
      const R o = __shfl(total, g);
      rank += o > total || (o == total && g < lane);
    }
    const bool keep = lane < p.groups && rank < p.kept;
    const uint64_t kept = __ballot(keep);
    if (FAST) {
      // the last group that is kept against the first that isn't
      float low = keep ? (float)total - e1 : INFINITY;
      float high = lane < p.groups && !keep && total > NONE
                       ? (float)total + e1 : -INFINITY;
      low = -wave_max(-low);
      high = wave_max(high);
      safe = !(low <= high);
    }
#pragma unroll
    for (int v = 0; v < V; ++v)
      if (!(kept >> ((v * 64 + lane) / size & 63) & 1)) key[v] = NONE;
  }

  // k times the largest key, and once more for the one that just fails
  R mine = 0, sum = 0, last_key = 0;
  int id = -1;
  float last_e = 0, last_x = 0, last_b = 0;
  for (int j = 0; j <= p.k; ++j) {
    R y = key[0];
    int at = lane, v_at = 0;
#pragma unroll
    for (int v = 1; v < V; ++v)
      if (key[v] > y) y = key[v], at = v * 64 + lane, v_at = v;
    R top = y;
    int e = at;
#pragma unroll
    for (int d = 32; d; d >>= 1) {
      const R o = __shfl_xor(top, d);
      const int oe = __shfl_xor(e, d);
      if (o > top || (o == top && oe < e)) top = o, e = oe;
    }
    if (!(top > NONE)) break;
    // what the chosen one's lane holds of it
    R sv = 0;
    float xv = 0, bv = 0;
#pragma unroll
    for (int v = 0; v < V; ++v)
      if (v == v_at) {
        sv = s[v], xv = x[v], bv = b[v];
        if (at == e) key[v] = NONE;
      }
    sv = __shfl(sv, e & 63);
    if (FAST) {
      xv = __shfl(xv, e & 63), bv = __shfl(bv, e & 63);
      const float err = error_of((float)sv, (float)top);
      // equal logits and biases tie in any precision
      if (j && !(last_key - top > last_e + err) &&
          !(xv == last_x && bv == last_b))
        safe = false;
      last_key = top, last_e = err, last_x = xv, last_b = bv;
    }
    if (j == p.k) break;
    if (lane == j) mine = sv, id = e;
    sum += sv;
  }
  // scores that leave the range of f32 still have their ratios
  if (FAST && p.renorm && __shfl(id, 0) >= 0 && !(sum > (R)1e-30f))
    safe = false;
  if (FAST && !safe) return false;
  if (lane < p.k) {
    R w = mine;
    if (p.renorm) w = sum > 0 ? w / sum : 0;
    p.ids[t * p.k + lane] = id;
    p.weights[t * p.k + lane] = (float)(w * (R)p.scale);
  }
  return true;
}

// 4 rows a workgroup, a wave each
template <typename T, int V>
__global__ __launch_bounds__(256) void route_kernel(Route p) {
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t t = (int64_t)blockIdx.x * 4 + wave;
  if (t >= p.T) return;
  float x[V], b[V];
#pragma unroll
  for (int v = 0; v < V; ++v) {
    const int e = v * 64 + lane;
    const bool in = e < p.E;
    x[v] = in ? (float)((const T*)p.x)[t * p.ldx + e] : -INFINITY;
    if (!(x[v] > -INFINITY)) x[v] = -INFINITY;  // NaN: not to be chosen
    b[v] = in && p.bias ? p.bias[e] : 0.f;
  }
  double* lds = (double*)smem + wave * p.E;
  if (!route_row<float, V>(p, t, x, b, (float*)lds, lane))
    route_row<double, V>(p, t, x, b, lds, lane);
}

// ----------------------------------------------------------------- plan

constexpr int PLAN_THREADS = 256, PLAN_ROWS = 4096;

struct Plan {
  const int* ids;
  int* counts;  // [blocks][E]: how many of a block's rows go to an expert
  int* order;   // [N]: the assignments, by expert; behind them nothing
  int4* tiles;  // {expert, first place in order, rows, 0}; expert -1: none
  int N, E, BM, n_tiles, blocks;
};

__global__ __launch_bounds__(PLAN_THREADS) void plan_count_kernel(Plan p) {
  extern __shared__ int count[];
  for (int e = threadIdx.x; e < p.E; e += PLAN_THREADS) count[e] = 0;
  __syncthreads();
  const int a0 = blockIdx.x * PLAN_ROWS;
  for (int i = threadIdx.x; i < PLAN_ROWS && a0 + i < p.N; i += PLAN_THREADS) {
    const unsigned e = (unsigned)p.ids[a0 + i];
    if (e < (unsigned)p.E) atomicAdd(&count[e], 1);
  }
  __syncthreads();
  for (int e = threadIdx.x; e < p.E; e += PLAN_THREADS)
    p.counts[blockIdx.x * p.E + e] = count[e];
}

// out[i] = sum of in[0..i), for i up to n: by the first wave, 64 a turn
__device__ __forceinline__ void scan(const int* in, int* out, int n) {
  if (threadIdx.x < 64) {
    const int lane = threadIdx.x;
    int before = 0;
    for (int i = 0; i < n; i += 64) {
      int v = i + lane < n ? in[i + lane] : 0, s = v;
#pragma unroll
      for (int d = 1; d < 64; d <<= 1) {
        const int o = __shfl_up(s, d);
        if (lane >= d) s += o;
      }
      if (i + lane < n) out[i + lane] = before + s - v;
      before += __shfl(s, 63);
    }
    if (lane == 0) out[n] = before;
  }
}

// Each workgroup puts its rows behind those of the workgroups before it; the
// first one lists the tiles. Which place a row gets among its workgroup's of
// the same expert is left to chance: no result hangs on it, as a row's
// products don't on the rows beside it.
__global__ __launch_bounds__(PLAN_THREADS) void plan_place_kernel(Plan p) {
  extern __shared__ int lds[];
  int* total = lds;             // [E], later tiles of each expert
  int* next = lds + p.E;        // [E]
  int* start = lds + 2 * p.E;   // [E + 1]
  int* tile0 = lds + 3 * p.E + 1;  // [E + 1]
  const int a0 = blockIdx.x * PLAN_ROWS;
  if (p.blocks == 1) {
    for (int e = threadIdx.x; e < p.E; e += PLAN_THREADS) total[e] = 0;
    __syncthreads();
    for (int i = threadIdx.x; i < p.N; i += PLAN_THREADS) {
      const unsigned e = (unsigned)p.ids[i];
      if (e < (unsigned)p.E) atomicAdd(&total[e], 1);
    }
  } else {
    for (int e = threadIdx.x; e < p.E; e += PLAN_THREADS) {
      int before = 0, sum = 0;
      for (int b = 0; b < p.blocks; ++b) {
        const int c = p.counts[b * p.E + e];
        if (b < (int)blockIdx.x) before += c;
        sum += c;
      }
      total[e] = sum;
      next[e] = before;
    }
  }
  __syncthreads();
  scan(total, start, p.E);
  __syncthreads();
  for (int e = threadIdx.x; e < p.E; e += PLAN_THREADS) {
    next[e] = start[e] + (p.blocks == 1 ? 0 : next[e]);
    total[e] = (total[e] + p.BM - 1) / p.BM;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < PLAN_ROWS && a0 + i < p.N; i += PLAN_THREADS) {
    const unsigned e = (unsigned)p.ids[a0 + i];
    if (e < (unsigned)p.E) p.order[atomicAdd(&next[e], 1)] = a0 + i;
  }
  if (blockIdx.x != 0) return;
  scan(total, tile0, p.E);
  __syncthreads();
  for (int i = threadIdx.x; i < p.n_tiles; i += PLAN_THREADS) {
    int4 t = make_int4(-1, 0, 0, 0);
    if (i < tile0[p.E]) {
      int lo = 0, hi = p.E;  // the expert with tile0[e] <= i < tile0[e + 1]
      while (hi - lo > 1) {
        const int mid = (lo + hi) / 2;
        if (tile0[mid] <= i)
          lo = mid;
        else
          hi = mid;
      }
      const int at = start[lo] + (i - tile0[lo]) * p.BM;
      t = make_int4(lo, at, min(p.BM, start[lo + 1] - at), 0);
    }
    p.tiles[i] = t;
  }
}

// rows of bf16 that no 16-byte load can take as they are: copied once, filled
// up with zeros to whole steps
__global__ __launch_bounds__(256) void pad_rows_kernel(
    const __bf16* __restrict__ X, int64_t ldx, int D, __bf16* __restrict__ Y,
    int Dp, int64_t n) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= n) return;
  const int64_t t = i / Dp;
  const int c = (int)(i - t * Dp);
  Y[i] = c < D ? X[t * ldx + c] : (__bf16)0.f;
}

// ------------------------------------------------------ grouped products

struct Experts {
  const int4* tiles;
  const int* order;
  int k, N, n_tiles, tiles_n;
  const uint8_t* A;  // rows by token (first product) or by place (second)
  const float* SA;   // [steps][rows]
  uint32_t a_bytes, sa_rows;
  int64_t a_row;     // bytes from row to row
  const uint8_t* B;  // [E][n][steps * 128 bytes]
  const float* SB;   // [E][ceil(n / 128)][steps]
  const float* bias;  // [E][n]
  int n, np, steps, act;
  void* H;            // first: [N][np] bf16 or e4m3
  float* SH;          // first: [np / 128][N]
  const float* w;     // second: [N] by assignment
  float* Y;           // second: [N][n] by assignment
};

// The rows of one tile, all of one expert, times its weights. FIRST: rows are
// gathered by token, the result is activated, rounded to the layer's type and
// kept in the order of the experts. Otherwise: rows as they lie, the result
// is weighted and goes to its assignment's place, in f32.
template <class S, bool FIRST>
__global__ __launch_bounds__(S::THREADS, 2) void experts_kernel(Experts p) {
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const Place at_tile = place_of(blockIdx.x, p.n_tiles, p.tiles_n);
  const int4 tile = p.tiles[at_tile.m];
  const int e = __builtin_amdgcn_readfirstlane(tile.x);
  if (e < 0) return;
  const int at0 = __builtin_amdgcn_readfirstlane(tile.y);
  const int rows = __builtin_amdgcn_readfirstlane(tile.z);
  const int n0 = at_tile.n * S::BN;
  const int64_t b_row = (int64_t)p.steps * STEP;
  const int blocks_n = (p.n + 127) / 128;

  // at least 1: no tile consists of columns alone that only fill up H, as BN
  // is a multiple of what H is filled up to
  const int cols = min(S::BN, p.n - n0);
  const auto rb = buffer(p.B + ((int64_t)e * p.n + n0) * b_row,
                         (uint32_t)(cols * b_row));
  const auto ra = FIRST ? buffer(p.A, p.a_bytes)
                        : buffer(p.A + at0 * p.a_row,
                                 (uint32_t)(rows * p.a_row));
  const auto rs = buffer(p.SA, p.sa_rows * 4 * p.steps);
  // the row of A and SA behind row r of the tile
  auto place = [&](int r) {
    r = min(r, rows - 1);
    return FIRST ? p.order[at0 + r] / p.k : r;
  };
  const Rows<S> at = rows_of<S>(
      wave, lane, [&](int r) { return (uint32_t)(place(r) * p.a_row); },
      [&](int r) { return (uint32_t)(min(r, cols - 1) * b_row); },
      [&](int r) { return (uint32_t)(place(r) + (FIRST ? 0 : at0)) * 4; });
  const int wm = wave / S::WN, wn = wave % S::WN;
  const int wave_n0 = n0 + wn * S::NT * 16;
  f32x4 acc[S::MT][S::NT];
  product<S>(smem, ra, rb, rs, at, 0, p.steps, p.sa_rows * 4,
             S::FP8 ? p.SB + ((int64_t)e * blocks_n +
                              min(wave_n0 / 128, blocks_n - 1)) * p.steps
                    : nullptr,
             wave, lane, acc);

  const float* bias = p.bias ? p.bias + (int64_t)e * p.n : nullptr;
  auto row = [&](int i) { return wm * S::MT * 16 + i * 16 + (lane & 15); };
  auto column = [&](int q) { return wave_n0 + run_column<S>(q, lane); };
  auto load_bias = [&](int q, float(&b)[S::W]) {
    load_run(bias + column(q), bias ? p.n - column(q) : 0, b);
  };

  if constexpr (FIRST) {
    // activated in place; the columns that only fill up H stay 0
#pragma unroll
    for (int q = 0; q < S::RUNS; ++q) {
      float b[S::W];
      load_bias(q, b);
#pragma unroll
      for (int i = 0; i < S::MT; ++i) {
        float v[S::W];
        run_of<S>(acc[i], q, v);
#pragma unroll
        for (int c = 0; c < S::W; ++c) v[c] += b[c];
        activate_by(v, p.act);
#pragma unroll
        for (int c = 0; c < S::W; ++c)
          acc[i][q * (S::W / 4) + c / 4][c % 4] =
              column(q) + c < p.n ? v[c] : 0.f;
      }
    }
  }
  if constexpr (FIRST && S::FP8) {
    // a block of 128 columns is spread over SHARE waves: each leaves the
    // largest value of its rows in LDS
    constexpr int SHARE = 128 / (S::NT * 16);
    uint32_t* top = (uint32_t*)smem;  // [WN][BM]
    __syncthreads();
#pragma unroll
    for (int i = 0; i < S::MT; ++i) {
      uint32_t m = 0;
#pragma unroll
      for (int q = 0; q < S::RUNS; ++q) {
        float v[S::W];
        run_of<S>(acc[i], q, v);
        m = max(m, amax_bits(v));
      }
      m = max(m, (uint32_t)__shfl_xor((int)m, 16));
      m = max(m, (uint32_t)__shfl_xor((int)m, 32));
      if (lane < 16) top[wn * S::BM + row(i)] = m;
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < S::MT; ++i) {
      const int r = row(i);
      uint32_t m = 0;
#pragma unroll
      for (int w = 0; w < SHARE; ++w)
        m = max(m, top[(wn / SHARE * SHARE + w) * S::BM + r]);
      if (r >= rows || wave_n0 >= p.np) continue;
      const float s = scale_of(m);
#pragma unroll
      for (int q = 0; q < S::RUNS; ++q) {
        float v[S::W];
        run_of<S>(acc[i], q, v);
        uint2 h[S::W / 8];
#pragma unroll
        for (int c = 0; c < S::W / 8; ++c) {
          float u[8];
#pragma unroll
          for (int j = 0; j < 8; ++j) u[j] = v[c * 8 + j];
          h[c] = to_fp8(u, s);
        }
        uint8_t* to = (uint8_t*)p.H + (int64_t)(at0 + r) * p.np + column(q);
        __builtin_memcpy(__builtin_assume_aligned(to, sizeof(h)), h,
                         sizeof(h));
      }
      if (lane < 16 && wn % SHARE == 0)
        p.SH[(int64_t)(wave_n0 / 128) * p.N + at0 + r] = s;
    }
  } else if constexpr (FIRST) {
#pragma unroll
    for (int q = 0; q < S::RUNS; ++q)
#pragma unroll
      for (int i = 0; i < S::MT; ++i) {
        if (row(i) >= rows || column(q) >= p.np) continue;
        float v[S::W];
        run_of<S>(acc[i], q, v);
        // rounded to bf16 here: the second product takes no wider operand
        __bf16 t[S::W];
#pragma unroll
        for (int c = 0; c < S::W; ++c) t[c] = (__bf16)v[c];
        __bf16* h =
            (__bf16*)p.H + (int64_t)(at0 + row(i)) * p.np + column(q);
        __builtin_memcpy(__builtin_assume_aligned(h, 16), t, sizeof(t));
      }
  } else {
#pragma unroll
    for (int i = 0; i < S::MT; ++i) {
      if (row(i) >= rows) continue;
      const int a = p.order[at0 + row(i)];
      const float w = p.w[a];
#pragma unroll
      for (int q = 0; q < S::RUNS; ++q) {
        float v[S::W], b[S::W];
        load_bias(q, b);
        run_of<S>(acc[i], q, v);
#pragma unroll
        for (int c = 0; c < S::W; ++c) v[c] = (v[c] + b[c]) * w;
        store_run(p.Y + (int64_t)a * p.n + column(q), p.n - column(q), v);
      }
    }
  }
}

// each token adds up its experts' rows, in the order of its list
__global__ __launch_bounds__(256) void combine_kernel(
    const float* __restrict__ P, const int* __restrict__ ids, int E, int k,
    int D, const __bf16* residual, int64_t ldr, __bf16* Y, int64_t ldy,
    int64_t n) {
  const int per = (D + 3) / 4;
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= n) return;
  const int64_t t = i / per;
  const int c = (int)(i - t * per) * 4;
  const int have = min(4, D - c);
  float v[4] = {0.f, 0.f, 0.f, 0.f};
  for (int j = 0; j < k; ++j) {
    if ((unsigned)ids[t * k + j] >= (unsigned)E) continue;
    const float* y = P + (t * k + j) * D + c;
    if (have == 4) {
      float u[4];
      __builtin_memcpy(u, y, sizeof(u));
#pragma unroll
      for (int q = 0; q < 4; ++q) v[q] += u[q];
    } else {
      for (int q = 0; q < have; ++q) v[q] += y[q];
    }
  }
  for (int q = 0; q < have; ++q) {
    if (residual) v[q] += (float)residual[t * ldr + c + q];
    Y[t * ldy + c + q] = (__bf16)v[q];
  }
}

template <bool FP8, bool FIRST>
using Tile = Shape<FP8, 128, 128, 2, 2, 2, FIRST ? (FP8 ? 16 : 8) : 4>;

template <class S, bool FIRST>
void run(Experts p, hipStream_t stream) {
  p.tiles_n = up(FIRST ? p.np : p.n, S::BN);
  hipLaunchKernelGGL((experts_kernel<S, FIRST>), dim3(p.n_tiles * p.tiles_n),
                     dim3(S::THREADS), S::LDS, stream, p);
}

int64_t up256(int64_t bytes) { return (bytes + 255) & ~int64_t(255); }

// where a call's intermediate data lie
struct Layout {
  int64_t counts, order, tiles, x, sx, h, sh, y, bytes;
  int n_tiles, blocks, BM, Dp, Hp;
  bool copy;  // the rows of x are brought into whole steps first
};

Layout layout(const MoeMlp& m) {
  Layout l{};
  const int64_t N = (int64_t)m.T * m.k;
  l.BM = 128;
  l.n_tiles = (int)(N / l.BM + std::min<int64_t>(N, m.E));
  l.blocks = up(N, PLAN_ROWS);
  const int unit = m.fp8 ? 128 : 64, size = m.fp8 ? 1 : 2;
  l.Dp = up(m.D, unit) * unit;
  l.Hp = up(m.H, unit) * unit;
  l.copy = m.fp8 || m.D != l.Dp || m.ldx % 8 || (uintptr_t)m.X % 16 ||
           (m.T - 1) * m.ldx * 2 + l.Dp * 2 > UINT32_MAX;
  int64_t at = 0;
  auto take = [&](int64_t bytes) {
    const int64_t was = at;
    at += up256(bytes);
    return was;
  };
  l.counts = take(l.blocks > 1 ? (int64_t)l.blocks * m.E * 4 : 0);
  l.order = take(N * 4);
  l.tiles = take((int64_t)l.n_tiles * 16);
  l.x = take(l.copy ? (int64_t)m.T * l.Dp * size : 0);
  l.sx = take(m.fp8 ? (int64_t)m.T * (l.Dp / 128) * 4 : 0);
  l.h = take(N * l.Hp * size);
  l.sh = take(m.fp8 ? N * (l.Hp / 128) * 4 : 0);
  l.y = take(N * m.D * 4);
  l.bytes = at;
  return l;
}

template <bool FP8>
void run_mlp(const MoeMlp& m, const Layout& l, char* ws, hipStream_t stream) {
  const int N = m.T * m.k;
  Plan plan{m.ids, (int*)(ws + l.counts), (int*)(ws + l.order),
            (int4*)(ws + l.tiles), N, m.E, l.BM, l.n_tiles, l.blocks};
  if (l.blocks > 1)
    hipLaunchKernelGGL(plan_count_kernel, dim3(l.blocks), dim3(PLAN_THREADS),
                       m.E * 4, stream, plan);
  hipLaunchKernelGGL(plan_place_kernel, dim3(l.blocks), dim3(PLAN_THREADS),
                     (4 * m.E + 2) * 4, stream, plan);

  Experts p{};
  p.tiles = plan.tiles;
  p.order = plan.order;
  p.k = m.k;
  p.N = N;
  p.n_tiles = l.n_tiles;
  const int size = FP8 ? 1 : 2;
  if (FP8)
    launch_quant_fp8(m.X, false, m.ldx, m.T, m.D, ws + l.x, l.Dp,
                     (float*)(ws + l.sx), 1, stream);
  else if (l.copy)
    hipLaunchKernelGGL(pad_rows_kernel, dim3(up((int64_t)m.T * l.Dp, 256)),
                       dim3(256), 0, stream, (const __bf16*)m.X, m.ldx, m.D,
                       (__bf16*)(ws + l.x), l.Dp, (int64_t)m.T * l.Dp);
  p.A = l.copy ? (const uint8_t*)ws + l.x : (const uint8_t*)m.X;
  p.a_row = l.copy ? (int64_t)l.Dp * size : m.ldx * 2;
  p.a_bytes = (uint32_t)((m.T - 1) * p.a_row + (int64_t)l.Dp * size);
  p.SA = (const float*)(ws + l.sx);
  p.sa_rows = m.T;
  p.B = (const uint8_t*)m.W1;
  p.SB = m.S1;
  p.bias = m.b1;
  p.n = m.H;
  p.np = l.Hp;
  p.steps = l.Dp * size / STEP;
  p.act = m.act;
  p.H = ws + l.h;
  p.SH = (float*)(ws + l.sh);
  run<Tile<FP8, true>, true>(p, stream);

  p.A = (const uint8_t*)ws + l.h;
  p.a_row = (int64_t)l.Hp * size;
  p.SA = p.SH;
  p.sa_rows = N;
  p.B = (const uint8_t*)m.W2;
  p.SB = m.S2;
  p.bias = m.b2;
  p.n = p.np = m.D;
  p.steps = l.Hp * size / STEP;
  p.w = m.weights;
  p.Y = (float*)(ws + l.y);
  run<Tile<FP8, false>, false>(p, stream);

  const int64_t work = (int64_t)m.T * ((m.D + 3) / 4);
  hipLaunchKernelGGL(combine_kernel, dim3(up(work, 256)), dim3(256), 0, stream,
                     p.Y, m.ids, m.E, m.k, m.D, (const __bf16*)m.residual,
                     m.ldr, (__bf16*)m.Y, m.ldy, work);
}

}  // namespace

void launch_moe_route(const void* X, bool f32, int64_t ldx, const float* bias,
                      int* ids, float* weights, int T, int E, int k,
                      bool sigmoid, int groups, int kept, int best,
                      bool renorm, float scale, hipStream_t stream) {
  const Route p{X, bias, ids, weights, ldx, T, E, k, groups, kept, best,
                sigmoid, renorm, scale};
  const dim3 grid(up(T, 4));
  const int lds = 4 * E * 8;
  auto go = [&](auto x) {
    using V = decltype(x);
    if (E <= 64)
      hipLaunchKernelGGL((route_kernel<V, 1>), grid, dim3(256), lds, stream, p);
    else if (E <= 128)
      hipLaunchKernelGGL((route_kernel<V, 2>), grid, dim3(256), lds, stream, p);
    else if (E <= 256)
      hipLaunchKernelGGL((route_kernel<V, 4>), grid, dim3(256), lds, stream, p);
    else
      hipLaunchKernelGGL((route_kernel<V, 8>), grid, dim3(256), lds, stream, p);
  };
  if (f32)
    go(0.f);
  else
    go((__bf16)0.f);
}

int64_t moe_mlp_workspace(const MoeMlp& m) { return layout(m).bytes; }

void launch_moe_mlp(const MoeMlp& m, void* ws, hipStream_t stream) {
  const Layout l = layout(m);
  if (m.fp8)
    run_mlp<true>(m, l, (char*)ws, stream);
  else
    run_mlp<false>(m, l, (char*)ws, stream);
}
