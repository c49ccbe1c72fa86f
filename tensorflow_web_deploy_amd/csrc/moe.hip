// Mixture-of-experts layers.
//   moe_logits logits = x W^T, W in f32
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
#include <cmath>
#include <cstdint>
#include <type_traits>

#include "kernels.h"
#include "quant_fp8.h"
#include "tile_gemm.h"

namespace {

using namespace tile;

int up(int64_t a, int64_t b) { return (int)((a + b - 1) / b); }

// ----------------------------------------------------------- moe_logits

struct Logits {
  const __bf16 *X, *W;  // W: [3][E][Dp], the parts of each weight
  float* Y;
  int64_t ldx;
  int T, D, Dp, E;
};

// 8 values of a row from p on, the ones from `have` on as 0; rows may start
// anywhere
__device__ __forceinline__ bf16x8 row8(const __bf16* p, int have) {
  bf16x8 r;
  if (have >= 8) {
    __builtin_memcpy(&r, p, sizeof(r));
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) r[e] = e < have ? p[e] : (__bf16)0.f;
  }
  return r;
}

// The router's product. Two logits that are close decide which expert runs, so
// neither the weights nor the result are rounded to bf16: each weight is the
// sum of three bf16 numbers, whose products with x are exact in f32, and a
// matrix instruction more for each costs little beside the loads. A wave takes
// RT x NT tiles of 16 rows and 16 experts, KS of them share K. The two small
// parts are summed apart: with an infinite value of x they, being 0 as a rule,
// would make NaN of it. Bound by how long its loads from the L2 take: 196 x
// 768, 64 experts 4.8 us, 12544 x 768, 64 19 (0.2 PFLOP/s of its instructions);
// the product into bf16 takes 14 and 23.
template <int RT, int NT, int KS>
__global__ __launch_bounds__(512) void logits_kernel(Logits p) {
  __shared__ __attribute__((aligned(16))) float part[KS > 1 ? 2 * 8 * 256 : 1];
  const int lane = threadIdx.x & 63, l = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int tiles_n = (p.E + NT * 16 - 1) / (NT * 16);
  const int64_t rows = blockIdx.x / tiles_n;
  const int n0 = (int)(blockIdx.x - rows * tiles_n) * NT * 16;
  const int ks = wave % KS;
  const int64_t m0 = (rows * (8 / KS) + wave / KS) * RT * 16;
  f32x4 acc[RT][NT] = {}, rest[RT][NT] = {};
  const __bf16 *x[RT], *w[NT];
#pragma unroll
  for (int i = 0; i < RT; ++i)
    x[i] = p.X + min(m0 + i * 16 + l, (int64_t)p.T - 1) * p.ldx;
#pragma unroll
  for (int t = 0; t < NT; ++t)
    w[t] = p.W + (int64_t)min(n0 + t * 16 + l, p.E - 1) * p.Dp;
  const int64_t next = (int64_t)p.E * p.Dp;
  const int steps = m0 < p.T ? p.Dp / 32 : 0;
#pragma unroll 2
  for (int s = steps * ks / KS; s < steps * (ks + 1) / KS; ++s) {
    const int k = s * 32 + g * 8;
    bf16x8 a[RT], b[NT][3];
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int j = 0; j < 3; ++j)
        b[t][j] = *(const bf16x8*)(w[t] + j * next + k);
#pragma unroll
    for (int i = 0; i < RT; ++i) a[i] = row8(x[i] + k, p.D - k);
#pragma unroll
    for (int i = 0; i < RT; ++i)
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        acc[i][t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
            b[t][0], a[i], acc[i][t], 0, 0, 0);
        rest[i][t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
            b[t][2], a[i], rest[i][t], 0, 0, 0);
        rest[i][t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
            b[t][1], a[i], rest[i][t], 0, 0, 0);
      }
  }
#pragma unroll
  for (int i = 0; i < RT; ++i)
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      if (KS > 1 && (i || t)) __syncthreads();  // the last sum has been read
      const f32x4 sum = few_join<KS>(acc[i][t], part, wave / KS, ks, lane);
      const f32x4 more =
          few_join<KS>(rest[i][t], part + 8 * 256, wave / KS, ks, lane);
      const int64_t m = m0 + i * 16 + l;
      const int n = n0 + t * 16 + g * 4;
      if (ks || m >= p.T) continue;
      float v[4];
#pragma unroll
      for (int c = 0; c < 4; ++c)
        v[c] = fabsf(sum[c]) < INFINITY ? sum[c] + more[c] : sum[c];
      store_run(p.Y + m * p.E + n, p.E - n, v);
    }
}

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

// How far the f32 score p and key = p + bias may be off. exp's argument d is
// rounded three times, which moves exp by 3 * 2^-24 |d| of itself. Softmax:
// |d| is no more than |ln p|; the sum of up to 512 terms in 32 + 4 steps, the
// terms' own errors in it, exp and the quotient stay within 64 * 2^-24.
// Sigmoid: exp counts by 1 - p, |d| (1 - p) is less than |ln p| + 1, and 8
// roundings cover the rest. Adding the bias rounds the key.
__device__ __forceinline__ float error_of(float p, float key, bool sigmoid) {
  const float d = fabsf(__builtin_amdgcn_logf(fmaxf(p, 1e-37f)));  // log2
  return 0x1p-24f * ((sigmoid ? 8.f : 64.f) + 2.1f * d) * p +
         0x1p-23f * fabsf(key) + 1e-37f;
}

// The largest value, the sum, .. of 16 neighbouring lanes, in all of them
template <int ROR>
__device__ __forceinline__ float turned(float v) {
  static_assert(ROR > 0 && ROR < 16);
  return __builtin_bit_cast(
      float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v),
                                         0x120 + ROR, 0xf, 0xf, true));
}
__device__ __forceinline__ float max16(float v) {
  v = fmaxf(v, turned<8>(v));
  v = fmaxf(v, turned<4>(v));
  v = fmaxf(v, turned<2>(v));
  return fmaxf(v, turned<1>(v));
}
__device__ __forceinline__ float sum16(float v) {
  v += turned<8>(v);
  v += turned<4>(v);
  v += turned<2>(v);
  return v + turned<1>(v);
}

// Between what lanes of a wave write to LDS and what others read of it: the
// hardware keeps the order, the compiler has to be told to.
__device__ __forceinline__ void wave_turn() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// what the lanes before this one of its 16 add up to
template <int SHR>
__device__ __forceinline__ int shifted(int v) {
  return __builtin_amdgcn_update_dpp(0, v, 0x110 + SHR, 0xf, 0xf, true);
}
__device__ __forceinline__ int before16(int v) {
  int s = v + shifted<1>(v);
  s += shifted<2>(s);
  s += shifted<4>(s);
  s += shifted<8>(s);
  return s - v;
}

// how many of the other 15 lanes hold a larger number
template <int R = 1>
__device__ __forceinline__ int above16(float v) {
  if constexpr (R == 16)
    return 0;
  else
    return (turned<R>(v) > v) + above16<R + 1>(v);
}

// how many of the 16 lanes' (o, oid) come before (v, id): a larger number, or
// the same one with a smaller id
template <int R = 0>
__device__ __forceinline__ int rank16(float v, float id, float o, float oid) {
  if constexpr (R == 16) {
    return 0;
  } else {
    float u = o, uid = oid;
    if constexpr (R > 0) u = turned<R>(o), uid = turned<R>(oid);
    return (u > v || (u == v && uid < id)) + rank16<R + 1>(v, id, o, oid);
  }
}

// The largest of a wave's numbers, one that is uniform over the wave
template <int CTRL, int ROWS>
__device__ __forceinline__ double moved(double v) {
  const int2 u = __builtin_bit_cast(int2, v);
  return __builtin_bit_cast(
      double, make_int2(__builtin_amdgcn_update_dpp(u.x, u.x, CTRL, ROWS, 0xf,
                                                    false),
                        __builtin_amdgcn_update_dpp(u.y, u.y, CTRL, ROWS, 0xf,
                                                    false)));
}
__device__ __forceinline__ double lane_of(double v, int lane) {
  const int2 u = __builtin_bit_cast(int2, v);
  return __builtin_bit_cast(
      double, make_int2(__builtin_amdgcn_readlane(u.x, lane),
                        __builtin_amdgcn_readlane(u.y, lane)));
}
__device__ __forceinline__ double wave_max(double v) {
  v = fmax(v, moved<0x128, 0xf>(v));  // within rows of 16: row_ror 8, 4, 2, 1
  v = fmax(v, moved<0x124, 0xf>(v));
  v = fmax(v, moved<0x122, 0xf>(v));
  v = fmax(v, moved<0x121, 0xf>(v));
  return fmax(fmax(lane_of(v, 0), lane_of(v, 16)),
              fmax(lane_of(v, 32), lane_of(v, 48)));
}

// One row by one wave in 64 bits, lane l with the experts l + 64 v
template <typename T, int V>
__device__ __forceinline__ void route_exactly(const Route& p, int64_t t,
                                              double* lds, int lane) {
  const double NONE = -INFINITY;
  float x[V];
  double s[V], key[V];
  float top = -INFINITY;
#pragma unroll
  for (int v = 0; v < V; ++v) {
    const int e = v * 64 + lane;
    x[v] = e < p.E ? (float)((const T*)p.x)[t * p.ldx + e] : -INFINITY;
    if (!(x[v] > -INFINITY)) x[v] = -INFINITY;
    top = fmaxf(top, x[v]);
  }
  if (p.sigmoid) {
#pragma unroll
    for (int v = 0; v < V; ++v)
      s[v] = x[v] > -INFINITY ? 1 / (1 + exp(-(double)x[v])) : 0;
  } else {
    top = (float)wave_max((double)top);
    double sum = 0;
#pragma unroll
    for (int v = 0; v < V; ++v) {
      // an infinite logit leaves nothing to the finite ones
      s[v] = x[v] == top ? 1 : exp((double)x[v] - (double)top);
      if (!(x[v] > -INFINITY)) s[v] = 0;
      sum += s[v];
    }
#pragma unroll
    for (int d = 32; d; d >>= 1) sum += __shfl_xor(sum, d);
#pragma unroll
    for (int v = 0; v < V; ++v) s[v] = sum > 0 ? s[v] / sum : 0;
  }
#pragma unroll
  for (int v = 0; v < V; ++v) {
    const int e = v * 64 + lane;
    key[v] = s[v] + (e < p.E && p.bias ? (double)p.bias[e] : 0);
    if (!(x[v] > -INFINITY) || !(key[v] > NONE)) key[v] = NONE;
  }
  if (p.groups > 1) {
    const int size = p.E / p.groups;
#pragma unroll
    for (int v = 0; v < V; ++v)
      if (v * 64 + lane < p.E) lds[v * 64 + lane] = key[v];
    wave_turn();
    double first = NONE, second = NONE;
    if (lane < p.groups) {
#pragma unroll 4
      for (int i = 0; i < size; ++i) {
        const double y = lds[lane * size + i];
        second = fmax(second, fmin(first, y));
        first = fmax(first, y);
      }
    }
    const double total =
        p.best == 2 && second > NONE ? first + second : first;
    int rank = 0;
    for (int g = 0; g < p.groups; ++g) {
      const double o = lane_of(total, g);
      rank += o > total || (o == total && g < lane);
    }
    const uint64_t kept = __ballot(lane < p.groups && rank < p.kept);
#pragma unroll
    for (int v = 0; v < V; ++v)
      if (!(kept >> ((v * 64 + lane) / size & 63) & 1)) key[v] = NONE;
  }
  double mine = 0, sum = 0;
  int id = -1;
  for (int j = 0; j < p.k; ++j) {
    double best = key[0];
#pragma unroll
    for (int v = 1; v < V; ++v) best = fmax(best, key[v]);
    best = wave_max(best);
    if (!(best > NONE)) break;
    double sv = 0;
    bool found = false;
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const uint64_t has = __ballot(key[v] == best);
      if (found || !has) continue;
      found = true;
      const int at = __builtin_ctzll(has);
      sv = lane_of(s[v], at);
      if (lane == at) key[v] = NONE;
      if (lane == j) mine = sv, id = v * 64 + at;
    }
    sum += sv;
  }
  if (lane < p.k) {
    if (p.renorm) mine = sum > 0 ? mine / sum : 0;
    p.ids[t * p.k + lane] = id;
    p.weights[t * p.k + lane] = (float)(mine * p.scale);
  }
}

// LDS of one row in f32: the scores, the keys (with groups), what the groups
// come to and the size of its parts, and the chosen ones
struct RouteLds {
  int p, key, total, round, list, floats;
  __host__ __device__ RouteLds(int V, int groups, int k) {
    p = 0;
    key = 16 * V;
    total = key + (groups > 1 ? 16 * V : 0);
    round = total + (groups > 1 ? groups : 0);
    list = (round + (groups > 1 ? groups : 0) + 1) & ~1;
    floats = (list + 2 * (k < 32 ? 32 : k + 1) + 3) & ~3;
  }
};

// Expert of a lane's place v: runs of 4 neighbours a lane (V >= 4), 64 a turn,
// so that each lane has some of every group of experts that is wide
template <int V>
__device__ __forceinline__ int expert_at(int l, int v) {
  return V >= 4 ? v / 4 * 64 + l * 4 + v % 4 : l;
}

// 16 lanes a row, 4 rows a wave: the steps across lanes stay within rows of
// the register file, and one instruction serves 4 rows (a wave a row took 47
// us where this takes 15). Everything is decided in f32; a row where rounding
// could change what is chosen or its order, or whose scores leave the range of
// f32, is then done again in 64 bits, so that the choice is that of the scores
// in 64 bits, the lower index first among equals. That is one row in some
// hundreds, unless logits repeat a lot. 12544 rows of 256 f32, 8 out of 4 of 8
// groups: 14.2 to 15.9 us, of which the rows in 64 bits take 2.5 at the end;
// bound by the VALU, busy for 63% of the cycles with 1250 instructions for 4
// rows.
template <typename T, int V>
__global__ __launch_bounds__(256) void route_kernel(Route p) {
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const float NONE = -INFINITY;
  const RouteLds at(V, p.groups, p.k);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int l = lane & 15;
  const int64_t t0 = ((int64_t)blockIdx.x * 4 + wave) * 4;
  if (t0 >= p.T) return;
  const int64_t t = t0 + (lane >> 4);
  float* wave_lds = (float*)smem + wave * 4 * at.floats;
  float* lds = wave_lds + (lane >> 4) * at.floats;
  constexpr int RUN = V >= 4 ? 4 : 1;
  const int E = t < p.T ? p.E : 0;

  float s[V], key[V];
#pragma unroll
  for (int v = 0; v < V; v += RUN) {
    const int e = expert_at<V>(l, v);
    const T* x = (const T*)p.x + (t < p.T ? t : t0) * p.ldx + e;
    if (e + RUN <= E) {
      T u[RUN];
      __builtin_memcpy(u, x, sizeof(u));
#pragma unroll
      for (int i = 0; i < RUN; ++i) key[v + i] = (float)u[i];
    } else {
#pragma unroll
      for (int i = 0; i < RUN; ++i)
        key[v + i] = e + i < E ? (float)x[i] : NONE;
    }
  }
#pragma unroll
  for (int v = 0; v < V; ++v)
    if (!(key[v] > NONE)) key[v] = NONE;  // NaN: not to be chosen
  auto to_lds = [&](int where, const float(&y)[V]) {
#pragma unroll
    for (int v = 0; v < V; v += RUN)
      __builtin_memcpy(__builtin_assume_aligned(
                           lds + where + expert_at<V>(l, v), RUN * 4),
                       y + v, RUN * 4);
  };
  constexpr float LOG2E = 1.44269504f;
  float most = 1.f;  // no score is larger
  if (p.sigmoid) {
#pragma unroll
    for (int v = 0; v < V; ++v)
      s[v] = __builtin_amdgcn_rcpf(
          1.f + __builtin_amdgcn_exp2f(key[v] * -LOG2E));
  } else {
    float top = key[0], sum = 0;
#pragma unroll
    for (int v = 1; v < V; ++v) top = fmaxf(top, key[v]);
    top = max16(top);
#pragma unroll
    for (int v = 0; v < V; ++v) {
      // an infinite logit leaves nothing to the finite ones
      s[v] = key[v] == top ? 1.f
                           : __builtin_amdgcn_exp2f((key[v] - top) * LOG2E);
      if (!(key[v] > NONE)) s[v] = 0.f;
      sum += s[v];
    }
    sum = 1.f / sum16(sum);
    most = fminf(sum, 1.f);
#pragma unroll
    for (int v = 0; v < V; ++v) s[v] = key[v] > NONE ? s[v] * sum : 0.f;
  }
  to_lds(at.p, s);
  if (p.bias) {
#pragma unroll
    for (int v = 0; v < V; v += RUN) {
      const int e = expert_at<V>(l, v);
      float b[RUN];
      load_run(p.bias + e, E - e, b);
#pragma unroll
      for (int i = 0; i < RUN; ++i) {
        const float y = s[v + i] + b[i];
        key[v + i] = key[v + i] > NONE && y > NONE ? y : NONE;
      }
    }
  } else {
#pragma unroll
    for (int v = 0; v < V; ++v) key[v] = key[v] > NONE ? s[v] : NONE;
  }
  bool safe = true;

  if (p.groups > 1) {
    const int size = p.E / p.groups;
    to_lds(at.key, key);
    wave_turn();
    // no group's sum is off by more than two of the largest score could be
    const float err = 2 * error_of(most, 0.f, p.sigmoid);
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int g = q * 16 + l;
      if (g >= p.groups) break;
      float first = NONE, second = NONE;
      auto see = [&](float y) {
        second = fmaxf(second, fminf(first, y));
        first = fmaxf(first, y);
      };
      const float* in = lds + at.key + g * size;
      if (V >= 4 && size % 4 == 0) {
        int j = l * 4 % size;  // spread over banks
#pragma unroll 4
        for (int i = 0; i < size; i += 4) {
          f32x4 y;
          __builtin_memcpy(&y, __builtin_assume_aligned(in + j, 16), 16);
#pragma unroll
          for (int u = 0; u < 4; ++u) see(y[u]);
          j = j + 4 == size ? 0 : j + 4;
        }
      } else {
        int j = l % size;
#pragma unroll 4
        for (int i = 0; i < size; ++i) {
          see(in[j]);
          j = j + 1 == size ? 0 : j + 1;
        }
      }
      lds[at.total + g] = p.best == 2 && second > NONE ? first + second : first;
      lds[at.round + g] =
          fabsf(first) + (second > NONE ? fabsf(second) : 0.f);
    }
    wave_turn();
    float low = INFINITY, high = NONE;
    uint64_t kept = 0;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int g = q * 16 + l;
      if (q * 16 >= p.groups) break;
      bool keep = false;
      if (g < p.groups) {
        const float total = lds[at.total + g];
        int rank = 0;
#pragma unroll 8
        for (int h = 0; h < p.groups; ++h) {
          const float o = lds[at.total + h];
          rank += o > total || (o == total && h < g);
        }
        keep = rank < p.kept;
        // the last group that is kept against the first that isn't; one
        // without any expert left doesn't matter
        const float e = err + 0x1p-22f * lds[at.round + g];
        if (total > NONE) {
          if (keep)
            low = fminf(low, total - e);
          else
            high = fmaxf(high, total + e);
        }
      }
      kept |= (__ballot(keep) >> (lane & 48) & 0xffff) << (16 * q);
    }
    safe = !(-max16(-low) <= max16(high));
    const uint32_t over = (1u << 20) / size + 1;  // e / size for e < 512
#pragma unroll
    for (int v = 0; v < V; ++v)
      if (!(kept >> (min(expert_at<V>(l, v), p.E - 1) * over >> 20) & 1))
        key[v] = NONE;
  }

  // The k largest keys, and the one that just fails, into a list. Each lane's
  // own largest key counts: where k + 1 lanes reach a bound, no key below it
  // can be wanted. For 8 of 256 that leaves some 13 keys; with up to 32, two a
  // lane, each finds its place by itself. For 12544 rows of 256 that and the
  // largest key k + 1 times take, in us: k = 2: 7.7 / 7.6, 4: 8.2 / 9.2,
  // 8: 11.4 / 14.0, 12: 16.3 / 17.3, 15: 20.7 / 19.7; of 16 or 64, k = 2:
  // 4.8 / 4.1, 5.7 / 5.5, k = 12: 7.5 / 9.1, 9.5 / 10.2.
  int2* list = (int2*)(lds + at.list);
  bool few = p.k > 2 && p.k < 14;
  if (few) {
    float own = key[0];
#pragma unroll
    for (int v = 1; v < V; ++v) own = fmaxf(own, key[v]);
    const float bound =
        -max16(above16(own) <= p.k ? -own : NONE);
    int count = 0;
#pragma unroll
    for (int v = 0; v < V; ++v) count += key[v] >= bound && key[v] > NONE;
    int to = before16(count);
    few = !__any(to + count > 32);
    const bool two = __any(to + count > 16);
    if (few) {
      const int2 none = make_int2(-1, __builtin_bit_cast(int, NONE));
      list[l] = none;
      if (two) list[l + 16] = none;
      wave_turn();
#pragma unroll
      for (int v = 0; v < V; ++v)
        if (key[v] >= bound && key[v] > NONE)
          list[to++] = make_int2(expert_at<V>(l, v),
                                 __builtin_bit_cast(int, key[v]));
      wave_turn();
      // places that hold nothing come last, each at its own
      const int2 a = list[l];
      const float ka = __builtin_bit_cast(float, a.y);
      const float ia = a.x < 0 ? 1024.f + l : (float)a.x;
      int rank = rank16(ka, ia, ka, ia);
      if (two) {
        const int2 b = list[l + 16];
        const float kb = __builtin_bit_cast(float, b.y);
        const float ib = b.x < 0 ? 1040.f + l : (float)b.x;
        rank += rank16(ka, ia, kb, ib);
        const int other = rank16(kb, ib, kb, ib) + rank16(kb, ib, ka, ia);
        wave_turn();
        list[other] = b;
      }
      wave_turn();
      list[rank] = a;
    }
  }
  // else k times the largest key, and once more
  for (int j = 0; j <= p.k && !few; ++j) {
    float top = key[0];
#pragma unroll
    for (int v = 1; v < V; ++v) top = fmaxf(top, key[v]);
    top = max16(top);
    // the smallest index that has it
    int id = 1024;
#pragma unroll
    for (int v = V - 1; v >= 0; --v)
      if (key[v] == top) id = expert_at<V>(l, v);
    id = (int)-max16(-(float)id);
#pragma unroll
    for (int v = 0; v < V; ++v)
      if (expert_at<V>(l, v) == id) key[v] = NONE;
    if (l == 0)
      list[j] = make_int2(top > NONE ? id : -1, __builtin_bit_cast(int, top));
  }
  wave_turn();

  // equal logits and biases tie in any precision
  auto ties = [&](int a, int b) {
    const T* x = (const T*)p.x + t * p.ldx;
    return (float)x[a] == (float)x[b] && (!p.bias || p.bias[a] == p.bias[b]);
  };
  float w[4], sum = 0.f;
  int id[4];
  bool close = false;
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    const int j = q * 16 + l;
    id[q] = -1, w[q] = 0.f;
    if (j >= p.k) continue;
    const int2 a = list[j], b = list[j + 1];
    id[q] = a.x;
    if (a.x < 0) continue;
    w[q] = lds[at.p + a.x];
    sum += w[q];
    if (b.x < 0) continue;
    const float ka = __builtin_bit_cast(float, a.y);
    const float kb = __builtin_bit_cast(float, b.y);
    // Chosen keys that lie apart, each from the next, all lie above what the
    // last one may be at the least, and b, the largest that isn't chosen, below
    // it. So do the others where b would with the largest error that any of
    // them can have: that of the largest score, or, without a bias, b's own.
    const bool last = j + 1 == p.k;
    const float pb = last && p.bias ? most : lds[at.p + b.x];
    if (!(ka - kb >
          error_of(w[q], ka, p.sigmoid) + error_of(pb, kb, p.sigmoid))) {
      close = last;
      if (!ties(a.x, b.x)) safe = false;
    }
  }
  // Where b ties with the last one, each of the others has to lie below or tie.
  const uint64_t closely = __ballot(close && safe);
  if (closely >> (lane & 48) & 0xffff) {
    const int2 a = list[p.k - 1], b = list[p.k];
    const float ka = __builtin_bit_cast(float, a.y);
    const float low = ka - error_of(lds[at.p + a.x], ka, p.sigmoid);
    const float more =
        error_of(p.bias ? most : lds[at.p + b.x], 0.f, p.sigmoid);
#pragma unroll
    for (int v = 0; v < V; ++v) {
      // a list leaves the chosen keys in place, the other way takes them out
      const int e = expert_at<V>(l, v);
      const float y = key[v];
      if (y > NONE && !(y + 0x1p-23f * fabsf(y) + more < low) &&
          (y < ka || (y == ka && e > a.x)) && !ties(a.x, e))
        safe = false;
    }
  }
  sum = sum16(sum);
  if (p.renorm && id[0] >= 0 && !(sum > 1e-30f)) safe = false;
  const uint64_t unsafe = __ballot(!safe);
  const bool again = unsafe >> (lane & 48) & 0xffff;
  // of all the chosen: no more than 2^100, where the scale over the sum may
  // leave the range
  const float over = p.renorm ? (sum > 0.f ? 1.f / sum : 0.f) : 1.f;
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    const int j = q * 16 + l;
    if (j >= p.k || t >= p.T || again) continue;
    p.ids[t * p.k + j] = id[q];
    p.weights[t * p.k + j] = w[q] * over * p.scale;
  }
  if (!unsafe) return;
  // the rows of the wave are done with LDS: it now holds numbers of 64 bits
  wave_turn();
  for (int r = 0; r < 4; ++r)
    if (unsafe >> (16 * r) & 0xffff)
      route_exactly<T, (V + 3) / 4>(p, t0 + r, (double*)wave_lds, lane);
}

// ----------------------------------------------------------------- plan

constexpr int PLAN_THREADS = 256, PLAN_EACH = 8;
constexpr int PLAN_ROWS = PLAN_THREADS * PLAN_EACH;

struct Plan {
  const int* ids;
  int* counts;  // [blocks][E]: how many of a block's rows go to an expert
  int* order;   // [N]: the assignments, by expert; behind them nothing
  int4* tiles;  // {expert, first place in order, rows, 0}; [n_tiles].x: how
                // many there are
  int N, E, BM, n_tiles, blocks;
};

// the experts of the PLAN_EACH rows of a thread; one that isn't there is E
__device__ __forceinline__ void load_ids(const Plan& p, int a0,
                                         int (&e)[PLAN_EACH]) {
#pragma unroll
  for (int i = 0; i < PLAN_EACH; ++i) {
    const int a = a0 + i * PLAN_THREADS + threadIdx.x;
    e[i] = a < p.N ? p.ids[a] : p.E;
  }
#pragma unroll
  for (int i = 0; i < PLAN_EACH; ++i)
    if ((unsigned)e[i] >= (unsigned)p.E) e[i] = p.E;
}

__device__ __forceinline__ void plan_count(const Plan& p, int* count) {
  int e[PLAN_EACH];
  load_ids(p, blockIdx.x * PLAN_ROWS, e);
  for (int i = threadIdx.x; i < p.E; i += PLAN_THREADS) count[i] = 0;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < PLAN_EACH; ++i)
    if (e[i] < p.E) atomicAdd(&count[e[i]], 1);
  __syncthreads();
  for (int i = threadIdx.x; i < p.E; i += PLAN_THREADS)
    p.counts[blockIdx.x * p.E + i] = count[i];
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
__device__ __forceinline__ void plan_place(const Plan& p, int* lds) {
  int* total = lds;             // [E], later tiles of each expert
  int* next = lds + p.E;        // [E]
  int* start = lds + 2 * p.E;   // [E + 1]
  int* tile0 = lds + 3 * p.E + 1;  // [E + 1]
  int mine[PLAN_EACH];
  load_ids(p, blockIdx.x * PLAN_ROWS, mine);
  if (p.blocks == 1) {
    for (int e = threadIdx.x; e < p.E; e += PLAN_THREADS)
      total[e] = next[e] = 0;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < PLAN_EACH; ++i)
      if (mine[i] < p.E) atomicAdd(&total[mine[i]], 1);
  } else {
    for (int e = threadIdx.x; e < p.E; e += PLAN_THREADS) {
      int before = 0, sum = 0;
#pragma unroll 8
      for (int b = 0; b < p.blocks; ++b) {
        const int c = p.counts[b * p.E + e];
        before += b < (int)blockIdx.x ? c : 0;
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
    next[e] += start[e];
    total[e] = (total[e] + p.BM - 1) / p.BM;
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < PLAN_EACH; ++i)
    if (mine[i] < p.E)
      p.order[atomicAdd(&next[mine[i]], 1)] =
          blockIdx.x * PLAN_ROWS + i * PLAN_THREADS + threadIdx.x;
  if (blockIdx.x != 0) return;
  scan(total, tile0, p.E);
  __syncthreads();
  const int tiles = tile0[p.E];
  for (int i = threadIdx.x; i < tiles; i += PLAN_THREADS) {
    int lo = 0, hi = p.E;  // the expert with tile0[e] <= i < tile0[e + 1]
    while (hi - lo > 1) {
      const int mid = (lo + hi) / 2;
      if (tile0[mid] <= i)
        lo = mid;
      else
        hi = mid;
    }
    const int at = start[lo] + (i - tile0[lo]) * p.BM;
    p.tiles[i] = make_int4(lo, at, min(p.BM, start[lo + 1] - at), 0);
  }
  if (threadIdx.x == 0) p.tiles[p.n_tiles] = make_int4(tiles, 0, 0, 0);
}

// Rows of bf16 that no 16-byte load can take as they are: copied once, filled
// up with zeros to whole steps, 8 values a thread
struct PadRows {
  const __bf16* X;
  int64_t ldx, T;
  int D;
  __bf16* Y;
  int Dp;

  int64_t workgroups() const { return (T * (Dp / 8) + 255) / 256; }
  __device__ __forceinline__ void run(int64_t block) const {
    const int64_t i = block * 256 + threadIdx.x, t = i / (Dp / 8);
    if (t >= T) return;
    const int c = (int)(i - t * (Dp / 8)) * 8;
    float v[8];
    load8(X + t * ldx + c, D - c, v);
    __bf16 o[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) o[e] = (__bf16)v[e];
    __builtin_memcpy(__builtin_assume_aligned(Y + t * Dp + c, 16), o,
                     sizeof(o));
  }
};

// The first plan_blocks workgroups count, or place where one of them does it
// all; the others bring the layer's input into its form in the same launch,
// which a launch more made 2 us longer.
template <class Rows>
__global__ __launch_bounds__(PLAN_THREADS) void prepare_kernel(
    Plan p, int plan_blocks, Rows rows) {
  extern __shared__ int lds[];
  if ((int)blockIdx.x >= plan_blocks)
    rows.run(blockIdx.x - plan_blocks);
  else if (p.blocks > 1)
    plan_count(p, lds);
  else
    plan_place(p, lds);
}

// 12544 rows, 2 of 32 experts: 6 us, bound by its steps' latency
__global__ __launch_bounds__(PLAN_THREADS) void plan_place_kernel(Plan p) {
  extern __shared__ int lds[];
  plan_place(p, lds);
}

// ------------------------------------------------------ grouped products

struct Experts {
  const int4* tiles;
  const int* order;
  const int* ids;    // without a plan: each row is a tile of its own
  int E;
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
  _Float16* Y;        // second: [N][up64(n)] by assignment, over a power of
  float* SY;          // two for each 64 columns, [N][up64(n) / 64]
};

// A row's 64 columns of a term share a power of two that brings the largest
// finite one under 2^15, and go out in 16 bits: 2^-12 of a value is lost where
// the sum's own rounding to bf16 loses 2^-9 (a value below 2^-29 of the largest
// loses 2^-40 of that one), and the terms, the most that a layer of many rows
// moves, take half the bytes.
constexpr uint32_t INF_BITS = 0x7f800000;
__device__ __forceinline__ int power_over(uint32_t top) {  // its biased form
  return max((int)(top >> 23), 15) - 14;
}
__device__ __forceinline__ float power(int biased) {
  return __builtin_bit_cast(float, biased << 23);
}
template <int R>
__device__ __forceinline__ void store_terms(_Float16* to, const float (&v)[R],
                                            int up) {
  const float down = power(254 - up);
  _Float16 h[R];
#pragma unroll
  for (int c = 0; c < R; ++c) h[c] = (_Float16)(v[c] * down);
  __builtin_memcpy(__builtin_assume_aligned(to, R * 2), h, sizeof(h));
}

// What becomes of a tile's result; WHOLE: all its rows and columns are there,
// and it goes a straight way without a test.
template <class S, bool FIRST, int KIND, bool WHOLE>
__device__ __forceinline__ void finish_experts(
    const Experts& p, int e, int at0, int rows, int row0, int wave_n0, int wn,
    int lane, char* smem, f32x4 (&acc)[S::MT][S::NT]) {
  const float* bias = p.bias ? p.bias + (int64_t)e * p.n : nullptr;
  auto row = [&](int i) { return row0 + i * 16 + (lane & 15); };
  auto column = [&](int q) { return wave_n0 + run_column<S>(q, lane); };
  float b[S::RUNS][S::W] = {};
  if (bias)
#pragma unroll
    for (int q = 0; q < S::RUNS; ++q)
      load_run(bias + column(q), WHOLE ? S::W : p.n - column(q), b[q]);
  // a run's values; what lies behind the last column is 0
  auto values = [&](int i, int q, float(&v)[S::W]) {
    run_of<S>(acc[i], q, v);
#pragma unroll
    for (int c = 0; c < S::W; ++c) v[c] += b[q][c];
    activate_kind<KIND>(v, p.act);
#pragma unroll
    for (int c = 0; c < S::W; ++c)
      if (!WHOLE && column(q) + c >= p.n) v[c] = 0.f;
  };

  if constexpr (FIRST && S::FP8) {
    // a block of 128 columns is spread over SHARE waves: each leaves the
    // largest value of its rows in LDS, and its values in the accumulators
    constexpr int SHARE = 128 / (S::NT * 16);
    uint32_t* top = (uint32_t*)smem;  // [WN][BM]
    __syncthreads();
#pragma unroll
    for (int i = 0; i < S::MT; ++i) {
      uint32_t m = 0;
#pragma unroll
      for (int q = 0; q < S::RUNS; ++q) {
        float v[S::W];
        values(i, q, v);
        m = max(m, amax_bits(v));
#pragma unroll
        for (int c = 0; c < S::W; ++c)
          acc[i][q * (S::W / 4) + c / 4][c % 4] = v[c];
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
      if (!WHOLE && (r >= rows || wave_n0 >= p.np)) continue;
      const float s = scale_of(m);
#pragma unroll
      for (int q = 0; q < S::RUNS; ++q) {
        float v[S::W];
        run_of<S>(acc[i], q, v);
        uint32_t h[S::W / 4];
        to_fp8(v, s, h);
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
        if (!WHOLE && (row(i) >= rows || column(q) >= p.np)) continue;
        float v[S::W];
        values(i, q, v);
        // rounded to bf16 here: the second product takes no wider operand
        __bf16 t[S::W];
#pragma unroll
        for (int c = 0; c < S::W; ++c) t[c] = (__bf16)v[c];
        __bf16* h =
            (__bf16*)p.H + (int64_t)(at0 + row(i)) * p.np + column(q);
        __builtin_memcpy(__builtin_assume_aligned(h, 16), t, sizeof(t));
      }
  } else {
    int a[S::MT];
    float w[S::MT];
#pragma unroll
    for (int i = 0; i < S::MT; ++i)
      a[i] = p.order[at0 + (WHOLE ? row(i) : min(row(i), rows - 1))];
#pragma unroll
    for (int i = 0; i < S::MT; ++i) w[i] = p.w[a[i]];
#pragma unroll
    for (int i = 0; i < S::MT; ++i) {
      if (!WHOLE && row(i) >= rows) continue;
      uint32_t top = 0;
      float v[S::RUNS][S::W];
#pragma unroll
      for (int q = 0; q < S::RUNS; ++q) {
        values(i, q, v[q]);
#pragma unroll
        for (int c = 0; c < S::W; ++c) v[q][c] *= w[i];
        top = max(top, amax_bits(v[q]));
      }
      top = max(top, (uint32_t)__shfl_xor((int)top, 16));
      top = max(top, (uint32_t)__shfl_xor((int)top, 32));
      if (top >= INF_BITS) {  // the columns beside it are kept all the same
        top = 0;
#pragma unroll
        for (int q = 0; q < S::RUNS; ++q)
#pragma unroll
          for (int c = 0; c < S::W; ++c) {
            const uint32_t u =
                __builtin_bit_cast(uint32_t, v[q][c]) & ~(1u << 31);
            top = max(top, u < INF_BITS ? u : 0);
          }
        top = max(top, (uint32_t)__shfl_xor((int)top, 16));
        top = max(top, (uint32_t)__shfl_xor((int)top, 32));
      }
      const int up = power_over(top);
#pragma unroll
      for (int q = 0; q < S::RUNS; ++q)
        if (WHOLE || column(q) < p.np)
          store_terms(p.Y + (int64_t)a[i] * p.np + column(q), v[q], up);
      if (lane < 16 && (WHOLE || wave_n0 < p.np))
        p.SY[(int64_t)a[i] * (p.np / 64) + wave_n0 / 64] = power(up);
    }
  }
}

// The rows of one tile, all of one expert, times its weights. FIRST: rows are
// gathered by token, the result is activated, rounded to the layer's type and
// kept in the order of the experts. Otherwise: rows as they lie, the result is
// weighted and goes to its assignment's place, in 16 bits over a power of two.
// What a tile shares with its neighbours, rows of x or of the weights, comes
// from its XCD's L2. 25088 assignments of 32 experts, 768 x 1536, bf16, GELU:
// 80 to 95 us and 61 to 70 as the card's clock goes (0.57 and 0.76 PFLOP/s at
// best), half of it in the 12 and 24 steps, which run at 1.3 PFLOP/s, half in
// front of them and behind. 65536 of 64 experts, 2048 x 1024, e4m3: 215 to 230
// and 246 to 260 us (1.28 and 1.12 at best).
template <class S, bool FIRST, int KIND>
__global__ __launch_bounds__(S::THREADS, 2) void experts_kernel(Experts p) {
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  // the grid is for the most tiles there can be; those that there are get
  // spread over all XCDs
  const int tiles = __builtin_amdgcn_readfirstlane(p.tiles[p.n_tiles].x);
  if ((int)blockIdx.x >= tiles * p.tiles_n) return;
  const Place at_tile = place_of(blockIdx.x, tiles, p.tiles_n);
  const int4 tile = p.tiles[at_tile.m];
  const int e = __builtin_amdgcn_readfirstlane(tile.x);
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
  Rows<S> at;
  auto row_b = [&](int r) { return (uint32_t)(min(r, cols - 1) * b_row); };
  rows_of_b<S>(at, wave, lane, row_b);
  // The weights go ahead, as where the tile's rows lie is still to come: 33
  // rows of 1000 for 64 experts in e4m3 10.5 -> 9.4 us (8-bit products).
  int row[S::CA], scale = min(scale_row<S>(wave, lane), rows - 1);
#pragma unroll
  for (int i = 0; i < S::CA; ++i) {
    row[i] = min(staged_row(wave, S::CA, i, lane), rows - 1);
    if (FIRST) row[i] = p.order[at0 + row[i]];
  }
  scale = FIRST ? S::FP8 ? p.order[at0 + scale] : 0 : at0 + scale;
  send_b<S>(smem, rb, at, 0, p.steps, wave);
  if (FIRST) {
#pragma unroll
    for (int i = 0; i < S::CA; ++i) row[i] /= p.k;
    scale /= p.k;
  }
#pragma unroll
  for (int i = 0; i < S::CA; ++i)
    at.a[i] = (uint32_t)(row[i] * p.a_row) + chunk_a(wave, S::CA, i, lane);
  at.s = (uint32_t)scale * 4;
  const int wm = wave / S::WN, wn = wave % S::WN;
  const int wave_n0 = n0 + wn * S::NT * 16;
  f32x4 acc[S::MT][S::NT];
  // Hidden values that lie on a border between two e4m3 numbers fall to either
  // side by the sums' error, and each counts as a step of 2^-4: where rows are
  // so few that the weights' way from memory bounds, the sums keep all of f32:
  // 33 rows for 64 experts are off by 0.0017 in all, as bf16's rounding alone,
  // and not by up to 0.0037, for 1 to 2 us of 27.
  constexpr bool EXACT = FIRST && S::FP8 && S::BM == 32;
  const float* sb = S::FP8 ? p.SB + ((int64_t)e * blocks_n +
                                     min(wave_n0 / 128, blocks_n - 1)) * p.steps
                           : nullptr;
  const bool odd =
      product<S, true, EXACT>(smem, ra, rb, rs, at, 0, p.steps, p.sa_rows * 4,
                              sb, wave, lane, acc);
  if constexpr (S::FP8) {
    auto row_of = [&](int r) {
      r = at0 + min(r, rows - 1);
      return FIRST ? p.order[r] / p.k : r;
    };
    mend_sums<S, EXACT>(
        ra, rb, rs,
        [&](int r) {
          return (uint32_t)((row_of(r) - (FIRST ? 0 : at0)) * p.a_row);
        },
        row_b, [&](int r) { return (uint32_t)row_of(r) * 4; }, 0, p.steps,
        p.sa_rows * 4, sb, wave, lane, odd, acc);
  }

  const int row0 = wm * S::MT * 16;
  if (rows == S::BM && n0 + S::BN <= p.n)
    finish_experts<S, FIRST, KIND, true>(p, e, at0, rows, row0, wave_n0, wn,
                                         lane, smem, acc);
  else
    finish_experts<S, FIRST, KIND, false>(p, e, at0, rows, row0, wave_n0, wn,
                                          lane, smem, acc);
}

// Without a plan, the first product: CW * 16 columns of an assignment a
// workgroup, K cut into KS parts, a wave each. The 16 rows are all the same.
// Bound by the time its weights take to come: 2 assignments, 768 x 1536 in
// bf16, 4.2 us. One tile of 16 columns with K in 8 parts, or two with 4, for a
// layer of 1 row: 9.9 / 10.5 us, 2 of 8 experts of 2048 x 2048 13.3 / 15.1;
// where half as wide workgroups are more than CUs, 2 rows of 4 experts, 1024 x
// 704, 11.3 / 11.1. 16 waves (e4m3, K in 2 parts: 13.6 -> 14.6) and 4 were
// slower.
template <bool FP8, int CW, int KS>
__global__ __launch_bounds__(512, 4) void experts_hidden_kernel(Experts p) {
  static_assert(CW * KS == 8 && (!FP8 || CW == 8));
  __shared__ __attribute__((aligned(16))) float part[8 * 256];
  __shared__ uint32_t top[CW];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int cw = wave / KS, ks = wave % KS;
  const int64_t a = blockIdx.x / p.tiles_n;
  const int n0 = ((int)(blockIdx.x - a * p.tiles_n) * CW + cw) * 16;
  const int e = p.ids[a];
  if ((unsigned)e >= (unsigned)p.E) return;
  const int64_t row = a / p.k;
  const int col = min(n0 + (lane & 15), p.n - 1);
  const int n = n0 + (lane >> 4) * 4;
  const int blocks_n = (p.n + 127) / 128;
  float b[4];  // on its way with the weights
  load_run(p.bias + (int64_t)e * p.n + n, p.bias ? p.n - n : 0, b);
  const f32x4 acc = few_product<FP8, FP8>(
      p.A + row * p.a_row + (lane >> 4) * 16,
      p.B + ((int64_t)e * p.n + col) * ((int64_t)p.steps * STEP) +
          (lane >> 4) * 16,
      p.SA + row, p.sa_rows,
      p.SB + ((int64_t)e * blocks_n + min(n0 / 128, blocks_n - 1)) * p.steps,
      p.steps * ks / KS, p.steps * (ks + 1) / KS);
  const f32x4 sum = few_join<KS>(acc, part, cw, ks, lane);
  float v[4] = {sum[0], sum[1], sum[2], sum[3]};
#pragma unroll
  for (int c = 0; c < 4; ++c) v[c] += b[c];
  activate(v, p.act);
#pragma unroll
  for (int c = 0; c < 4; ++c)
    if (n + c >= p.n) v[c] = 0.f;
  const bool mine = ks == 0 && (lane & 15) == 0 && n0 < p.np;
  if constexpr (FP8) {
    uint32_t m = amax_bits(v);
    m = max(m, (uint32_t)__shfl_xor((int)m, 16));
    m = max(m, (uint32_t)__shfl_xor((int)m, 32));
    if (lane == 0) top[cw] = m;
    __syncthreads();
#pragma unroll
    for (int c = 0; c < CW; ++c) m = max(m, top[c]);
    if (!mine) return;
    const float s = scale_of(m);
    uint32_t h[1];
    to_fp8(v, s, h);
    *(uint32_t*)((uint8_t*)p.H + a * p.np + n) = h[0];
    if (cw == 0 && lane == 0) p.SH[(int64_t)(n0 / 128) * p.N + a] = s;
  } else if (mine) {
    // rounded to bf16 as with a plan. Kept in two parts, what bf16 holds and
    // the rest, the result would be off by bf16's own rounding alone, 0.0017
    // for 0.0024, but 1 us of 11 later.
    __bf16 h[4];
#pragma unroll
    for (int c = 0; c < 4; ++c) h[c] = (__bf16)v[c];
    __builtin_memcpy(
        __builtin_assume_aligned((__bf16*)p.H + a * p.np + n, 8), h,
        sizeof(h));
  }
}

// Without a plan, the second product and the sum over a token's experts: 16
// columns of a token a workgroup, its waves share the experts and, if there
// are fewer than 8, K. The 16 rows are all the same one. Bound as above: 1 row
// of 2 experts, 1536 x 768 in bf16, 6.0 us, 0.7 more with K in one piece.
template <bool FP8>
__global__ __launch_bounds__(512, 4) void experts_sum_kernel(
    Experts p, const __bf16* residual, int64_t ldr, __bf16* Y, int64_t ldy) {
  __shared__ __attribute__((aligned(16))) float part[8 * 256];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t t = blockIdx.x / p.tiles_n;
  const int n0 = (int)(blockIdx.x - t * p.tiles_n) * 16;
  const int col = min(n0 + (lane & 15), p.n - 1);
  const int n = n0 + (lane >> 4) * 4;
  const int blocks_n = (p.n + 127) / 128;
  f32x4 total = {0.f, 0.f, 0.f, 0.f};
  const int parts = max(1, 8 / p.k);
  for (int u = wave; u < p.k * parts; u += 8) {
    const int j = u / parts, ks = u - j * parts;
    const int64_t a = t * p.k + j;
    const int e = p.ids[a];
    if ((unsigned)e >= (unsigned)p.E) continue;
    const float w = p.w[a];
    float b[4];
    load_run(p.bias + (int64_t)e * p.n + n, p.bias && ks == 0 ? p.n - n : 0,
             b);
    const f32x4 acc = few_product<FP8, false>(
        p.A + a * p.a_row + (lane >> 4) * 16,
        p.B + ((int64_t)e * p.n + col) * ((int64_t)p.steps * STEP) +
            (lane >> 4) * 16,
        p.SA + a, p.sa_rows,
        p.SB + ((int64_t)e * blocks_n + n0 / 128) * p.steps,
        p.steps * ks / parts, p.steps * (ks + 1) / parts);
#pragma unroll
    for (int c = 0; c < 4; ++c)
      total[c] = __builtin_fmaf(acc[c] + b[c], w, total[c]);
  }
  const f32x4 sum = few_join<8>(total, part, 0, wave, lane);
  if (wave || lane & 15) return;
#pragma unroll
  for (int c = 0; c < 4; ++c)
    if (n + c < p.n)
      Y[t * ldy + n + c] = (__bf16)(
          sum[c] + (residual ? (float)residual[t * ldr + n + c] : 0.f));
}

// Each token adds up its experts' rows, in the order of its list: 8 columns a
// thread. Bound by HBM: 8192 rows of 8 x 2048 57 us, 5.3 TB/s. Where Y and the
// residual allow 16 bytes at a time, 12544 x 768 takes 12 to 13 us, else 16.
__global__ __launch_bounds__(256) void combine_kernel(
    const _Float16* __restrict__ P, const float* __restrict__ SP,
    const int* __restrict__ ids, int E, int k, int D, int Dp,
    const __bf16* residual, int64_t ldr, __bf16* Y, int64_t ldy, bool vec,
    int64_t n) {
  const int per = (D + 7) / 8;
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= n) return;
  const int64_t t = i / per;
  const int c = (int)(i - t * per) * 8;
  float v[8] = {};
#pragma unroll 4
  for (int j = 0; j < k; ++j) {
    if ((unsigned)ids[t * k + j] >= (unsigned)E) continue;
    const int64_t a = t * k + j;
    _Float16 u[8];
    __builtin_memcpy(u, __builtin_assume_aligned(P + a * Dp + c, 16),
                     sizeof(u));
    const float s = SP[a * (Dp / 64) + c / 64];
#pragma unroll
    for (int q = 0; q < 8; ++q) v[q] = __builtin_fmaf((float)u[q], s, v[q]);
  }
  const __bf16* r = residual + t * ldr + c;
  __bf16* y = Y + t * ldy + c;
  __bf16 o[8];
  if (vec && c + 8 <= D) {
    if (residual) {
      __builtin_memcpy(o, __builtin_assume_aligned(r, 16), sizeof(o));
#pragma unroll
      for (int q = 0; q < 8; ++q) v[q] += (float)o[q];
    }
#pragma unroll
    for (int q = 0; q < 8; ++q) o[q] = (__bf16)v[q];
    __builtin_memcpy(__builtin_assume_aligned(y, 16), o, sizeof(o));
  } else {
#pragma unroll
    for (int q = 0; q < 8; ++q)
      if (c + q < D) y[q] = (__bf16)(v[q] + (residual ? (float)r[q] : 0.f));
  }
}

template <bool FP8, bool FIRST>
using Tile128 = Shape<FP8, 128, 128, 2, 2, 2, FIRST && FP8 ? 16 : 8>;
// Few rows an expert: what counts is how much of the weights is on its way.
// As many stages as let two workgroups onto a CU: with one more, so that each
// lies alone, 33 rows of 1000 for 64 experts in e4m3 took 34.7 us, not 28.5.
// Tiles of 64 rows in e4m3 go three to a CU with 2 stages: 3000 rows of 1024,
// 8 of 128 experts, 127 us, with 3 stages 137; in bf16 it is 186 and 189, but
// 52 and 44 where each lies alone (256 rows of 2048, 2 of 8).
template <bool FP8, bool FIRST>
using Tile32 =
    Shape<FP8, 32, 128, 2, 2, FP8 ? 3 : 4, FIRST && FP8 ? 16 : 8>;
template <bool FP8, bool FIRST>
using Tile64 = Shape<FP8, 64, 128, 2, 2, FP8 ? 2 : 3, FIRST && FP8 ? 16 : 8>;

template <class S, bool FIRST, int KIND>
void run(Experts p, hipStream_t stream) {
  p.tiles_n = up(FIRST ? p.np : p.n, S::BN);
  hipLaunchKernelGGL((experts_kernel<S, FIRST, KIND>),
                     dim3(p.n_tiles * p.tiles_n), dim3(S::THREADS), S::LDS,
                     stream, p);
}

template <class S>
void run_first(Experts p, hipStream_t stream) {
  switch (kind_of(p.act)) {
    case PLAIN:
      return run<S, true, PLAIN>(p, stream);
    case CLAMP:
      return run<S, true, CLAMP>(p, stream);
    case GELU:
      return run<S, true, GELU>(p, stream);
  }
}

int64_t up256(int64_t bytes) { return (bytes + 255) & ~int64_t(255); }

// where a call's intermediate data lie
// direct: so few rows that a plan isn't worth its launches, two products and
// no more
struct Layout {
  bool direct;
  int64_t counts, order, tiles, x, sx, h, sh, y, sy, bytes;
  int n_tiles, blocks, BM, Dp, Hp;
  bool copy;  // the rows of x are brought into whole steps first
};

// Few rows go without a plan, each with its own expert's weights: two launches
// less, but experts that rows share are read for each of them. In us, without
// and with a plan: 64 experts of 1024 x 704 in bf16, N = 8: 11.4 / 23.1, 16:
// 14.7 / 25.0; 16 of 768 x 1536, N = 16: 20.4 / 26.3, 32: 30.7 / 26.6; 128 of
// 1024 x 704 in e4m3, N = 32: 18.1 / 25.7; 32 of 768 x 1536, N = 32:
// 24.4 / 24.2.
bool goes_directly(int64_t N, int64_t E) {
  return N <= 16 ? N <= E : N <= 32 && 2 * N <= E;
}

// Rows of a tile: 32, 64 or 128, whatever costs least. Both products take as
// many rounds over the chip as their tiles need, two of them a CU (of 64 rows
// in e4m3 three, which then take 1.27 times as long), a little less than a
// whole one if each lies alone; a round takes its steps and what lies before
// and behind them. Measured, in us, for 32 / 64 / 128 rows and N rows in all:
// 16 experts of 768 x 1536 in bf16, N = 256: 29.4 / 33.3 / 41.9, N = 2048:
// 44.7 / 39.1 / 49.6, N = 6000: 88 / 72 / 67; 128 of 1024 x 704 in e4m3,
// N = 128: 36.7 / 35.5 / 43.3, N = 8192: 79 / 70 / 82, N = 48000:
// 302 / 211 / 207. Over 124 such cases the costs below chose a tile that is
// 0.2% off the best one on average, 5% at most.
int tile_rows(const MoeMlp& m, int64_t N, int unit) {
  struct {
    int rows;
    double step, fixed;
  } const shapes[] = {{32, 0.7, 0.2}, {64, 0.92, 0.4}, {128, 1.25, 2.6}};
  const double used = (double)std::min<int64_t>(N, m.E);
  double least = 1e30;
  int best = 0;
  for (const auto& s : shapes) {
    // half a tile an expert is left over, and each has one at least
    const double rows = std::max(used, (double)N / s.rows + used / 2);
    auto product = [&](int k, int n) {
      const double tiles = rows * up(n, 128);
      const double rounds = tiles <= 256 ? 0.8
                            : tiles > 512 && s.rows == 64 && m.fp8
                                ? std::ceil(tiles / 768) * 1.27
                                : std::ceil(tiles / 512);
      return rounds * (up(k, unit) * s.step + s.fixed);
    };
    const double t = product(m.D, m.H) + product(m.H, m.D);
    if (t < least) least = t, best = s.rows;
  }
  return best;
}

Layout layout(const MoeMlp& m) {
  Layout l{};
  const int64_t N = (int64_t)m.T * m.k;
  l.direct = goes_directly(N, m.E);
  const int unit = m.fp8 ? 128 : 64, size = m.fp8 ? 1 : 2;
  l.BM = tile_rows(m, N, unit);
  l.n_tiles = (int)(N / l.BM + std::min<int64_t>(N, m.E));
  l.blocks = up(N, PLAN_ROWS);
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
  l.tiles = take((int64_t)(l.n_tiles + 1) * 16);
  l.x = take(l.copy ? (int64_t)m.T * l.Dp * size : 0);
  l.sx = take(m.fp8 ? (int64_t)m.T * (l.Dp / 128) * 4 : 0);
  l.h = take(N * l.Hp * size);
  l.sh = take(m.fp8 ? N * (l.Hp / 128) * 4 : 0);
  l.y = take(N * up(m.D, 64) * 64 * 2);
  l.sy = take(N * up(m.D, 64) * 4);
  l.bytes = at;
  return l;
}

template <bool FP8>
void run_mlp(const MoeMlp& m, const Layout& l, char* ws, hipStream_t stream) {
  const int N = m.T * m.k;
  const Plan plan{m.ids, (int*)(ws + l.counts), (int*)(ws + l.order),
            (int4*)(ws + l.tiles), N, m.E, l.BM, l.n_tiles, l.blocks};
  const int plan_lds = (4 * m.E + 2) * 4;
  auto prepare = [&](auto rows, bool some) {
    const int plan_blocks = l.direct ? 0 : l.blocks;
    const int64_t blocks = plan_blocks + (some ? rows.workgroups() : 0);
    if (blocks)
      hipLaunchKernelGGL((prepare_kernel<decltype(rows)>),
                         dim3((uint32_t)blocks), dim3(PLAN_THREADS), plan_lds,
                         stream, plan, plan_blocks, rows);
  };
  const auto x = (const __bf16*)m.X;
  if (FP8)
    prepare(QuantRows<__bf16>::of(x, m.ldx, m.T, m.D, ws + l.x, l.Dp,
                                  (float*)(ws + l.sx)),
            true);
  else
    prepare(PadRows{x, m.ldx, m.T, m.D, (__bf16*)(ws + l.x), l.Dp}, l.copy);
  if (!l.direct && l.blocks > 1)
    hipLaunchKernelGGL(plan_place_kernel, dim3(l.blocks), dim3(PLAN_THREADS),
                       plan_lds, stream, plan);

  Experts p{};
  p.tiles = plan.tiles;
  p.order = plan.order;
  p.ids = l.direct ? m.ids : nullptr;
  p.E = m.E;
  p.k = m.k;
  p.N = N;
  p.n_tiles = l.n_tiles;
  const int size = FP8 ? 1 : 2;
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
  if (l.direct) {
    auto hidden = [&](auto cw, auto ks) {
      constexpr int CW = decltype(cw)::value, KS = decltype(ks)::value;
      p.tiles_n = up(p.np, CW * 16);
      hipLaunchKernelGGL((experts_hidden_kernel<FP8, CW, KS>),
                         dim3(N * p.tiles_n), dim3(CW * KS * 64), 0, stream,
                         p);
    };
    using std::integral_constant;
    if constexpr (FP8)  // the waves share the scale of a block of columns
      hidden(integral_constant<int, 8>(), integral_constant<int, 1>());
    else if (N * up(p.np, 32) <= 128)  // twice as many fit, one to a CU
      hidden(integral_constant<int, 1>(), integral_constant<int, 8>());
    else
      hidden(integral_constant<int, 2>(), integral_constant<int, 4>());
  } else if (l.BM == 32) {
    run_first<Tile32<FP8, true>>(p, stream);
  } else if (l.BM == 64) {
    run_first<Tile64<FP8, true>>(p, stream);
  } else {
    run_first<Tile128<FP8, true>>(p, stream);
  }

  p.A = (const uint8_t*)ws + l.h;
  p.a_row = (int64_t)l.Hp * size;
  p.SA = p.SH;
  p.sa_rows = N;
  p.B = (const uint8_t*)m.W2;
  p.SB = m.S2;
  p.bias = m.b2;
  p.n = m.D;
  p.np = up(m.D, 64) * 64;
  p.steps = l.Hp * size / STEP;
  p.w = m.weights;
  p.Y = (_Float16*)(ws + l.y);
  p.SY = (float*)(ws + l.sy);
  const auto residual = (const __bf16*)m.residual;
  if (l.direct) {
    p.tiles_n = up(m.D, 16);
    hipLaunchKernelGGL((experts_sum_kernel<FP8>), dim3(m.T * p.tiles_n),
                       dim3(512), 0, stream, p, residual, m.ldr, (__bf16*)m.Y,
                       m.ldy);
    return;
  }
  if (l.BM == 32)
    run<Tile32<FP8, false>, false, PLAIN>(p, stream);
  else if (l.BM == 64)
    run<Tile64<FP8, false>, false, PLAIN>(p, stream);
  else
    run<Tile128<FP8, false>, false, PLAIN>(p, stream);

  const int64_t work = (int64_t)m.T * up(m.D, 8);
  const bool vec = (uintptr_t)m.Y % 16 == 0 && m.ldy % 8 == 0 &&
                   (uintptr_t)m.residual % 16 == 0 && m.ldr % 8 == 0;
  hipLaunchKernelGGL(combine_kernel, dim3(up(work, 256)), dim3(256), 0, stream,
                     p.Y, p.SY, m.ids, m.E, m.k, m.D, p.np,
                     residual, m.ldr, (__bf16*)m.Y, m.ldy, vec, work);
}

}  // namespace

void launch_moe_logits(const void* X, int64_t ldx, const void* W, float* Y,
                       int T, int D, int E, hipStream_t stream) {
  const Logits p{(const __bf16*)X, (const __bf16*)W, Y, ldx, T, D,
                 up(D, 64) * 64, E};
  auto go = [&](auto rt, auto nt, auto ks) {
    constexpr int RT = decltype(rt)::value, NT = decltype(nt)::value,
                  KS = decltype(ks)::value;
    hipLaunchKernelGGL((logits_kernel<RT, NT, KS>),
                       dim3(up(T, 8 / KS * RT * 16) * up(E, NT * 16)),
                       dim3(512), 0, stream, p);
  };
  // Few tiles: all 8 waves share K; many: each load serves more products. In
  // us, for <1, 1, 8> / <2, 1, 4> / <4, 2, 4>: 1 x 768, 64 experts: 4.2 / 4.9 /
  // 9.6, 1568 x 768, 64: 7.6 / 9.1 / 18, 12544 x 768, 8: 9.7 / 7.7 / 14,
  // 3136 x 768, 64: 12.9 / 9.2 / 18, 12544 x 768, 64: 36 / 29 / 19, 256:
  // 130 / 88 / 72.
  using std::integral_constant;
  const int64_t tiles = (int64_t)up(T, 16) * up(E, 16);
  if (tiles <= 512)
    go(integral_constant<int, 1>(), integral_constant<int, 1>(),
       integral_constant<int, 8>());
  else if (tiles <= 1536)
    go(integral_constant<int, 2>(), integral_constant<int, 1>(),
       integral_constant<int, 4>());
  else
    go(integral_constant<int, 4>(), integral_constant<int, 2>(),
       integral_constant<int, 4>());
}

void launch_moe_route(const void* X, bool f32, int64_t ldx, const float* bias,
                      int* ids, float* weights, int T, int E, int k,
                      bool sigmoid, int groups, int kept, int best,
                      bool renorm, float scale, hipStream_t stream) {
  const Route p{X, bias, ids, weights, ldx, T, E, k, groups, kept, best,
                sigmoid, renorm, scale};
  const dim3 grid(up(T, 16));
  auto go = [&](auto x, auto v) {
    using X_ = decltype(x);
    constexpr int V = decltype(v)::value;
    const int lds = RouteLds(V, groups, k).floats * 16 * 4;
    hipLaunchKernelGGL((route_kernel<X_, V>), grid, dim3(256), lds, stream, p);
  };
  auto by_type = [&](auto v) {
    if (f32)
      go(0.f, v);
    else
      go((__bf16)0.f, v);
  };
  if (E <= 16)
    by_type(std::integral_constant<int, 1>());
  else if (E <= 64)
    by_type(std::integral_constant<int, 4>());
  else if (E <= 128)
    by_type(std::integral_constant<int, 8>());
  else if (E <= 256)
    by_type(std::integral_constant<int, 16>());
  else
    by_type(std::integral_constant<int, 32>());
}

int64_t moe_mlp_workspace(const MoeMlp& m) { return layout(m).bytes; }

void launch_moe_mlp(const MoeMlp& m, void* ws, hipStream_t stream) {
  const Layout l = layout(m);
  if (m.fp8)
    run_mlp<true>(m, l, (char*)ws, stream);
  else
    run_mlp<false>(m, l, (char*)ws, stream);
}
