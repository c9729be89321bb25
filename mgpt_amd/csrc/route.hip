// route.hip -- the choice of experts from a router's logits and its gradient: softmax or
// sigmoid scores, a bias for balance, groups of experts, renormalised weights.
//
// For a token's logits l (each at most FLT_MAX; an expert whose logit is -infinity or
// NaN, or whose key is, takes no part):
//   s = softmax(l) or 1 / (1 + exp(-l)),   key = l, or s + bias where there is a bias
//   a group's size is the sum of the scores (s or s + bias) of its best one or two; the
//   top_groups largest groups take part, and of their experts the k largest keys, in
//   descending order, the lower id first where equal; where fewer are left, the lowest of the other ids
//   follow, with weight 0:
//   w_j = c s_j / D,  D = sum_j s_j + 1e-20 (renormalised) or 1;  a score below 2^-126 may count as 0 here
// Backward, for the upstream gradients dw of the weights and g_e of expert e's score in every token:
//   d_j = (c dw_j - sum_i dw_i w_i) / D (or c dw_j),  ds = g + d scattered to the chosen ones
//   sigmoid: dl = ds s (1 - s),   softmax: dl = s (ds - sum_e ds_e s_e)
//
// A token's experts lie in LP lanes of a wave, V neighbouring ones in each, so that 64 / LP tokens
// share a wave, and stay in registers; the token's own LDS holds what lanes look up by expert (logits, the
// gradient's scatter) and pass between groups.
//
// The choice: keys as whole numbers, (key - the largest) in a fixed unit, with the expert's id below them, so that
// no two are equal.  Every lane sorts its own by a network of minima and maxima; k rounds then take the largest of the
// lanes' first ones, by moves within rows of 16 lanes, and pop it.
//
// Keys with a bias, and sizes of groups, are those of 64 bits, and logits may have the same number without being equal:
// where what is compared is not further apart than its rounding, the wave does its tokens again in 64 bits (few steps),
// by code that is short, since a wave that comes to it alone waits for every fetch of it, and whose
// invariants are formed there (ahead of the loop they took a hundred registers).  At 32768 x 256 (8 groups, a bias), us:
// 64 bits throughout 52, a wave to a token that searches for each maximum 57, again in 64 bits by unrolled code 64, by
// loops that load the logits one by one 43, so 30, 8 of them for those tokens.  1100 vector instructions a step of four tokens
// bound it, 15 us.  The backward, whose next step's loads are on their way, takes 22 (67 MB, 13 at a copy's rate);
// 40001 x 160 bf16 (8 groups of 20, softmax) 37 and 22 (28 MB, 5.6 at that rate: 256 places for 160 experts, and in bf16
// a lane's loads and stores are 8 bytes, 32 apart), 16384 x 16 4 and 3.4.
#include <algorithm>
#include <cfloat>
#include <cmath>
#include <type_traits>

#include "capi_internal.hpp"
#include "route.hpp"

namespace mgpt {

namespace {

constexpr float kNone = -INFINITY;

// exp to 1.5 ulp: the elementary split of log2 e, its float and what that leaves (log2 e - fl(log2 e) = 1.92596299e-8),
// around the hardware's exponential of 2; the remainder enters by the exponential's slope.
__device__ __forceinline__ float exp_full(float x) {
  const float y = x * 1.44269504088896340736f;
  const float r = __builtin_fmaf(x, 1.44269504088896340736f, -y) + x * 1.92596299e-8f;
  const float e = __builtin_amdgcn_exp2f(y);
  return y > -INFINITY && y < 128.0f ? __builtin_fmaf(e, r * 0.693147180559945f, e) : e;
}

// (bounds as the hardware's zeros, so that the move folds into the operation; every lane has a source)
template <int CTRL>
__device__ __forceinline__ int dpp(int v) {
  return __builtin_amdgcn_update_dpp(0, v, CTRL, 0xf, 0xf, true);
}
template <int CTRL>
__device__ __forceinline__ uint32_t dpp(uint32_t v) {
  return (uint32_t)dpp<CTRL>((int)v);
}
template <int CTRL>
__device__ __forceinline__ float dpp(float v) {
  return __int_as_float(dpp<CTRL>(__float_as_int(v)));
}
template <int CTRL>
__device__ __forceinline__ double dpp(double v) {
  return __hiloint2double(dpp<CTRL>(__double2hiint(v)), dpp<CTRL>(__double2loint(v)));
}

// Step D of a butterfly over lanes: the value of lane ^ 1, ^ 2, or of a lane in the other
// 4 (8) of its 8 (16), or of lane ^ 16, ^ 32.  After the steps 1 .. L / 2 of a symmetric operation all of
// L neighbouring lanes hold its result.
__device__ __forceinline__ int partner16(int v) {
  const auto r = __builtin_amdgcn_permlane16_swap(v, v, false, false);
  return (lane_id() & 16) ? r[0] : r[1];
}
__device__ __forceinline__ int partner32(int v) {
  const auto r = __builtin_amdgcn_permlane32_swap(v, v, false, false);
  return (lane_id() & 32) ? r[0] : r[1];
}
__device__ __forceinline__ uint32_t partner16(uint32_t v) { return (uint32_t)partner16((int)v); }
__device__ __forceinline__ uint32_t partner32(uint32_t v) { return (uint32_t)partner32((int)v); }
__device__ __forceinline__ float partner16(float v) { return __int_as_float(partner16(__float_as_int(v))); }
__device__ __forceinline__ float partner32(float v) { return __int_as_float(partner32(__float_as_int(v))); }
__device__ __forceinline__ double partner16(double v) {
  return __hiloint2double(partner16(__double2hiint(v)), partner16(__double2loint(v)));
}
__device__ __forceinline__ double partner32(double v) {
  return __hiloint2double(partner32(__double2hiint(v)), partner32(__double2loint(v)));
}
template <int D, typename T>
__device__ __forceinline__ T partner(T v) {
  if constexpr (D == 1) return dpp<0xB1>(v);
  else if constexpr (D == 2) return dpp<0x4E>(v);
  else if constexpr (D == 4) return dpp<0x141>(v);   // row_half_mirror
  else if constexpr (D == 8) return dpp<0x140>(v);   // row_mirror
  else if constexpr (D == 16) return partner16(v);
  else return partner32(v);
}
template <int L, typename T, typename Op>
__device__ __forceinline__ T across(T v, Op op) {
  if constexpr (L > 1) v = op(v, partner<1>(v));
  if constexpr (L > 2) v = op(v, partner<2>(v));
  if constexpr (L > 4) v = op(v, partner<4>(v));
  if constexpr (L > 8) v = op(v, partner<8>(v));
  if constexpr (L > 16) v = op(v, partner<16>(v));
  if constexpr (L > 32) v = op(v, partner<32>(v));
  return v;
}
__device__ __forceinline__ float inverse(float x) { return __builtin_amdgcn_rcpf(x); }   // 1 ulp

// Orders a wave's own LDS accesses across its lanes.
__device__ __forceinline__ void wave_sync() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// The number, of which the compiler knows nothing here: what follows from it is not computed ahead of a loop, where it
// would take registers for code that hardly ever runs.
__device__ __forceinline__ int here(int x) {
  asm volatile("" : "+s"(x));
  return x;
}
__device__ __forceinline__ int here_lane(int x) {
  asm volatile("" : "+v"(x));
  return x;
}

// A lane's V logits of a token, e0 .. e0 + V - 1; experts past E have -infinity.
template <typename T, int V>
__device__ __forceinline__ void load_logits(const RouteArgs& g, size_t t, int e0, bool live, float (&l)[V]) {
  const T* p = reinterpret_cast<const T*>(g.logits) + t * g.E;
#pragma unroll
  for (int v = 0; v < V; ++v) l[v] = kNone;
  if (!live) return;
  if (g.vec) {   // E is a multiple of 4 and rows are aligned to 4 experts
#pragma unroll
    for (int q = 0; q < V; q += 4) {
      if (e0 + q < g.E) {
        if constexpr (sizeof(T) == 4) {
          const float4 x = *reinterpret_cast<const float4*>(p + e0 + q);
          l[q] = x.x, l[q + 1] = x.y, l[q + 2] = x.z, l[q + 3] = x.w;
        } else {
          const uint2 x = *reinterpret_cast<const uint2*>(p + e0 + q);
          l[q] = __uint_as_float(x.x << 16), l[q + 1] = __uint_as_float(x.x & 0xFFFF0000u);
          l[q + 2] = __uint_as_float(x.y << 16), l[q + 3] = __uint_as_float(x.y & 0xFFFF0000u);
        }
      }
    }
  } else {
    const int n = here(g.E) - e0;
#pragma unroll
    for (int v = 0; v < V; ++v)
      if (v < n) l[v] = to_f32(p[e0 + v]);
  }
}

// An infinity or a NaN among the logits, out of the way.
// (The hardware's median of three with a NaN is their minimum; the compiler would make a minimum of two of it.)
__device__ __forceinline__ float clean(float l) {
  float r;
  asm("v_med3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(l), "v"(kNone), "v"(FLT_MAX));
  return r;
}

// A maximum of numbers that are none a signalling NaN (fmaxf would first make sure of that).
__device__ __forceinline__ float max32(float a, float b) {
  float r;
  asm("v_max_f32 %0, %1, %2" : "=v"(r) : "v"(a), "v"(b));
  return r;
}

template <int LP, int V>
__device__ __forceinline__ float largest(const float (&l)[V]) {
  float m = l[0];
#pragma unroll
  for (int v = 1; v < V; ++v) m = max32(m, l[v]);
  return max32(across<LP>(m, [](float a, float b) { return max32(a, b); }), -FLT_MAX);   // (a row without experts)
}

// Softmax to some 2^-22.
template <int LP, int V>
__device__ __forceinline__ void softmax_of(const float (&l)[V], float (&s)[V]) {
  const float m = largest<LP, V>(l);
  float z = 0.0f;
#pragma unroll
  for (int v = 0; v < V; ++v) {
    s[v] = exp_full(l[v] - m);
    z += s[v];
  }
  z = across<LP>(z, [](float a, float b) { return a + b; });
  const float r = z > 0.0f ? inverse(z) : 0.0f;
#pragma unroll
  for (int v = 0; v < V; ++v) s[v] *= r;
}

// exp(x) in 64 bits to 2^-51, x <= 0 (down to 0 itself): 2^t by its whole part and a polynomial of degree 10 on [-1/2, 1/2]
// (least maximum relative error, 2^-52).
__device__ __forceinline__ double exp64(double x) {
  const double t = fmax(x * 1.4426950408889634, -1100.0);
  const double n = (t + 0x1.8p52) - 0x1.8p52, f = t - n;
  double q = 0x1.e3992178bd0ddp-28;
  q = __builtin_fma(q, f, 0x1.b6740fb0785eap-24);
  q = __builtin_fma(q, f, 0x1.62c157ec7ee12p-20);
  q = __builtin_fma(q, f, 0x1.ffcb55e844f93p-17);
  q = __builtin_fma(q, f, 0x1.43091260573e4p-13);
  q = __builtin_fma(q, f, 0x1.5d87fe9cc5ce9p-10);
  q = __builtin_fma(q, f, 0x1.3b2ab6fbde0f3p-7);
  q = __builtin_fma(q, f, 0x1.c6b08d703d48ap-5);
  q = __builtin_fma(q, f, 0x1.ebfbdff82c3b9p-3);
  q = __builtin_fma(q, f, 0x1.62e42fefa3a17p-1);
  q = __builtin_fma(q, f, 1.0);
  return __builtin_ldexp(q, (int)n);
}
// 1 / x to 2^-52: the hardware's and two Newton steps.
__device__ __forceinline__ double inverse64(double x) {
  double r = __builtin_amdgcn_rcp(x);
  r = __builtin_fma(r, __builtin_fma(-x, r, 1.0), r);
  return __builtin_fma(r, __builtin_fma(-x, r, 1.0), r);
}

__device__ __forceinline__ void order2(uint32_t& a, uint32_t& b) {
  const uint32_t x = max(a, b);
  b = min(a, b);
  a = x;
}
// The largest min(V, 8) of V numbers, descending.
template <int V>
__device__ __forceinline__ void sort_lane(const uint32_t* x, uint32_t* y) {
  if constexpr (V == 16) {
    uint32_t z[8];
    sort_lane<8>(x, y);
    sort_lane<8>(x + 8, z);
#pragma unroll
    for (int i = 0; i < 8; ++i) y[i] = max(y[i], z[7 - i]);   // the 8 largest, up and down
#pragma unroll
    for (int d = 4; d >= 1; d /= 2)
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (!(i & d)) order2(y[i], y[i + d]);
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) y[i] = x[i];
    // odd-even merges
    constexpr int kNet8[19][2] = {{0, 1}, {2, 3}, {4, 5}, {6, 7}, {0, 2}, {1, 3}, {4, 6}, {5, 7}, {1, 2}, {5, 6},
                                  {0, 4}, {1, 5}, {2, 6}, {3, 7}, {2, 4}, {3, 5}, {1, 2}, {3, 4}, {5, 6}};
    constexpr int kNet4[5][2] = {{0, 1}, {2, 3}, {0, 2}, {1, 3}, {1, 2}};
    if constexpr (V == 8) {
#pragma unroll
      for (int i = 0; i < 19; ++i) order2(y[kNet8[i][0]], y[kNet8[i][1]]);
    } else {
#pragma unroll
      for (int i = 0; i < 5; ++i) order2(y[kNet4[i][0]], y[kNet4[i][1]]);
    }
  }
}

// What a wave keeps in LDS: for each of its tokens the logits (32 bits) or keys (64) by expert, the sizes
// of the groups, and the chosen experts, as packed numbers or (64 bits) ids.
template <int LP, int V>
struct Space {
  static constexpr int kTokens = kWave / LP;
  static constexpr int kGroups = LP * V < kMaxExperts ? LP * V : kMaxExperts;
  double key[kWave * V];
  double size[kTokens][kGroups];
  uint8_t on[kTokens][kGroups];
  uint32_t pick[kTokens][kMaxTopK + 2];
};

constexpr double kOut = -1e300;   // in 64 bits: takes no part; places past E are below

// The groups that take part, in 32 bits: the keys of the others become -infinity.  Returns whether the last of them and
// the first that does not are further apart than tol.
template <int LP, int V>
__device__ __forceinline__ bool choose_groups(const RouteArgs& g, float (&key)[V], int e0, int tok, int lp, float tol,
                                              Space<LP, V>& sp) {
  float* sizes = reinterpret_cast<float*>(sp.size[tok]);
  float a = kNone, b = kNone;
  auto take = [&](float x) {
    b = __builtin_amdgcn_fmed3f(a, b, x);   // (a >= b)
    a = max32(a, x);
  };
  auto join = [&](float a2, float b2) {
    b = __builtin_amdgcn_fmed3f(a, a2, max32(b, b2));   // (the larger second is under both firsts, or between them)
    a = max32(a, a2);
  };
  const int lanes = g.S / V;
  const bool whole = g.S % V == 0 && (lanes & (lanes - 1)) == 0 && lanes <= 16;
  int mine = lp;   // the lane's group, or of a loop's first turn
  if (whole) {
    // a group fills whole lanes, a power of two of them: by those themselves
#pragma unroll
    for (int v = 0; v < V; ++v) take(key[v]);
    if (lanes > 1) join(partner<1>(a), partner<1>(b));
    if (lanes > 2) join(partner<2>(a), partner<2>(b));
    if (lanes > 4) join(partner<4>(a), partner<4>(b));
    if (lanes > 8) join(partner<8>(a), partner<8>(b));
    mine = lp / lanes;
    if (lp % lanes == 0 && mine < g.G) sizes[mine] = g.best > 1 && b > kNone ? a + b : a;
  } else {
    const int G = here(g.G), S = here(g.S);
    lp = here_lane(lp);
    float* keys = reinterpret_cast<float*>(sp.key) + tok * LP * V;
#pragma unroll
    for (int v = 0; v < V; v += 4)
      *reinterpret_cast<float4*>(keys + e0 + v) = make_float4(key[v], key[v + 1], key[v + 2], key[v + 3]);
    wave_sync();
    // P lanes to a group, a power of two (at most 16)
    int P = 1;
    while (2 * P * G <= LP && P < 16) P *= 2;
    for (int gr0 = 0; gr0 < G; gr0 += LP / P) {
      const int gr = gr0 + lp / P;
      a = b = kNone;
      if (gr < G)
        for (int i = lp % P; i < S; i += P) take(keys[gr * S + i]);
      if (P > 1) join(partner<1>(a), partner<1>(b));
      if (P > 2) join(partner<2>(a), partner<2>(b));
      if (P > 4) join(partner<4>(a), partner<4>(b));
      if (P > 8) join(partner<8>(a), partner<8>(b));
      if (gr < G && lp % P == 0) sizes[gr] = g.best > 1 && b > kNone ? a + b : a;
    }
  }
  wave_sync();
  float last = INFINITY, next = kNone;
  bool in = false;
  for (int gr = mine; gr < g.G; gr += LP) {
    const float x = sizes[gr];
    int rank = 0;
    for (int o = 0; o < g.G; ++o) {
      const float y = sizes[o];
      rank += y > x || (y == x && o < gr);
    }
    in = rank < g.top_groups;
    if (in) last = fminf(last, x);
    else next = fmaxf(next, x);
    if (whole) break;
    sp.on[tok][gr] = in;
  }
  last = across<LP>(last, [](float p, float q) { return fminf(p, q); });
  next = across<LP>(next, [](float p, float q) { return fmaxf(p, q); });
  if (whole) {
#pragma unroll
    for (int v = 0; v < V; ++v) key[v] = in ? key[v] : kNone;
  } else {
    wave_sync();
    const int G = here(g.G), S = here(g.S);
    int gr = here_lane(e0) / S, r = e0 - gr * S;
#pragma unroll
    for (int v = 0; v < V; ++v) {
      key[v] = gr < G && sp.on[tok][gr] ? key[v] : kNone;
      if (++r == S) {
        r = 0;
        ++gr;
      }
    }
  }
  return next == kNone || last - next > tol;
}

// A step's tokens in 64 bits, from their (clean) logits: the chosen ids into sp.pick (bit 30: takes no part).  Scores and
// sizes in rolled loops over LDS, the k rounds from registers.  bias: in LDS.
template <int LP, int V, bool SOFTMAX>
__device__ __forceinline__ void choose_exactly(RouteArgs g, const float (&l)[V], const float* bias, int tok, int lp,
                                               Space<LP, V>& sp) {
  constexpr int kAll = LP * V;
  g.E = here(g.E);
  g.G = here(g.G);
  g.S = here(g.S);
  g.k = here(g.k);
  g.top_groups = here(g.top_groups);
  lp = here_lane(lp);
  tok = here_lane(tok);
  const int e0 = lp * V;
  double* key = sp.key + tok * kAll;
  double* sizes = sp.size[tok];
  const bool scores = g.bias || g.G > 1;
#pragma unroll
  for (int v = 0; v < V; ++v) key[e0 + v] = e0 + v < g.E ? (double)l[v] : -INFINITY;
  double m = 0.0, r = 1.0;
  if (SOFTMAX && scores) m = largest<LP, V>(l);
  wave_sync();
  if (scores) {
    if constexpr (SOFTMAX) {
      double z = 0.0;
#pragma unroll 2
      for (int e = lp; e < kAll; e += LP) {
        const double x = key[e];
        z += x > -INFINITY ? exp64(x - m) : 0.0;
      }
      z = across<LP>(z, [](double a, double b) { return a + b; });
      r = inverse64(fmax(z, 1.0));
    }
#pragma unroll 2
    for (int e = lp; e < kAll; e += LP) {
      const double x = key[e];
      const double q = exp64(SOFTMAX ? x - m : -fabs(x)), i = SOFTMAX ? r : inverse64(1.0 + q);
      double s = SOFTMAX || x < 0.0 ? q * i : i;
      if (g.bias) s += (double)bias[e];
      // (a NaN is not above)
      key[e] = e >= g.E ? -INFINITY : x > -INFINITY && s > -INFINITY ? fmin(s, 1e300) : kOut;
    }
    wave_sync();
  }
  if (g.G > 1) {
#pragma unroll 1
    for (int gr = lp; gr < g.G; gr += LP) {
      double a = kOut, b = kOut;
#pragma unroll 4
      for (int i = 0; i < g.S; ++i) {
        const double x = key[gr * g.S + i];
        b = fmax(b, fmin(a, x));
        a = fmax(a, x);
      }
      sizes[gr] = g.best > 1 && b > kOut ? a + b : a;
    }
    wave_sync();
#pragma unroll 1
    for (int gr = lp; gr < g.G; gr += LP) {
      const double x = sizes[gr];
      int rank = 0;
#pragma unroll 4
      for (int o = 0; o < g.G; ++o) {
        const double y = sizes[o];
        rank += y > x || (y == x && o < gr);
      }
      sp.on[tok][gr] = rank < g.top_groups;
    }
    wave_sync();
  }
  double kd[V];
  {
    int gr = g.G > 1 ? e0 / g.S : 0, i = g.G > 1 ? e0 % g.S : 0;
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const bool in = e0 + v < g.E;
      double x = key[e0 + v];
      if (!(x > -INFINITY)) x = kOut;
      if (g.G > 1) {
        if (in && !sp.on[tok][gr]) x = kOut;
        if (++i == g.S) {
          i = 0;
          ++gr;
        }
      }
      if (!g.bias && x > kOut) x = (double)l[v];   // the order of the logits
      kd[v] = in ? x : -INFINITY;
    }
  }
#pragma unroll 1
  for (int j = 0; j < g.k; ++j) {
    double best = kd[0];
#pragma unroll
    for (int v = 1; v < V; ++v) best = fmax(best, kd[v]);
    const double top = across<LP>(best, [](double a, double b) { return fmax(a, b); });
    int at = kAll;
#pragma unroll
    for (int v = V - 1; v >= 0; --v) at = kd[v] == top ? e0 + v : at;
    at = across<LP>(at, [](int a, int b) { return min(a, b); });
#pragma unroll
    for (int v = 0; v < V; ++v) kd[v] = at == e0 + v ? -INFINITY : kd[v];
    if (lp == 0) sp.pick[tok][j] = (uint32_t)at | (top > kOut ? 0u : 1u << 30);
  }
  wave_sync();
}

// (Three blocks a CU: with two or four 33 and 34 us at 32768 x 256.)
// NEAR: a bias or groups, for which the scores of all experts are needed.
template <typename T, int LP, int V, bool SOFTMAX, bool NEAR>
__global__ __launch_bounds__(256, 3) void route_kernel(RouteArgs g) {
  constexpr int kTokens = kWave / LP, kAll = LP * V, L = V < 8 ? V : 8;
  constexpr int kAgain = 64;   // steps of a wave that wait for their 64-bit turn
  constexpr int kIdBits = kAll == 16 ? 4 : kAll == 32 ? 5 : kAll == 64 ? 6 : kAll == 128 ? 7 : kAll == 256 ? 8 : 9;
  static_assert(1 << kIdBits == kAll, "a power of two of places");
  constexpr float kTop = (float)((1 << (kIdBits < 8 ? 23 : 31 - kIdBits)) - 2);   // the largest key's number, exact as a float
  constexpr int kSlots = kMaxTopK / LP + 1;   // of k + 1 chosen ones a lane keeps
  constexpr float kLog2e = 1.44269504088896340736f;
  __shared__ Space<LP, V> space[4];
  __shared__ int s_count[kMaxExpertsWide];
  __shared__ int s_again[4][kAgain];
  __shared__ float s_bias[NEAR ? kAll : 1];
  const int w = threadIdx.x / kWave, lane = lane_id();
  const int tok = lane / LP, lp = lane % LP, e0 = lp * V;
  Space<LP, V>& sp = space[w];
  float* logits = reinterpret_cast<float*>(sp.key) + tok * kAll;   // a token's, by expert
  if (g.counts) {
    for (int e = threadIdx.x; e < g.E; e += 256) s_count[e] = 0;
  }
  if (NEAR && g.bias)
    for (int e = threadIdx.x; e < kAll; e += 256) {
      const float b = e < g.E ? g.bias[e] : 0.0f;   // (past E there is no logit)
      s_bias[e] = b == b ? b : kNone;
    }
  __syncthreads();
  float bias[V], most_bias = 0.0f;   // -infinity for one that is none
  // The unit of the keys' numbers: of logits, 32 below the largest have numbers of their own; of scores with
  // a bias, all.
  float per = (kTop - 2.0f) / 32.0f;
  if (NEAR && g.bias) {
    float lo = 0.0f, hi = 0.0f;
#pragma unroll
    for (int v = 0; v < V; ++v) {
      bias[v] = s_bias[e0 + v];
      lo = bias[v] > kNone ? fminf(lo, bias[v]) : lo;
      hi = fmaxf(hi, bias[v]);
    }
    lo = across<LP>(lo, [](float a, float b) { return fminf(a, b); });
    hi = across<LP>(hi, [](float a, float b) { return fmaxf(a, b); });
    per = (kTop - 2.0f) / (1.0f + (hi - lo));
    most_bias = fmaxf(hi, -lo);
  }
  // The outputs of token t0 + tok's chosen ones (entry i LP + lp of the k): id, logit, whether it takes part; m and z the softmax's.
  auto finish = [&](int t0, const int (&id)[kSlots], const float (&x)[kSlots], const bool (&on)[kSlots], float m, float z)
      __attribute__((always_inline)) {
    const int t = t0 + tok;
    float sc[kSlots], D = 0.0f;
#pragma unroll
    for (int i = 0; i < kSlots; ++i) {
      if constexpr (SOFTMAX) sc[i] = exp_full(x[i] - m) * inverse(z);
      else sc[i] = inverse(1.0f + exp_full(-x[i]));
      sc[i] = on[i] ? sc[i] : 0.0f;
      D += sc[i];
    }
    D = across<(LP < 8 ? LP : 8)>(D, [](float a, float b) { return a + b; });   // (lanes 8 .. hold zeros)
    const float r = g.how & kRouteRenorm ? g.scale / (D + 1e-20f) : g.scale;
#pragma unroll
    for (int i = 0; i < kSlots; ++i) {
      const int j = i * LP + lp;
      if (j < g.k && t < g.N) {
        g.idx[(size_t)t * g.k + j] = id[i] | (on[i] ? 0 : g.how >> 31);
        g.weights[(size_t)t * g.k + j] = sc[i] * r;
        if (g.counts && on[i]) atomicAdd(&s_count[id[i]], 1);
      }
    }
    wave_sync();   // before the next token's
  };
  auto request = [&](int t0, float (&l)[V]) __attribute__((always_inline)) {
    const int t = t0 + tok;
    load_logits<T, V>(g, t < g.N ? t : 0, here_lane(e0), t < g.N, l);
  };
  auto sums = [&](float (&l)[V], float& m, float& z) __attribute__((always_inline)) {
#pragma unroll
    for (int v = 0; v < V; ++v) l[v] = clean(l[v]);
    m = SOFTMAX || NEAR ? largest<LP, V>(l) : 0.0f;
    z = 0.0f;
    if constexpr (SOFTMAX) {
#pragma unroll
      for (int v = 0; v < V; ++v) z += __builtin_amdgcn_exp2f((l[v] - m) * kLog2e);
      z = across<LP>(z, [](float a, float b) { return a + b; });
    }
  };

  const int step = gridDim.x * 4 * kTokens;
  int t0 = (blockIdx.x * 4 + w) * kTokens;
  float ahead[V];   // the next step's logits
  request(t0, ahead);
  while (t0 < g.N) {
    int again = 0;
    for (; t0 < g.N && again < kAgain; t0 += step) {
      float l[V], m, z;
#pragma unroll
      for (int v = 0; v < V; ++v) l[v] = ahead[v];
      request(min(t0 + step, g.N), ahead);
      sums(l, m, z);
      float key[V], tol = 0.0f;
      bool sure = true;
      if constexpr (NEAR) {
        const float r = SOFTMAX ? (z > 0.0f ? inverse(z) : 0.0f) : 1.0f;
#pragma unroll
        for (int v = 0; v < V; ++v) {
          const float s = SOFTMAX ? __builtin_amdgcn_exp2f((l[v] - m) * kLog2e) * r
                                  : inverse(1.0f + __builtin_amdgcn_exp2f(l[v] * -kLog2e));
          key[v] = l[v] > kNone ? g.bias ? s + bias[v] : s : kNone;
        }
        // A key's rounding, of the largest score and bias.  sigmoid: the exponential's argument, 2^-24 |l|, which s (1 - s)
        // scales, |l| that of the largest score where all are small; 1 + e and the reciprocal 1.5 2^-23; the sum
        // 2^-24.  softmax: the arguments' 2^-23 |l - m| s, at most 0.4 2^-23 of the largest, the sum and its reciprocal
        // 2^-22, the rest 2^-23.
        const float big = (SOFTMAX ? r : inverse(1.0f + __builtin_amdgcn_exp2f(m * -kLog2e))) + most_bias;
        tol = big * (SOFTMAX ? 3 * 0x1p-22f : (1.5f + 0.25f * fabsf(m)) * 0x1p-22f);
        if (g.G > 1) sure = choose_groups<LP, V>(g, key, e0, tok, lp, 5 * tol, sp);
        if (!g.bias) {   // the order of the logits, which are exact
#pragma unroll
          for (int v = 0; v < V; ++v) key[v] = key[v] > kNone ? l[v] : kNone;
        }
      } else {
#pragma unroll
        for (int v = 0; v < V; ++v) key[v] = l[v];
      }
      float most = key[0];
#pragma unroll
      for (int v = 1; v < V; ++v) most = max32(most, key[v]);
      most = across<LP>(most, [](float a, float b) { return max32(a, b); });
      most = max32(most, -FLT_MAX);
      // (-infinity converts to 0, as does what is below the unit's reach)
      auto number = [&](float k) __attribute__((always_inline)) {
        return (uint32_t)__builtin_fmaf(k - most, per, kTop);
      };
      uint32_t list[V], head[L];
#pragma unroll
      for (int v = 0; v < V; ++v) {
        // (a place past E is none, and behind all experts that are none)
        list[v] = number(key[v]) << kIdBits | (uint32_t)(kAll - 1 - (e0 + v));
      }
      sort_lane<V>(list, head);
      const int lq = here_lane(lp);
      uint32_t pick[kSlots];
      int popped = 0;
#pragma unroll
      for (int i = 0; i < kSlots; ++i) pick[i] = 0;
#pragma unroll
      for (int j = 0; j <= kMaxTopK; ++j) {
        if (j <= g.k) {
          const uint32_t first = across<LP>(head[0], [](uint32_t a, uint32_t b) { return max(a, b); });
          const uint32_t mine = head[0] == first ? ~0u : 0u;
          // (as bits: a choice between neighbours would become a register index)
#pragma unroll
          for (int i = 0; i < L; ++i) head[i] = (i + 1 < L ? head[i + 1] & mine : 0) | (head[i] & ~mine);
          if constexpr (V > L) popped -= (int)mine;
          pick[j / LP] = lq == j % LP ? first : pick[j / LP];
        }
      }
      // (a list that gave all it had: what follows in the lane is not known)
      if constexpr (V > L) sure = sure && popped < L;
#pragma unroll
      for (int v = 0; v < V; v += 4)
        *reinterpret_cast<float4*>(logits + e0 + v) = make_float4(l[v], l[v + 1], l[v + 2], l[v + 3]);
#pragma unroll
      for (int i = 0; i < kSlots; ++i)
        if (i * LP + lp <= g.k) sp.pick[tok][i * LP + lp] = pick[i];
      wave_sync();
      int id[kSlots];
      float x[kSlots];
      bool on[kSlots];
      const uint32_t near = (uint32_t)fminf(2.0f * tol * per + 4.0f, 0x1p30f);
      float edge = kNone;   // the last chosen one's logit, where the next has the same number
      bool out = false;     // one is chosen that takes no part
#pragma unroll
      for (int i = 0; i < kSlots; ++i) {
        const int j = i * LP + lp;
        const bool in = j < g.k;
        const uint32_t p = in ? pick[i] : 0, n = in ? sp.pick[tok][j + 1] : 0;
        const uint32_t q = p >> kIdBits, qn = n >> kIdBits;
        id[i] = kAll - 1 - (int)(p & (kAll - 1));
        on[i] = q > 0;
        x[i] = in ? logits[id[i]] : kNone;
        // (out of the unit's reach, or of the groups': in no order)
        sure = sure && (q > 0 || x[i] == kNone);
        out = out || (in && q == 0);
        if (qn > 0) {
          if (NEAR && g.bias) {
            sure = sure && q - qn > near;
          } else if (q == qn) {   // equal logits are in order, others not
            sure = sure && x[i] == logits[kAll - 1 - (int)(n & (kAll - 1))];
            if (j + 1 == g.k) edge = x[i];
          }
        }
      }
      if (__ballot(out)) {
        // does one take part that is out of the unit's reach?
#pragma unroll
        for (int v = 0; v < V; ++v)
          if (key[v] > kNone && number(key[v]) == 0) sure = false;
      }
      if (__ballot(edge > kNone)) {
        // are all logits of that number equal?  (those that were not reached may be in any lane)
        const float ex = across<LP>(edge, [](float a, float b) { return fmaxf(a, b); });
        const uint32_t eq = number(ex);
#pragma unroll
        for (int v = 0; v < V; ++v)
          if (eq > 0 && number(key[v]) == eq && key[v] != ex) sure = false;
      }
      if (__ballot(t0 + tok < g.N && !sure)) {
        s_again[w][again++] = t0;
        wave_sync();
      } else {
        finish(t0, id, x, on, m, z);
      }
    }
#pragma unroll 1
    for (int i = 0; i < again; ++i) {
      const int ta = here(__builtin_amdgcn_readfirstlane(s_again[w][i]));
      float l[V], m, z;
      request(ta, l);
      sums(l, m, z);
      choose_exactly<LP, V, SOFTMAX>(g, l, s_bias, tok, lp, sp);
#pragma unroll
      for (int v = 0; v < V; ++v) logits[e0 + v] = l[v];
      wave_sync();
      int id[kSlots];
      float x[kSlots];
      bool on[kSlots];
#pragma unroll
      for (int c = 0; c < kSlots; ++c) {
        const int j = c * LP + lp;
        const uint32_t p = j < g.k ? sp.pick[tok][j] : 1u << 30;
        id[c] = (int)(p & (kAll - 1));
        on[c] = p >> 30 == 0;
        x[c] = logits[id[c]];
      }
      finish(ta, id, x, on, m, z);
    }
    wave_sync();
  }
  if (g.counts) {
    __syncthreads();
    for (int e = threadIdx.x; e < g.E; e += 256)
      if (s_count[e]) atomicAdd(g.counts + e, s_count[e]);
  }
}

template <typename T, int LP, int V, bool SOFTMAX>
__global__ __launch_bounds__(256) void route_backward_kernel(RouteArgs g) {
  constexpr int kTokens = kWave / LP, kSlots = (kMaxTopK + LP - 1) / LP;
  __shared__ float s_all[4][kWave * V];
  const int w = threadIdx.x / kWave, lane = lane_id();
  const int tok = lane / LP, lp = lane % LP, e0 = lp * V;
  float* mine = s_all[w] + tok * LP * V;
  float up[V];
#pragma unroll
  for (int v = 0; v < V; ++v) up[v] = g.dscore && e0 + v < g.E ? g.dscore[e0 + v] : 0.0f;
  const int step = gridDim.x * 4 * kTokens;
  // A step's logits, and the lane's chosen ones (entry i LP + lp of the k), a step ahead.
  struct Step {
    float l[V], w[kSlots], dw[kSlots];
    int e[kSlots];
  };
  auto request = [&](int t0, Step& x) __attribute__((always_inline)) {
    const int t = t0 + tok;
    const bool live = t < g.N;
    load_logits<T, V>(g, live ? t : 0, here_lane(e0), live, x.l);
#pragma unroll
    for (int i = 0; i < kSlots; ++i) {
      const int j = i * LP + lp;
      x.e[i] = 0;
      x.w[i] = x.dw[i] = 0.0f;
      if (j < g.k && live) {
        const size_t f = (size_t)t * g.k + j;
        x.e[i] = g.bidx[f];
        x.w[i] = g.bw[f];
        x.dw[i] = g.dw[f];
      }
    }
  };
  auto plus = [](float a, float b) { return a + b; };
  int t0 = (blockIdx.x * 4 + w) * kTokens;
  Step ahead;
  request(t0, ahead);
  for (; t0 < g.N; t0 += step) {
    const int t = t0 + tok;
    const bool live = t < g.N;
    const Step now = ahead;
    request(min(t0 + step, g.N), ahead);
    float l[V], s[V];
#pragma unroll
    for (int v = 0; v < V; ++v) l[v] = clean(now.l[v]);
    if constexpr (SOFTMAX) {
      softmax_of<LP, V>(l, s);
#pragma unroll
      for (int v = 0; v < V; ++v) mine[e0 + v] = s[v];
    } else {
      // e = exp(-|l|), r = 1 / (1 + e): s = r or e r, and s (1 - s) = e r^2, without a difference
#pragma unroll
      for (int v = 0; v < V; ++v) {
        const float e = exp_full(-fabsf(l[v])), r = inverse(1.0f + e), er = e * r;
        mine[e0 + v] = l[v] >= 0.0f ? r : er;
        s[v] = er * r;
      }
    }
    wave_sync();
    bool on[kSlots];
    float sc[kSlots], D = 0.0f, dot = 0.0f;
#pragma unroll
    for (int i = 0; i < kSlots; ++i) {
      on[i] = now.w[i] != 0.0f && (unsigned)now.e[i] < (unsigned)g.E;
      sc[i] = on[i] ? mine[now.e[i]] : 0.0f;
      D += sc[i];
    }
    float inv = 1.0f;
    if (g.how & kRouteRenorm) {
      D = across<LP>(D, plus);
      inv = 1.0f / (D + 1e-20f);
#pragma unroll
      for (int i = 0; i < kSlots; ++i) dot += on[i] ? now.dw[i] * (sc[i] * inv) : 0.0f;
      dot = across<LP>(dot, plus);
    }
    wave_sync();
#pragma unroll
    for (int v = 0; v < V; ++v) mine[e0 + v] = 0.0f;
    wave_sync();
    const float c = g.scale * inv;
    float sum = 0.0f;   // of ds_e s_e
#pragma unroll
    for (int i = 0; i < kSlots; ++i) {
      const float d = c * (now.dw[i] - dot);
      if (on[i]) {
        mine[now.e[i]] = d;
        sum += d * sc[i];
      }
    }
    // (renormalised, the chosen ones' terms cancel but for 1e-20 of c dot)
    if (g.how & kRouteRenorm) sum = c * dot * 1e-20f;
    else sum = across<LP>(sum, plus);
    wave_sync();
    float ds[V];
#pragma unroll
    for (int v = 0; v < V; ++v) ds[v] = mine[e0 + v] + up[v];
    if constexpr (SOFTMAX) {
      if (g.dscore) {
        float a = 0.0f;
#pragma unroll
        for (int v = 0; v < V; ++v) a += l[v] > kNone ? up[v] * s[v] : 0.0f;
        sum += across<LP>(a, [](float x, float y) { return x + y; });
      }
    }
    float o[V];
#pragma unroll
    for (int v = 0; v < V; ++v) {
      if constexpr (SOFTMAX) o[v] = s[v] * (ds[v] - sum);
      else o[v] = ds[v] * s[v];   // (s (1 - s) there)
      if (!(l[v] > kNone)) o[v] = 0.0f;
    }
    if (live) {
      T* p = reinterpret_cast<T*>(g.dlogits) + (size_t)t * g.E;
      if (g.vec) {
#pragma unroll
        for (int q = 0; q < V; q += 4)
          if (e0 + q < g.E) {
            if constexpr (sizeof(T) == 4)
              *reinterpret_cast<float4*>(p + e0 + q) = make_float4(o[q], o[q + 1], o[q + 2], o[q + 3]);
            else
              *reinterpret_cast<uint2*>(p + e0 + q) =
                  make_uint2(pack_bf16x2(o[q], o[q + 1]), pack_bf16x2(o[q + 2], o[q + 3]));
          }
      } else {
#pragma unroll
        for (int v = 0; v < V; ++v)
          if (e0 + v < g.E) store_act(p + e0 + v, o[v]);
      }
    }
    wave_sync();
  }
}

// bias_e += rate sign(mean count - count_e): experts with more than their share of tokens lose, the others gain.
__global__ __launch_bounds__(512) void route_balance_kernel(const int32_t* __restrict__ counts, int E, float rate,
                                                            float* __restrict__ bias) {
  __shared__ long long s_sum[8];
  const int e = threadIdx.x;
  const long long c = e < E ? counts[e] : 0;
  long long sum = c;
#pragma unroll
  for (int d = 32; d >= 1; d >>= 1) sum += __shfl_xor(sum, d, kWave);
  if (lane_id() == 0) s_sum[e / kWave] = sum;
  __syncthreads();
  sum = 0;
  for (int i = 0; i < 8; ++i) sum += s_sum[i];
  if (e < E && c * E != sum) bias[e] += c * E < sum ? rate : -rate;
}

// (a block: 64 tokens)
__global__ __launch_bounds__(256) void route_take_kernel(const int32_t* from, const float* from_w, int N, int E, int k,
                                                         int32_t* idx, float* w, int32_t* hist, int nb) {
  __shared__ int s_hist[kMaxExpertsWide];
  for (int e = threadIdx.x; e < E; e += 256) s_hist[e] = 0;
  __syncthreads();
  const size_t f0 = (size_t)blockIdx.x * kRouterTokens * k;
  const int n = min(kRouterTokens, N - (int)blockIdx.x * kRouterTokens) * k;
  for (int f = threadIdx.x; f < n; f += 256) {
    int e;
    if (from) {
      e = from[f0 + f];
      const float p = from_w[f0 + f];
      const bool in = (unsigned)e < (unsigned)E && p != 0.0f;
      w[f0 + f] = in ? p : 0.0f;
      e = in ? e : -1;
      idx[f0 + f] = e;
    } else {
      e = idx[f0 + f];
    }
    if (hist && e >= 0) atomicAdd(&s_hist[e], 1);
  }
  if (!hist) return;
  __syncthreads();
  for (int e = threadIdx.x; e < E; e += 256) hist[(size_t)e * nb + blockIdx.x] = s_hist[e];
}

__global__ __launch_bounds__(512) void route_dscore_kernel(const int32_t* __restrict__ counts, int E, int N,
                                                           float alpha, float* __restrict__ dscore) {
  const int e = threadIdx.x;
  if (e < E) dscore[e] = (alpha * (float)E * ((float)counts[e] / (float)N)) / (float)N;
}

// Calls go(lanes per token, experts per lane, softmax) for the config.
template <typename Go>
hipError_t for_route(const mgpt_route_config* cfg, Go go) {
  auto with = [&](auto lp, auto v) {
    cfg->score == MGPT_SCORE_SOFTMAX ? go(lp, v, std::true_type{}) : go(lp, v, std::false_type{});
  };
  auto of = [&](auto lp, auto v) { with(lp, v); };
  const int E = cfg->num_experts;
  typedef std::integral_constant<int, 4> C4;
  typedef std::integral_constant<int, 8> C8;
  typedef std::integral_constant<int, 16> C16;
  typedef std::integral_constant<int, 32> C32;
  if (E <= 16) of(C4{}, C4{});
  else if (E <= 32) of(C4{}, C8{});
  else if (E <= 64) of(C8{}, C8{});
  else if (E <= 128) of(C16{}, C8{});
  else if (E <= 256) of(C16{}, C16{});
  else of(C32{}, C16{});
  return hipGetLastError();
}

}  // namespace

int check_route(const mgpt_route_config* cfg, int N) {
  if (!cfg) return fail(MGPT_ERR_INVALID_ARGUMENT, "config is null");
  if (N < 0) return fail(MGPT_ERR_INVALID_ARGUMENT, "negative num_tokens");
  if (N > 1 << 28) return fail(MGPT_ERR_UNSUPPORTED, "num_tokens %d > 2^28", N);
  if (cfg->num_experts < 1 || cfg->top_k < 1 || cfg->top_k > cfg->num_experts)
    return fail(MGPT_ERR_INVALID_ARGUMENT, "invalid num_experts=%d top_k=%d", cfg->num_experts, cfg->top_k);
  if (cfg->num_experts > kMaxExpertsWide)
    return fail(MGPT_ERR_UNSUPPORTED, "num_experts %d > %d", cfg->num_experts, kMaxExpertsWide);
  if (cfg->top_k > kMaxTopK) return fail(MGPT_ERR_UNSUPPORTED, "top_k %d > %d", cfg->top_k, kMaxTopK);
  if (cfg->score != MGPT_SCORE_SOFTMAX && cfg->score != MGPT_SCORE_SIGMOID)
    return fail(MGPT_ERR_INVALID_ARGUMENT, "unknown score %d", cfg->score);
  if (cfg->groups < 1 || cfg->num_experts % cfg->groups != 0 || cfg->top_groups < 1 || cfg->top_groups > cfg->groups)
    return fail(MGPT_ERR_INVALID_ARGUMENT, "groups %d must divide num_experts %d, top_groups %d be 1 .. groups",
                cfg->groups, cfg->num_experts, cfg->top_groups);
  if (cfg->groups > kMaxExperts) return fail(MGPT_ERR_UNSUPPORTED, "groups %d > %d", cfg->groups, kMaxExperts);
  if (cfg->group_best != 1 && cfg->group_best != 2)
    return fail(MGPT_ERR_INVALID_ARGUMENT, "group_best must be 1 or 2, not %d", cfg->group_best);
  if (!std::isfinite(cfg->scale) || cfg->scale == 0.0f)
    return fail(MGPT_ERR_INVALID_ARGUMENT, "scale must be finite and not 0");
  if (cfg->dtype != MGPT_DTYPE_F32 && cfg->dtype != MGPT_DTYPE_BF16)
    return fail(MGPT_ERR_UNSUPPORTED, "unsupported dtype %d", cfg->dtype);
  return MGPT_OK;
}

RouteArgs route_args(const mgpt_route_config* cfg, const void* logits, const void* dlogits, int N) {
  RouteArgs g{};
  g.logits = logits;
  g.N = N;
  g.E = cfg->num_experts;
  g.k = cfg->top_k;
  g.G = cfg->groups;
  g.S = g.E / g.G;
  g.top_groups = cfg->top_groups;
  g.best = cfg->group_best;
  g.scale = cfg->scale;
  g.how = cfg->renormalise ? kRouteRenorm : 0;
  const uintptr_t row = cfg->dtype == MGPT_DTYPE_F32 ? 16 : 8;
  g.vec = g.E % 4 == 0 && (((uintptr_t)logits | (uintptr_t)dlogits) & (row - 1)) == 0;
  return g;
}

hipError_t launch_route_take(const int32_t* from, const float* from_w, int N, int E, int k, int32_t* idx, float* w,
                             int32_t* hist, hipStream_t st) {
  const int nb = (N + kRouterTokens - 1) / kRouterTokens;
  if (nb <= 0) return hipSuccess;
  if (E > kMaxExpertsWide) return hipErrorInvalidValue;
  hipLaunchKernelGGL(route_take_kernel, dim3(nb), dim3(256), 0, st, from, from_w, N, E, k, idx, w, hist, nb);
  return hipGetLastError();
}

hipError_t launch_route_dscore(const int32_t* counts, int E, int N, float alpha, float* dscore, hipStream_t st) {
  if (E > kMaxExpertsWide) return hipErrorInvalidValue;
  hipLaunchKernelGGL(route_dscore_kernel, dim3(1), dim3(512), 0, st, counts, E, N, alpha, dscore);
  return hipGetLastError();
}

hipError_t launch_route(const mgpt_route_config* cfg, const RouteArgs& g, bool backward, hipStream_t st) {
  return for_route(cfg, [&](auto lp, auto v, auto softmax) {
    constexpr int kLP = decltype(lp)::value, kV = decltype(v)::value;
    constexpr bool kSoftmax = decltype(softmax)::value;
    const int per = 4 * (kWave / kLP);
    const int grid = (int)std::min<long>(((long)g.N + per - 1) / per, (long)compute_units() * (backward ? 8 : 3));
    auto launch = [&](auto kernel) { hipLaunchKernelGGL(kernel, dim3(grid), dim3(256), 0, st, g); };
    const bool f32 = cfg->dtype == MGPT_DTYPE_F32;
    if (backward)
      f32 ? launch(route_backward_kernel<float, kLP, kV, kSoftmax>)
          : launch(route_backward_kernel<bf16_t, kLP, kV, kSoftmax>);
    else if (g.bias || g.G > 1)
      f32 ? launch(route_kernel<float, kLP, kV, kSoftmax, true>) : launch(route_kernel<bf16_t, kLP, kV, kSoftmax, true>);
    else
      f32 ? launch(route_kernel<float, kLP, kV, kSoftmax, false>)
          : launch(route_kernel<bf16_t, kLP, kV, kSoftmax, false>);
  });
}

}  // namespace mgpt

using namespace mgpt;

extern "C" {

int mgpt_route_forward(const mgpt_route_config* cfg, const void* logits, const float* bias, int32_t* idx,
                       float* weights, int32_t* counts, int num_tokens, void* stream) {
  if (int rc = check_route(cfg, num_tokens)) return rc;
  if (num_tokens == 0) return MGPT_OK;
  if (!logits || !idx || !weights) return fail(MGPT_ERR_INVALID_ARGUMENT, "null logits, idx or weights");
  RouteArgs g = route_args(cfg, logits, nullptr, num_tokens);
  g.bias = bias;
  g.idx = idx;
  g.weights = weights;
  g.counts = counts;
  HIP_TRY(launch_route(cfg, g, false, (hipStream_t)stream));
  return MGPT_OK;
}

int mgpt_route_backward(const mgpt_route_config* cfg, const void* logits, const int32_t* idx, const float* weights,
                        const float* dweights, const float* dscores, void* dlogits, int num_tokens, void* stream) {
  if (int rc = check_route(cfg, num_tokens)) return rc;
  if (num_tokens == 0) return MGPT_OK;
  if (!logits || !idx || !weights || !dweights || !dlogits)
    return fail(MGPT_ERR_INVALID_ARGUMENT, "null logits, idx, weights, dweights or dlogits");
  RouteArgs g = route_args(cfg, logits, dlogits, num_tokens);
  g.bidx = idx;
  g.bw = weights;
  g.dw = dweights;
  g.dscore = dscores;
  g.dlogits = dlogits;
  HIP_TRY(launch_route(cfg, g, true, (hipStream_t)stream));
  return MGPT_OK;
}

int mgpt_route_balance(int num_experts, const int32_t* counts, float rate, float* bias, void* stream) {
  if (num_experts < 1) return fail(MGPT_ERR_INVALID_ARGUMENT, "invalid num_experts %d", num_experts);
  if (num_experts > kMaxExpertsWide)
    return fail(MGPT_ERR_UNSUPPORTED, "num_experts %d > %d", num_experts, kMaxExpertsWide);
  if (!std::isfinite(rate)) return fail(MGPT_ERR_INVALID_ARGUMENT, "rate must be finite");
  if (!counts || !bias) return fail(MGPT_ERR_INVALID_ARGUMENT, "null counts or bias");
  hipLaunchKernelGGL(route_balance_kernel, dim3(1), dim3(512), 0, (hipStream_t)stream, counts, num_experts, rate,
                     bias);
  HIP_TRY(hipGetLastError());
  return MGPT_OK;
}

}  // extern "C"
