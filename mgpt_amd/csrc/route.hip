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
//   w_j = c s_j / D,  D = sum_j s_j + 1e-20 (renormalised) or 1
// Backward, for the upstream gradients dw of the weights and g_e of expert e's score in every token:
//   d_j = (c dw_j - sum_i dw_i w_i) / D (or c dw_j),  ds = g + d scattered to the chosen ones
//   sigmoid: dl = ds s (1 - s),   softmax: dl = s (ds - sum_e ds_e s_e)
//
// A token's experts lie in LP lanes of a wave, V neighbouring ones in each, so that 64 / LP tokens
// share a wave, and stay in registers; the token's own LDS holds what lanes look up by expert (scores
// for the groups, the gradient's scatter).  A choice is k rounds of a maximum over V registers and LP lanes.
//
// Keys with a bias, and sizes of groups, are those of 64 bits: fp32 ones, 2^-20 of a score off at
// most, decide where the values that are compared are further apart than that, and otherwise the
// wave does the token again in 64 bits.
#include <algorithm>
#include <cfloat>
#include <cmath>
#include <type_traits>

#include "capi_internal.hpp"
#include "route.hpp"

namespace mgpt {

namespace {

constexpr float kNone = -INFINITY;

// exp to 1.5 ulp: the product with log2 e in two parts around the hardware's exponential.
__device__ __forceinline__ float exp_full(float x) {
  const float y = x * 1.44269504088896340736f;
  const float r = __builtin_fmaf(x, 1.44269504088896340736f, -y) + x * 1.925963033500869e-8f;
  const float e = __builtin_amdgcn_exp2f(y);
  return y > -INFINITY && y < 128.0f ? __builtin_fmaf(e, r * 0.693147180559945f, e) : e;
}

template <int CTRL>
__device__ __forceinline__ float dpp(float v) {
  return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, 0xf, 0xf, false));
}
template <int CTRL>
__device__ __forceinline__ int dpp(int v) {
  return __builtin_amdgcn_update_dpp(0, v, CTRL, 0xf, 0xf, false);
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
__device__ __forceinline__ float larger(float a, float b) { return fmaxf(a, b); }
__device__ __forceinline__ double larger(double a, double b) { return fmax(a, b); }
__device__ __forceinline__ float smaller(float a, float b) { return fminf(a, b); }
__device__ __forceinline__ double smaller(double a, double b) { return fmin(a, b); }
__device__ __forceinline__ float exp_of(float x) { return exp_full(x); }
__device__ __forceinline__ double exp_of(double x) { return exp(x); }
__device__ __forceinline__ float inverse(float x) { return 1.0f / x; }
__device__ __forceinline__ double inverse(double x) { return 1.0 / x; }

// Orders a wave's own LDS accesses across its lanes.
__device__ __forceinline__ void wave_sync() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
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
#pragma unroll
    for (int v = 0; v < V; ++v)
      if (e0 + v < g.E) l[v] = to_f32(p[e0 + v]);
  }
}

// An infinity or a NaN among the logits, out of the way.
__device__ __forceinline__ float clean(float l) { return l != l ? kNone : fminf(l, FLT_MAX); }

template <int LP, int V, bool SOFTMAX, typename K>
__device__ __forceinline__ void scores_of(const float (&l)[V], K (&s)[V]) {
  if constexpr (SOFTMAX) {
    float m = l[0];
#pragma unroll
    for (int v = 1; v < V; ++v) m = fmaxf(m, l[v]);
    m = across<LP>(m, [](float a, float b) { return fmaxf(a, b); });
    m = fmaxf(m, -FLT_MAX);   // a row without experts
    K z = 0;
#pragma unroll
    for (int v = 0; v < V; ++v) {
      s[v] = exp_of((K)l[v] - (K)m);
      z += s[v];
    }
    z = across<LP>(z, [](K a, K b) { return a + b; });
    const K r = z > 0 ? inverse(z) : (K)0;
#pragma unroll
    for (int v = 0; v < V; ++v) s[v] *= r;
  } else {
#pragma unroll
    for (int v = 0; v < V; ++v) s[v] = inverse((K)1 + exp_of(-(K)l[v]));
  }
}

// What a wave keeps in LDS: for each of its tokens the scores (or gradients) by expert, the sizes of the
// groups, and the chosen experts with their scores.
template <int LP, int V>
struct Space {
  static constexpr int kTokens = kWave / LP;
  static constexpr int kGroups = LP * V < kMaxExperts ? LP * V : kMaxExperts;
  double key[kWave * V];
  double size[kTokens][kGroups + 2];
  int on[kTokens][kGroups];
  int id[kTokens][kMaxTopK];
  float score[kTokens][kMaxTopK];
};

// The groups that take part, in sp.on; returns whether the last of them and the first that does
// not are further apart than `tol`.
template <int LP, int V, typename K>
__device__ __forceinline__ bool choose_groups(const RouteArgs& g, const K (&key)[V], int e0, int tok, int lp, K tol,
                                              Space<LP, V>& sp) {
  K* keys = reinterpret_cast<K*>(sp.key) + tok * LP * V;
  K* sizes = reinterpret_cast<K*>(sp.size[tok]);
#pragma unroll
  for (int v = 0; v < V; ++v) keys[e0 + v] = key[v];
  wave_sync();
  // P lanes to a group, a power of two
  int P = 1;
  while (2 * P * g.G <= LP) P *= 2;
  const K none = -INFINITY;
  for (int gr0 = 0; gr0 < g.G; gr0 += LP / P) {
    const int gr = gr0 + lp / P;
    K a = none, b = none;
    if (gr < g.G)
      for (int i = lp % P; i < g.S; i += P) {
        const K x = keys[gr * g.S + i];
        b = larger(b, smaller(a, x));
        a = larger(a, x);
      }
    auto join = [&](K a2, K b2) {
      b = larger(smaller(a, a2), larger(b, b2));
      a = larger(a, a2);
    };
    if (P > 1) join(partner<1>(a), partner<1>(b));
    if (P > 2) join(partner<2>(a), partner<2>(b));
    if (P > 4) join(partner<4>(a), partner<4>(b));
    if (P > 8) join(partner<8>(a), partner<8>(b));
    if constexpr (LP > 16)
      if (P > 16) join(partner<16>(a), partner<16>(b));
    if (gr < g.G && lp % P == 0) sizes[gr] = g.best > 1 && b > none ? a + b : a;
  }
  if (lp == 0) sizes[g.G] = sizes[g.G + 1] = none;
  wave_sync();
  for (int gr = lp; gr < g.G; gr += LP) {
    const K x = sizes[gr];
    int rank = 0;
    for (int o = 0; o < g.G; ++o) rank += sizes[o] > x || (sizes[o] == x && o < gr);
    sp.on[tok][gr] = rank < g.top_groups;
    // (a lane of another group reads only the first G)
    if (rank == g.top_groups - 1) sizes[g.G] = x;
    if (rank == g.top_groups) sizes[g.G + 1] = x;
  }
  wave_sync();
  const K last = sizes[g.G], next = sizes[g.G + 1];
  return next == none || last - next > tol;
}

// k rounds over the keys; the chosen ids and scores into sp.  Returns whether neighbours
// in the order, the first that was not chosen among them, are further apart than `tol`
// (tol < 0: whether equal ones are in order is known).
template <int LP, int V, typename K>
__device__ __forceinline__ bool choose(const RouteArgs& g, K (&key)[V], const float (&s)[V], unsigned taken, int e0,
                                       int tok, int lp, K tol, Space<LP, V>& sp) {
  const K none = -INFINITY;
  bool sure = true;
  K last = INFINITY;
  const int rounds = tol >= 0 ? g.k + 1 : g.k;
  for (int j = 0; j < rounds; ++j) {
    K m = none;
#pragma unroll
    for (int v = 0; v < V; ++v)
      if (!(taken >> v & 1)) m = larger(m, key[v]);
    m = across<LP>(m, [](K a, K b) { return larger(a, b); });
    if (tol >= 0 && j > 0) sure &= m == none || last - m > tol;
    last = m;
    if (j == g.k) break;
    int e = INT_MAX;
#pragma unroll
    for (int v = V - 1; v >= 0; --v)
      if (!(taken >> v & 1) && key[v] == m) e = e0 + v;
    const int mine = e;
    e = across<LP>(e, [](int a, int b) { return min(a, b); });
    if (mine == e) {
#pragma unroll
      for (int v = 0; v < V; ++v)
        if (e == e0 + v) {
          taken |= 1u << v;
          sp.id[tok][j] = e;
          sp.score[tok][j] = m > none ? s[v] : -1.0f;   // (-1: takes no part)
        }
    }
  }
  return sure;
}

template <typename T, int LP, int V, bool SOFTMAX>
__global__ __launch_bounds__(256) void route_kernel(RouteArgs g) {
  constexpr int kTokens = kWave / LP;
  __shared__ Space<LP, V> space[4];
  __shared__ int s_count[kMaxExpertsWide];
  const int w = threadIdx.x / kWave, lane = lane_id();
  const int tok = lane / LP, lp = lane % LP, e0 = lp * V;
  Space<LP, V>& sp = space[w];
  if (g.counts) {
    for (int e = threadIdx.x; e < g.E; e += 256) s_count[e] = 0;
    __syncthreads();
  }
  float bias[V];
  int grp[V];
#pragma unroll
  for (int v = 0; v < V; ++v) {
    const bool in = e0 + v < g.E;
    bias[v] = in && g.bias ? g.bias[e0 + v] : 0.0f;
    grp[v] = in ? (e0 + v) / g.S : 0;
  }
  unsigned out = 0;   // lanes' places past E
#pragma unroll
  for (int v = 0; v < V; ++v) out |= (unsigned)(e0 + v >= g.E) << v;

  const int step = gridDim.x * 4 * kTokens;
  for (int t0 = (blockIdx.x * 4 + w) * kTokens; t0 < g.N; t0 += step) {
    const int t = t0 + tok;
    const bool live = t < g.N;
    float l[V], s[V];
    load_logits<T, V>(g, live ? t : 0, e0, live, l);
#pragma unroll
    for (int v = 0; v < V; ++v) l[v] = clean(l[v]);
    scores_of<LP, V, SOFTMAX, float>(l, s);

    // keys of one precision, the groups by them, the choice
    auto decide = [&](auto zero) {
      typedef decltype(zero) K;
      constexpr bool kExact = sizeof(K) == 8;
      K sk[V], key[V];
      if constexpr (kExact) {
        scores_of<LP, V, SOFTMAX, K>(l, sk);
      } else {
#pragma unroll
        for (int v = 0; v < V; ++v) sk[v] = s[v];
      }
      K big = 0;   // of what the rounding of fp32 keys goes by
#pragma unroll
      for (int v = 0; v < V; ++v) {
        const K x = sk[v] + (K)bias[v];
        key[v] = l[v] > kNone && x == x ? x : (K)kNone;
        if (!kExact && key[v] > kNone) big = larger(big, larger(sk[v], (K)fabsf((float)key[v])));
      }
      K tol = -1;
      if constexpr (!kExact) tol = across<LP>(big, [](K a, K b) { return larger(a, b); }) * (K)0x1p-18f;
      bool sure = true;
      if (g.G > 1) {
        sure = choose_groups<LP, V, K>(g, key, e0, tok, lp, 2 * tol, sp);
#pragma unroll
        for (int v = 0; v < V; ++v)
          if (!sp.on[tok][grp[v]]) key[v] = (K)kNone;
      }
      if (g.bias) return choose<LP, V, K>(g, key, s, out, e0, tok, lp, kExact ? (K)-1 : tol, sp) && sure;
      // the order of the logits, which fp32 holds exactly
      float lk[V];
#pragma unroll
      for (int v = 0; v < V; ++v) lk[v] = key[v] > (K)kNone ? l[v] : kNone;
      return choose<LP, V, float>(g, lk, s, out, e0, tok, lp, -1.0f, sp) && sure;
    };
    const bool sure = decide(0.0f);
    if (__ballot(live && !sure)) {
      wave_sync();
      decide(0.0);
    }
    wave_sync();
    float D = 0.0f;
    for (int j = 0; j < g.k; ++j) D += fmaxf(sp.score[tok][j], 0.0f);
    const float r = g.renorm ? g.scale / (D + 1e-20f) : g.scale;
    for (int j = lp; j < g.k; j += LP) {
      const float x = sp.score[tok][j];
      if (live) {
        g.idx[(size_t)t * g.k + j] = sp.id[tok][j];
        g.weights[(size_t)t * g.k + j] = x > 0.0f ? x * r : 0.0f;
        if (g.counts && x >= 0.0f) atomicAdd(&s_count[sp.id[tok][j]], 1);
      }
    }
    wave_sync();   // before the next token's
  }
  if (g.counts) {
    __syncthreads();
    for (int e = threadIdx.x; e < g.E; e += 256)
      if (s_count[e]) atomicAdd(g.counts + e, s_count[e]);
  }
}

template <typename T, int LP, int V, bool SOFTMAX>
__global__ __launch_bounds__(256) void route_backward_kernel(RouteArgs g) {
  constexpr int kTokens = kWave / LP;
  __shared__ float s_all[4][kWave * V];
  const int w = threadIdx.x / kWave, lane = lane_id();
  const int tok = lane / LP, lp = lane % LP, e0 = lp * V;
  float* mine = s_all[w] + tok * LP * V;
  float up[V];
#pragma unroll
  for (int v = 0; v < V; ++v) up[v] = g.dscore && e0 + v < g.E ? g.dscore[e0 + v] : 0.0f;
  const int step = gridDim.x * 4 * kTokens;
  for (int t0 = (blockIdx.x * 4 + w) * kTokens; t0 < g.N; t0 += step) {
    const int t = t0 + tok;
    const bool live = t < g.N;
    float l[V], s[V];
    load_logits<T, V>(g, live ? t : 0, e0, live, l);
#pragma unroll
    for (int v = 0; v < V; ++v) l[v] = clean(l[v]);
    scores_of<LP, V, SOFTMAX, float>(l, s);
#pragma unroll
    for (int v = 0; v < V; ++v) mine[e0 + v] = s[v];
    wave_sync();
    // the chosen experts, the same in all of the token's lanes
    int id[kMaxTopK];
    float sc[kMaxTopK], dw[kMaxTopK];
    float D = 0.0f, dot = 0.0f;
#pragma unroll
    for (int j = 0; j < kMaxTopK; ++j) {
      id[j] = -1;
      sc[j] = dw[j] = 0.0f;
      if (j < g.k && live) {
        const int e = g.bidx[(size_t)t * g.k + j];
        const float wj = g.bw[(size_t)t * g.k + j];
        if (wj != 0.0f && (unsigned)e < (unsigned)g.E) {
          id[j] = e;
          sc[j] = mine[e];
          dw[j] = g.dw[(size_t)t * g.k + j];
          D += sc[j];
        }
      }
    }
    float inv = 1.0f;
    if (g.renorm) {
      inv = 1.0f / (D + 1e-20f);
#pragma unroll
      for (int j = 0; j < kMaxTopK; ++j) dot += dw[j] * (sc[j] * inv);
    }
    wave_sync();
#pragma unroll
    for (int v = 0; v < V; ++v) mine[e0 + v] = 0.0f;
    wave_sync();
    const float c = g.scale * inv;
    float sum = 0.0f;   // of ds_e s_e
#pragma unroll
    for (int j = 0; j < kMaxTopK; ++j) {
      const float d = c * (dw[j] - dot);
      if (id[j] >= 0 && lp == j % LP) mine[id[j]] = d;
      // (renormalised, the chosen ones' terms cancel but for 1e-20 of c dot)
      if (!g.renorm && id[j] >= 0) sum += d * sc[j];
    }
    if (g.renorm) sum = c * dot * 1e-20f;
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
      // (1 - s from the other side: s may be near 1)
      if constexpr (SOFTMAX) o[v] = s[v] * (ds[v] - sum);
      else o[v] = ds[v] * (s[v] * inverse(1.0f + exp_full(l[v])));
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
      const bool in = (unsigned)e < (unsigned)E;
      w[f0 + f] = in ? from_w[f0 + f] : 0.0f;
      e = in ? e : 0;
      idx[f0 + f] = e;
    } else {
      e = idx[f0 + f];
    }
    if (hist) atomicAdd(&s_hist[e], 1);
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

int compute_units() {
  int dev = 0, n = 0;
  if (hipGetDevice(&dev) != hipSuccess ||
      hipDeviceGetAttribute(&n, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess || n <= 0)
    return 256;
  return n;
}

// Calls go(lanes per token, experts per lane, softmax) for the config.
template <typename Go>
hipError_t for_route(const mgpt_route_config* cfg, Go go) {
  auto with = [&](auto lp, auto v) {
    cfg->score == MGPT_SCORE_SOFTMAX ? go(lp, v, std::true_type{}) : go(lp, v, std::false_type{});
  };
  const int E = cfg->num_experts;
  if (E <= 16) with(std::integral_constant<int, 4>{}, std::integral_constant<int, 4>{});
  else if (E <= 32) with(std::integral_constant<int, 8>{}, std::integral_constant<int, 4>{});
  else if (E <= 64) with(std::integral_constant<int, 16>{}, std::integral_constant<int, 4>{});
  else if (E <= 128) with(std::integral_constant<int, 32>{}, std::integral_constant<int, 4>{});
  else if (E <= 256) with(std::integral_constant<int, 64>{}, std::integral_constant<int, 4>{});
  else with(std::integral_constant<int, 64>{}, std::integral_constant<int, 8>{});
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
  g.renorm = cfg->renormalise;
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
    const int grid = (int)std::min<long>(((long)g.N + per - 1) / per, (long)compute_units() * 8);
    auto launch = [&](auto kernel) { hipLaunchKernelGGL(kernel, dim3(grid), dim3(256), 0, st, g); };
    const bool f32 = cfg->dtype == MGPT_DTYPE_F32;
    if (backward)
      f32 ? launch(route_backward_kernel<float, kLP, kV, kSoftmax>)
          : launch(route_backward_kernel<bf16_t, kLP, kV, kSoftmax>);
    else
      f32 ? launch(route_kernel<float, kLP, kV, kSoftmax>) : launch(route_kernel<bf16_t, kLP, kV, kSoftmax>);
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
