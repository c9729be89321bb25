// sample.hip -- a token for each row of logits from a given random number, by temperature,
// top-k, top-p and min-p.
//
// Reference: the Generator's sampling (pipeline/Generator.cpp:13-36), which copies the logits to the host.  Here,
// with l the logits (NaN as -infinity, each at most FLT_MAX), ordered by (l descending, id ascending):
//   w_i = rint(2^40 exp((l_i - max l) / T))
//   kept: the first top_k; of those the ones before which less than top_p of their sum lies; of those
//         the ones with w_i >= min_p 2^40, and always the first
//   token: the first, by id, at which the running sum of the kept w exceeds u times their sum
// Weights are whole numbers, so that their sums, formed by many threads and atomics in LDS, have no
// order; exp is a polynomial in 64 bits, which this card runs at the rate of 32.  All three
// filters keep a prefix of the order, (a logit, how many of those equal to it), so nothing is sorted: the
// prefix's end is found in a histogram of 1024 bins along the exponent, and within its bin by the bits of the logits.
//
// A block takes a row and reads it once per pass: maximum, histogram (of counts, of weights), the bin's
// logits, and the draw, whose pieces of the row are summed and then searched.
#include <cfloat>
#include <cmath>

#include "../../include/mgpt_moe.h"
#include "capi_internal.hpp"
#include "common.hpp"

namespace mgpt {
namespace {

typedef unsigned long long u64;

constexpr int kThreads = 1024, kWaves = kThreads / kWave;
constexpr int kBins = 1024;          // of 1/16 of a power of two of weight; the last holds weights of 0
constexpr int kList = 4096;          // logits of a bin that LDS takes
constexpr int kMaxVocab = 1 << 20;
constexpr double kUnits = 0x1p40;

struct SampleArgs {
  const void* logits;      // [B][V]
  const float* u;          // [B]
  const float *T, *p, *m;  // [B], or null: the values below
  const int32_t* k;
  float T0, p0, m0;
  int k0;
  int32_t* token;          // [B]
  float* logp;             // [B] or null
  int V;
};

__device__ __forceinline__ float clean_logit(float l) { return l != l ? -INFINITY : fminf(l, FLT_MAX) + 0.0f; }
// Unsigned numbers in the order of floats (-0 is +0 by then).
__device__ __forceinline__ uint32_t order_of(float l) {
  const uint32_t b = __float_as_uint(l);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float logit_of(uint32_t k) {
  return __uint_as_float(k & 0x80000000u ? k & 0x7FFFFFFFu : ~k);
}

struct Scale {
  float top;       // the row's largest logit
  double c;        // log2(e) / T
  float c32;       // the same for the bins
};

// rint(2^40 2^t), t = (l - top) c <= 0: 2^t by its whole part and a polynomial of degree 10 on [-1/2, 1/2]
// (least maximum relative error, 2^-52).
__device__ __forceinline__ u64 weight_of(float l, const Scale& s) {
  const double t = ((double)l - (double)s.top) * s.c;
  if (!(t > -42.0)) return 0;   // (also -infinity, and its product with 0)
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
  // times 2^(n + 40), to the nearest whole number, in the low bits
  const double v = __builtin_ldexp(q, (int)n + 40) + 0x1p52;
  return (u64)__double_as_longlong(v) & 0xFFFFFFFFFFFFFull;
}

__device__ __forceinline__ int bin_of(float l, const Scale& s) {
  return (int)fminf((s.top - l) * s.c32 * 16.0f, (float)(kBins - 1));   // (NaN, from 0 times infinity: the last)
}

template <typename T>
__device__ __forceinline__ T wave_scan(T v) {   // inclusive
#pragma unroll
  for (int d = 1; d < kWave; d <<= 1) {
    const T o = __shfl_up(v, d, kWave);
    if (lane_id() >= d) v += o;
  }
  return v;
}

// 16 bytes at any element of a row.
typedef uint32_t vec_f32 __attribute__((ext_vector_type(4), aligned(4)));
typedef uint32_t vec_bf16 __attribute__((ext_vector_type(4), aligned(2)));
template <typename T> struct VecOf { typedef vec_f32 type; };
template <> struct VecOf<bf16_t> { typedef vec_bf16 type; };

// Eight (bf16) or four (fp32) neighbouring logits of a row at any element.
template <typename T>
struct Piece {
  static constexpr int N = 16 / sizeof(T);
  float l[N];
  __device__ __forceinline__ void load(const T* row, int i, int V) {
    if (i + N <= V) {
      const u32x4 w = *reinterpret_cast<const typename VecOf<T>::type*>(row + i);
#pragma unroll
      for (int q = 0; q < N; ++q) {
        if constexpr (sizeof(T) == 4) l[q] = __uint_as_float(w[q]);
        else l[q] = __uint_as_float(q & 1 ? w[q / 2] & 0xFFFF0000u : w[q / 2] << 16);
      }
    } else {
#pragma unroll
      for (int q = 0; q < N; ++q) l[q] = i + q < V ? to_f32(row[i + q]) : -INFINITY;
    }
#pragma unroll
    for (int q = 0; q < N; ++q) l[q] = clean_logit(l[q]);
  }
};

// The end of a prefix of the order: the logits above `key`, and the first n of those equal to it.
struct End {
  uint32_t key;
  int n;
};

struct Shared {
  u64 bins[kBins];
  int sizes[kBins];
  u64 digit[256];
  int digit_n[256];
  uint32_t list[kList];
  u64 red[kWaves];
  u64 found[4];
  int count;
};

template <typename T>
struct Row {
  const T* p;
  int V;
  // f(logit, id) of every logit of the row that the block's threads share out; past the end: -infinity
  template <typename F>
  __device__ __forceinline__ void each(F f) const {
    for (int i = threadIdx.x * Piece<T>::N; i < V; i += kThreads * Piece<T>::N) {
      Piece<T> x;
      x.load(p, i, V);
#pragma unroll
      for (int q = 0; q < Piece<T>::N; ++q) f(x.l[q], i + q);
    }
  }
};

// By wave 0: of n entries with sum(i) in all and size(i) items, `base` lying before the first, the last one with
// items before which less than `bound` lies, or the first with items: found[0] its index, [1] what lies before it,
// [2] the entries' sum.
template <typename Sum, typename Size>
__device__ __forceinline__ void find_end(int n, u64 base, double bound, Sum sum, Size size, u64* found) {
  const int lane = lane_id();
  const int per = n / kWave;   // (n is a multiple)
  u64 mine = 0;
  for (int i = 0; i < per; ++i) mine += sum(lane * per + i);
  const u64 incl = wave_scan(mine);
  u64 before = base + incl - mine, at_before = 0;
  int at = -1;
  for (int i = 0; i < per; ++i) {
    const int e = lane * per + i;
    if (size(e) > 0 && ((double)before < bound || before == base)) {
      at = e;
      at_before = before;
    }
    before += sum(e);
  }
  const unsigned long long m = __ballot(at >= 0);
  const int owner = m ? 63 - __builtin_clzll(m) : 0;
  const u64 all = __shfl(incl, kWave - 1, kWave);
  at = __shfl(at, owner, kWave);
  at_before = __shfl(at_before, owner, kWave);
  if (lane == 0) {
    found[0] = (u64)max(at, 0);
    found[1] = at_before;
    found[2] = all;
  }
}

// Of the logits that `in` admits, the end of the prefix whose items have less than `bound` of weight(l) before
// them, `before` lying before the first of all: the last such logit's key, how many have it, and what lies before
// it in *at.  Four rounds over 8 bits of the keys; from the list in LDS (n of them) or, n < 0, from
// the row.
template <typename T, typename In, typename W>
__device__ __forceinline__ End refine(const Row<T>& row, Shared& sh, int n, u64 before, double bound, In in, W weight,
                                      u64* at) {
  uint32_t prefix = 0;
  int equal = 0;
  for (int shift = 24; shift >= 0; shift -= 8) {
    __syncthreads();
    if (threadIdx.x < 256) {
      sh.digit[threadIdx.x] = 0;
      sh.digit_n[threadIdx.x] = 0;
    }
    __syncthreads();
    auto add = [&](uint32_t key) {
      if (shift < 24 && (key >> (shift + 8)) != (prefix >> (shift + 8))) return;
      const int d = 255 - (int)(key >> shift & 255);   // the largest first
      atomicAdd(&sh.digit[d], weight(logit_of(key)));
      atomicAdd(&sh.digit_n[d], 1);
    };
    if (n >= 0) {
      for (int i = threadIdx.x; i < n; i += kThreads) add(sh.list[i]);
    } else {
      row.each([&](float l, int i) {
        if (i < row.V && in(l)) add(order_of(l));
      });
    }
    __syncthreads();
    if (threadIdx.x < kWave)
      find_end(256, before, bound, [&](int i) { return sh.digit[i]; }, [&](int i) { return sh.digit_n[i]; }, sh.found);
    __syncthreads();
    const int d = (int)sh.found[0];
    before = sh.found[1];
    equal = sh.digit_n[d];
    prefix |= (uint32_t)(255 - d) << shift;
  }
  __syncthreads();
  *at = before;
  return {prefix, equal};
}

// How many of n items of weight w, `before` before the first, have less than `bound` before them.
__device__ __forceinline__ int under(u64 before, u64 w, int n, double bound) {
  int lo = 0, hi = n;   // the first of which it does not hold
  while (lo < hi) {
    const int mid = (lo + hi) / 2;
    if ((double)(before + (u64)mid * w) < bound) lo = mid + 1;
    else hi = mid;
  }
  return lo;
}

template <typename T>
__global__ __launch_bounds__(kThreads) void sample_kernel(SampleArgs g) {
  __shared__ Shared sh;
  extern __shared__ u64 pieces[];   // per piece of the row (a wave's load): its weights' sum, how many have the end's key
  const int b = blockIdx.x, tid = threadIdx.x, wave = tid / kWave, lane = lane_id();
  const Row<T> row{reinterpret_cast<const T*>(g.logits) + (size_t)b * g.V, g.V};
  const int V = g.V;
  const float temp = g.T ? g.T[b] : g.T0, min_p = g.m ? g.m[b] : g.m0, top_p = g.p ? g.p[b] : g.p0;
  int k = g.k ? g.k[b] : g.k0;
  const float ur = g.u[b];

  // the largest logit, and its lowest id
  u64 best = 0;   // key, then the id's complement
  row.each([&](float l, int i) {
    const u64 x = (u64)order_of(l) << 32 | (uint32_t)~(uint32_t)i;
    if (i < V && x > best) best = x;
  });
#pragma unroll
  for (int d = 32; d >= 1; d >>= 1) {
    const u64 o = __shfl_xor(best, d, kWave);
    best = o > best ? o : best;
  }
  if (lane == 0) sh.red[wave] = best;
  __syncthreads();
  best = sh.red[0];
#pragma unroll
  for (int i = 1; i < kWaves; ++i) best = sh.red[i] > best ? sh.red[i] : best;
  const float top = logit_of((uint32_t)(best >> 32));
  const bool empty = !(top > -INFINITY);
  if (empty || !(temp > 0.0f) || k == 1 || min_p > 1.0f) {
    if (tid == 0) {
      g.token[b] = empty ? -1 : (int)~(uint32_t)best;
      if (g.logp) g.logp[b] = empty ? -INFINITY : 0.0f;
    }
    return;
  }
  Scale s;
  s.top = top;
  s.c = 1.4426950408889634 / (double)temp;
  s.c32 = fminf((float)s.c, 1e30f);

  // top_k: the end of the first k
  End end{0, 0};   // everything
  if (k > 0 && k < V) {
    for (int i = tid; i < kBins; i += kThreads) sh.sizes[i] = 0;
    if (tid == 0) sh.count = 0;
    __syncthreads();
    row.each([&](float l, int i) {
      if (i < V) atomicAdd(&sh.sizes[bin_of(l, s)], 1);
    });
    __syncthreads();
    if (tid < kWave)
      find_end(kBins, 0, (double)k, [&](int i) { return (u64)sh.sizes[i]; }, [&](int i) { return sh.sizes[i]; }, sh.found);
    __syncthreads();
    const int bin = (int)sh.found[0];
    const u64 before = sh.found[1];
    const int n = sh.sizes[bin];
    // (the last bin's weights are 0: whether they are kept makes no difference)
    if (bin < kBins - 1) {
      auto in = [&](float l) { return bin_of(l, s) == bin; };
      if (n <= kList) {
        row.each([&](float l, int i) {
          if (i < V && in(l)) sh.list[atomicAdd(&sh.count, 1)] = order_of(l);
        });
      }
      u64 at;
      end = refine(row, sh, n <= kList ? n : -1, before, (double)k, in, [](float) { return (u64)1; }, &at);
      end.n = min(end.n, k - (int)at);
    }
  }
  const u64 w_k = end.key ? weight_of(logit_of(end.key), s) : 0;

  // top_p: the end of the prefix before whose items less than top_p of the sum lies
  if (top_p < 1.0f) {
    for (int i = tid; i < kBins; i += kThreads) {
      sh.bins[i] = 0;
      sh.sizes[i] = 0;
    }
    if (tid == 0) sh.count = 0;
    __syncthreads();
    row.each([&](float l, int i) {
      const u64 w = i < V && order_of(l) > end.key ? weight_of(l, s) : 0;
      if (w) {
        const int e = bin_of(l, s);
        atomicAdd(&sh.bins[e], w);
        atomicAdd(&sh.sizes[e], 1);
      }
    });
    __syncthreads();
    const int bin_k = end.key ? bin_of(logit_of(end.key), s) : kBins - 1;
    if (tid == 0 && w_k) {
      sh.bins[bin_k] += (u64)end.n * w_k;
      sh.sizes[bin_k] += end.n;
    }
    __syncthreads();
    auto sum = [&](int i) { return sh.bins[i]; };
    auto size = [&](int i) { return sh.sizes[i]; };
    if (tid < kWave) find_end(kBins, 0, 0.0, sum, size, sh.found);
    __syncthreads();
    const double bound = fmax((double)top_p * (double)sh.found[2], 0.0);
    __syncthreads();
    if (tid < kWave) find_end(kBins, 0, bound, sum, size, sh.found);
    __syncthreads();
    const int bin = (int)sh.found[0];
    const u64 before = sh.found[1];
    const int ties = w_k && bin == bin_k ? end.n : 0;   // of the k's last logit, the bin's smallest
    const int n = sh.sizes[bin] - ties;
    u64 tie_before = before;
    End cut = end;
    bool found = false;
    auto in = [&](float l) { return bin_of(l, s) == bin && order_of(l) > end.key && weight_of(l, s) > 0; };
    if (n > 0) {
      if (n <= kList) {
        row.each([&](float l, int i) {
          if (i < V && in(l)) sh.list[atomicAdd(&sh.count, 1)] = order_of(l);
        });
      }
      u64 at;
      const End e = refine(row, sh, n <= kList ? n : -1, before, bound, in, [&](float l) { return weight_of(l, s); }, &at);
      const u64 w = weight_of(logit_of(e.key), s);
      cut = {e.key, max(1, under(at, w, e.n, bound))};
      tie_before = before + sh.bins[bin] - (u64)ties * w_k;
      found = true;
    }
    if (ties > 0 && (!found || (double)tie_before < bound)) cut = {end.key, max(found ? 0 : 1, under(tie_before, w_k, ties, bound))};
    end = cut;
    __syncthreads();
  }

  // The draw: sums of the kept weights above the end's key, and the numbers of that key, by piece.
  constexpr int kPiece = kWave * Piece<T>::N;
  const int num_pieces = (V + kPiece - 1) / kPiece;
  int* piece_n = reinterpret_cast<int*>(pieces + num_pieces);
  const double least = (double)min_p * kUnits;
  const u64 w_end = end.key ? weight_of(logit_of(end.key), s) : 0;
  auto kept = [&](float l) -> u64 {   // of a logit above the end's key
    const u64 w = weight_of(l, s);
    return (double)w >= least ? w : 0;
  };
  const u64 tie = end.key && (double)w_end >= least ? w_end : 0;
  for (int c = wave; c < num_pieces; c += kWaves) {
    Piece<T> x;
    const int i = c * kPiece + lane * Piece<T>::N;
    u64 sum = 0;
    int eq = 0;
    if (i < V) {
      x.load(row.p, i, V);
#pragma unroll
      for (int q = 0; q < Piece<T>::N; ++q) {
        const uint32_t key = order_of(x.l[q]);
        if (i + q < V) {
          if (key > end.key) sum += kept(x.l[q]);
          eq += key == end.key;
        }
      }
    }
#pragma unroll
    for (int d = 32; d >= 1; d >>= 1) {
      sum += __shfl_xor(sum, d, kWave);
      eq += __shfl_xor(eq, d, kWave);
    }
    if (lane == 0) {
      pieces[c] = sum;
      piece_n[c] = eq;
    }
  }
  __syncthreads();
  if (wave > 0) return;

  // One wave: the piece, the lane, the logit where the running sum passes u times the whole.
  const int per = (num_pieces + kWave - 1) / kWave;
  const int c0 = min(lane * per, num_pieces), c1 = min(c0 + per, num_pieces);
  int eq = 0;
  for (int c = c0; c < c1; ++c) eq += piece_n[c];
  const int eq_before = wave_scan(eq) - eq;
  auto ties_of = [&](int before, int n) { return (u64)max(0, min(end.n - before, n)); };
  u64 mine = 0;
  {
    int e = eq_before;
    for (int c = c0; c < c1; ++c) {
      mine += pieces[c] + ties_of(e, piece_n[c]) * tie;
      e += piece_n[c];
    }
  }
  const u64 incl = wave_scan(mine);
  const u64 total = __shfl(incl, kWave - 1, kWave);
  const double target = (double)(ur > 0.0f ? ur : 0.0f) * (double)total;
  auto past = [&](u64 run) { return (double)run > target || run >= total; };
  const int owner = __ffsll((long long)__ballot(past(incl))) - 1;   // (the last lane's is the total)
  u64 run = __shfl(incl - mine, owner, kWave);
  int seen = __shfl(eq_before, owner, kWave);
  const int first = __shfl(c0, owner, kWave), last = __shfl(c1, owner, kWave);
  int c = first;
  for (; c < last - 1; ++c) {
    const u64 w = pieces[c] + ties_of(seen, piece_n[c]) * tie;
    if (past(run + w)) break;
    run += w;
    seen += piece_n[c];
  }
  const int i = c * kPiece + lane * Piece<T>::N;
  Piece<T> x;
  u64 w[Piece<T>::N];
  bool is_tie[Piece<T>::N];
  int le = 0;
#pragma unroll
  for (int q = 0; q < Piece<T>::N; ++q) {
    w[q] = 0;
    is_tie[q] = false;
    x.l[q] = -INFINITY;
  }
  if (i < V) {
    x.load(row.p, i, V);
#pragma unroll
    for (int q = 0; q < Piece<T>::N; ++q)
      if (i + q < V) {
        const uint32_t key = order_of(x.l[q]);
        if (key > end.key) w[q] = kept(x.l[q]);
        is_tie[q] = key == end.key;
        le += is_tie[q];
      }
  }
  int e = seen + wave_scan(le) - le;
  u64 sum = 0;
#pragma unroll
  for (int q = 0; q < Piece<T>::N; ++q) {
    if (is_tie[q]) {
      if (e < end.n) w[q] = tie;
      ++e;
    }
    sum += w[q];
  }
  u64 here = run + wave_scan(sum) - sum;
  int id = -1;
  float l = 0.0f;
#pragma unroll
  for (int q = 0; q < Piece<T>::N; ++q) {
    here += w[q];
    if (id < 0 && w[q] && past(here)) {
      id = i + q;
      l = x.l[q];
    }
  }
  const unsigned long long hit = __ballot(id >= 0);
  const int who = hit ? __ffsll((long long)hit) - 1 : 0;
  if (lane == who) {
    g.token[b] = id;
    if (g.logp) {
      const double z = ((double)l - (double)top) / (double)temp;
      g.logp[b] = (float)(z - log((double)total / kUnits));
    }
  }
}

}  // namespace
}  // namespace mgpt

using namespace mgpt;

extern "C" {

int mgpt_sample(const mgpt_sample_config* cfg, const void* logits, const float* u, const float* temperature,
                const int32_t* top_k, const float* top_p, const float* min_p, int32_t* token, float* logp, int num_rows,
                void* stream) {
  if (!cfg) return fail(MGPT_ERR_INVALID_ARGUMENT, "config is null");
  if (num_rows < 0) return fail(MGPT_ERR_INVALID_ARGUMENT, "negative num_rows");
  if (num_rows > 1 << 24) return fail(MGPT_ERR_UNSUPPORTED, "num_rows %d > 2^24", num_rows);
  if (cfg->vocab_size < 1) return fail(MGPT_ERR_INVALID_ARGUMENT, "invalid vocab_size=%d", cfg->vocab_size);
  if (cfg->vocab_size > kMaxVocab) return fail(MGPT_ERR_UNSUPPORTED, "vocab_size %d > %d", cfg->vocab_size, kMaxVocab);
  if (cfg->dtype != MGPT_DTYPE_F32 && cfg->dtype != MGPT_DTYPE_BF16)
    return fail(MGPT_ERR_UNSUPPORTED, "unsupported dtype %d", cfg->dtype);
  if (!temperature && !(cfg->temperature >= 0.0f))
    return fail(MGPT_ERR_INVALID_ARGUMENT, "temperature must be >= 0");
  if (!top_p && !(cfg->top_p >= 0.0f)) return fail(MGPT_ERR_INVALID_ARGUMENT, "top_p must be >= 0");
  if (!min_p && !(cfg->min_p >= 0.0f)) return fail(MGPT_ERR_INVALID_ARGUMENT, "min_p must be >= 0");
  if (num_rows == 0) return MGPT_OK;
  if (!logits || !u || !token) return fail(MGPT_ERR_INVALID_ARGUMENT, "null logits, u or token");
  SampleArgs g{};
  g.logits = logits;
  g.u = u;
  g.T = temperature;
  g.p = top_p;
  g.m = min_p;
  g.k = top_k;
  g.T0 = cfg->temperature;
  g.p0 = cfg->top_p;
  g.m0 = cfg->min_p;
  g.k0 = cfg->top_k;
  g.token = token;
  g.logp = logp;
  g.V = cfg->vocab_size;
  const bool f32 = cfg->dtype == MGPT_DTYPE_F32;
  const int piece = kWave * (f32 ? 4 : 8);
  const size_t lds = ((size_t)(g.V + piece - 1) / piece) * 12;
  if (f32) hipLaunchKernelGGL(sample_kernel<float>, dim3(num_rows), dim3(kThreads), lds, (hipStream_t)stream, g);
  else hipLaunchKernelGGL(sample_kernel<bf16_t>, dim3(num_rows), dim3(kThreads), lds, (hipStream_t)stream, g);
  HIP_TRY(hipGetLastError());
  return MGPT_OK;
}

}  // extern "C"
