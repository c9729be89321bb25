// sample.hip -- a token for each row of logits from a given random number, by temperature,
// top-k, top-p and min-p.
//
// Reference: the Generator's sampling (pipeline/Generator.cpp:13-36), which copies the logits to the host.  Here,
// with l the logits (NaN as -infinity, each at most FLT_MAX), ordered by (l descending, id ascending):
//   w_i = rint(2^40 exp((l_i - max l) / T))
//   kept: the first top_k; of those the ones before which less than top_p of their sum lies; of those
//         the ones with w_i >= min_p 2^40, and always the first
//   token: the first, by id, at which the running sum of the kept w exceeds u times their sum
// Weights are whole numbers, so that their sums, formed by many threads and atomics, have no
// order; exp is a polynomial in 64 bits, which this card runs at the rate of 32.  All three
// filters keep a prefix of the order, (a logit, how many of those equal to it), so nothing but a short list is ever
// sorted: the prefix's end is found in a histogram of 1024 bins along the exponent, and within its bin by the bits of the
// logits.
//
// Long rows are cut into chunks, a block each, and the steps are launches (a row's parameters, which may lie on the
// device, say which of them it needs):
//   max:   the chunks' largest logits
//   scan:  top-k: histogram of counts; else top-p: of weights; else: the weights' sums, by piece (a wave's load)
//   list:  top-k: the logits down to its bin, else top-p: those of its bin; the rest: the draw
//   cut:   top-k: a block does all else from the list; top-p: the end from the list, then the pieces' sums
//   draw:  top-p: the draw; and whole rows by one block where a list did not hold (top_k above kFew, thousands
//          of equal logits)
// Short rows are done whole, by a block each, in one launch.
//
// Measured: 256 rows of 131072 bf16 with top_p and min_p 101 us, of it max 14 (4.7 TB/s), scan 26 (38 with the 26 vector
// instructions of a weight for every logit), list 24, cut 35, draw 8; 64 rows of 100003 fp32, all open, 32 us; one
// row of 50257 with top_k 25 us, of it five launches' latency; one of 8192 16 us.  A block for each row and all
// steps took 191, 71 and 61 us for the first three.
#include <algorithm>
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
constexpr int kList = 4096;          // logits that a list takes
constexpr int kMaxVocab = 1 << 20;
constexpr double kUnits = 0x1p40;

constexpr int kFew = 1024;           // top_k up to which the list serves
constexpr int kFewer = 256;          // logits of a list that need no sorting
constexpr uint32_t kValues = 4096;   // of bf16, counted by themselves: 16 powers of two of either sign
constexpr uint32_t kLeastValue = (127 - 8) << 7;   // 2^-8
constexpr int kCopies = 4;           // of a block's histogram, so that a wave's lanes meet less
constexpr int kChunkThreads = 256, kChunkWaves = kChunkThreads / kWave;
constexpr int kMaxChunks = 64;

struct End;
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
  // in chunks: workspace
  int chunks, pieces;      // of a row
  u64* best;               // [B][chunks]: key, then the id's complement
  u64* bins;               // [B][kBins]
  u64* list;               // [B][kList]: as best
  u64* sums;               // [B][pieces]
  int* ties;               // [B][pieces]
  int* list_n;             // [B]
  End* cut;                // [B]
};

// NaN counts as -infinity, infinity as the largest number (of a NaN and two numbers the median is the smaller one;
// in assembly, since the compiler makes a minimum of it, which is not).  -0 stays.
__device__ __forceinline__ float clean_logit(float l) {
  float r;
  asm("v_med3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(l), "v"(-INFINITY), "v"(FLT_MAX));
  return r;
}
// Unsigned numbers in the order of floats, -0 as +0.
__device__ __forceinline__ uint32_t order_of(float l) {
  const uint32_t b = __float_as_uint(l + 0.0f);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float logit_of(uint32_t k) {
  return __uint_as_float(k & 0x80000000u ? k & 0x7FFFFFFFu : ~k);
}

struct Scale {
  float top;            // the row's largest logit
  float c32;            // log2(e) / T, for counts
  double c;             // log2(e) / T
  const double* pow;    // 2^(40 + j/16), in LDS: 16 of them lie on 32 banks
};
__constant__ double kPow[16] = {
    0x1.0000000000000p+40, 0x1.0b5586cf9890fp+40, 0x1.172b83c7d517bp+40, 0x1.2387a6e756238p+40,
    0x1.306fe0a31b715p+40, 0x1.3dea64c123422p+40, 0x1.4bfdad5362a27p+40, 0x1.5ab07dd485429p+40,
    0x1.6a09e667f3bcdp+40, 0x1.7a11473eb0187p+40, 0x1.8ace5422aa0dbp+40, 0x1.9c49182a3f090p+40,
    0x1.ae89f995ad3adp+40, 0x1.c199bdd85529cp+40, 0x1.d5818dcfba487p+40, 0x1.ea4afa2a490dap+40};
__device__ __forceinline__ void lay_out_pow(double* pow) {   // (before a __syncthreads)
  if (threadIdx.x < 16) pow[threadIdx.x] = kPow[threadIdx.x];
}

// rint(2^40 2^t), t = (l - top) c <= 0, and its bin, -16 t to the nearest: 2^t by its sixteenths and a polynomial of
// degree 6 on [-1/32, 1/32] (least maximum relative error, 2^-57).
__device__ __forceinline__ u64 weight_of(float l, const Scale& s, int* bin) {
  const double t = fmax(((double)l - (double)s.top) * s.c, -60.0);   // (also -infinity, and its product with 0)
  const double m = t + 0x1.8p48, f = t - (m - 0x1.8p48);
  const int j = (int)__double_as_longlong(m);   // 16 t
  double q = 0x1.4307dc964c652p-13;
  q = __builtin_fma(q, f, 0x1.5d89be48923e6p-10);
  q = __builtin_fma(q, f, 0x1.3b2ab6feace08p-7);
  q = __builtin_fma(q, f, 0x1.c6b08d6e8a411p-5);
  q = __builtin_fma(q, f, 0x1.ebfbdff82c53cp-3);
  q = __builtin_fma(q, f, 0x1.62e42fefa39fdp-1);
  q = __builtin_fma(q, f, 1.0);
  *bin = -j;
  // to the nearest whole number, in the low bits
  const double v = __builtin_ldexp(q * s.pow[j & 15], j >> 4) + 0x1p52;
  return (u64)__double_as_longlong(v) & 0xFFFFFFFFFFFFFull;
}
__device__ __forceinline__ u64 weight_of(float l, const Scale& s) {
  int bin;
  return weight_of(l, s, &bin);
}

// The bins of counts, which need no weight: by 32 bits, and cut off instead of rounded.
__device__ __forceinline__ int bin_of(float l, const Scale& s) {
  return (int)fminf((s.top - l) * (s.c32 * 16.0f), (float)(kBins - 1));   // (NaN, from 0 times infinity: the last)
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

__device__ __forceinline__ uint32_t bits_of(float x) { return __float_as_uint(x); }
__device__ __forceinline__ uint32_t bits_of(bf16_t x) { return __builtin_bit_cast(uint16_t, x); }

// Eight (bf16) or four (fp32) neighbouring logits of a row at any element.
template <typename T>
struct Piece {
  static constexpr int N = 16 / sizeof(T);
  u32x4 w;
  // (past the row's end: -infinity)
  __device__ __forceinline__ void load(const T* row, int i, int V) {
    if (i + N <= V) {
      w = *reinterpret_cast<const typename VecOf<T>::type*>(row + i);
    } else {
      constexpr uint32_t kNone = sizeof(T) == 4 ? 0xFF800000u : 0xFF80u;
#pragma unroll
      for (int q = 0; q < 4; ++q) w[q] = 0;
#pragma unroll
      for (int q = 0; q < N; ++q) {
        uint32_t x = kNone;
        if (i + q < V) x = bits_of(row[i + q]);
        if constexpr (sizeof(T) == 4) w[q] = x;
        else w[q / 2] |= x << 16 * (q & 1);
      }
    }
  }
  __device__ __forceinline__ float raw(int q) const {
    if constexpr (sizeof(T) == 4) return __uint_as_float(w[q]);
    else return __uint_as_float(q & 1 ? w[q / 2] & 0xFFFF0000u : w[q / 2] << 16);
  }
  __device__ __forceinline__ uint32_t bits(int q) const {   // T's own
    if constexpr (sizeof(T) == 4) return w[q];
    else return q & 1 ? w[q / 2] >> 16 : w[q / 2] & 0xFFFF;
  }
  __device__ __forceinline__ float operator[](int q) const { return clean_logit(raw(q)); }
};

// Pieces first, first + step, ... below last of a row, by a wave, two on their way from the start on.
template <typename T>
struct Pieces {
  const T* row;
  int V, first, last, step;
  Piece<T> x[2];
  __device__ __forceinline__ int at(int c) const { return (c * kWave + lane_id()) * Piece<T>::N; }
  __device__ __forceinline__ void start() {
    if (first >= last) return;
    x[0].load(row, at(first), V);
    x[1] = x[0];
    if (first + step < last) x[1].load(row, at(first + step), V);
  }
  // f(piece, its number)
  template <typename F>
  __device__ __forceinline__ void run(F f) {
    for (int c = first; c < last; c += step) {
      Piece<T> then = x[1];
      if (c + 2 * step < last) then.load(row, at(c + 2 * step), V);
      f(x[0], c);
      x[0] = x[1];
      x[1] = then;
    }
  }
  // f(logit, id) of every logit; past the row's end: -infinity
  template <typename F>
  __device__ __forceinline__ void each(F f) {
    run([&](const Piece<T>& p, int c) {
#pragma unroll
      for (int q = 0; q < Piece<T>::N; ++q) f(p[q], at(c) + q);
    });
  }
};

// f(logit, its place, whether it is one) of the logits in `hits`, each lane's next one in every round: in a piece there
// are few as a rule.
template <typename T, typename F>
__device__ __forceinline__ void each_hit(const Piece<T>& x, uint32_t hits, F f) {
  while (__any(hits != 0)) {
    const int q = __ffs(hits) - 1;
    uint32_t w = x.w[0];
    constexpr int kPer = Piece<T>::N / 4;
#pragma unroll
    for (int k = 1; k < 4; ++k) w = q >= k * kPer ? x.w[k] : w;
    if constexpr (kPer == 2) w = q & 1 ? w & 0xFFFF0000u : w << 16;
    f(clean_logit(__uint_as_float(w)), q, hits != 0);
    hits &= hits - 1;
  }
}

// The end of a prefix of the order: the logits above `key`, and the first n of those equal to it.
struct End {
  uint32_t key;
  int n;
};

// LDS of finish_few.
template <int WAVES>
struct FewShared {
  u64 key[kFewer], weight[kFewer];
  u64 red[WAVES];
};

struct Shared {
  union {
    u64 bins[kBins];
    FewShared<kWaves> few;
  };
  int sizes[kBins];
  u64 digit[256];
  int digit_n[256];
  uint32_t list[kList];
  u64 red[kWaves];
  u64 found[4];
  double pow[16];
  int count;
};

struct Params {
  float temp, top_p, min_p, u;
  int k;
};
__device__ __forceinline__ Params params_of(const SampleArgs& g, int b) {
  const float m = g.m ? g.m[b] : g.m0;
  return {g.T ? g.T[b] : g.T0, g.p ? g.p[b] : g.p0, m > 0.0f ? m : 0.0f, g.u[b], g.k ? g.k[b] : g.k0};
}
__device__ __forceinline__ Scale scale_of(float top, float temp, const double* pow) {
  Scale s;
  s.top = top;
  s.c = 1.4426950408889634 / (double)temp;
  s.c32 = fminf((float)s.c, 1e30f);
  s.pow = pow;
  return s;
}
// Whether the row is its largest logit, or nothing; then its outputs, by one thread.
__device__ __forceinline__ bool settled(const SampleArgs& g, int b, const Params& p, u64 best, bool writer) {
  const bool empty = !(logit_of((uint32_t)(best >> 32)) > -INFINITY);
  if (!empty && p.temp > 0.0f && p.k != 1 && !(p.min_p > 1.0f)) return false;
  if (writer) {
    g.token[b] = empty ? -1 : (int)~(uint32_t)best;
    if (g.logp) g.logp[b] = empty ? -INFINITY : 0.0f;
  }
  return true;
}
__device__ __forceinline__ u64 larger(u64 a, u64 b) { return a > b ? a : b; }

// What the draw goes by: the weights kept above the end's key, and of each with that key.
struct Kept {
  Scale s;
  End end;
  float at;       // the end's logit, or NaN
  float from;     // below it, no logit above the end has `least`
  u64 least;      // min_p in units
  u64 tie;
  __device__ __forceinline__ u64 operator()(float l) const {
    const u64 w = weight_of(l, s);
    return w >= least ? w : 0;
  }
};
__device__ __forceinline__ Kept kept_of(const Scale& s, End end, float min_p) {
  Kept k;
  k.s = s;
  k.end = end;
  const double least = (double)min_p * kUnits;   // (at most kUnits: more has been settled)
  k.least = (u64)ceil(least);
  // (a weight is the nearest whole number, so it has `least` units from half a unit below on; wider by more than the
  // logarithm's error; the difference's rounding to 32 bits passes no logit)
  const double span = k.least > 0 ? 40.01 - (double)log2f((float)((double)k.least - 0.5)) : 42.0;
  k.from = fmaxf((float)((double)s.top - span / s.c), -FLT_MAX);
  k.at = __builtin_nanf("");
  k.tie = 0;
  if (end.key) {
    k.at = logit_of(end.key);
    k.from = fmaxf(k.from, logit_of(end.key + 1));
    k.tie = k(k.at);
  }
  return k;
}

// The kept weights of a piece above the end's key, and how many have that key: in every lane of the wave.
template <typename T>
__device__ __forceinline__ void piece_sum(const Piece<T>& piece, const Kept& kept, u64* sum, int* ties) {
  constexpr int N = Piece<T>::N;
  float x[N];
  u64 w = 0;
  int eq = 0;
  uint32_t hits = 0;
#pragma unroll
  for (int q = 0; q < N; ++q) {   // (past V: -infinity, below all)
    x[q] = piece[q];
    hits |= x[q] >= kept.from ? 1u << q : 0;
    eq += x[q] == kept.at;
  }
  if (__any(__popc(hits) > N / 2)) {
#pragma unroll
    for (int q = 0; q < N; ++q)
      if (hits >> q & 1) w += kept(x[q]);
  } else {
    each_hit(piece, hits, [&](float l, int, bool is) { w += is ? kept(l) : 0; });
  }
  if (__any(w != 0))
#pragma unroll
    for (int d = 32; d >= 1; d >>= 1) w += __shfl_xor(w, d, kWave);
  if (__any(eq != 0))
#pragma unroll
    for (int d = 32; d >= 1; d >>= 1) eq += __shfl_xor(eq, d, kWave);
  *sum = w;
  *ties = eq;
}

// The same of pieces, into sums and ties.
template <typename T>
__device__ __forceinline__ void piece_sums(Pieces<T>& pieces, const Kept& kept, u64* sums, int* ties) {
  pieces.run([&](const Piece<T>& x, int c) {
    u64 sum;
    int eq;
    piece_sum(x, kept, &sum, &eq);
    if (lane_id() == 0) {
      sums[c] = sum;
      ties[c] = eq;
    }
  });
}

// By one wave: the piece, the lane, the logit at which the running sum passes u times the whole.
template <typename T>
__device__ __forceinline__ void draw(const SampleArgs& g, int b, const T* row, const Params& p, const Kept& kept,
                                     const u64* sums, const int* ties, int num) {
  constexpr int N = Piece<T>::N;
  const int lane = lane_id();
  const int per = (num + kWave - 1) / kWave;
  const int c0 = min(lane * per, num), c1 = min(c0 + per, num);
  int eq = 0;
  for (int c = c0; c < c1; ++c) eq += ties[c];
  const int eq_before = wave_scan(eq) - eq;
  auto ties_of = [&](int before, int n) { return (u64)max(0, min(kept.end.n - before, n)); };
  u64 mine = 0;
  {
    int e = eq_before;
    for (int c = c0; c < c1; ++c) {
      mine += sums[c] + ties_of(e, ties[c]) * kept.tie;
      e += ties[c];
    }
  }
  const u64 incl = wave_scan(mine);
  const u64 total = __shfl(incl, kWave - 1, kWave);
  const double target = (double)(p.u > 0.0f ? p.u : 0.0f) * (double)total;
  auto past = [&](u64 run) { return (double)run > target || run >= total; };
  const int owner = __ffsll((long long)__ballot(past(incl))) - 1;   // (the last lane's is the total)
  u64 run = __shfl(incl - mine, owner, kWave);
  int seen = __shfl(eq_before, owner, kWave);
  const int last = __shfl(c1, owner, kWave);
  int c = __shfl(c0, owner, kWave);
  for (; c < last - 1; ++c) {
    const u64 w = sums[c] + ties_of(seen, ties[c]) * kept.tie;
    if (past(run + w)) break;
    run += w;
    seen += ties[c];
  }
  const int i = (c * kWave + lane) * N;
  Piece<T> piece;
  float x[N];
  u64 w[N];
  bool is_tie[N];
  int le = 0;
#pragma unroll
  for (int q = 0; q < N; ++q) {
    w[q] = 0;
    is_tie[q] = false;
    x[q] = -INFINITY;
  }
  if (i < g.V) {
    piece.load(row, i, g.V);
#pragma unroll
    for (int q = 0; q < N; ++q)
      if (i + q < g.V) {
        x[q] = piece[q];
        if (x[q] >= kept.from) w[q] = kept(x[q]);
        is_tie[q] = x[q] == kept.at;
        le += is_tie[q];
      }
  }
  int e = seen + wave_scan(le) - le;
  u64 sum = 0;
#pragma unroll
  for (int q = 0; q < N; ++q) {
    if (is_tie[q]) {
      if (e < kept.end.n) w[q] = kept.tie;
      ++e;
    }
    sum += w[q];
  }
  u64 here = run + wave_scan(sum) - sum;
  int id = -1;
  float l = 0.0f;
#pragma unroll
  for (int q = 0; q < N; ++q) {
    here += w[q];
    if (id < 0 && w[q] && past(here)) {
      id = i + q;
      l = x[q];
    }
  }
  const unsigned long long hit = __ballot(id >= 0);
  if (lane == (hit ? __ffsll((long long)hit) - 1 : 0)) {
    g.token[b] = id;
    if (g.logp) {
      const double z = ((double)l - (double)kept.s.top) / (double)p.temp;
      g.logp[b] = (float)(z - log((double)total / kUnits));
    }
  }
}

template <typename T, int THREADS>
struct Row {
  const T* p;
  int V;
  __device__ __forceinline__ Pieces<T> pieces() const {
    constexpr int kPiece = kWave * Piece<T>::N;
    Pieces<T> x{p, V, (int)threadIdx.x / kWave, (V + kPiece - 1) / kPiece, THREADS / kWave};
    x.start();
    return x;
  }
  // f(logit, id) of every logit of the row that the block's threads share out; past the end: -infinity
  template <typename F>
  __device__ __forceinline__ void each(F f) const {
    Pieces<T> x = pieces();
    x.each(f);
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
// it in *at.  Rounds over up to 8 bits of the keys in which they differ; from the list in LDS (n of them, at least one)
// or, n < 0, from the row.
template <int THREADS, typename T, typename S, typename In, typename W>
__device__ __forceinline__ End refine(const Row<T, THREADS>& row, S& sh, int n, u64 before, double bound, In in, W weight,
                                      u64* at) {
  uint32_t prefix = 0;
  int equal = 0, high = 32, low = 0;   // the bits to be found: [low, high)
  if (n >= 0) {
    if (threadIdx.x == 0) sh.digit_n[0] = 0;
    __syncthreads();   // (the list is written)
    prefix = sh.list[0];
    uint32_t differ = 0;
    for (int i = threadIdx.x; i < n; i += THREADS) differ |= sh.list[i] ^ prefix;
#pragma unroll
    for (int d = 32; d >= 1; d >>= 1) differ |= __shfl_xor(differ, d, kWave);
    if (lane_id() == 0) atomicOr(&sh.digit_n[0], (int)differ);
    __syncthreads();
    differ = (uint32_t)sh.digit_n[0];
    if (differ == 0) differ = 1;   // (one round, for its sums)
    high = 32 - __builtin_clz(differ);
    low = __builtin_ctz(differ);
    prefix &= ~((u64)(1ull << high) - 1) | ((1u << low) - 1);
  }
  while (high > low) {
    const int width = min(8, high - low), shift = high - width;
    __syncthreads();
    if (threadIdx.x < 256) {
      sh.digit[threadIdx.x] = 0;
      sh.digit_n[threadIdx.x] = 0;
    }
    __syncthreads();
    const uint32_t ones = (1u << width) - 1;
    auto add = [&](uint32_t key) {
      if (((u64)(key ^ prefix) >> high) != 0) return;
      const int d = (int)(ones - (key >> shift & ones));   // the largest first
      atomicAdd(&sh.digit[d], weight(logit_of(key)));
      atomicAdd(&sh.digit_n[d], 1);
    };
    if (n >= 0) {
      for (int i = threadIdx.x; i < n; i += THREADS) add(sh.list[i]);
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
    prefix |= (ones - (uint32_t)d) << shift;
    high = shift;
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

// Sums of v over the threads before this one, and of all, in the order of the threads.
template <int WAVES>
__device__ __forceinline__ u64 block_scan(u64 v, u64* red, u64* all) {
  const u64 incl = wave_scan(v);
  __syncthreads();
  if (lane_id() == kWave - 1) red[threadIdx.x / kWave] = incl;
  __syncthreads();
  u64 before = incl - v;
  *all = 0;
#pragma unroll
  for (int i = 0; i < WAVES; ++i) {
    if (i < (int)threadIdx.x / kWave) before += red[i];
    *all += red[i];
  }
  return before;
}

// The token of a row from the running sums of its kept weights: this logit's, `before` it, of `all`.
__device__ __forceinline__ void draw_one(const SampleArgs& g, int b, const Params& p, const Scale& s, u64 x, u64 w,
                                         u64 before, u64 all) {
  const double target = (double)(p.u > 0.0f ? p.u : 0.0f) * (double)all;
  auto past = [&](u64 r) { return (double)r > target || r >= all; };
  if (!w || (before > 0 && past(before)) || !past(before + w)) return;
  g.token[b] = (int)~(uint32_t)x;
  if (g.logp) {
    const double z = ((double)logit_of((uint32_t)(x >> 32)) - (double)s.top) / (double)p.temp;
    g.logp[b] = (float)(z - log((double)all / kUnits));
  }
}

// The rest of a top_k row from a short list, x a thread's logit of it: places and sums of a logit by comparison with all others.
template <int THREADS>
__device__ __forceinline__ void finish_few(const SampleArgs& g, int b, const Params& p, const Scale& s, int n, u64 x,
                                           FewShared<THREADS / kWave>& sh) {
  static_assert(kFewer <= THREADS, "a logit a thread");
  const int t = threadIdx.x;
  u64 w = t < n ? weight_of(logit_of((uint32_t)(x >> 32)), s) : 0;
  if (t < kFewer) {
    sh.key[t] = x;
    sh.weight[t] = w;
  }
  __syncthreads();
  int place = 0;
  u64 before = 0;
#pragma unroll 4
  for (int j = 0; j < n; ++j) {
    const bool above = sh.key[j] > x;
    place += above;
    before += above ? sh.weight[j] : 0;
  }
  u64 all;
  block_scan<THREADS / kWave>(place < p.k ? w : 0, sh.red, &all);   // (its syncs end the reads above)
  const bool keep = place < p.k && (place == 0 || (((double)before < (double)p.top_p * (double)all || !(p.top_p < 1.0f)) &&
                                                   (double)w >= (double)p.min_p * kUnits));
  if (!keep) w = 0;
  if (t < kFewer) sh.weight[t] = w;
  __syncthreads();
  before = 0;
  all = 0;
#pragma unroll 4
  for (int j = 0; j < n; ++j) {
    const u64 o = sh.weight[j];
    all += o;
    before += (uint32_t)sh.key[j] > (uint32_t)x ? o : 0;   // (the ids' complements)
  }
  draw_one(g, b, p, s, x, w, before, all);
}

// The end of top_p among n <= kList logits of a bin (sh.list) and the `ties` that are its smallest, `before` lying
// before them; weights' sum of the bin.
template <int THREADS, typename T, typename S, typename In>
__device__ __forceinline__ End end_of_mass(const Row<T, THREADS>& row, S& sh, int n, bool listed, u64 bin_sum, u64 before,
                                           double bound, End end, u64 w_end, int ties, const Scale& s, In in) {
  End cut = end;
  u64 tie_before = before;
  if (n > 0) {
    u64 at;
    const End e = refine<THREADS>(row, sh, listed ? n : -1, before, bound, in,
                                  [&](float l) { return weight_of(l, s); }, &at);
    cut = {e.key, max(1, under(at, weight_of(logit_of(e.key), s), e.n, bound))};
    tie_before = before + bin_sum - (u64)ties * w_end;
  }
  if (ties > 0 && (n <= 0 || (double)tie_before < bound))
    cut = {end.key, max(n > 0 ? 0 : 1, under(tie_before, w_end, ties, bound))};
  return cut;
}

// A row by one block.  FEW: a short list may do for a top_k.
template <typename T, int THREADS, bool FEW>
__device__ void whole_row(const SampleArgs& g, int b, Shared& sh, u64* sums, int* piece_ties) {
  const int tid = threadIdx.x, wave = tid / kWave, lane = lane_id();
  const Row<T, THREADS> row{reinterpret_cast<const T*>(g.logits) + (size_t)b * g.V, g.V};
  const int V = g.V;
  const Params p = params_of(g, b);

  // the largest logit, and its lowest id
  u64 best = 0;
  row.each([&](float l, int i) {
    if (i < V) best = larger(best, (u64)order_of(l) << 32 | (uint32_t)~(uint32_t)i);
  });
#pragma unroll
  for (int d = 32; d >= 1; d >>= 1) best = larger(best, __shfl_xor(best, d, kWave));
  if (lane == 0) sh.red[wave] = best;
  lay_out_pow(sh.pow);
  __syncthreads();
  best = sh.red[0];
#pragma unroll
  for (int i = 1; i < (THREADS / kWave); ++i) best = larger(best, sh.red[i]);
  if (settled(g, b, p, best, tid == 0)) return;
  const Scale s = scale_of(logit_of((uint32_t)(best >> 32)), p.temp, sh.pow);

  // top_k: the end of the first k
  End end{0, 0};   // everything
  if (p.k > 0 && p.k < V) {
    for (int i = tid; i < kBins; i += THREADS) sh.sizes[i] = 0;
    if (tid == 0) sh.count = 0;
    __syncthreads();
    row.each([&](float l, int i) {
      if (i < V) atomicAdd(&sh.sizes[bin_of(l, s)], 1);
    });
    __syncthreads();
    auto size = [&](int i) { return sh.sizes[i]; };
    if (tid < kWave) find_end(kBins, 0, (double)p.k, [&](int i) { return (u64)sh.sizes[i]; }, size, sh.found);
    __syncthreads();
    const int bin = (int)sh.found[0];
    const u64 before = sh.found[1];
    const int n = sh.sizes[bin];
    if (const int last = min(bin, kBins - 2), few = (int)before + (bin == last ? n : 0); FEW && before + n <= kFewer) {
      __syncthreads();   // (bins is free, sizes has been read)
      u64* keys = sh.bins;
      row.each([&](float l, int i) {
        if (i < V && bin_of(l, s) <= last) keys[atomicAdd(&sh.count, 1)] = (u64)order_of(l) << 32 | (uint32_t)~(uint32_t)i;
      });
      __syncthreads();
      const u64 x = tid < few ? keys[tid] : 0;
      __syncthreads();
      finish_few<THREADS>(g, b, p, s, few, x, sh.few);
      return;
    }
    // (the last bin's weights are 0: whether they are kept makes no difference)
    if (bin < kBins - 1) {
      auto in = [&](float l) { return bin_of(l, s) == bin; };
      if (n <= kList) {
        row.each([&](float l, int i) {
          if (i < V && in(l)) sh.list[atomicAdd(&sh.count, 1)] = order_of(l);
        });
      }
      u64 at;
      end = refine<THREADS>(row, sh, n <= kList ? n : -1, before, (double)p.k, in, [](float) { return (u64)1; }, &at);
      end.n = min(end.n, p.k - (int)at);
    }
  }

  // top_p: the end of the prefix before whose items less than top_p of the sum lies
  if (p.top_p < 1.0f) {
    int bin_k = kBins - 1;
    const u64 w_end = end.key ? weight_of(logit_of(end.key), s, &bin_k) : 0;
    for (int i = tid; i < kBins; i += THREADS) {
      sh.bins[i] = 0;
      sh.sizes[i] = 0;
    }
    if (tid == 0) sh.count = 0;
    __syncthreads();
    row.each([&](float l, int i) {
      int e = 0;
      const u64 w = order_of(l) > end.key ? weight_of(l, s, &e) : 0;
      if (w) {
        atomicAdd(&sh.bins[e], w);
        atomicAdd(&sh.sizes[e], 1);
      }
    });
    __syncthreads();
    if (tid == 0 && w_end) {
      sh.bins[bin_k] += (u64)end.n * w_end;
      sh.sizes[bin_k] += end.n;
    }
    __syncthreads();
    auto sum = [&](int i) { return sh.bins[i]; };
    auto size = [&](int i) { return sh.sizes[i]; };
    if (tid < kWave) find_end(kBins, 0, 0.0, sum, size, sh.found);
    __syncthreads();
    const double bound = fmax((double)p.top_p * (double)sh.found[2], 0.0);
    __syncthreads();
    if (tid < kWave) find_end(kBins, 0, bound, sum, size, sh.found);
    __syncthreads();
    const int bin = (int)sh.found[0];
    const u64 before = sh.found[1], bin_sum = sh.bins[bin];
    const int ties = w_end && bin == bin_k ? end.n : 0;   // of the k's last logit, the bin's smallest
    const int n = sh.sizes[bin] - ties;
    const End old = end;
    auto in = [&](float l) {
      int e = 0;
      return order_of(l) > old.key && weight_of(l, s, &e) > 0 && e == bin;
    };
    if (n > 0 && n <= kList)
      row.each([&](float l, int i) {
        if (i < V && in(l)) sh.list[atomicAdd(&sh.count, 1)] = order_of(l);
      });
    end = end_of_mass<THREADS>(row, sh, n, n <= kList, bin_sum, before, bound, old, w_end, ties, s, in);
    __syncthreads();
  }

  // the draw
  constexpr int kPiece = kWave * Piece<T>::N;
  const Kept kept = kept_of(s, end, p.min_p);
  Pieces<T> pieces = row.pieces();
  piece_sums(pieces, kept, sums, piece_ties);
  __syncthreads();
  if (wave == 0) draw(g, b, row.p, p, kept, sums, piece_ties, (V + kPiece - 1) / kPiece);
}

template <typename T>
__global__ __launch_bounds__(kThreads) void sample_kernel(SampleArgs g) {
  __shared__ Shared sh;
  extern __shared__ u64 sums[];   // the pieces', then their ties
  whole_row<T, kThreads, true>(g, blockIdx.x, sh, sums, reinterpret_cast<int*>(sums + (g.V + kWave * Piece<T>::N - 1) / (kWave * Piece<T>::N)));
}

// ------------------------------------------------------------------ in chunks
// The steps that a row of the launches takes.
enum Mode { kWhole, kTopK, kTopP, kOpen };
__device__ __forceinline__ Mode mode_of(const SampleArgs& g, const Params& p) {
  if (p.k > 0 && p.k < g.V) return p.k <= kFew ? kTopK : kWhole;
  return p.top_p < 1.0f ? kTopP : kOpen;
}

// A chunk's pieces for this wave.
template <typename T>
__device__ __forceinline__ Pieces<T> pieces_of(const SampleArgs& g, int b, int chunk) {
  Pieces<T> x{reinterpret_cast<const T*>(g.logits) + (size_t)b * g.V, g.V,
              (int)((long)chunk * g.pieces / g.chunks) + (int)threadIdx.x / kWave,
              (int)((long)(chunk + 1) * g.pieces / g.chunks), kChunkWaves};
  x.start();
  return x;
}

// The row's largest logit from the chunks', by every wave for itself.
__device__ __forceinline__ u64 best_of(const SampleArgs& g, int b) {
  u64 best = lane_id() < g.chunks ? g.best[(size_t)b * g.chunks + lane_id()] : 0;
#pragma unroll
  for (int d = 32; d >= 1; d >>= 1) best = larger(best, __shfl_xor(best, d, kWave));
  return best;
}

template <typename T>
__global__ __launch_bounds__(kChunkThreads) void sample_max_kernel(SampleArgs g) {
  __shared__ u64 s_best[kChunkWaves];
  const int b = blockIdx.y, chunk = blockIdx.x;
  Pieces<T> part = pieces_of<T>(g, b, chunk);
  // what later steps add to
  for (int i = chunk * kChunkThreads + threadIdx.x; i < kBins; i += g.chunks * kChunkThreads) g.bins[(size_t)b * kBins + i] = 0;
  if (chunk == 0 && threadIdx.x == 0) g.list_n[b] = 0;
  // a lane's largest, and the first piece that has it
  float top = -INFINITY;
  int piece = -1;
  part.run([&](const Piece<T>& x, int c) {
    float most = -INFINITY;
#pragma unroll
    for (int q = 0; q < Piece<T>::N; ++q) most = x.raw(q) > most ? x.raw(q) : most;   // (not a NaN)
    most = most > FLT_MAX ? FLT_MAX : most;
    if (most > top) {
      top = most;
      piece = c;
    }
  });
  u64 best = 0;
  if (piece >= 0) {
    const int i = (piece * kWave + lane_id()) * Piece<T>::N;
    Piece<T> x;
    x.load(part.row, i, g.V);
    int id = i;
#pragma unroll
    for (int q = Piece<T>::N - 1; q >= 0; --q)
      if (x[q] == top) id = i + q;
    best = (u64)order_of(top) << 32 | (uint32_t)~(uint32_t)id;
  }
#pragma unroll
  for (int d = 32; d >= 1; d >>= 1) best = larger(best, __shfl_xor(best, d, kWave));
  if (lane_id() == 0) s_best[threadIdx.x / kWave] = best;
  __syncthreads();
  if (threadIdx.x == 0) {
#pragma unroll
    for (int i = 1; i < kChunkWaves; ++i) best = larger(best, s_best[i]);
    g.best[(size_t)b * g.chunks + chunk] = best;
  }
}

template <typename T>
__global__ __launch_bounds__(kChunkThreads) void sample_scan_kernel(SampleArgs g) {
  constexpr bool kByValue = sizeof(T) == 2;
  constexpr int kBinCopies = kByValue ? 1 : kCopies;
  __shared__ u64 s_bins[kBins * kBinCopies];
  __shared__ uint32_t s_value[kByValue ? kValues : 1];
  __shared__ double s_pow[16];
  const int b = blockIdx.y, chunk = blockIdx.x;
  Pieces<T> part = pieces_of<T>(g, b, chunk);
  const Params p = params_of(g, b);
  const u64 best = best_of(g, b);
  if (settled(g, b, p, best, chunk == 0 && threadIdx.x == 0)) return;
  lay_out_pow(s_pow);
  __syncthreads();
  const Scale s = scale_of(logit_of((uint32_t)(best >> 32)), p.temp, s_pow);
  const Mode mode = mode_of(g, p);
  if (mode == kWhole) return;
  if (mode == kOpen) {
    const Kept kept = kept_of(s, End{0, 0}, p.min_p);
    piece_sums(part, kept, g.sums + (size_t)b * g.pieces, g.ties + (size_t)b * g.pieces);
    return;
  }
  for (int i = threadIdx.x; i < kBinCopies * kBins; i += kChunkThreads) s_bins[i] = 0;
  if constexpr (kByValue)
    for (int i = threadIdx.x; i < kValues; i += kChunkThreads) s_value[i] = 0;
  __syncthreads();
  u64* mine = s_bins + threadIdx.x % kBinCopies;
  // `n` logits l
  auto add = [&](float l, uint32_t n) {
    if (mode == kTopK) {
      atomicAdd(reinterpret_cast<uint32_t*>(mine + bin_of(l, s) * kBinCopies), n);
    } else {
      int bin;
      const u64 w = weight_of(l, s, &bin);
      if (w) atomicAdd(mine + bin * kBinCopies, w * n);
    }
  };
  if constexpr (kByValue) {
    // bf16 has few values: those of 2^-8 to 2^8 in magnitude are counted, and weighed once each
    part.run([&](const Piece<T>& x, int) {
#pragma unroll
      for (int q = 0; q < Piece<T>::N; ++q) {
        const uint32_t bits = x.bits(q), i = (bits & 0x7FFF) - kLeastValue;
        if (i < kValues / 2) {
          atomicAdd(s_value + (i | (bits >> 15) * (kValues / 2)), 1u);
        } else {
          const float l = x[q];
          if (l > -INFINITY) add(l, 1);
        }
      }
    });
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < kValues; i += kChunkThreads) {
      const uint32_t bits = (i % (kValues / 2) + kLeastValue) | (i / (kValues / 2)) << 15;
      if (const uint32_t n = s_value[i]) add(__uint_as_float(bits << 16), n);
    }
  } else if (mode == kTopK) {
    part.each([&](float l, int i) {
      if (i < g.V) add(l, 1);
    });
  } else {
    part.each([&](float l, int) { add(l, 1); });
  }
  __syncthreads();
  for (int i = threadIdx.x; i < kBins; i += kChunkThreads) {
    u64 w = 0;
#pragma unroll
    for (int c = 0; c < kBinCopies; ++c) w += s_bins[i * kBinCopies + c];
    if (w) atomicAdd(g.bins + (size_t)b * kBins + i, w);
  }
}

// Where the end lies: the last bin with items before which less than `bound` lies.
struct Place {
  int bin;
  u64 before, sum;   // sum: of the bin
  double bound;
};
struct PlaceShared {
  u64 red[kChunkWaves];
  u64 before[kChunkWaves], sum[kChunkWaves];
  int bin[kChunkWaves];
};
__device__ __forceinline__ Place place_of(const SampleArgs& g, int b, const Params& p, Mode mode, PlaceShared& sh) {
  static_assert(kBins == 4 * kChunkThreads, "the bins' share of a thread");
  const u64* bins = g.bins + (size_t)b * kBins + 4 * threadIdx.x;
  u64 w[4], sum = 0, all;
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    w[q] = bins[q];
    sum += w[q];
  }
  u64 run = block_scan<kChunkWaves>(sum, sh.red, &all);
  Place at{-1, 0, 0, mode == kTopP ? fmax((double)p.top_p * (double)all, 0.0) : (double)p.k};
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    if (w[q] && ((double)run < at.bound || run == 0)) {
      at.bin = 4 * threadIdx.x + q;
      at.before = run;
      at.sum = w[q];
    }
    run += w[q];
  }
  const unsigned long long m = __ballot(at.bin >= 0);
  const int wave = threadIdx.x / kWave;
  if (lane_id() == (m ? 63 - __builtin_clzll(m) : 0)) {
    sh.bin[wave] = at.bin;
    sh.before[wave] = at.before;
    sh.sum[wave] = at.sum;
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kChunkWaves; ++i)
    if (sh.bin[i] >= 0) {
      at.bin = sh.bin[i];
      at.before = sh.before[i];
      at.sum = sh.sum[i];
    }
  return at;
}

template <typename T>
__global__ __launch_bounds__(kChunkThreads) void sample_list_kernel(SampleArgs g) {
  __shared__ PlaceShared s_place;
  __shared__ u64 s_list[kList];
  __shared__ int s_n, s_base;
  __shared__ double s_pow[16];
  const int b = blockIdx.y, chunk = blockIdx.x;
  Pieces<T> part = pieces_of<T>(g, b, chunk);
  const Params p = params_of(g, b);
  const u64 best = best_of(g, b);
  if (settled(g, b, p, best, false)) return;
  lay_out_pow(s_pow);
  __syncthreads();
  const Scale s = scale_of(logit_of((uint32_t)(best >> 32)), p.temp, s_pow);
  const Mode mode = mode_of(g, p);
  if (mode == kOpen) {
    if (chunk == 0 && threadIdx.x < kWave)
      draw(g, b, part.row, p, kept_of(s, End{0, 0}, p.min_p), g.sums + (size_t)b * g.pieces,
           g.ties + (size_t)b * g.pieces, g.pieces);
    return;
  }
  if (mode == kWhole) return;
  if (threadIdx.x == 0) s_n = 0;
  const Place at = place_of(g, b, p, mode, s_place);
  // top_k: what lies before the bin too; the last bin's weights are 0, and left out.  A cheap test first, of an
  // interval of logits that is wider than the bin (by far more than the roundings).
  const int last = min(at.bin, kBins - 2);
  double below, above = -1.0;   // in bins
  if (mode == kTopK) {
    below = (last + 1.01) / (16.0 * (double)s.c32);
  } else {
    below = (last + 0.6) / (16.0 * s.c);
    if (last > 0) above = (last - 0.6) / (16.0 * s.c);
  }
  const float from = fmaxf((float)((double)s.top - below), -FLT_MAX);
  const float to = above < 0.0 ? INFINITY : (float)((double)s.top - above);
  part.run([&](const Piece<T>& x, int c) {
    uint32_t hits = 0;
#pragma unroll
    for (int q = 0; q < Piece<T>::N; ++q) hits |= x.raw(q) >= from && x.raw(q) <= to ? 1u << q : 0;   // (no NaN)
    each_hit(x, hits, [&](float l, int q, bool in) {
      const int i = (c * kWave + lane_id()) * Piece<T>::N + q;
      int bin;
      if (mode == kTopK) bin = bin_of(l, s);
      else weight_of(l, s, &bin);
      in = in && (mode == kTopK ? bin <= last : bin == last);
      const unsigned long long m = __ballot(in);
      if (!m) return;
      int base = 0;
      if (lane_id() == 0) base = atomicAdd(&s_n, __popcll(m));
      base = __builtin_amdgcn_readfirstlane(base);
      const int slot = base + __popcll(m & ((1ull << lane_id()) - 1));
      if (in && slot < kList) s_list[slot] = (u64)order_of(l) << 32 | (uint32_t)~(uint32_t)i;
    });
  });
  __syncthreads();
  const int n = s_n;   // (of more than kList, so are the row's)
  if (n == 0) return;
  if (threadIdx.x == 0) s_base = atomicAdd(g.list_n + b, n);
  __syncthreads();
  u64* list = g.list + (size_t)b * kList;
  for (int i = threadIdx.x; i < n && s_base + i < kList; i += kChunkThreads) list[s_base + i] = s_list[min(i, kList - 1)];
}

// Sorts n (a power of two) numbers in LDS, descending.
template <int THREADS>
__device__ __forceinline__ void sort_down(u64* x, int n) {
  for (int size = 2; size <= n; size *= 2)
    for (int d = size / 2; d >= 1; d /= 2) {
      __syncthreads();
      for (int t = threadIdx.x; t < n / 2; t += THREADS) {
        const int i = 2 * t - (t & (d - 1)), j = i + d;
        const u64 a = x[i], c = x[j];
        if ((a < c) == ((i & size) == 0)) {
          x[i] = c;
          x[j] = a;
        }
      }
    }
  __syncthreads();
}

// LDS of the cut: a row's list (top_k), or what refine needs (top_p).
struct CutShared {
  union {
    u64 key[kList];
    FewShared<kChunkWaves> few;
    struct {
      uint32_t list[kList];
      u64 digit[256];
      int digit_n[256];
      u64 found[4];
    };
  };
  u64 red[kChunkWaves];
  PlaceShared place;
};

// The rest of a top_k row, from the list of its logits: by a block.
__device__ __forceinline__ void finish_top_k(const SampleArgs& g, int b, const Params& p, const Scale& s, int n,
                                             CutShared& sh) {
  const u64* list = g.list + (size_t)b * kList;
  int size = 2;
  while (size < n) size *= 2;
  for (int i = threadIdx.x; i < size; i += kChunkThreads) sh.key[i] = i < n ? list[i] : 0;
  sort_down<kChunkThreads>(sh.key, size);
  n = min(n, p.k);
  // four neighbours a thread (n <= kFew)
  static_assert(kFew <= 4 * kChunkThreads, "the chosen ones' share of a thread");
  u64 w[4], x[4], sum = 0, all;
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    const int i = 4 * threadIdx.x + q;
    x[q] = i < n ? sh.key[i] : 0;
    w[q] = i < n ? weight_of(logit_of((uint32_t)(x[q] >> 32)), s) : 0;
    sum += w[q];
  }
  u64 run = block_scan<kChunkWaves>(sum, sh.red, &all);
  const double bound = (double)p.top_p * (double)all, least = (double)p.min_p * kUnits;
  // the kept ones, by id: their order's complement is the number's lower half
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    const int i = 4 * threadIdx.x + q;
    const bool keep = i < n && (i == 0 || (((double)run < bound || !(p.top_p < 1.0f)) && (double)w[q] >= least));
    run += w[q];
    if (!keep) w[q] = 0;
    x[q] = keep && w[q] ? (u64)(uint32_t)x[q] << 32 | x[q] >> 32 : 0;
  }
  __syncthreads();
  int m = 2;
  while (m < n) m *= 2;
#pragma unroll
  for (int q = 0; q < 4; ++q)
    if (4 * (int)threadIdx.x + q < m) sh.key[4 * threadIdx.x + q] = x[q];
  sort_down<kChunkThreads>(sh.key, m);   // ids ascending, then zeros
  sum = 0;
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    const int i = 4 * threadIdx.x + q;
    x[q] = i < m ? sh.key[i] : 0;
    w[q] = x[q] ? weight_of(logit_of((uint32_t)x[q]), s) : 0;
    sum += w[q];
  }
  run = block_scan<kChunkWaves>(sum, sh.red, &all);
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    draw_one(g, b, p, s, x[q] << 32 | x[q] >> 32, w[q], run, all);
    run += w[q];
  }
}

template <typename T>
__global__ __launch_bounds__(kChunkThreads) void sample_cut_kernel(SampleArgs g) {
  __shared__ CutShared sh;
  __shared__ double s_pow[16];
  const int b = blockIdx.y, chunk = blockIdx.x;
  Pieces<T> part = pieces_of<T>(g, b, chunk);
  const Params p = params_of(g, b);
  const u64 best = best_of(g, b);
  if (settled(g, b, p, best, false)) return;
  lay_out_pow(s_pow);
  __syncthreads();
  const Scale s = scale_of(logit_of((uint32_t)(best >> 32)), p.temp, s_pow);
  const Mode mode = mode_of(g, p);
  const int n = g.list_n[b];
  if (mode == kOpen || mode == kWhole) return;
  if (n > kList) return;
  if (mode == kTopK) {
    if (chunk == 0 && n <= kFewer)
      finish_few<kChunkThreads>(g, b, p, s, n, (int)threadIdx.x < n ? g.list[(size_t)b * kList + threadIdx.x] : 0, sh.few);
    else if (chunk == 0)
      finish_top_k(g, b, p, s, n, sh);
    return;
  }
  // (every block of the row finds the end for itself)
  const Place at = place_of(g, b, p, mode, sh.place);
  for (int i = threadIdx.x; i < n; i += kChunkThreads) sh.list[i] = (uint32_t)(g.list[(size_t)b * kList + i] >> 32);
  const Row<T, kChunkThreads> none{nullptr, 0};
  const End end = end_of_mass<kChunkThreads>(none, sh, n, true, at.sum, at.before, at.bound, End{0, 0}, 0, 0, s,
                                             [](float) { return false; });
  if (chunk == 0 && threadIdx.x == 0) g.cut[b] = end;
  const Kept kept = kept_of(s, end, p.min_p);
  piece_sums(part, kept, g.sums + (size_t)b * g.pieces, g.ties + (size_t)b * g.pieces);
}

template <typename T>
__global__ __launch_bounds__(kThreads) void sample_draw_kernel(SampleArgs g) {
  __shared__ Shared sh;
  const int b = blockIdx.x;
  const Params p = params_of(g, b);
  const u64 best = best_of(g, b);
  if (settled(g, b, p, best, false)) return;
  const Mode mode = mode_of(g, p);
  u64* sums = g.sums + (size_t)b * g.pieces;
  int* ties = g.ties + (size_t)b * g.pieces;
  if (mode == kWhole || (mode != kOpen && g.list_n[b] > kList)) {
    whole_row<T, kThreads, false>(g, b, sh, sums, ties);
  } else if (mode == kTopP && threadIdx.x < kWave) {
    lay_out_pow(sh.pow);   // (written and read by this wave alone, in order)
    __builtin_amdgcn_wave_barrier();
    const Scale s = scale_of(logit_of((uint32_t)(best >> 32)), p.temp, sh.pow);
    draw(g, b, reinterpret_cast<const T*>(g.logits) + (size_t)b * g.V, p, kept_of(s, g.cut[b], p.min_p), sums, ties,
         g.pieces);
  }
}

}  // namespace
}  // namespace mgpt

using namespace mgpt;

namespace {

// Rows of a launch in chunks.  Of workspace each has 40 KB (bins and list), 8 bytes a chunk and 12 bytes for every 256 (fp32)
// or 512 (bf16) logits: up to 89 KB, at 2^20 fp32 logits, and 89 MB for all of them.
constexpr int kSlice = 1024;
constexpr int kWholeSlice = 1 << 20;   // rows of a launch by whole blocks (a launch takes fewer than 2^32 threads)

// Rows of up to 8192 are whole blocks' work in one launch.
bool in_chunks(const mgpt_sample_config* cfg) { return cfg->vocab_size > 8192; }

struct SampleLayout {
  int rows, chunks, pieces;
  size_t best, bins, list, sums, ties, list_n, cut, total;
};
SampleLayout sample_layout(const mgpt_sample_config* cfg, int num_rows, int cus) {
  SampleLayout l{};
  if (!in_chunks(cfg) || num_rows == 0) return l;
  l.rows = std::min(num_rows, kSlice);
  const int piece = kWave * (cfg->dtype == MGPT_DTYPE_F32 ? 4 : 8);
  l.pieces = (cfg->vocab_size + piece - 1) / piece;
  // about four blocks a CU, of eight pieces at least
  l.chunks = std::max(1, std::min({(4 * cus + l.rows - 1) / l.rows, l.pieces / 8, kMaxChunks}));
  size_t off = 0;
  auto take = [&](size_t bytes) {
    const size_t at = off;
    off += (bytes + 255) / 256 * 256;
    return at;
  };
  const size_t R = l.rows;
  l.best = take(R * l.chunks * 8);
  l.bins = take(R * kBins * 8);
  l.list = take(R * kList * 8);
  l.sums = take(R * l.pieces * 8);
  l.ties = take(R * l.pieces * 4);
  l.list_n = take(R * 4);
  l.cut = take(R * sizeof(End));
  l.total = off;
  return l;
}

int check_sample(const mgpt_sample_config* cfg, int num_rows) {
  if (!cfg) return fail(MGPT_ERR_INVALID_ARGUMENT, "config is null");
  if (num_rows < 0) return fail(MGPT_ERR_INVALID_ARGUMENT, "negative num_rows");
  if (num_rows > 1 << 24) return fail(MGPT_ERR_UNSUPPORTED, "num_rows %d > 2^24", num_rows);
  if (cfg->vocab_size < 1) return fail(MGPT_ERR_INVALID_ARGUMENT, "invalid vocab_size=%d", cfg->vocab_size);
  if (cfg->vocab_size > kMaxVocab) return fail(MGPT_ERR_UNSUPPORTED, "vocab_size %d > %d", cfg->vocab_size, kMaxVocab);
  if (cfg->dtype != MGPT_DTYPE_F32 && cfg->dtype != MGPT_DTYPE_BF16)
    return fail(MGPT_ERR_UNSUPPORTED, "unsupported dtype %d", cfg->dtype);
  return MGPT_OK;
}

template <typename T>
hipError_t launch_sample(SampleArgs g, const SampleLayout& l, int num_rows, char* ws, bool cut, hipStream_t st) {
  if (l.rows > 0) {
    g.chunks = l.chunks;
    g.pieces = l.pieces;
    g.best = (u64*)(ws + l.best);
    g.bins = (u64*)(ws + l.bins);
    g.list = (u64*)(ws + l.list);
    g.sums = (u64*)(ws + l.sums);
    g.ties = (int*)(ws + l.ties);
    g.list_n = (int*)(ws + l.list_n);
    g.cut = (End*)(ws + l.cut);
  }
  const int slice = l.rows > 0 ? l.rows : kWholeSlice;
  for (int r = 0; r < num_rows; r += slice) {
    const int n = std::min(slice, num_rows - r);
    SampleArgs a = g;
    a.logits = (const T*)g.logits + (size_t)r * g.V;
    a.u += r;
    if (a.T) a.T += r;
    if (a.p) a.p += r;
    if (a.m) a.m += r;
    if (a.k) a.k += r;
    a.token += r;
    if (a.logp) a.logp += r;
    if (l.rows == 0) {
      const int piece = kWave * Piece<T>::N;
      const size_t lds = (size_t)((g.V + piece - 1) / piece) * 12;
      hipLaunchKernelGGL(sample_kernel<T>, dim3(n), dim3(kThreads), lds, st, a);
      continue;
    }
    const dim3 grid(l.chunks, n), block(kChunkThreads);
    hipLaunchKernelGGL(sample_max_kernel<T>, grid, block, 0, st, a);
    hipLaunchKernelGGL(sample_scan_kernel<T>, grid, block, 0, st, a);
    hipLaunchKernelGGL(sample_list_kernel<T>, grid, block, 0, st, a);
    if (cut) {
      hipLaunchKernelGGL(sample_cut_kernel<T>, grid, block, 0, st, a);
      hipLaunchKernelGGL(sample_draw_kernel<T>, dim3(n), dim3(kThreads), 0, st, a);
    }
  }
  return hipGetLastError();
}

}  // namespace

extern "C" {

int mgpt_sample_workspace_bytes(const mgpt_sample_config* cfg, int num_rows, size_t* bytes) {
  if (int rc = check_sample(cfg, num_rows)) return rc;
  if (!bytes) return fail(MGPT_ERR_INVALID_ARGUMENT, "null bytes");
  *bytes = sample_layout(cfg, num_rows, compute_units()).total;
  return MGPT_OK;
}

int mgpt_sample(const mgpt_sample_config* cfg, const void* logits, const float* u, const float* temperature,
                const int32_t* top_k, const float* top_p, const float* min_p, int32_t* token, float* logp, int num_rows,
                void* workspace, size_t workspace_bytes, void* stream) {
  if (int rc = check_sample(cfg, num_rows)) return rc;
  if (!temperature && !(cfg->temperature >= 0.0f))
    return fail(MGPT_ERR_INVALID_ARGUMENT, "temperature must be >= 0");
  if (!top_p && !(cfg->top_p >= 0.0f)) return fail(MGPT_ERR_INVALID_ARGUMENT, "top_p must be >= 0");
  if (!min_p && !(cfg->min_p >= 0.0f)) return fail(MGPT_ERR_INVALID_ARGUMENT, "min_p must be >= 0");
  if (num_rows == 0) return MGPT_OK;
  if (!logits || !u || !token) return fail(MGPT_ERR_INVALID_ARGUMENT, "null logits, u or token");
  const SampleLayout l = sample_layout(cfg, num_rows, compute_units());
  if (l.total > 0 && !workspace) return fail(MGPT_ERR_INVALID_ARGUMENT, "null workspace");
  if ((uintptr_t)workspace & 255) return fail(MGPT_ERR_INVALID_ARGUMENT, "workspace must be 256-byte aligned");
  if (workspace_bytes < l.total)
    return fail(MGPT_ERR_WORKSPACE_TOO_SMALL, "workspace needs %zu bytes, got %zu", l.total, workspace_bytes);
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
  // (known here: no row has a list)
  const bool cut = top_k || cfg->top_k > 0 || top_p || cfg->top_p < 1.0f;
  HIP_TRY(cfg->dtype == MGPT_DTYPE_F32
              ? launch_sample<float>(g, l, num_rows, (char*)workspace, cut, (hipStream_t)stream)
              : launch_sample<bf16_t>(g, l, num_rows, (char*)workspace, cut, (hipStream_t)stream));
  return MGPT_OK;
}

}  // extern "C"
