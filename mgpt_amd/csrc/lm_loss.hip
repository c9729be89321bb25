// lm_loss.hip -- softmax cross entropy of a language model's head over its
// vocabulary, and its gradients, without ever holding the logits.
//
// Reference: LinearLayer lm_head, then CrossEntropyLossLayer (layers/LinearLayer.cpp,
// layers/CrossEntropyLossLayer.cpp), which keep logits, probabilities and their
// gradients, three [N][V] arrays.  Here, with z = x W^T + b (x [N][C], W [V][C]):
//   forward:  lse_n = log sum_v exp(z_nv),  loss_n = lse_n - z_n,t(n)
//   backward: d_nv = (exp(z_nv - lse_n) - [v = t(n)]) g_n, with g_n row n's upstream
//             gradient (0 where it has no target),
//             dx = d W,  dW = d^T x,  db_v = sum_n d_nv
//
// Forward: one product whose epilogue reduces every 64 columns of a row to (max, sum of
// exponentials) and picks the target's logit; join_kernel adds them up.
// Backward, for a piece of the vocabulary at a time: the product again, whose epilogue
// forms d, in the inputs' type, as rows [N][piece] and transposed [piece][N] (both
// from registers, so that every product has both operands contiguous along its
// contraction), and its column sums; then dx += d W_piece and dW_piece = d^T x.
//
// All four products are one kernel (ring_kernel): a persistent block per CU walks 256 x
// 256 tiles, operands go HBM -> LDS by untracked 1 KB loads into a ring of 5 units (an
// operand's 128-byte slabs of a tile), 8 waves of 64 columns x 128 rows run D = B . A^T by
// v_mfma_f32_32x32x16_bf16 (gemm_dma.hip describes the ring and its measurements); fp32
// operands are split in registers into three bf16 numbers (Split).  Rows past an operand's
// last re-read the last, so that nothing behind a caller's tensor is touched.  Few tiles
// take 128 x 128 or 64 x 128 ones, two blocks of 4 waves a CU, or 64 x 64 ones, and products
// of few tiles (dx, dW) split their contraction, the parts added in order (plan_gemm).
//
// What bounds it: the matrix rate, 2 N C V operations forward and 6 N C V backward (a
// third of them to form the logits again), except for few rows, where reading W does.
// MI355X, kernel times: 16384 x 1024 x 32000 bf16 (1.07 T operations a product): logits
// forward 939 us, again with d's epilogue 1275, dx 842, dW 822 (1140, 840, 1275, 1305
// TFLOP/s; a library product of 8192^3 1373).  The logits' epilogues are what those lack:
// an exponential per logit on the vector unit, and for d 2 GB of stores, which a wave's
// next loads wait behind.  64 rows x 2048 x 50257: 45 us from memory (206
// MB, 4.6 TB/s; a library's sum reads 3.8), 36 from the last-level cache (5.8).
// Logits, sums and their logarithms are fp32.  With bf16 inputs d is rounded to bf16, as
// the operand of two bf16 products (dx and dW 0.0021 off against 64 bits where targets are drawn
// from the softmax, with d in fp32 and the results in bf16 0.0017); db is summed before that.
#include <algorithm>
#include <type_traits>

#include "../../include/mgpt_moe.h"
#include "capi_internal.hpp"
#include "gemm_ring.hpp"

namespace mgpt {

template <typename T>
hipError_t launch_copy_cols(const T*, int, T*, int, int, int, int, hipStream_t);   // pack.hip
hipError_t launch_fill_zero(float* p, size_t n, hipStream_t stream);              // wgrad.hip

namespace {

enum LossEpilogue {
  kLse,      // (max, sum of exponentials) per row and 64 columns, the target's logit
  kDLogit,   // d and its transpose
  kDLogitSum,   // and d's column sums
  kPart,     // fp32 partial product, stored or added
  kStore,    // the product in the inputs' type, rows as 16-byte vectors
  kStoreOdd  // the same for rows that are not: a lane has a column, so that a row's neighbours are stored together
};

constexpr float kLog2e = 1.44269504088896340736f;

struct LossArgs {
  const char *A, *B;     // A [M][lda], B [Nf][ldb], contiguous along the contraction
  size_t lda, ldb;       // bytes; multiples of 16
  int M, Nf, KT;         // rows, columns, 128-byte slabs of the contraction
  int mt, nt, parts;     // tiles; parts of the contraction
  int turn, once;        // UNITS even: a power of 2 up to a part's slabs, less 1 (see slab_of); B past the caches
  // kLse and kDLogit: bias of the columns (or null), targets counted from column 0
  const float* bias;
  const int32_t* targets;
  int target0;           // the piece's first column
  float2* part_lse;      // [columns of a wave][ld_lse]
  int ld_lse;
  float* picked;         // [M]
  int* counter;          // set to 0 for join_kernel's blocks
  const float *lse, *scale;
  char *d, *dt;          // [M][ldd], [.][lddt] in T
  size_t ldd, lddt;      // elements
  int rows_t;            // rows that the transpose holds (zeros past M)
  float* colsum;         // [2 mt][ldd]
  // kPart: out [parts][M][ldo] fp32; kStore, kStoreOdd: out [M][ldo] in T
  char* out;
  size_t ldo;
  int add;
  const float* factor;   // kStore, kStoreOdd: of the product
};

// fp32 operands as three bf16 numbers each, x = h + m + l exactly (rounded to nearest, 8 of
// its 24 bits each): six of the nine products keep all but some 2^-24 of the factors'
// magnitudes.  Six v_mfma_f32_32x32x16_bf16 of 32 cycles contract 16 columns, where
// v_mfma_f32_32x32x2_f32 takes eight of 64; the splitting, 5.5 vector instructions a value,
// then runs beside them (999 x 500 x 8003: products of 73 to 143 us became 57 to 67; the
// error against 64 bits fell from 5.7e-7 to 2.7e-7).  An infinity, or a magnitude above
// bf16's largest, splits into NaN.
struct Split {
  bf16x8 h, m, l;
};
__device__ __forceinline__ Split split(f32x4 a, f32x4 b) {
  uint32_t w[3][4];
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    float x = q < 2 ? a[2 * q] : b[2 * q - 4], y = q < 2 ? a[2 * q + 1] : b[2 * q - 3];
#pragma unroll
    for (int p = 0; p < 3; ++p) {
      w[p][q] = pack_bf16x2(x, y);
      if (p < 2) {
        x -= __uint_as_float(w[p][q] << 16);
        y -= __uint_as_float(w[p][q] & 0xFFFF0000u);
      }
    }
  }
  Split s;
  __builtin_memcpy(&s.h, w[0], 16);
  __builtin_memcpy(&s.m, w[1], 16);
  __builtin_memcpy(&s.l, w[2], 16);
  return s;
}
__device__ __forceinline__ f32x16 contract(bf16x8 w, bf16x8 x, f32x16 acc) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(w, x, acc, 0, 0, 0);
}
__device__ __forceinline__ f32x16 contract(const Split& w, const Split& x, f32x16 acc) {
  acc = contract(w.l, x.h, acc);   // the smallest first
  acc = contract(w.m, x.m, acc);
  acc = contract(w.h, x.l, acc);
  acc = contract(w.m, x.h, acc);
  acc = contract(w.h, x.m, acc);
  return contract(w.h, x.h, acc);
}

// A 1 KB direct-to-LDS load (see dma16) from a uniform base and a lane's offset.
__device__ __forceinline__ void dma16_base(const char* base, uint32_t off, uint32_t lds) {
  asm volatile("global_load_lds_dwordx4 %0, %1" ::"v"(off), "s"(base), "{m0}"(lds) : "memory");
}

// The same past the caches.
__device__ __forceinline__ void dma16_once(const char* base, uint32_t off, uint32_t lds) {
  asm volatile("global_load_lds_dwordx4 %0, %1 nt" ::"v"(off), "s"(base), "{m0}"(lds) : "memory");
}

// A wave-uniform address, in scalar registers.
__device__ __forceinline__ const char* uniform(const char* p) {
  const uint64_t u = (uint64_t)(uintptr_t)p;
  const uint32_t lo = __builtin_amdgcn_readfirstlane((uint32_t)u);
  const uint32_t hi = __builtin_amdgcn_readfirstlane((uint32_t)(u >> 32));
  return reinterpret_cast<const char*>((uintptr_t)(((uint64_t)hi << 32) | lo));
}

__device__ __forceinline__ float other_half_max(float v) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float other_half_sum(float v) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// Sum over the 32 lanes of each half, in its last lane.
template <int CTRL, int ROWS>
__device__ __forceinline__ float dpp_fadd(float v) {
  return v + __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, ROWS, 0xf, false));
}
__device__ __forceinline__ float half_sum(float v) {
  v = dpp_fadd<0x111, 0xf>(v);
  v = dpp_fadd<0x112, 0xf>(v);
  v = dpp_fadd<0x114, 0xf>(v);
  v = dpp_fadd<0x118, 0xf>(v);
  return dpp_fadd<0x142, 0xa>(v);
}

// Lane r of each four holds the 4 bf16 features of token r; afterwards it holds feature r
// of the 4 tokens.
__device__ __forceinline__ uint2 transpose4(uint2 u, int lane) {
  const uint32_t p0 = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)u.x, 0xB1, 0xf, 0xf, false);   // lane ^ 1
  const uint32_t p1 = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)u.y, 0xB1, 0xf, 0xf, false);
  // even lanes: both lanes' first feature of the pair; odd ones: their second
  const uint32_t sel = lane & 1 ? 0x07060302u : 0x01000504u;
  const uint32_t a0 = __builtin_amdgcn_perm(u.x, p0, sel), a1 = __builtin_amdgcn_perm(u.y, p1, sel);
  const bool upper = lane & 2;
  const uint32_t r = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(upper ? a0 : a1), 0x4E, 0xf, 0xf, false);   // lane ^ 2
  return upper ? make_uint2(r, a1) : make_uint2(a0, r);
}

template <typename W>
using Acc = f32x16[W::TN][W::TM];

// The accumulators of a wave's columns fw .. start from their biases (column 8k + 4h + q
// of a group of 32 in register 4k + q) or, past the last column, from -inf: no
// probability, no gradient.  Whole groups are read by scalar loads; a vector load would
// wait for the ring's, which the compiler does not track.
template <typename W>
__device__ __forceinline__ void start_from_bias(const LossArgs& g, Acc<W>& acc, int fw, int lhalf) {
#pragma unroll
  for (int j = 0; j < W::TN; ++j) {
    const int f0 = fw + 32 * j;
    f32x16 b;
    if (f0 + 32 <= g.Nf) {
      if (g.bias) {
        typedef const __attribute__((address_space(4))) float* cptr;
        const cptr u = (cptr)(uintptr_t)(g.bias + f0);
#pragma unroll
        for (int k = 0; k < 4; ++k)
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const float lo = u[8 * k + q], hi = u[8 * k + 4 + q];
            b[4 * k + q] = lhalf ? hi : lo;
          }
      } else {
#pragma unroll
        for (int v = 0; v < 16; ++v) b[v] = 0.0f;
      }
    } else {
#pragma unroll
      for (int v = 0; v < 16; ++v) {
        const int f = f0 + 8 * (v / 4) + 4 * lhalf + v % 4;
        b[v] = g.bias ? g.bias[min(f, g.Nf - 1)] : 0.0f;
        if (f >= g.Nf) b[v] = -INFINITY;
      }
    }
#pragma unroll
    for (int i = 0; i < W::TM; ++i) acc[j][i] = b;
    __builtin_amdgcn_sched_barrier(0);   // one group at a time (scalar registers)
  }
}

// exp(z - s) of a register: one fma into the hardware's exponential; `huge` (a lane's s at
// kHuge and beyond, where the rounding of s log2 e would be some and at last all of the
// exponent): difference first.  (By lane: a row's bits do not depend on its neighbours.)
__device__ __forceinline__ float exp_less(float z, float s, float ns, bool huge) {
  return __builtin_amdgcn_exp2f(huge ? (z - s) * kLog2e : __builtin_fmaf(z, kLog2e, ns));
}
constexpr float kHuge = 0x1p20f;   // (half a step of 1.44 kHuge is 1/16)

// What exp_less's ns = -s log2 e lost to rounding, as the factor that all exponentials of
// the row lack: half a step of 1.44 |s|, 5e-6 of them for an s near 100.  (The fma is
// exact.)  It goes to the row's sum or upstream gradient, so no exponential costs more.
__device__ __forceinline__ float lost_in_product(float s, float ns, bool huge) {
  return huge ? 1.0f : __builtin_amdgcn_exp2f(-__builtin_fmaf(s, kLog2e, ns));
}

// a * b, 0 where either is 0, whatever the other.
__device__ __forceinline__ float mul_zero(float a, float b) {
  float r;
  asm("v_mul_legacy_f32 %0, %1, %2" : "=v"(r) : "v"(a), "v"(b));
  return r;
}

template <typename T, typename W>
__device__ __forceinline__ void emit_lse(const LossArgs& g, Acc<W>& acc, int row0, int fw, int lrow, int lhalf) {
  if (fw >= g.Nf) return;
#pragma unroll
  for (int i = 0; i < W::TM; ++i) {
    const int row = row0 + 32 * i + lrow;
    const bool live = row < g.M;
    const int t = live ? g.targets[row] : -1;
    float m = -INFINITY;
#pragma unroll
    for (int j = 0; j < W::TN; ++j)
#pragma unroll
      for (int v = 0; v < 16; v += 2) m = fmaxf(fmaxf(acc[j][i][v], acc[j][i][v + 1]), m);
    m = other_half_max(m);
    const float top = m == -INFINITY ? 0.0f : m, ntop = -top * kLog2e;
    float s = 0.0f;
    const bool huge = !(fabsf(top) < kHuge);
    if (__ballot(huge)) {
#pragma unroll
      for (int j = 0; j < W::TN; ++j)
#pragma unroll
        for (int v = 0; v < 16; ++v) s += exp_less(acc[j][i][v], top, ntop, huge);
    } else {
#pragma unroll
      for (int j = 0; j < W::TN; ++j)
#pragma unroll
        for (int v = 0; v < 16; ++v) s += exp_less(acc[j][i][v], top, ntop, false);
    }
    s = other_half_sum(s) * lost_in_product(top, ntop, huge);
    if (live && lhalf == 0) g.part_lse[(size_t)(fw / W::WTN) * g.ld_lse + row] = make_float2(m, s);
    const int fl = t >= fw && t < min(fw + W::WTN, g.Nf) ? t - fw : -1;
    const bool mine = fl >= 0 && ((fl >> 2) & 1) == lhalf;
    if (__ballot(mine)) {
      float z = 0.0f;
#pragma unroll
      for (int j = 0; j < W::TN; ++j)
#pragma unroll
        for (int v = 0; v < 16; ++v)
          if (fl == 32 * j + 8 * (v / 4) + 4 * lhalf + v % 4) z = acc[j][i][v];
      if (mine) g.picked[row] = z;
    }
    __builtin_amdgcn_sched_barrier(0);
  }
}

template <typename T, typename W, bool SUM>
__device__ __forceinline__ void emit_dlogit(const LossArgs& g, Acc<W>& acc, int row0, int fw, int lrow, int lhalf,
                                            int sum_row) {
  float lse[W::TM], sc[W::TM], psc[W::TM];   // psc: of the probabilities
  int tl[W::TM];   // the target's column in the wave's
  bool huge = false;
#pragma unroll
  for (int i = 0; i < W::TM; ++i) {
    const int row = row0 + 32 * i + lrow, r = min(row, g.M - 1);
    sc[i] = row < g.M ? g.scale[r] : 0.0f;
    lse[i] = sc[i] == 0.0f ? 0.0f : g.lse[r];
    psc[i] = sc[i] * lost_in_product(lse[i], -lse[i] * kLog2e, !(fabsf(lse[i]) < kHuge));
    tl[i] = g.targets[r] - g.target0 - fw;
    huge |= !(fabsf(lse[i]) < kHuge);
  }
  const bool slow = __ballot(huge) != 0;
  // (uniform addresses and a lane's 32-bit offsets: a tile's rows are within 4 GB, as
  // launch_ring checks)
  const uint32_t d_off = ((uint32_t)lrow * (uint32_t)g.ldd + 4 * lhalf) * (uint32_t)sizeof(T);
  uint32_t t_off[4];
#pragma unroll
  for (int k = 0; k < 4; ++k)
    t_off[k] = sizeof(T) == 2
                   ? ((uint32_t)(8 * k + 4 * lhalf + (lrow & 3)) * (uint32_t)g.lddt + (uint32_t)(lrow & ~3)) * 2
                   : ((uint32_t)(8 * k + 4 * lhalf) * (uint32_t)g.lddt + (uint32_t)lrow) * 4;
#pragma unroll
  for (int j = 0; j < W::TN; ++j) {
    const int f0 = fw + 32 * j;
    float cs[16];
#pragma unroll
    for (int v = 0; v < 16; ++v) cs[v] = 0.0f;
#pragma unroll
    for (int i = 0; i < W::TM; ++i) {
      const int row = row0 + 32 * i + lrow;
      const float nl = -lse[i] * kLog2e;
      float d[16];
      if (slow) {
#pragma unroll
        for (int v = 0; v < 16; ++v) d[v] = exp_less(acc[j][i][v], lse[i], nl, !(fabsf(lse[i]) < kHuge));
      } else {
#pragma unroll
        for (int v = 0; v < 16; ++v) d[v] = exp_less(acc[j][i][v], lse[i], nl, false);
      }
      // the target's entry apart: (p - 1) times the upstream gradient, which may be infinite
      const bool hit = __ballot(tl[i] >= 32 * j && tl[i] < 32 * j + 32) != 0;
      float at = 0.0f;
      if (hit) {
#pragma unroll
        for (int v = 0; v < 16; ++v)
          if (tl[i] == 32 * j + 8 * (v / 4) + 4 * lhalf + v % 4) at = d[v];
        at = mul_zero(at * lost_in_product(lse[i], nl, !(fabsf(lse[i]) < kHuge)) - 1.0f, sc[i]);
      }
      // (0 times anything is 0 here: a row without a target has no gradient even where its
      // logits are not finite)
#pragma unroll
      for (int v = 0; v < 16; ++v) d[v] = mul_zero(d[v], psc[i]);
      if (hit) {
#pragma unroll
        for (int v = 0; v < 16; ++v)
          if (tl[i] == 32 * j + 8 * (v / 4) + 4 * lhalf + v % 4) d[v] = at;
      }
      if constexpr (SUM) {
#pragma unroll
        for (int v = 0; v < 16; ++v) cs[v] += d[v];
      }
      char* dm = g.d + ((size_t)(row0 + 32 * i) * g.ldd + f0) * sizeof(T);
      char* dt = g.dt + ((size_t)f0 * g.lddt + (row0 + 32 * i)) * sizeof(T);
      if constexpr (sizeof(T) == 2) {
        uint2 q[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) q[k] = pack4_bf16(d[4 * k], d[4 * k + 1], d[4 * k + 2], d[4 * k + 3]);
        store_group32(reinterpret_cast<bf16_t*>(dm + (d_off - 8 * lhalf)), q, lhalf, row < g.M);
        if ((row & ~3) < g.rows_t) {
          // (past the caches: 695 -> 637 us at 16384 x 1024 x 16128, where both write 256 KB a
          // tile; d's own stores too: 685)
#pragma unroll
          for (int k = 0; k < 4; ++k) store_once(reinterpret_cast<uint2*>(dt + t_off[k]), transpose4(q[k], lrow));
        }
      } else {
        if (row < g.M) {
#pragma unroll
          for (int k = 0; k < 4; ++k)
            *reinterpret_cast<float4*>(dm + d_off + 32 * k) =
                make_float4(d[4 * k], d[4 * k + 1], d[4 * k + 2], d[4 * k + 3]);
        }
        if (row < g.rows_t) {
#pragma unroll
          for (int k = 0; k < 4; ++k)
#pragma unroll
            for (int q = 0; q < 4; ++q)
              *reinterpret_cast<float*>(dt + (size_t)q * g.lddt * 4 + t_off[k]) = d[4 * k + q];
        }
      }
      __builtin_amdgcn_sched_barrier(0);
    }
    if constexpr (SUM) {
#pragma unroll
      for (int v = 0; v < 16; ++v) {
        const float s = half_sum(cs[v]);
        if (lrow == 31) g.colsum[(size_t)sum_row * g.ldd + f0 + 8 * (v / 4) + 4 * lhalf + v % 4] = s;
      }
    }
  }
}

template <typename W>
__device__ __forceinline__ void emit_part(const LossArgs& g, Acc<W>& acc, int part, int row0, int fw, int lrow,
                                          int lhalf) {
  float* out = reinterpret_cast<float*>(g.out) + (size_t)part * g.M * g.ldo;
#pragma unroll
  for (int j = 0; j < W::TN; ++j) {
    const int f0 = fw + 32 * j + 4 * lhalf;
    if (fw + 32 * j >= g.Nf) continue;
#pragma unroll
    for (int i = 0; i < W::TM; ++i) {
      const int row = row0 + 32 * i + lrow;
      if (row < g.M) {
        float4* o = reinterpret_cast<float4*>(out + (size_t)row * g.ldo + f0);   // (ldo covers whole tiles)
        float4 old[4];
        if (g.add) {
#pragma unroll
          for (int k = 0; k < 4; ++k) old[k] = o[2 * k];
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          float4 r = make_float4(acc[j][i][4 * k], acc[j][i][4 * k + 1], acc[j][i][4 * k + 2], acc[j][i][4 * k + 3]);
          if (g.add) {
            r.x = old[k].x + r.x;
            r.y = old[k].y + r.y;
            r.z = old[k].z + r.z;
            r.w = old[k].w + r.w;
          }
          o[2 * k] = r;
        }
      }
      __builtin_amdgcn_sched_barrier(0);
    }
  }
}

template <typename T, typename W>
__device__ __forceinline__ void emit_store(const LossArgs& g, Acc<W>& acc, int row0, int fw, int lrow, int lhalf) {
  T* out = reinterpret_cast<T*>(g.out);
  const float factor = uniform_load(g.factor);
#pragma unroll
  for (int j = 0; j < W::TN; ++j) {
    const int f0 = fw + 32 * j;
    if (f0 >= g.Nf) continue;
    const bool whole = f0 + 32 <= g.Nf;
#pragma unroll
    for (int i = 0; i < W::TM; ++i) {
      const int row = row0 + 32 * i + lrow;
      T* o = out + (size_t)row * g.ldo + f0;
#pragma unroll
      for (int v = 0; v < 16; ++v) acc[j][i][v] *= factor;
      if (whole && sizeof(T) == 2) {
        uint2 q[4];
#pragma unroll
        for (int k = 0; k < 4; ++k)
          q[k] = pack4_bf16(acc[j][i][4 * k], acc[j][i][4 * k + 1], acc[j][i][4 * k + 2], acc[j][i][4 * k + 3]);
        store_group32(reinterpret_cast<bf16_t*>(o), q, lhalf, row < g.M);
      } else if (row < g.M) {   // (a row is a multiple of 8 columns: quads are whole)
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const int f = 8 * k + 4 * lhalf;
          if (f0 + f >= g.Nf) continue;
          if constexpr (sizeof(T) == 2)
            *reinterpret_cast<uint2*>(o + f) =
                pack4_bf16(acc[j][i][4 * k], acc[j][i][4 * k + 1], acc[j][i][4 * k + 2], acc[j][i][4 * k + 3]);
          else
            *reinterpret_cast<float4*>(o + f) =
                make_float4(acc[j][i][4 * k], acc[j][i][4 * k + 1], acc[j][i][4 * k + 2], acc[j][i][4 * k + 3]);
        }
      }
      __builtin_amdgcn_sched_barrier(0);
    }
  }
}

// Accumulators of A . B^T: register v of a tile holds row 8 (v / 4) + 4 h + v % 4, column
// lane % 32.
template <typename T, typename W>
__device__ __forceinline__ void emit_store_odd(const LossArgs& g, Acc<W>& acc, int row0, int fw, int lrow,
                                               int lhalf) {
  T* out = reinterpret_cast<T*>(g.out);
  const float factor = uniform_load(g.factor);
#pragma unroll
  for (int j = 0; j < W::TN; ++j) {
    const int f = fw + 32 * j + lrow;
#pragma unroll
    for (int i = 0; i < W::TM; ++i) {
#pragma unroll
      for (int v = 0; v < 16; ++v) {
        const int row = row0 + 32 * i + 8 * (v / 4) + 4 * lhalf + v % 4;
        if (f < g.Nf && row < g.M) store_act(out + (size_t)row * g.ldo + f, acc[j][i][v] * factor);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
  }
}

struct Item {
  int row0, n0, k0, k1, part;
};

template <int BM, int BN>
__device__ __forceinline__ bool locate_item(const LossArgs& g, int v, Item* it) {
  const int tiles = g.mt * g.nt;
  if (v >= tiles * g.parts) return false;
  const int part = v / tiles, u = v % tiles;
  // groups of kGroupM row tiles x all column tiles, rows fastest (as locate_tile)
  const int grp = u / (kGroupM * g.nt), gsize = min(kGroupM, g.mt - grp * kGroupM);
  const int idx = u - grp * kGroupM * g.nt;
  it->row0 = __builtin_amdgcn_readfirstlane((grp * kGroupM + idx % gsize) * BM);
  it->n0 = __builtin_amdgcn_readfirstlane(idx / gsize * BN);
  it->part = __builtin_amdgcn_readfirstlane(part);
  // (parts <= 128 and KT < 2^17: no overflow)
  it->k0 = __builtin_amdgcn_readfirstlane(part * g.KT / g.parts);
  it->k1 = __builtin_amdgcn_readfirstlane((part + 1) * g.KT / g.parts);
  return true;
}

// The slab in memory of an item's slab kt, with neighbouring tiles a slab apart.
template <int BN>
__device__ __forceinline__ int slab_of(const LossArgs& g, const Item& it, int kt) {
  const int k = kt + ((it.n0 / BN) & g.turn);
  return k < it.k1 ? k : k - (it.k1 - it.k0);
}

// D[m][f] = sum_k A[m][k] B[f][k].  Ring, swizzle and schedule as gemm_ring5_kernel: units
// A0 B0 A1 B1 .. of consecutive slabs in UNITS slots; barrier s frees slab s - 1's two for
// the columns of slab s + (UNITS - 3) / 2 and the rows of the one after, whose loads go
// out in quarters between the matrix instructions.  Five slots; nine where a block is
// alone on its CU anyway, whose slabs are then requested early enough for the memory's
// latency.
//
// UNITS even: for one row of tiles, where reading B, once, is what takes the time.  Slots of
// the units' own sizes, so that three slabs fit (six where a block is alone on its CU), and
// barrier s frees slab s - 1's for both units of slab s + UNITS / 2 - 1.  Neighbouring
// tiles start a slab apart: in step, all blocks read the same few columns of every row,
// which memory has on a few of its channels.  B that no cache could hold for its next
// use is read past them.  W from memory, the forward's us with 5 or 9 units / these: 64 x 2048
// x 50257 62 / 55, 64 x 4096 x 32000 (262 MB) 68 / 56, 64 x 2048 x 32000 44 / 38; past the caches
// where they could hold it, 64 x 2048 x 50257 takes 52, but 55 and not 46 from the caches.
template <typename T, int EPI, int BM, int BN, int NW, int UNITS>
__global__ __launch_bounds__(NW * 64, NW == 8 || UNITS <= 6 ? 2 : 1) void ring_kernel(LossArgs g) {
  using W = Waves<NW, BM, BN>;
  constexpr int kTN = W::TN, kTM = W::TM, kUnits = UNITS, kRow = 128;
  constexpr bool kOdd = kUnits % 2 == 1;
  static_assert(kUnits >= 5, "a slab worked on, the next one on its way");
  constexpr int kSlot = (BM > BN ? BM : BN) * kRow;
  constexpr int kDA = BM * kRow / 1024 / NW, kDB = BN * kRow / 1024 / NW;   // loads per wave and unit
  auto slot_at = [](int slot) __attribute__((always_inline)) {
    return kOdd ? slot * kSlot : (slot / 2 * (BM + BN) + (slot & 1) * BM) * kRow;
  };
  __shared__ __attribute__((aligned(1024))) char smem[kOdd ? kUnits * kSlot : kUnits / 2 * (BM + BN) * kRow];

  const int G = gridDim.x, items = g.mt * g.nt * g.parts;
  int t = blockIdx.x;
  if (G % kNumXcd == 0) {   // each XCD a contiguous run of each round
    const int run = (min(G, items) + kNumXcd - 1) / kNumXcd, in_xcd = (int)blockIdx.x / kNumXcd;
    t = in_xcd < run ? (int)(blockIdx.x % kNumXcd) * run + in_xcd : items;
  }
  Item cur;
  if (!locate_item<BM, BN>(g, t, &cur)) return;

  const int tid = threadIdx.x;
  if (EPI == kLse && blockIdx.x == 0 && tid == 0) *g.counter = 0;
  const int w = __builtin_amdgcn_readfirstlane(tid / kWave), lane = lane_id();
  const int wn = w % W::WN, wm = w / W::WN;
  const int lrow = lane & 31, lhalf = lane >> 5;
  const uint32_t lds0 = (uint32_t)(uintptr_t)(lds_char*)smem;
  const uint32_t lds_a = lds0 + (uint32_t)(w * kDA * 1024), lds_b = lds0 + (uint32_t)(w * kDB * 1024);

  // Cursors of the two operands (UNITS odd: the rows' a slab ahead of the columns').  Past the
  // block's last slab they stay on it (in bounds, into a slot that is no longer read).
  struct Cursor {
    Item it;
    int v, kt;
    bool valid;
  };
  Cursor ca = {cur, t, cur.k0, true}, cb = ca;
  uint32_t a_off[kDA], b_off[kDB];
  const char *a_base, *b_base;
  auto enter_a = [&]() __attribute__((always_inline)) {
    a_base = g.A + (size_t)ca.it.row0 * g.lda;
    const int last = g.M - 1 - ca.it.row0;
#pragma unroll
    for (int i = 0; i < kDA; ++i) {
      const int r = (w * kDA + i) * 8 + lane / 8;
      a_off[i] = (uint32_t)min(r, last) * (uint32_t)g.lda + (uint32_t)(((lane % 8) ^ ((r >> 1) & 7)) << 4);
    }
  };
  auto enter_b = [&]() __attribute__((always_inline)) {
    b_base = g.B + (size_t)cb.it.n0 * g.ldb;
    const int last = g.Nf - 1 - cb.it.n0;
#pragma unroll
    for (int i = 0; i < kDB; ++i) {
      const int r = (w * kDB + i) * 8 + lane / 8;
      b_off[i] = (uint32_t)min(r, last) * (uint32_t)g.ldb + (uint32_t)(((lane % 8) ^ ((r >> 1) & 7)) << 4);
    }
  };
  // moves a cursor past the slab that was just taken; true: to another item
  auto advance = [&](Cursor& c) __attribute__((always_inline)) {
    if (!c.valid || ++c.kt < c.it.k1) return false;
    Item nx;
    c.v += G;
    c.valid = locate_item<BM, BN>(g, c.v, &nx);
    if (!c.valid) {
      --c.kt;
      return false;
    }
    c.it = nx;
    c.kt = nx.k0;
    return true;
  };
  enter_a();
  enter_b();
  int dslot = 0;
  bool fresh_a = false, fresh_b = false;   // the cursor's item has no offsets yet
  const char *ua, *ub;
  uint32_t da, db;
  auto take_a = [&]() __attribute__((always_inline)) {
    if (fresh_a) enter_a();
    ua = uniform(a_base + (size_t)(kOdd ? ca.kt : slab_of<BN>(g, ca.it, ca.kt)) * kRow);
    da = lds_a + (uint32_t)slot_at(dslot);
    dslot = dslot + 1 == kUnits ? 0 : dslot + 1;
    fresh_a = advance(ca);
  };
  auto take_b = [&]() __attribute__((always_inline)) {
    if (fresh_b) enter_b();
    ub = uniform(b_base + (size_t)(kOdd ? cb.kt : slab_of<BN>(g, cb.it, cb.kt)) * kRow);
    db = lds_b + (uint32_t)slot_at(dslot);
    dslot = dslot + 1 == kUnits ? 0 : dslot + 1;
    fresh_b = advance(cb);
  };
  // loads d0 .. d1 - 1 of the taken units, the columns' first
  auto issue = [&](int d0, int d1) __attribute__((always_inline)) {
#pragma unroll
    for (int d = d0; d < d1; ++d) {
      if (d < kDB && !kOdd && g.once)
        dma16_once(ub, b_off[d], db + d * 1024);
      else if (d < kDB)
        dma16_base(ub, b_off[d], db + d * 1024);
      else
        dma16_base(ua, a_off[d - kDB], da + (d - kDB) * 1024);
    }
  };
  constexpr int kD = kDA + kDB;
  auto quarter = [&](int q) __attribute__((always_inline)) { issue(q * kD / 4, (q + 1) * kD / 4); };
  auto slab_wait = [&]() __attribute__((always_inline)) {
    if constexpr (kOdd) {
      slab_barrier<(kUnits - 3) / 2 * kDA + (kUnits - 5) / 2 * kDB>();   // all but the slabs after the next one's columns
      take_b();
      take_a();
    } else {
      slab_barrier<(kUnits / 2 - 2) * kD>();
      take_a();
      take_b();
    }
  };

  const int swz = (lrow >> 1) & 7;
  const char* x_base = smem + (wm * W::WTM + lrow) * kRow;
  const char* w_base = smem + (wn * W::WTN + lrow) * kRow;
  // bf16: the fragments of a k-step (16 columns), a 16-byte vector a lane; fp32: of two (8
  // vectors of 4 columns in the slab), which together contract 16 columns.
  constexpr bool kF32 = sizeof(T) == 4, kRowsFirst = EPI == kStoreOdd;
  constexpr int kSteps = kF32 ? 2 : 4, kVec = kF32 ? 2 : 1;
  typedef std::conditional_t<kF32, f32x4, bf16x8> F;
  F xf[2][kTM][kVec], wf[2][kTN][kVec];
  auto frags = [&](int aslot, int step, F (&xs)[kTM][kVec], F (&ws)[kTN][kVec]) __attribute__((always_inline)) {
    const int bslot = aslot + 1 == kUnits ? 0 : aslot + 1;
#pragma unroll
    for (int c = 0; c < kVec; ++c) {
      const int cofs = ((((step * kVec + c) * 2 + lhalf) ^ swz) << 4);
#pragma unroll
      for (int i = 0; i < kTM; ++i)
        xs[i][c] = *reinterpret_cast<const F*>(x_base + slot_at(aslot) + i * 32 * kRow + cofs);
#pragma unroll
      for (int j = 0; j < kTN; ++j)
        ws[j][c] = *reinterpret_cast<const F*>(w_base + slot_at(bslot) + j * 32 * kRow + cofs);
    }
  };

  if constexpr (kOdd) {
    take_a();
    issue(kDB, kD);
#pragma unroll
    for (int u = 1; u < kUnits - 2; u += 2) {
      take_b();
      issue(0, kDB);
      take_a();
      issue(kDB, kD);
    }
  } else {
#pragma unroll
    for (int u = 0; u < kUnits - 2; u += 2) {
      take_a();
      take_b();
      issue(0, kD);
    }
  }
  slab_wait();
  quarter(0);
  frags(0, 0, xf[0], wf[0]);
  int aslot = 0;

  for (;;) {
    f32x16 acc[kTN][kTM];
    if constexpr (EPI == kLse || EPI == kDLogit || EPI == kDLogitSum) {
      start_from_bias<W>(g, acc, cur.n0 + wn * W::WTN, lhalf);
    } else {
#pragma unroll
      for (int j = 0; j < kTN; ++j)
#pragma unroll
        for (int i = 0; i < kTM; ++i)
#pragma unroll
          for (int v = 0; v < 16; ++v) acc[j][i][v] = 0.0f;
    }
    for (int kt = cur.k0; kt < cur.k1; ++kt) {
#pragma unroll
      for (int ks = 0; ks < kSteps; ++ks) {
        if (ks + 1 < kSteps) {
#pragma unroll
          for (int q = ks * 3 / (kSteps - 1); q < (ks + 1) * 3 / (kSteps - 1); ++q) quarter(q + 1);
          frags(aslot, ks + 1, xf[(ks + 1) & 1], wf[(ks + 1) & 1]);
        } else {
          aslot += 2;
          if (aslot >= kUnits) aslot -= kUnits;
          slab_wait();
          quarter(0);
          frags(aslot, 0, xf[0], wf[0]);
        }
        auto& xs = xf[ks & 1];
        auto& ws = wf[ks & 1];
        if constexpr (kF32) {
          Split sw[kTN];
#pragma unroll
          for (int j = 0; j < kTN; ++j) sw[j] = split(ws[j][0], ws[j][1]);
#pragma unroll
          for (int i = 0; i < kTM; ++i) {
            const Split sx = split(xs[i][0], xs[i][1]);
#pragma unroll
            for (int j = 0; j < kTN; ++j)
              acc[j][i] = kRowsFirst ? contract(sx, sw[j], acc[j][i]) : contract(sw[j], sx, acc[j][i]);
          }
        } else {
#pragma unroll
          for (int j = 0; j < kTN; ++j)
#pragma unroll
            for (int i = 0; i < kTM; ++i)
              acc[j][i] = kRowsFirst ? contract(xs[i][0], ws[j][0], acc[j][i]) : contract(ws[j][0], xs[i][0], acc[j][i]);
          constexpr int kReads = kTM + kTN, kMfma = kTN * kTM;
          constexpr int kPairs = kReads < kMfma ? kReads : kMfma;
#pragma unroll
          for (int q = 0; q < kPairs; ++q) {
            __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);   // one MFMA
            __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);   // one LDS read
          }
          if constexpr (kMfma > kPairs) __builtin_amdgcn_sched_group_barrier(0x008, kMfma - kPairs, 0);
          if constexpr (kReads > kPairs) __builtin_amdgcn_sched_group_barrier(0x100, kReads - kPairs, 0);
        }
      }
    }
    // (the lane formed again rather than kept live across the loop: the 256 x 256 tiles
    // run at the register limit)
    int lane_now;
    asm volatile("v_mbcnt_lo_u32_b32 %0, -1, 0\n\tv_mbcnt_hi_u32_b32 %0, -1, %0" : "=v"(lane_now));
    const int lr = lane_now & 31, lh = lane_now >> 5;
    const int row0 = cur.row0 + wm * W::WTM, fw = cur.n0 + wn * W::WTN;
    if constexpr (EPI == kLse)
      emit_lse<T, W>(g, acc, row0, fw, lr, lh);
    else if constexpr (EPI == kDLogit || EPI == kDLogitSum)
      emit_dlogit<T, W, EPI == kDLogitSum>(g, acc, row0, fw, lr, lh, cur.row0 / BM * W::WM + wm);
    else if constexpr (EPI == kPart)
      emit_part<W>(g, acc, cur.part, row0, fw, lr, lh);
    else if constexpr (EPI == kStore)
      emit_store<T, W>(g, acc, row0, fw, lr, lh);
    else
      emit_store_odd<T, W>(g, acc, row0, fw, lr, lh);
    t += G;
    if (!locate_item<BM, BN>(g, t, &cur)) break;
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");   // the repeated tail loads
}

// (max, sum) of two sets of exponentials, as one.
__device__ __forceinline__ void merge(float& m, float& s, float m2, float s2) {
  const float n = fmaxf(m, m2);
  if (n == -INFINITY) return;   // both empty
  s = s * __builtin_amdgcn_exp2f((m - n) * kLog2e) + s2 * __builtin_amdgcn_exp2f((m2 - n) * kLog2e);
  m = n;
}

__device__ __forceinline__ float wave_max(float v) {
#pragma unroll
  for (int d = 32; d >= 1; d >>= 1) v = fmaxf(v, __shfl_xor(v, d, kWave));
  return v;
}
template <typename S>
__device__ __forceinline__ S wave_total(S v) {
#pragma unroll
  for (int d = 32; d >= 1; d >>= 1) v += __shfl_xor(v, d, kWave);
  return v;
}

struct JoinSum {
  double loss;
  int count, pad;
};

// TOK tokens a block, SLICES threads each: 16 and 64; 64 and 4 where a row has up to 64 sums to
// add up (1024 rows of 8 sums 8.5 -> 5.2 us); 4 and 64, with more loads in flight, for few
// rows (64 rows of 786 sums 9 -> 7 us, but 2000 rows of 470 12 -> 21).
// mean[0]: the mean over the rows with a target, 0 if there is none; mean[1]: their
// number; the last block to end adds the blocks' sums up, in their order.
template <int TOK, int SLICES>
__global__ __launch_bounds__(TOK * SLICES) void join_kernel(const float2* __restrict__ part, int P, int ld, int N, int V,
                                                    const float* __restrict__ picked,
                                                    const int32_t* __restrict__ targets, float* __restrict__ loss,
                                                    float* __restrict__ lse, float* __restrict__ mean,
                                                    JoinSum* __restrict__ sums, int* counter) {
  constexpr int kThreads = TOK * SLICES;
  __shared__ float2 red[SLICES][TOK + 1];
  __shared__ JoinSum total[kThreads / kWave];
  __shared__ bool last;
  const int tok = threadIdx.x % TOK, slice = threadIdx.x / TOK, n = blockIdx.x * TOK + tok;
  float m = -INFINITY, s = 0.0f;
  bool nan = false;
  if (n < N) {
    constexpr int kAhead = TOK == 4 ? 16 : 4;   // loads in flight
    for (int p0 = slice; p0 < P; p0 += SLICES * kAhead) {
      float2 v[kAhead];
#pragma unroll
      for (int u = 0; u < kAhead; ++u)
        v[u] = p0 + SLICES * u < P ? part[(size_t)(p0 + SLICES * u) * ld + n] : make_float2(-INFINITY, 0.0f);
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        nan |= v[u].y != v[u].y;   // (the maximum passes over NaN)
        merge(m, s, v[u].x, v[u].y);
      }
    }
    if (nan) s = __uint_as_float(0x7FC00000u);
  }
  red[slice][tok] = make_float2(m, s);
  __syncthreads();
  for (int d = SLICES / 2; d >= 1; d >>= 1) {
    if (slice < d) {
      const float2 o = red[slice + d][tok];
      float2 v = red[slice][tok];
      const bool bad = v.y != v.y || o.y != o.y;
      merge(v.x, v.y, o.x, o.y);
      if (bad) v.y = __uint_as_float(0x7FC00000u);
      red[slice][tok] = v;
    }
    __syncthreads();
  }
  if (threadIdx.x < kWave) {   // (the first TOK lanes have a token)
    float l = 0.0f;
    bool has = false;
    if (slice == 0 && n < N) {
      const float2 v = red[0][tok];
      const float z = v.x == -INFINITY && v.y == 0.0f ? -INFINITY : v.x + logf(v.y);
      const int t = targets[n];
      has = t >= 0 && t < V;
      l = has ? z - picked[n] : 0.0f;
      lse[n] = z;
      loss[n] = l;
    }
    if (mean) {
      const double sum = wave_total((double)l);
      const int count = wave_total(has ? 1 : 0);
      if (threadIdx.x == 0) {
        sums[blockIdx.x] = {sum, count, 0};
        __threadfence();
        last = atomicAdd(counter, 1) == (int)gridDim.x - 1;
      }
    }
  }
  if (!mean) return;
  __syncthreads();
  if (!last) return;
  __threadfence();
  JoinSum a = {0.0, 0, 0};
  for (int b = threadIdx.x; b < (int)gridDim.x; b += kThreads) {
    a.loss += sums[b].loss;
    a.count += sums[b].count;
  }
  a.loss = wave_total(a.loss);
  a.count = wave_total(a.count);
  if (lane_id() == 0) total[threadIdx.x / kWave] = a;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int i = 1; i < kThreads / kWave; ++i) {
      a.loss += total[i].loss;
      a.count += total[i].count;
    }
    mean[0] = a.count ? (float)(a.loss / (double)a.count) : 0.0f;
    mean[1] = (float)a.count;
  }
}

// What a backward's products read, by ranges of blocks of 256 threads: the rows' upstream
// gradients, and transposes of x and of the first piece of W (for a later piece that
// alone), zeros past their rows, through 64 x 64 tiles.
//
// The upstream gradients as scale[n] times *factor, the largest magnitude (1 for each row
// of a mean): so d = (p - onehot) scale rounds to bf16 as p - onehot does; one common odd
// factor within d would round all its targets' entries the same way, an error that adds
// up over the rows.  scale is 0 where row n has no target.
template <typename T>
struct PrepareArgs {
  int scale_blocks, rows_per_block;
  const int32_t* targets;
  const float *dloss, *dmean;
  int N, V;
  float *scale, *factor;
  struct {
    const T* src;   // [rows][cols]
    T* dst;         // [cols][ld]
    int rows, cols, ld, blocks, vec;
  } t[2];
};

// The kV elements p[0 .. kV - 1] of a row, those from the n-th on as zeros, for a row that
// starts anywhere: by dwords where all that they hold is the row's own.
template <typename T>
__device__ __forceinline__ uint4 load_odd(const T* p, int n, bool before) {
  constexpr int kV = 16 / (int)sizeof(T);
  struct __attribute__((packed, aligned(4))) Words {
    uint32_t w[4];
  };
  if (((uintptr_t)p & 3) == 0 && n >= kV) {
    const Words d = *reinterpret_cast<const Words*>(p);
    return make_uint4(d.w[0], d.w[1], d.w[2], d.w[3]);
  }
  if constexpr (sizeof(T) == 2) {
    if (before && n > kV) {   // (an odd row: the elements from -1 to kV, shifted)
      const Words d = *reinterpret_cast<const Words*>(p - 1);
      const uint32_t last = *reinterpret_cast<const uint32_t*>(p + 7);
      return make_uint4(__builtin_amdgcn_alignbyte(d.w[1], d.w[0], 2), __builtin_amdgcn_alignbyte(d.w[2], d.w[1], 2),
                        __builtin_amdgcn_alignbyte(d.w[3], d.w[2], 2), __builtin_amdgcn_alignbyte(last, d.w[3], 2));
    }
  }
  T v[kV];
#pragma unroll
  for (int q = 0; q < kV; ++q) v[q] = q < n ? p[q] : T(0);
  uint4 u;
  __builtin_memcpy(&u, v, 16);
  return u;
}

// dst [rows][ld] = src [rows][cols], zeros past a row; ld a multiple of a 16-byte vector.
template <typename T>
__global__ __launch_bounds__(256) void pad_kernel(const T* __restrict__ src, int rows, int cols,
                                                  T* __restrict__ dst, int ld) {
  constexpr int kV = 16 / (int)sizeof(T);
  const int per = ld / kV;
  const size_t total = (size_t)rows * per;
  for (size_t i = (size_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (size_t)gridDim.x * 256) {
    const size_t r = i / per;
    const int c = (int)(i % per) * kV;
    const uint4 u = c < cols ? load_odd(src + r * cols + c, cols - c, c > 0) : make_uint4(0u, 0u, 0u, 0u);
    *reinterpret_cast<uint4*>(dst + i * kV) = u;
  }
}

template <typename T>
__global__ __launch_bounds__(256) void prepare_kernel(PrepareArgs<T> a) {
  constexpr int kV = 16 / (int)sizeof(T);   // elements a vector
  __shared__ __attribute__((aligned(16))) T tile[64][64 + kV];
  __shared__ float rm[4];
  __shared__ int rc[4];
  int b = blockIdx.x;
  if (b < a.scale_blocks) {
    int c = 0;
    float m = 0.0f;
    for (int n = threadIdx.x; n < a.N; n += 256) {
      const int t = a.targets[n];
      if (t >= 0 && t < a.V) {
        ++c;
        if (a.dloss) m = fmaxf(m, fabsf(a.dloss[n]));
      }
    }
    c = wave_total(c);
    m = wave_max(m);
    if (lane_id() == 0) {
      rc[threadIdx.x / kWave] = c;
      rm[threadIdx.x / kWave] = m;
    }
    __syncthreads();
    c = rc[0] + rc[1] + rc[2] + rc[3];
    m = fmaxf(fmaxf(rm[0], rm[1]), fmaxf(rm[2], rm[3]));
    float f;
    if (a.dloss)
      f = m > 0.0f && m < INFINITY ? m : 1.0f;
    else
      f = c ? (a.dmean ? *a.dmean : 1.0f) / (float)c : 0.0f;
    if (b == 0 && threadIdx.x == 0) *a.factor = f;
    const int n1 = min(a.N, (b + 1) * a.rows_per_block);
    for (int n = b * a.rows_per_block + threadIdx.x; n < n1; n += 256) {
      const int t = a.targets[n];
      a.scale[n] = t >= 0 && t < a.V ? (a.dloss ? a.dloss[n] / f : 1.0f) : 0.0f;
    }
    return;
  }
  b -= a.scale_blocks;
  const int k = b < a.t[0].blocks ? 0 : 1;
  if (k) b -= a.t[0].blocks;
  const auto& t = a.t[k];
  const int nx = (t.cols + 63) / 64;   // tiles across; columns fastest: whole rows of the source
  const int c0 = b % nx * 64, r0 = b / nx * 64;
  // rows r0 .. of src into the tile; a row of x without a target as zeros, whatever it
  // holds (its d is 0, and 0 times what is not finite would not be)
  for (int i = threadIdx.x; i < 64 * 64 / kV; i += 256) {
    const int r = i / (64 / kV), c = i % (64 / kV) * kV;
    bool in = r0 + r < t.rows;
    if (k == 0 && in) {
      const int target = a.targets[r0 + r];
      in = target >= 0 && target < a.V;
    }
    const T* p = t.src + (size_t)(r0 + r) * t.cols + c0 + c;
    uint4 v = make_uint4(0u, 0u, 0u, 0u);
    if (in && c0 + c < t.cols) {
      if (t.vec) v = *reinterpret_cast<const uint4*>(p);   // (a vector is within the row or past it)
      else v = load_odd(p, t.cols - c0 - c, c0 + c > 0);
    }
    *reinterpret_cast<uint4*>(&tile[r][c]) = v;
  }
  __syncthreads();
  // (ld is a multiple of 64: every tile's columns of dst exist)
  for (int i = threadIdx.x; i < 64 * 64 / kV; i += 256) {
    const int c = i / (64 / kV), r = i % (64 / kV) * kV;
    if (c0 + c >= t.cols) continue;
    T v[kV];
#pragma unroll
    for (int q = 0; q < kV; ++q) v[q] = tile[r + q][c];
    uint4 u;
    __builtin_memcpy(&u, v, 16);
    *reinterpret_cast<uint4*>(t.dst + (size_t)(c0 + c) * t.ld + r0 + r) = u;
  }
}

// out[m][c] = *factor times the sum of part[.][m][c], in order; a quad of columns a thread.
template <typename T>
__global__ __launch_bounds__(256) void reduce_kernel(const float* __restrict__ part, int parts, int M, int C, size_t ld,
                                                     const float* __restrict__ factor, T* __restrict__ out, int vec) {
  const int quads = (C + 3) / 4;
  const float f = *factor;
  for (size_t i = (size_t)blockIdx.x * 256 + threadIdx.x; i < (size_t)M * quads; i += (size_t)gridDim.x * 256) {
    const size_t m = i / quads;
    const int c = (int)(i % quads) * 4;
    float4 s = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 4
    for (int p = 0; p < parts; ++p) {
      const float4 v = *reinterpret_cast<const float4*>(part + ((size_t)p * M + m) * ld + c);
      s.x += v.x; s.y += v.y; s.z += v.z; s.w += v.w;
    }
    s.x *= f; s.y *= f; s.z *= f; s.w *= f;
    T* o = out + m * C + c;
    if (vec) {
      if constexpr (sizeof(T) == 4) *reinterpret_cast<float4*>(o) = s;
      else *reinterpret_cast<uint2*>(o) = pack4_bf16(s.x, s.y, s.z, s.w);
    } else {
      const float v[4] = {s.x, s.y, s.z, s.w};
#pragma unroll
      for (int q = 0; q < 4; ++q)
        if (c + q < C) store_act(o + q, v[q]);
    }
  }
}

// db[f] = *factor times the sum of the rows of colsum, 64 columns a block of 16 waves.
__global__ __launch_bounds__(1024) void colsum_kernel(const float* __restrict__ src, int rows, size_t ld, int n,
                                                      const float* __restrict__ factor, float* __restrict__ db) {
  __shared__ float lds[16][kWave];
  const int w = threadIdx.x / kWave, lane = lane_id(), f = blockIdx.x * kWave + lane;
  float s = 0.0f;
  if (f < n)
    for (int r = w; r < rows; r += 16) s += src[(size_t)r * ld + f];
  lds[w][lane] = s;
  __syncthreads();
  if (w == 0 && f < n) {
    float t = 0.0f;
    for (int i = 0; i < 16; ++i) t += lds[i][lane];
    db[f] = t * *factor;
  }
}

int compute_units() {
  int dev = 0, n = 0;
  if (hipGetDevice(&dev) != hipSuccess ||
      hipDeviceGetAttribute(&n, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess || n <= 0)
    return 256;
  return n;
}

size_t align_up(size_t v, size_t a) { return (v + a - 1) / a * a; }
int div_up(int a, int b) { return (a + b - 1) / b; }

// Tile size and parts of a product of M rows, Nf columns, KT slabs: the least of the
// estimated times over the sizes and, where the contraction may be split, 1 .. 128 parts of
// at least 4 slabs.  A CU takes ceil(items / CUs) items one after the other (the
// smaller tiles two at a time, at the same rate); a part costs its fp32 sums' way to memory and
// back, all of them a launch.  Rates: the large tile's, 1250 TFLOP/s in bf16 and 180 in fp32 over
// 256 CUs, times what the smaller ones reach of it (16384 x 1024 x 16128, bf16, dW: 411 /
// 524 / 769 us; 4096 x 512 x 8000, fp32, forward: 185 / 220 / 294).  The smallest tile is
// for products that leave CUs without one, whose waves then do half as much each: 1024 x
// 128 x 256 fp32, the forward 10.3 us with 64 x 128 tiles, 8.2 with 64 x 64, d 13.2 / 10.3,
// dx 12.9 / 10.2.
enum TileSize { kTiny, kSmall, kMid, kLarge };   // 64 x 64, 64 x 128, 128 x 128 (two blocks a CU), 256 x 256
int tile_rows(TileSize t) { return t == kLarge ? 256 : t == kMid ? 128 : 64; }
int tile_cols(TileSize t) { return t == kLarge ? 256 : t == kTiny ? 64 : 128; }
int wave_cols(TileSize t) { return t == kTiny ? 32 : 64; }
struct GemmPlan {
  TileSize tile;
  int parts;
};
template <typename T>
GemmPlan plan_gemm(int M, int Nf, int KT, bool split, TileSize most, int cus) {
  const double rate = (sizeof(T) == 2 ? 1250e6 : 180e6) / 256;   // operations a us and CU
  GemmPlan best{kSmall, 1};
  double least = 1e300;
  for (int t = kTiny; t <= most; ++t) {
    const TileSize tile = (TileSize)t;
    const double reach = tile == kLarge ? 1.0 : tile == kMid ? 0.82 : tile == kSmall ? 0.6 : 0.5;
    const long tiles = (long)div_up(M, tile_rows(tile)) * div_up(Nf, tile_cols(tile));
    const double one = 2.0 * tile_rows(tile) * tile_cols(tile) * KT * (128 / sizeof(T)) / (rate * reach);
    for (int p = 1; p <= (split ? std::max(1, std::min(128, KT / 4)) : 1); ++p) {
      const long rounds = (tiles * p + cus - 1) / cus;
      if (rounds > 1 && tile == kTiny) break;
      double us = (double)rounds * one / p;
      if (rounds == 1 && tile != kLarge) us *= 1.35;   // a block alone does not cover its waits
      if (p > 1) us += p * ((double)M * Nf * 8 / 5e6 + 0.25) + 4;
      if (us < least) {
        least = us;
        best = {tile, p};
      }
    }
  }
  return best;
}

template <typename T, int EPI>
hipError_t launch_ring(LossArgs g, const GemmPlan& p, int cus, hipStream_t st) {
  g.parts = std::min(p.parts, g.KT);   // (every part has a slab; a short last piece adds to fewer)
  g.mt = div_up(g.M, tile_rows(p.tile));
  g.nt = div_up(g.Nf, tile_cols(p.tile));
  for (g.turn = 1; 2 * g.turn <= g.KT / g.parts;) g.turn *= 2;
  --g.turn;
  g.once = (size_t)g.Nf * g.ldb >= (size_t)256 << 20;   // (what the last-level cache has no room for)
  const long items = (long)g.mt * g.nt * g.parts;
  if (items > 0x3FFFFFFF || std::max(g.lda, g.ldb) * 256 > 0xFFFFFFFFu ||
      std::max(g.ldd, g.lddt) * 32 * sizeof(T) > 0xFFFFFFFFu)
    return hipErrorInvalidValue;
  const int grid =
      (int)std::min<long>((items + kNumXcd - 1) / kNumXcd * kNumXcd, p.tile == kLarge ? cus : 2 * cus);
  auto go = [&](auto kernel, int threads) {
    hipLaunchKernelGGL(kernel, dim3(grid), dim3(threads), 0, st, g);
  };
  const bool alone = items <= cus;
  if (p.tile == kTiny) {
    go(ring_kernel<T, EPI, 64, 64, 4, 9>, 256);
  } else if (p.tile == kSmall) {
    if (g.mt == 1 && alone) go(ring_kernel<T, EPI, 64, 128, 4, 12>, 256);
    else if (g.mt == 1) go(ring_kernel<T, EPI, 64, 128, 4, 6>, 256);
    else if (alone) go(ring_kernel<T, EPI, 64, 128, 4, 9>, 256);
    else go(ring_kernel<T, EPI, 64, 128, 4, 5>, 256);
  } else if (p.tile == kMid) {
    if (alone) go(ring_kernel<T, EPI, 128, 128, 4, 9>, 256);
    else go(ring_kernel<T, EPI, 128, 128, 4, 5>, 256);
  } else {
    if constexpr (!(sizeof(T) == 4 && (EPI == kDLogit || EPI == kDLogitSum)))
      go(ring_kernel<T, EPI, 256, 256, 8, 5>, 512);
    else
      return hipErrorInvalidValue;   // (its epilogue beside the split operands spills registers)
  }
  return hipGetLastError();
}

template <typename T>
hipError_t launch_store(const LossArgs& g, const GemmPlan& p, int cus, hipStream_t st) {
  const bool vec = g.Nf % 8 == 0 && ((uintptr_t)g.out & 15) == 0;
  return vec ? launch_ring<T, kStore>(g, p, cus, st) : launch_ring<T, kStoreOdd>(g, p, cus, st);
}

// The type's elements per 128-byte slab.
template <typename T> constexpr int kSlab = 128 / (int)sizeof(T);

struct LossLayout {
  // forward
  int ld_lse;
  size_t part_lse, picked, sums, counter, xpad, wpad, total;
  // backward
  int piece, pieces, vpad, nk;   // columns a piece, pieces, columns of d, of its transpose
  size_t scale, factor, xt, wt, d, dt, colsum, dxp, dwp;
  GemmPlan dl, dx, dw;
  bool dx_part;
  int ldx;   // columns of the fp32 partial products
};

constexpr size_t kPieceBytes = (size_t)1 << 30;

template <typename T>
LossLayout loss_layout(int N, int C, int V, bool backward, bool pad, int cus) {
  LossLayout l{};
  size_t off = 0;
  auto take = [&](size_t bytes) {
    const size_t o = off;
    off = align_up(off + bytes, 256);
    return o;
  };
  const int kp = (int)align_up((size_t)C, kSlab<T>);
  if (!backward) {
    l.ld_lse = (int)align_up((size_t)N, 64);
    l.dl = plan_gemm<T>(N, V, kp / kSlab<T>, false, kLarge, cus);
    l.part_lse = take((size_t)div_up(V, wave_cols(l.dl.tile)) * l.ld_lse * sizeof(float2));
    l.picked = take((size_t)N * 4);
    l.sums = take((size_t)std::max(32, div_up(N, 16)) * sizeof(JoinSum));
    l.counter = take(4);
    l.xpad = take(pad ? (size_t)N * kp * sizeof(T) : 0);
    l.wpad = take(pad ? (size_t)V * kp * sizeof(T) : 0);
    l.total = off;
    return l;
  }
  // d and its transpose within kPieceBytes, pieces of equal size
  l.nk = (int)align_up((size_t)N, 64);
  const size_t most = std::max<size_t>(256, kPieceBytes / (2 * sizeof(T) * (size_t)l.nk) / 256 * 256);
  l.pieces = (int)(((size_t)V + most - 1) / most);
  l.piece = (int)align_up((size_t)div_up(V, l.pieces), 256);
  l.pieces = div_up(V, l.piece);
  l.vpad = l.piece;
  l.ldx = (int)align_up((size_t)C, 256);
  l.dl = plan_gemm<T>(N, l.piece, kp / kSlab<T>, false, sizeof(T) == 4 ? kMid : kLarge, cus);
  l.dx = plan_gemm<T>(N, C, div_up(std::min(V, l.piece), kSlab<T>), true, kLarge, cus);
  // (few rows: little but dW's stores, which two blocks a CU overlap; with gradients, 1 x 1024 x
  // 100000 341 -> 327 us, 64 x 4096 x 20000 280 -> 266)
  l.dw = plan_gemm<T>(std::min(V, l.piece), C, l.nk / kSlab<T>, true, l.nk / kSlab<T> <= 2 ? kMid : kLarge, cus);
  l.dx_part = l.pieces > 1 || l.dx.parts > 1;
  l.scale = take((size_t)N * 4);
  l.factor = take(4);
  l.xpad = take(pad ? (size_t)N * kp * sizeof(T) : 0);
  l.wpad = take(pad ? (size_t)l.piece * kp * sizeof(T) : 0);
  l.xt = take((size_t)C * l.nk * sizeof(T));
  l.wt = take((size_t)C * l.vpad * sizeof(T));
  l.d = take((size_t)N * l.vpad * sizeof(T));
  l.dt = take((size_t)l.vpad * l.nk * sizeof(T));
  l.colsum = take((size_t)div_up(N, tile_rows(l.dl.tile)) * 2 * l.vpad * 4);
  l.dxp = take(l.dx_part ? (size_t)l.dx.parts * N * l.ldx * 4 : 0);
  l.dwp = take(l.dw.parts > 1 ? (size_t)l.dw.parts * l.piece * l.ldx * 4 : 0);
  l.total = off;
  return l;
}

template <typename T>
bool needs_pad(int C, const void* x, const void* W) {
  return C % kSlab<T> != 0 || (((uintptr_t)x | (uintptr_t)W) & 15) != 0;
}

template <typename T>
hipError_t launch_pad(const T* src, int rows, int cols, T* dst, int ld, hipStream_t st) {
  const size_t blocks = ((size_t)rows * (ld / (16 / sizeof(T))) + 255) / 256;
  hipLaunchKernelGGL(pad_kernel<T>, dim3((unsigned)std::min<size_t>(blocks, 1 << 16)), dim3(256), 0, st, src, rows,
                     cols, dst, ld);
  return hipGetLastError();
}

template <typename T>
hipError_t forward_impl(const mgpt_lm_loss_config* cfg, const T* x, const T* W, const float* bias,
                        const int32_t* targets, int N, float* loss, float* lse, float* mean, char* ws, bool pad,
                        const LossLayout& l, int cus, hipStream_t st) {
  const int C = cfg->embed_dim, V = cfg->vocab_size, kp = (int)align_up((size_t)C, kSlab<T>);
  hipError_t e;
  if (pad) {
    if ((e = launch_pad<T>(x, N, C, (T*)(ws + l.xpad), kp, st)) != hipSuccess) return e;
    if ((e = launch_pad<T>(W, V, C, (T*)(ws + l.wpad), kp, st)) != hipSuccess) return e;
    x = (const T*)(ws + l.xpad);
    W = (const T*)(ws + l.wpad);
  }
  LossArgs g{};
  g.A = (const char*)x;
  g.B = (const char*)W;
  g.lda = g.ldb = (size_t)kp * sizeof(T);
  g.M = N;
  g.Nf = V;
  g.KT = kp / kSlab<T>;
  g.bias = bias;
  g.targets = targets;
  g.part_lse = (float2*)(ws + l.part_lse);
  g.ld_lse = l.ld_lse;
  g.picked = (float*)(ws + l.picked);
  g.counter = (int*)(ws + l.counter);
  if ((e = launch_ring<T, kLse>(g, l.dl, cus, st)) != hipSuccess) return e;
  const int P = div_up(V, wave_cols(l.dl.tile));
  auto join = [&](auto kernel, int tokens, int threads) {
    hipLaunchKernelGGL(kernel, dim3(div_up(N, tokens)), dim3(threads), 0, st, g.part_lse, P, l.ld_lse, N, V,
                        g.picked, targets, loss, lse, mean, (JoinSum*)(ws + l.sums), g.counter);
  };
  if (P <= 64) join(join_kernel<64, 4>, 64, 256);
  else if (N <= 128) join(join_kernel<4, 64>, 4, 256);
  else join(join_kernel<16, 64>, 16, 1024);
  return hipGetLastError();
}

template <typename T>
hipError_t reduce_parts(const float* part, int parts, int M, int C, int ld, const float* factor, T* out,
                        hipStream_t st) {
  const size_t n = (size_t)M * ((C + 3) / 4);
  const int vec = C % 4 == 0 && ((uintptr_t)out & (4 * sizeof(T) - 1)) == 0;
  hipLaunchKernelGGL(reduce_kernel<T>, dim3((unsigned)std::min<size_t>((n + 255) / 256, 1 << 20)), dim3(256), 0, st,
                     part, parts, M, C, (size_t)ld, factor, out, vec);
  return hipGetLastError();
}

template <typename T>
hipError_t backward_impl(const mgpt_lm_loss_config* cfg, const T* x, const T* W, const float* bias,
                         const int32_t* targets, const float* lse, const float* dloss, const float* dmean, int N,
                         T* dx, T* dW, float* db, char* ws, bool pad, const LossLayout& l, int cus,
                         hipStream_t st) {
  const int C = cfg->embed_dim, V = cfg->vocab_size, kp = (int)align_up((size_t)C, kSlab<T>);
  hipError_t e;
  float *scale = (float*)(ws + l.scale), *factor = (float*)(ws + l.factor);
  const T* xk = x;
  if (pad) {
    if ((e = launch_pad<T>(x, N, C, (T*)(ws + l.xpad), kp, st)) != hipSuccess) return e;
    xk = (const T*)(ws + l.xpad);
  }
  T *xt = (T*)(ws + l.xt), *wt = (T*)(ws + l.wt);
  auto prepare = [&](int piece) -> hipError_t {
    PrepareArgs<T> a{};
    auto transpose = [&](int k, const T* src, int rows, T* dst, int ld) {
      a.t[k] = {src, dst, rows, C, ld, div_up(C, 64) * (ld / 64), C % (16 / (int)sizeof(T)) == 0 && ((uintptr_t)src & 15) == 0};
    };
    if (piece == 0) {
      a.rows_per_block = std::max(256, div_up(N, 64));
      a.scale_blocks = div_up(N, a.rows_per_block);
      a.targets = targets;
      a.dloss = dloss;
      a.dmean = dmean;
      a.N = N;
      a.V = V;
      a.scale = scale;
      a.factor = factor;
      if (dW) transpose(0, x, N, xt, l.nk);
    }
    const int v0 = piece * l.piece;
    if (dx) transpose(1, W + (size_t)v0 * C, std::min(l.piece, V - v0), wt, l.vpad);
    const long blocks = (long)a.scale_blocks + a.t[0].blocks + a.t[1].blocks;
    if (blocks == 0) return hipSuccess;
    if (blocks > 0xFFFFFF) return hipErrorInvalidValue;
    hipLaunchKernelGGL(prepare_kernel<T>, dim3((unsigned)blocks), dim3(256), 0, st, a);
    return hipGetLastError();
  };
  for (int i = 0; i < l.pieces; ++i) {
    const int v0 = i * l.piece, vn = std::min(l.piece, V - v0);
    if ((e = prepare(i)) != hipSuccess) return e;
    const T* wp = W + (size_t)v0 * C;
    const T* wk = wp;
    if (pad) {
      if ((e = launch_pad<T>(wp, vn, C, (T*)(ws + l.wpad), kp, st)) != hipSuccess) return e;
      wk = (const T*)(ws + l.wpad);
    }
    LossArgs g{};
    g.A = (const char*)xk;
    g.B = (const char*)wk;
    g.lda = g.ldb = (size_t)kp * sizeof(T);
    g.M = N;
    g.Nf = vn;
    g.KT = kp / kSlab<T>;
    g.bias = bias ? bias + v0 : nullptr;
    g.targets = targets;
    g.target0 = v0;
    g.lse = lse;
    g.scale = scale;
    g.d = ws + l.d;
    g.ldd = l.vpad;
    g.dt = ws + l.dt;
    g.lddt = l.nk;
    g.rows_t = l.nk;
    g.colsum = db ? (float*)(ws + l.colsum) : nullptr;
    e = db ? launch_ring<T, kDLogitSum>(g, l.dl, cus, st) : launch_ring<T, kDLogit>(g, l.dl, cus, st);
    if (e != hipSuccess) return e;
    if (db) {
      hipLaunchKernelGGL(colsum_kernel, dim3(div_up(vn, kWave)), dim3(1024), 0, st, g.colsum,
                         div_up(N, tile_rows(l.dl.tile)) * 2, g.ldd, vn, factor, db + v0);
      if ((e = hipGetLastError()) != hipSuccess) return e;
    }
    if (dx) {
      LossArgs p{};
      p.A = ws + l.d;
      p.lda = (size_t)l.vpad * sizeof(T);
      p.B = (const char*)wt;
      p.ldb = (size_t)l.vpad * sizeof(T);
      p.M = N;
      p.factor = factor;
      p.Nf = C;
      p.KT = div_up(vn, kSlab<T>);
      p.out = l.dx_part ? ws + l.dxp : (char*)dx;
      p.ldo = l.dx_part ? l.ldx : C;
      p.add = i > 0;
      GemmPlan plan = l.dx;
      if (l.dx_part)
        e = launch_ring<T, kPart>(p, plan, cus, st);
      else
        e = launch_store<T>(p, plan, cus, st);
      if (e != hipSuccess) return e;
    }
    if (dW) {
      LossArgs p{};
      p.A = ws + l.dt;
      p.lda = (size_t)l.nk * sizeof(T);
      p.B = (const char*)xt;
      p.ldb = (size_t)l.nk * sizeof(T);
      p.M = vn;
      p.factor = factor;
      p.Nf = C;
      p.KT = l.nk / kSlab<T>;
      T* out = dW + (size_t)v0 * C;
      p.out = l.dw.parts > 1 ? ws + l.dwp : (char*)out;
      p.ldo = l.dw.parts > 1 ? l.ldx : C;
      if (l.dw.parts > 1) {
        if ((e = launch_ring<T, kPart>(p, l.dw, cus, st)) != hipSuccess) return e;
        e = reduce_parts<T>((const float*)(ws + l.dwp), l.dw.parts, vn, C, l.ldx, factor, out, st);
      } else {
        e = launch_store<T>(p, l.dw, cus, st);
      }
      if (e != hipSuccess) return e;
    }
  }
  if (dx && l.dx_part) return reduce_parts<T>((const float*)(ws + l.dxp), l.dx.parts, N, C, l.ldx, factor, dx, st);
  return hipSuccess;
}

int check_loss(const mgpt_lm_loss_config* cfg, int N) {
  if (!cfg) return fail(MGPT_ERR_INVALID_ARGUMENT, "config is null");
  if (N < 0) return fail(MGPT_ERR_INVALID_ARGUMENT, "negative num_tokens");
  if (cfg->embed_dim <= 0 || cfg->vocab_size <= 0)
    return fail(MGPT_ERR_INVALID_ARGUMENT, "embed_dim %d, vocab_size %d", cfg->embed_dim, cfg->vocab_size);
  if (cfg->dtype != MGPT_DTYPE_F32 && cfg->dtype != MGPT_DTYPE_BF16)
    return fail(MGPT_ERR_UNSUPPORTED, "unsupported dtype %d", cfg->dtype);
  // (row offsets within a tile are 32 bits, tile numbers too)
  if (cfg->embed_dim > 1 << 20 || cfg->vocab_size > 1 << 24 || N > 1 << 21)
    return fail(MGPT_ERR_UNSUPPORTED, "embed_dim %d > 2^20, vocab_size %d > 2^24 or num_tokens %d > 2^21",
                cfg->embed_dim, cfg->vocab_size, N);
  return MGPT_OK;
}

LossLayout layout_of(const mgpt_lm_loss_config* cfg, int N, bool backward, bool pad, int cus) {
  return cfg->dtype == MGPT_DTYPE_F32
             ? loss_layout<float>(N, cfg->embed_dim, cfg->vocab_size, backward, pad, cus)
             : loss_layout<bf16_t>(N, cfg->embed_dim, cfg->vocab_size, backward, pad, cus);
}

int workspace(const mgpt_lm_loss_config* cfg, int N, bool backward, size_t* bytes) {
  if (!bytes) return fail(MGPT_ERR_INVALID_ARGUMENT, "null bytes");
  if (int rc = check_loss(cfg, N)) return rc;
  // as if x or W were not 16-byte aligned, which no caller's size tells
  *bytes = N == 0 ? 0 : layout_of(cfg, N, backward, true, compute_units()).total;
  return MGPT_OK;
}

int check_workspace(const void* ws, size_t have, size_t need) {
  if (!ws) return fail(MGPT_ERR_INVALID_ARGUMENT, "null workspace");
  if ((uintptr_t)ws & 255) return fail(MGPT_ERR_INVALID_ARGUMENT, "workspace must be 256-byte aligned");
  if (have < need) return fail(MGPT_ERR_WORKSPACE_TOO_SMALL, "workspace needs %zu bytes, got %zu", need, have);
  return MGPT_OK;
}

}  // namespace
}  // namespace mgpt

using namespace mgpt;

extern "C" {

int mgpt_lm_loss_workspace_bytes(const mgpt_lm_loss_config* cfg, int num_tokens, size_t* bytes) {
  return workspace(cfg, num_tokens, false, bytes);
}

int mgpt_lm_loss_backward_workspace_bytes(const mgpt_lm_loss_config* cfg, int num_tokens, size_t* bytes) {
  return workspace(cfg, num_tokens, true, bytes);
}

int mgpt_lm_loss_forward(const mgpt_lm_loss_config* cfg, const void* x, const void* W, const float* bias,
                         const int32_t* targets, float* loss, float* lse, float* mean, int num_tokens,
                         void* workspace, size_t workspace_bytes, void* stream) {
  if (int rc = check_loss(cfg, num_tokens)) return rc;
  hipStream_t st = (hipStream_t)stream;
  if (num_tokens == 0) {
    if (mean) HIP_TRY(launch_fill_zero(mean, 2, st));
    return MGPT_OK;
  }
  if (!x || !W || !targets || !loss || !lse)
    return fail(MGPT_ERR_INVALID_ARGUMENT, "null x, W, targets, loss or lse");
  const int cus = compute_units();
  const bool f32 = cfg->dtype == MGPT_DTYPE_F32;
  const bool pad = f32 ? needs_pad<float>(cfg->embed_dim, x, W) : needs_pad<bf16_t>(cfg->embed_dim, x, W);
  const LossLayout l = layout_of(cfg, num_tokens, false, pad, cus);
  if (int rc = check_workspace(workspace, workspace_bytes, l.total)) return rc;
  HIP_TRY(f32 ? forward_impl<float>(cfg, (const float*)x, (const float*)W, bias, targets, num_tokens, loss, lse,
                                    mean, (char*)workspace, pad, l, cus, st)
              : forward_impl<bf16_t>(cfg, (const bf16_t*)x, (const bf16_t*)W, bias, targets, num_tokens, loss, lse,
                                     mean, (char*)workspace, pad, l, cus, st));
  return MGPT_OK;
}

int mgpt_lm_loss_backward(const mgpt_lm_loss_config* cfg, const void* x, const void* W, const float* bias,
                          const int32_t* targets, const float* lse, const float* dloss, const float* dmean,
                          void* dx, void* dW, float* dbias, int num_tokens, void* workspace,
                          size_t workspace_bytes, void* stream) {
  if (int rc = check_loss(cfg, num_tokens)) return rc;
  if (dloss && dmean) return fail(MGPT_ERR_INVALID_ARGUMENT, "dloss and dmean exclude each other");
  hipStream_t st = (hipStream_t)stream;
  const bool f32 = cfg->dtype == MGPT_DTYPE_F32;
  const size_t C = cfg->embed_dim, V = cfg->vocab_size;
  if (num_tokens == 0) {   // no token adds to the weights' gradients
    if (dW && f32) HIP_TRY(launch_fill_zero((float*)dW, V * C, st));
    if (dW && !f32)
      HIP_TRY(launch_copy_cols<bf16_t>((const bf16_t*)dW, 0, (bf16_t*)dW, (int)C, (int)V, 0, (int)C, st));
    if (dbias) HIP_TRY(launch_fill_zero(dbias, V, st));
    return MGPT_OK;
  }
  if (!x || !W || !targets || !lse) return fail(MGPT_ERR_INVALID_ARGUMENT, "null x, W, targets or lse");
  if (!dx && !dW && !dbias) return MGPT_OK;
  const int cus = compute_units();
  const bool pad = f32 ? needs_pad<float>(cfg->embed_dim, x, W) : needs_pad<bf16_t>(cfg->embed_dim, x, W);
  const LossLayout l = layout_of(cfg, num_tokens, true, pad, cus);
  if (int rc = check_workspace(workspace, workspace_bytes, l.total)) return rc;
  HIP_TRY(f32 ? backward_impl<float>(cfg, (const float*)x, (const float*)W, bias, targets, lse, dloss, dmean,
                                     num_tokens, (float*)dx, (float*)dW, dbias, (char*)workspace, pad, l, cus, st)
              : backward_impl<bf16_t>(cfg, (const bf16_t*)x, (const bf16_t*)W, bias, targets, lse, dloss, dmean,
                                      num_tokens, (bf16_t*)dx, (bf16_t*)dW, dbias, (char*)workspace, pad, l, cus,
                                      st));
  return MGPT_OK;
}

}  // extern "C"
