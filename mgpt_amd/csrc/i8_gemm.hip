// i8_gemm.hip -- products in 8-bit integers with a scale for each row and each output:
//   y[n][m] = (sum_k qa[n][k] qb[m][k]) sa[n] sb[m] + bias[m]
// for one weight or for the segments of several experts, and the experts' gate/up product with SwiGLU
// in its epilogue.  The integer sums are exact (K up to 2^17), so their order does not matter.
//
// Operands are row blocks of operand tiles (i8.hpp).  Two kernels:
//  * ring: persistent blocks walk BM x BN output tiles; operands go HBM -> LDS by 1 KB loads
//    into a ring of 5 units (a tile's rows, or its outputs, of a slab of 128 columns), whose
//    barrier frees a slab's two units for the loads of the next outputs and of the rows after them.
//    v_mfma_i32_32x32x32_i8 takes the same bytes a cycle as bf16's 32x32x16 and contracts
//    twice the columns.
//  * stream: few rows a segment; every wave reads the outputs' tiles from memory straight into the
//    registers that the matrix instruction takes, a slab ahead, the rows' from the caches. Waves split a
//    long contraction, add their integers up in LDS and take the outputs' row blocks in turn.
//
// Measured: ring, 16384 x 2048 x 8192 250 us (2200 TOP/s; a library's int8 product of 8192^3 2090); gate/up of 32768 rows x
// 1024 x 5632 in 16 segments 263 us (1440), of it some 70 the epilogue, which a block that fills the CU has nothing to
// hide behind (row scales loaded in it, behind the ring's loads, cost 25 more); down, x 2816 x 1024, 127; the two of an fp32
// caller 302 (a full exponential and a division for each unit, 32 bytes of a row a store) and 140.  Stream, 1 x
// 2048 x 50257 21 us (4.9 TB/s), 512 rows of 64 experts, 2048 x 2816 80 (4.6), 1408 x 2048 35 (5.2); 999 x 500 x 1003 8
// (ring of 128 x 128 tiles: 15).
#include <algorithm>
#include <type_traits>

#include "../../include/mgpt_moe.h"
#include "capi_internal.hpp"
#include "gemm_ring.hpp"
#include "i8.hpp"

namespace mgpt {
namespace {

constexpr int kTileBytes = 1024;             // 32 x 32
constexpr int kSlabBytes = 4 * kTileBytes;   // of a row block

__device__ __forceinline__ i32x16 contract8(i32x4 a, i32x4 b, i32x16 c) {
  return __builtin_amdgcn_mfma_i32_32x32x32_i8(a, b, c, 0, 0, 0);
}

// Where a tile of rows lies: rows row0 .. row_end - 1 of the output, row blocks blk0 .. of A (blk_end:
// past the segment's last).
struct RowTile {
  int expert, row0, row_end, blk0, blk_end;
};

// Lane l holds expert e_base + l of the block's group (at most 64 experts).
template <int BM>
struct Segments {
  int cnt, rows_incl, blks_incl, tiles_incl, tm;
  __device__ __forceinline__ void init(const I8Args& g, int E, int e_base) {
    const int l = lane_id();
    if (!g.counts) {
      cnt = l == 0 ? g.N : 0;
    } else {
      cnt = l < E ? g.counts[e_base + l] : 0;
    }
    int rows = 0, blks = 0;   // of the experts before the group
    for (int e = l; e < e_base; e += kWave) {
      const int c = g.counts[e];
      rows += c;
      blks += (c + kI8Rows - 1) / kI8Rows;
    }
    if (e_base > 0) {
      rows = __builtin_amdgcn_readfirstlane(__shfl(wave_incl_scan(rows), kWave - 1, kWave));
      blks = __builtin_amdgcn_readfirstlane(__shfl(wave_incl_scan(blks), kWave - 1, kWave));
    }
    rows_incl = wave_incl_scan(cnt) + rows;
    blks_incl = wave_incl_scan((cnt + kI8Rows - 1) / kI8Rows) + blks;
    tiles_incl = wave_incl_scan((cnt + BM - 1) / BM);
    tm = __builtin_amdgcn_readfirstlane(__shfl(tiles_incl, kWave - 1, kWave));
  }
  // row tile mt < tm
  __device__ __forceinline__ void find(int mt, RowTile* out) const {
    const int tiles = (cnt + BM - 1) / BM, excl = tiles_incl - tiles;
    const unsigned long long m = __ballot(mt >= excl && mt < tiles_incl);
    const int owner = __ffsll((long long)m) - 1;
    auto of = [&](int v) { return __builtin_amdgcn_readfirstlane(__shfl(v, owner, kWave)); };
    const int t = mt - of(excl);
    out->expert = owner;
    out->row_end = of(rows_incl);
    out->row0 = out->row_end - of(cnt) + t * BM;
    out->blk_end = of(blks_incl);
    out->blk0 = out->blk_end - (of(cnt) + kI8Rows - 1) / kI8Rows + t * (BM / kI8Rows);
  }
};

struct I8Tile {
  RowTile r;
  int n0;
};

template <int BM, int BN>
__device__ __forceinline__ bool locate8(const Segments<BM>& sc, int nbx, int v, I8Tile* out) {
  if (v >= sc.tm * nbx) return false;
  // groups of kGroupM row tiles x all output tiles, rows fastest (as locate_tile)
  const int grp = v / (kGroupM * nbx), gsize = min(kGroupM, sc.tm - grp * kGroupM);
  const int idx = v - grp * kGroupM * nbx;
  sc.find(grp * kGroupM + idx % gsize, &out->r);
  out->n0 = idx / gsize * BN;
  return true;
}

// 32 floats at a uniform address, of which a lane takes those of its half's rows of an
// accumulator: value v is element 8 (v / 4) + 4 half + v % 4.  Scalar loads: a vector load here
// would wait for the ring's loads, which the compiler does not track.
__device__ __forceinline__ f32x16 take32(const float* p, int half) {
  typedef const __attribute__((address_space(4))) float* cptr;
  const uint64_t a = (uint64_t)(uintptr_t)p;
  const uint32_t lo = __builtin_amdgcn_readfirstlane((uint32_t)a), hi = __builtin_amdgcn_readfirstlane((uint32_t)(a >> 32));
  const cptr u = (cptr)(uintptr_t)(((uint64_t)hi << 32) | lo);
  f32x16 r;
#pragma unroll
  for (int k = 0; k < 4; ++k)
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const float x = u[8 * k + q], y = u[8 * k + 4 + q];
      r[4 * k + q] = half ? y : x;
    }
  return r;
}

// The same for outputs f0 .. f0 + 31 of which n exist; zeros past them or without an array.
__device__ __forceinline__ f32x16 take_outputs(const float* p, int n, int half) {
  if (p && n >= 32) return take32(p, half);
  f32x16 r;
#pragma unroll
  for (int v = 0; v < 16; ++v) {
    const int f = 8 * (v / 4) + 4 * half + v % 4;
    r[v] = p && f < n ? p[f] : 0.0f;
  }
  return r;
}

// The scales of a lane's rows row0 + 32 i + lrow of the tile t.
template <int TM>
__device__ __forceinline__ void row_scales(const I8Args& g, const RowTile& t, int row0, int blk, int lrow, float (&sa)[TM]) {
#pragma unroll
  for (int i = 0; i < TM; ++i)
    sa[i] = row0 + 32 * i + lrow < t.row_end ? g.sa[(size_t)(blk + i) * kI8Rows + lrow] : 0.0f;
}

// Columns col .. col + 31 of a row of HiddenRows: a lane of each half has 16 values, as an accumulator does, and their
// largest magnitude's bits.
__device__ __forceinline__ void put_hidden(const HiddenRows& to, const float (&x)[16], uint32_t top, int row, int col,
                                           int half, bool live) {
  constexpr int kBits = 20;
  const auto o = __builtin_amdgcn_permlane32_swap(top, top, false, false);
  top = max(o[0], o[1]);
  const int e = max((int)(top >> 23), kBits);
  // to units of 2^(e - 125 - kBits), in the low bits of a sum; a magnitude that would round to 2^(kBits - 1) of them stays
  // below
  const float f = __uint_as_float((uint32_t)max(252 + kBits - e, 1) << 23);
  const float most = __uint_as_float((uint32_t)(e + 2 - kBits) << 23) * (float)((1 << (kBits - 1)) - 1);
  uint32_t q[16];
#pragma unroll
  for (int v = 0; v < 16; ++v)
    q[v] = __float_as_uint(fmaf(__builtin_amdgcn_fmed3f(x[v], -most, most), f, 0x1.8p23f));
  uint2 hi[4];
  uint32_t low[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const uint32_t* w = q + 4 * k;
    hi[k] = make_uint2(__builtin_amdgcn_perm(w[1] << 12, w[0] << 12, 0x07060302),
                       __builtin_amdgcn_perm(w[3] << 12, w[2] << 12, 0x07060302));
    low[k] = __builtin_amdgcn_perm(__builtin_amdgcn_perm(w[3], w[2], 0x0c0c0400),
                                   __builtin_amdgcn_perm(w[1], w[0], 0x0c0c0400), 0x05040100) & 0x0F0F0F0Fu;
  }
  store_group32(reinterpret_cast<bf16_t*>(to.q) + (size_t)row * to.ld + col, hi, half, live);
  const auto n = __builtin_amdgcn_permlane32_swap(low[0] | low[1] << 4, low[2] | low[3] << 4, false, false);
  if (live) *reinterpret_cast<uint2*>(to.n + (size_t)row * (to.ld / 2) + col / 2 + 8 * half) = make_uint2(n[0], n[1]);
  if (live && half == 0) to.top[(size_t)row * (to.ld / 32) + col / 32] = top;
}

// The same of Rows24.
__device__ __forceinline__ void put24(const Rows24& to, const float (&x)[16], int row, int col, int half, bool live) {
  uint2 hi[4];
  uint32_t low[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    uint32_t w[4];
#pragma unroll
    for (int q = 0; q < 4; ++q) w[q] = __float_as_uint(x[4 * k + q]) + (x[4 * k + q] == x[4 * k + q] ? 0x80u : 0u);   // (a NaN stays one)
    hi[k] = make_uint2(__builtin_amdgcn_perm(w[1], w[0], 0x07060302), __builtin_amdgcn_perm(w[3], w[2], 0x07060302));
    low[k] = __builtin_amdgcn_perm(w[1], w[0], 0x0c0c0501) | __builtin_amdgcn_perm(w[3], w[2], 0x05010c0c);
  }
  store_group32(to.hi + (size_t)row * to.ld + col, hi, half, live);
  const auto a = __builtin_amdgcn_permlane32_swap(low[0], low[2], false, false);   // columns 16 half .. + 3, + 4 .. 7
  const auto b = __builtin_amdgcn_permlane32_swap(low[1], low[3], false, false);
  if (live) *reinterpret_cast<uint4*>(to.low + (size_t)row * to.ld + col + 16 * half) = make_uint4(a[0], a[1], b[0], b[1]);
}

// The outputs' scales come first: those of rows reach from the smallest to the largest numbers, and a product of the two
// scales alone would leave them (0 times infinity for a sum of 0, bits lost below 2^-126).
//
// Accumulators of TN x TM tiles: outputs fw + 32 j, rows row0 + 32 i of the tile t (row blocks
// blk + i of A), and the rows' scales.
template <int KIND, int TN, int TM>
__device__ __forceinline__ void emit8(const I8Args& g, const i32x16 (&acc)[TN][TM], const float (&sa)[TM], const RowTile& t,
                                      int row0, int fw, int lrow, int half) {
  const size_t eb = (size_t)(g.e_base + t.expert);
  const float* sb = g.sb + eb * g.ldsb;
  if constexpr (KIND == kI8GateUp || KIND == kI8GateUpF32) {
#pragma unroll
    for (int gi = 0; gi < TN / 2; ++gi) {
      const int f0 = fw + 64 * gi, hb = f0 / 2;
      if (f0 >= g.Nf) continue;
      const f32x16 sg = take32(sb + f0, half), su = take32(sb + f0 + 32, half);
      const f32x16 bg = take32(g.bias0 + eb * g.bias_ld + hb, half), bu = take32(g.bias1 + eb * g.bias_ld + hb, half);
#pragma unroll
      for (int i = 0; i < TM; ++i) {
        const int row = row0 + 32 * i + lrow;
        float h[16];
        uint32_t top = 0;
#pragma unroll
        for (int v = 0; v < 16; ++v) {
          const float ag = (float)acc[2 * gi][i][v], au = (float)acc[2 * gi + 1][i][v];
          if constexpr (KIND == kI8GateUpF32) {
            // each operation's own rounding: the integers of h are those of the formula in 32 bits, scales included
            // (QuantizeArgs::by_product)
            const float x = ag * sa[i] * sg[v] + bg[v], u = au * sa[i] * su[v] + bu[v];
            h[v] = x / (1.0f + expf(-x)) * u;
          } else {   // (some 2^-22 off, a quarter of what 20 bits are)
            const float x = fmaf(ag * sg[v], sa[i], bg[v]), u = fmaf(au * su[v], sa[i], bu[v]);
            h[v] = x * __builtin_amdgcn_rcpf(1.0f + __expf(-x)) * u;
          }
          top = max(top, __float_as_uint(h[v]) & 0x7FFFFFFFu);   // (a NaN lies above all)
        }
        if constexpr (KIND == kI8GateUpF32) {
          if (row < t.row_end)
#pragma unroll
            for (int k = 0; k < 4; ++k)
              *reinterpret_cast<float4*>(reinterpret_cast<float*>(g.out) + (size_t)row * g.ldo + hb + 8 * k + 4 * half) =
                  make_float4(h[4 * k], h[4 * k + 1], h[4 * k + 2], h[4 * k + 3]);
        } else {
          put_hidden(g.h, h, top, row, hb, half, row < t.row_end);
        }
        __builtin_amdgcn_sched_barrier(0);
      }
    }
  } else {
#pragma unroll
    for (int j = 0; j < TN; ++j) {
      const int f0 = fw + 32 * j, n = g.Nf - f0;
      if (n <= 0) continue;
      const f32x16 s = take_outputs(sb + f0, n, half);
      const f32x16 b = take_outputs(g.bias0 ? g.bias0 + eb * g.bias_ld + f0 : nullptr, n, half);
#pragma unroll
      for (int i = 0; i < TM; ++i) {
        const int row = row0 + 32 * i + lrow;
        float y[16];
#pragma unroll
        for (int v = 0; v < 16; ++v) y[v] = (float)acc[j][i][v] * s[v] * sa[i] + b[v];
        const bool live = row < t.row_end;
        if constexpr (KIND == kI8Rows24) {
          put24(g.o, y, row, f0, half, live);
        } else if constexpr (KIND == kI8Bf16) {
          bf16_t* o = reinterpret_cast<bf16_t*>(g.out) + (size_t)row * g.ldo + f0;
          uint2 q[4];
#pragma unroll
          for (int k = 0; k < 4; ++k) q[k] = pack4_bf16(y[4 * k], y[4 * k + 1], y[4 * k + 2], y[4 * k + 3]);
          if (n >= 32) {
            store_group32(o, q, half, live);
          } else if (live) {   // (outputs are a multiple of 8: quads are whole)
#pragma unroll
            for (int k = 0; k < 4; ++k)
              if (8 * k + 4 * half < n) *reinterpret_cast<uint2*>(o + 8 * k + 4 * half) = q[k];
          }
        } else {
          float* o = reinterpret_cast<float*>(g.out) + (size_t)row * g.ldo + f0;
          if (live)
#pragma unroll
            for (int k = 0; k < 4; ++k)
              if (8 * k + 4 * half < n)
                *reinterpret_cast<float4*>(o + 8 * k + 4 * half) =
                    make_float4(y[4 * k], y[4 * k + 1], y[4 * k + 2], y[4 * k + 3]);
        }
        __builtin_amdgcn_sched_barrier(0);
      }
    }
  }
}

// The same for accumulators of A B^T (a lane has output fw + 32 j + lrow, value v row 8 (v / 4) + 4 half +
// v % 4): outputs whose rows are not aligned to vectors.
template <int KIND, int TN, int TM>
__device__ __forceinline__ void emit8_odd(const I8Args& g, const i32x16 (&acc)[TN][TM], const RowTile& t, int row0,
                                          int blk, int fw, int lrow, int half) {
  const size_t eb = (size_t)(g.e_base + t.expert);
#pragma unroll
  for (int j = 0; j < TN; ++j) {
    const int f = fw + 32 * j + lrow;
    const bool in = f < g.Nf;
    const float s = in ? g.sb[eb * g.ldsb + f] : 0.0f;
    const float b = in && g.bias0 ? g.bias0[eb * g.bias_ld + f] : 0.0f;
#pragma unroll
    for (int i = 0; i < TM; ++i) {
      if (blk + i >= t.blk_end) continue;
      const f32x16 sa = take32(g.sa + (size_t)(blk + i) * kI8Rows, half);
#pragma unroll
      for (int v = 0; v < 16; ++v) {
        const int row = row0 + 32 * i + 8 * (v / 4) + 4 * half + v % 4;
        const float y = (float)acc[j][i][v] * s * sa[v] + b;
        if (in && row < t.row_end) {
          if constexpr (KIND == kI8Bf16) store_act(reinterpret_cast<bf16_t*>(g.out) + (size_t)row * g.ldo + f, y);
          else reinterpret_cast<float*>(g.out)[(size_t)row * g.ldo + f] = y;
        }
      }
      __builtin_amdgcn_sched_barrier(0);
    }
  }
}

// A 1 KB direct-to-LDS load (see dma16) from a uniform base.
__device__ __forceinline__ void dma_tile(const char* base, uint32_t off, uint32_t lds) {
  asm volatile("global_load_lds_dwordx4 %0, %1" ::"v"(off), "s"(base), "{m0}"(lds) : "memory");
}
__device__ __forceinline__ const char* uniform_address(const char* p) {
  const uint64_t u = (uint64_t)(uintptr_t)p;
  const uint32_t lo = __builtin_amdgcn_readfirstlane((uint32_t)u);
  const uint32_t hi = __builtin_amdgcn_readfirstlane((uint32_t)(u >> 32));
  return reinterpret_cast<const char*>((uintptr_t)(((uint64_t)hi << 32) | lo));
}

template <int KIND, bool ODD, int BM, int BN, int NW>
__global__ __launch_bounds__(NW * kWave, 2) void i8_ring_kernel(I8Args g, int group) {
  using W = Waves<NW, BM, BN>;
  constexpr int TN = W::TN, TM = W::TM, kUnits = 5;
  constexpr int kSlot = (BM > BN ? BM : BN) * kI8Slab;
  constexpr int kDA = BM / 8 / NW, kDB = BN / 8 / NW;   // 1 KB loads of a wave and unit
  static_assert(kDA >= 1 && 4 % kDA == 0, "a wave's loads of a unit lie in one row block");
  static_assert(kDA == kDB, "a repeated unit's loads stay in its row block, whichever operand's they repeat");
  __shared__ __attribute__((aligned(1024))) char smem[kUnits * kSlot];

  const int G = gridDim.x;
  const int nbx = (g.Nf + BN - 1) / BN;
  int E = g.E;
  g.e_base = 0;
  if (gridDim.y > 1) {
    g.e_base = (int)blockIdx.y * group;
    E = min(group, g.E - g.e_base);
  }
  Segments<BM> sc;
  sc.init(g, E, g.e_base);
  // the blocks of an XCD take neighbouring tiles
  int t = G % kNumXcd == 0 ? (int)(blockIdx.x % kNumXcd) * (G / kNumXcd) + (int)blockIdx.x / kNumXcd : (int)blockIdx.x;
  if (sc.tm * nbx < G && G % kNumXcd == 0) {
    const int run = (sc.tm * nbx + kNumXcd - 1) / kNumXcd, in = (int)blockIdx.x / kNumXcd;
    t = in < run ? (int)(blockIdx.x % kNumXcd) * run + in : sc.tm * nbx;
  }
  I8Tile cur;
  if (!locate8<BM, BN>(sc, nbx, t, &cur)) return;

  const int w = __builtin_amdgcn_readfirstlane((int)threadIdx.x / kWave), lane = lane_id();
  const int wn = w % W::WN, wm = w / W::WN;
  const size_t row_block = (size_t)g.KT * kSlabBytes;
  const uint32_t off = (uint32_t)lane * 16;
  const uint32_t lds0 = (uint32_t)(uintptr_t)(lds_char*)smem;
  const uint32_t lds_a = lds0 + (uint32_t)(w * kDA) * kTileBytes, lds_b = lds0 + (uint32_t)(w * kDB) * kTileBytes;
  // a wave's first load of a unit: the row block, past the last one the last, and the place in its slab
  auto rows_at = [&](const I8Tile& c) __attribute__((always_inline)) {
    const int b = min(c.r.blk0 + w * kDA / 4, c.r.blk_end - 1);
    return g.A + (size_t)b * row_block + (w * kDA % 4) * kTileBytes;
  };
  auto outs_at = [&](const I8Tile& c) __attribute__((always_inline)) {
    const int b = min(c.n0 / kI8Rows + w * kDB / 4, g.b_blocks - 1);
    return g.B + (size_t)(g.e_base + c.r.expert) * g.b_expert + (size_t)b * row_block + (w * kDB % 4) * kTileBytes;
  };

  // Cursor over the units A0 B0 A1 B1 .. of the block's tiles.  Past the last one it repeats
  // it (in bounds, into a slot that is free), so that every slab issues the same loads.
  I8Tile dtile;
  int dt = t, dk = 0, dop = 0, dslot = 0;
  bool valid = true;
  const char *da = rows_at(cur), *db = outs_at(cur), *last = da;
  auto next_unit = [&](const char*& src, uint32_t& dst) __attribute__((always_inline)) {
    const bool outs = dop != 0;
    if (valid) last = (outs ? db : da) + (size_t)dk * kSlabBytes;
    src = uniform_address(last);
    dst = (outs ? lds_b : lds_a) + (uint32_t)(dslot * kSlot);
    dslot = dslot + 1 == kUnits ? 0 : dslot + 1;
    dop ^= 1;
    if (outs && valid && ++dk == g.KT) {
      dt += G;
      valid = locate8<BM, BN>(sc, nbx, dt, &dtile);
      if (valid) {
        dk = 0;
        da = rows_at(dtile);
        db = outs_at(dtile);
      }
    }
  };
  const char *ua, *ub;   // the two units that are being loaded: outputs, then rows
  uint32_t la, lb;
  constexpr int kD = kDA + kDB;
  auto issue = [&](int d0, int d1) __attribute__((always_inline)) {
#pragma unroll
    for (int d = d0; d < d1; ++d) {
      if (d < kDB) dma_tile(ub + d * kTileBytes, off, lb + d * kTileBytes);
      else dma_tile(ua + (d - kDB) * kTileBytes, off, la + (d - kDB) * kTileBytes);
    }
  };
  auto quarter = [&](int q) __attribute__((always_inline)) { issue(q * kD / 4, (q + 1) * kD / 4); };
  // (a unit past the end may be rows where outputs are due: both loads stay in their own slot)
  auto slab_wait = [&]() __attribute__((always_inline)) {
    slab_barrier<kDA>();   // all but the next slab's rows have landed
    next_unit(ub, lb);
    next_unit(ua, la);
  };

  i32x4 xf[2][TM], wf[2][TN];
  const char* x_base = smem + wm * TM * kSlabBytes + lane * 16;
  const char* w_base = smem + wn * TN * kSlabBytes + lane * 16;
  auto frags = [&](int aslot, int ks, i32x4 (&xs)[TM], i32x4 (&ws)[TN]) __attribute__((always_inline)) {
    const int bslot = aslot + 1 == kUnits ? 0 : aslot + 1;
#pragma unroll
    for (int i = 0; i < TM; ++i)
      xs[i] = *reinterpret_cast<const i32x4*>(x_base + aslot * kSlot + i * kSlabBytes + ks * kTileBytes);
#pragma unroll
    for (int j = 0; j < TN; ++j)
      ws[j] = *reinterpret_cast<const i32x4*>(w_base + bslot * kSlot + j * kSlabBytes + ks * kTileBytes);
  };

  // A tile's row scales are loaded a tile ahead: a load waits for the ring's loads before it.
  float sa[TM];
  auto scales = [&](const I8Tile& c, float (&to)[TM]) __attribute__((always_inline)) {
    if constexpr (!ODD) row_scales<TM>(g, c.r, c.r.row0 + wm * W::WTM, c.r.blk0 + wm * TM, lane_id() & 31, to);
  };
  scales(cur, sa);
  if constexpr (!ODD)
#pragma unroll
    for (int i = 0; i < TM; ++i) asm volatile("" : "+v"(sa[i]));

  // units A0 B0 A1
  next_unit(ua, la);
  issue(kDB, kD);
  next_unit(ub, lb);
  issue(0, kDB);
  next_unit(ua, la);
  issue(kDB, kD);
  slab_wait();
  quarter(0);
  frags(0, 0, xf[0], wf[0]);
  int aslot = 0;

  for (;;) {
    i32x16 acc[TN][TM];
#pragma unroll
    for (int j = 0; j < TN; ++j)
#pragma unroll
      for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int v = 0; v < 16; ++v) acc[j][i][v] = 0;
    // MT row blocks of the wave hold rows
    auto kloop = [&](auto mt) __attribute__((always_inline)) {
      constexpr int MT = decltype(mt)::value;
      constexpr int kReads = TM + TN, kMfma = TN * MT, kPairs = kReads < kMfma ? kReads : kMfma;
      for (int kt = 0; kt < g.KT; ++kt) {
#pragma unroll
        for (int ks = 0; ks < 4; ++ks) {
          if (ks < 3) {
            quarter(ks + 1);
            frags(aslot, ks + 1, xf[(ks + 1) & 1], wf[(ks + 1) & 1]);
          } else {
            aslot += 2;
            if (aslot >= kUnits) aslot -= kUnits;
            slab_wait();
            quarter(0);
            frags(aslot, 0, xf[0], wf[0]);
          }
#pragma unroll
          for (int j = 0; j < TN; ++j)
#pragma unroll
            for (int i = 0; i < MT; ++i)
              acc[j][i] = ODD ? contract8(xf[ks & 1][i], wf[ks & 1][j], acc[j][i])
                              : contract8(wf[ks & 1][j], xf[ks & 1][i], acc[j][i]);
#pragma unroll
          for (int q = 0; q < kPairs; ++q) {
            __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);   // one MFMA
            __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);   // one LDS read
          }
          if constexpr (kMfma > kPairs) __builtin_amdgcn_sched_group_barrier(0x008, kMfma - kPairs, 0);
          if constexpr (kReads > kPairs) __builtin_amdgcn_sched_group_barrier(0x100, kReads - kPairs, 0);
        }
      }
    };
    const int rows = cur.r.row_end - (cur.r.row0 + wm * W::WTM);
    const int live = rows <= 0 ? 0 : min(TM, (rows + 31) / 32);
    if constexpr (TM == 4) {
      if (live == 3) kloop(IntC<3>{});
      else if (live == 4) kloop(IntC<4>{});
    }
    if constexpr (TM >= 2)
      if (live == 2) kloop(IntC<2>{});
    if (live == 1) kloop(IntC<1>{});
    if (live == 0) kloop(IntC<0>{});
    // (the lane formed again rather than kept across the loop)
    int lane_now;
    asm volatile("v_mbcnt_lo_u32_b32 %0, -1, 0\n\tv_mbcnt_hi_u32_b32 %0, -1, %0" : "=v"(lane_now));
    const int row0 = cur.r.row0 + wm * W::WTM, blk = cur.r.blk0 + wm * TM, fw = cur.n0 + wn * W::WTN;
    t += G;
    I8Tile next;
    const bool more = locate8<BM, BN>(sc, nbx, t, &next);
    float ahead[TM];
    if (more) scales(next, ahead);
    if constexpr (ODD) emit8_odd<KIND, TN, TM>(g, acc, cur.r, row0, blk, fw, lane_now & 31, lane_now >> 5);
    else emit8<KIND, TN, TM>(g, acc, sa, cur.r, row0, fw, lane_now & 31, lane_now >> 5);
    if (!more) break;
    cur = next;
    if constexpr (!ODD)
#pragma unroll
      for (int i = 0; i < TM; ++i) {
        sa[i] = ahead[i];
        asm volatile("" : "+v"(sa[i]));   // (waited for here)
      }
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");   // the repeated loads at the end
}

// Row tile of 32 MT rows number mt, by every thread of the block (LDS); false past the last.
template <int BM>
__device__ __forceinline__ bool find_rows(const I8Args& g, int mt, RowTile* out) {
  if (!g.counts) {
    const int row0 = mt * BM;
    *out = {0, row0, g.N, row0 / kI8Rows, (g.N + kI8Rows - 1) / kI8Rows};
    return row0 < g.N;
  }
  __shared__ int s_info[5];
  if (threadIdx.x < kWave) {
    const int l = lane_id();
    int rows = 0, blks = 0, tiles = 0, found = -1;
    for (int e0 = 0; e0 < g.E && found < 0; e0 += kWave) {
      const int c = e0 + l < g.E ? g.counts[e0 + l] : 0;
      const int ri = wave_incl_scan(c) + rows, bi = wave_incl_scan((c + kI8Rows - 1) / kI8Rows) + blks;
      const int n = (c + BM - 1) / BM, ti = wave_incl_scan(n) + tiles;
      const bool mine = mt >= ti - n && mt < ti;
      if (mine) {
        const int t = mt - (ti - n);
        s_info[1] = ri - c + t * BM;
        s_info[2] = ri;
        s_info[3] = bi - (c + kI8Rows - 1) / kI8Rows + t * (BM / kI8Rows);
        s_info[4] = bi;
      }
      const unsigned long long m = __ballot(mine);
      if (m) found = e0 + __ffsll((long long)m) - 1;
      rows = __shfl(ri, kWave - 1, kWave);
      blks = __shfl(bi, kWave - 1, kWave);
      tiles = __shfl(ti, kWave - 1, kWave);
    }
    if (l == 0) s_info[0] = found;
  }
  __syncthreads();
  *out = {s_info[0], s_info[1], s_info[2], s_info[3], s_info[4]};
  return out->expert >= 0;
}

constexpr int kStreamWaves = 8;
constexpr int kStreamFB = 2;   // row blocks of outputs a wave

// A wave: FB row blocks of outputs, MT of rows, one KS-th of the slabs.
template <int KIND, bool ODD, int MT, int KS>
__global__ __launch_bounds__(kStreamWaves * kWave) void i8_stream_kernel(I8Args g) {
  constexpr int FB = kStreamFB, F = kStreamWaves / KS;   // waves of a block with different outputs
  __shared__ int s_acc[KS > 1 ? F * FB * MT * 16 * kWave : 1];
  g.e_base = 0;
  RowTile t;
  if (!find_rows<32 * MT>(g, blockIdx.y, &t)) return;
  const int w = __builtin_amdgcn_readfirstlane((int)threadIdx.x / kWave), lane = lane_id();
  const int f = w / KS, s = w % KS;
  const int fb = (blockIdx.x * F + f) * FB;
  const size_t row_block = (size_t)g.KT * kSlabBytes;
  const int k0 = s * g.KT / KS, k1 = (s + 1) * g.KT / KS;
  if constexpr (KS > 1) {
    for (int i = threadIdx.x; i < F * FB * MT * 16 * kWave; i += kStreamWaves * kWave) s_acc[i] = 0;
    __syncthreads();
  }
  const char *wp[FB], *xp[MT];
#pragma unroll
  for (int j = 0; j < FB; ++j)
    wp[j] = g.B + (size_t)t.expert * g.b_expert + (size_t)min(fb + j, g.b_blocks - 1) * row_block + lane * 16;
#pragma unroll
  for (int i = 0; i < MT; ++i) xp[i] = g.A + (size_t)min(t.blk0 + i, t.blk_end - 1) * row_block + lane * 16;
  i32x16 acc[FB][MT];
#pragma unroll
  for (int j = 0; j < FB; ++j)
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int v = 0; v < 16; ++v) acc[j][i][v] = 0;
  const bool busy = fb * kI8Rows < g.Nf;
  if (busy) {
    i32x4 wf[2][4][FB], xf[2][4][MT];
    auto load = [&](int kt, i32x4 (&ws)[4][FB], i32x4 (&xs)[4][MT]) __attribute__((always_inline)) {
#pragma unroll
      for (int ks = 0; ks < 4; ++ks) {
        const size_t at = (size_t)kt * kSlabBytes + ks * kTileBytes;
#pragma unroll
        for (int j = 0; j < FB; ++j) ws[ks][j] = __builtin_nontemporal_load(reinterpret_cast<const i32x4*>(wp[j] + at));
#pragma unroll
        for (int i = 0; i < MT; ++i) xs[ks][i] = *reinterpret_cast<const i32x4*>(xp[i] + at);
      }
    };
    auto work = [&](i32x4 (&ws)[4][FB], i32x4 (&xs)[4][MT]) __attribute__((always_inline)) {
#pragma unroll
      for (int ks = 0; ks < 4; ++ks)
#pragma unroll
        for (int j = 0; j < FB; ++j)
#pragma unroll
          for (int i = 0; i < MT; ++i)
            acc[j][i] = ODD ? contract8(xs[ks][i], ws[ks][j], acc[j][i]) : contract8(ws[ks][j], xs[ks][i], acc[j][i]);
    };
    load(k0, wf[0], xf[0]);
    for (int kt = k0; kt < k1; kt += 2) {
      load(min(kt + 1, k1 - 1), wf[1], xf[1]);
      work(wf[0], xf[0]);
      if (kt + 1 >= k1) break;
      load(min(kt + 2, k1 - 1), wf[0], xf[0]);
      work(wf[1], xf[1]);
    }
  }
  if constexpr (KS > 1) {
    int* mine = s_acc + f * FB * MT * 16 * kWave + lane;
    if (busy)
#pragma unroll
      for (int j = 0; j < FB; ++j)
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
          for (int v = 0; v < 16; ++v) atomicAdd(mine + ((j * MT + i) * 16 + v) * kWave, acc[j][i][v]);
    __syncthreads();
  }
  if (!busy) return;
  // Outputs JF row blocks at a time (gate and up together).  The waves that share them take them in turn.
  constexpr int JF = KIND == kI8GateUp || KIND == kI8GateUpF32 ? 2 : 1;
  static_assert(FB % JF == 0, "gate and up are neighbours");
#pragma unroll
  for (int j = 0; j < FB; j += JF)
#pragma unroll
    for (int i = 0; i < MT; ++i) {
      if (KS > 1 && (j / JF * MT + i) % KS != s) continue;
      i32x16 part[JF][1];
#pragma unroll
      for (int q = 0; q < JF; ++q)
#pragma unroll
        for (int v = 0; v < 16; ++v)
          part[q][0][v] = KS > 1 ? s_acc[(((f * FB + j + q) * MT + i) * 16 + v) * kWave + lane] : acc[j + q][i][v];
      const int row0 = t.row0 + 32 * i, blk = t.blk0 + i, fw = (fb + j) * kI8Rows, lrow = lane & 31, half = lane >> 5;
      if constexpr (ODD) {
        emit8_odd<KIND, JF, 1>(g, part, t, row0, blk, fw, lrow, half);
      } else {
        float sa[1];
        row_scales<1>(g, t, row0, blk, lrow, sa);
        emit8<KIND, JF, 1>(g, part, sa, t, row0, fw, lrow, half);
      }
    }
}

}  // namespace

hipError_t launch_i8_gemm(I8Out kind, const I8Args& args, int num_cus, hipStream_t st) {
  I8Args g = args;
  if (g.N <= 0 || g.Nf <= 0) return hipSuccess;
  const int E = g.counts ? g.E : 1;
  g.E = E;
  if (E < 1 || E > kMaxExpertsWide || g.KT < 1 || g.b_blocks < 1 || num_cus <= 0) return hipErrorInvalidValue;
  const bool gate_up = kind == kI8GateUp || kind == kI8GateUpF32;
  if (kind == kI8GateUp && (g.h.ld % 32 != 0 || g.h.ld < g.Nf / 2 || ((uintptr_t)g.h.q & 15) != 0 ||
                            ((uintptr_t)g.h.n & 7) != 0 || !g.h.n))
    return hipErrorInvalidValue;
  if (kind == kI8Rows24 && (g.o.ld % 32 != 0 || g.o.ld < g.Nf || (((uintptr_t)g.o.hi | (uintptr_t)g.o.low) & 15) != 0))
    return hipErrorInvalidValue;
  if (kind == kI8GateUpF32 && (g.ldo % 4 != 0 || (long)g.ldo < g.Nf / 2 || ((uintptr_t)g.out & 15) != 0))
    return hipErrorInvalidValue;
  if ((gate_up || kind == kI8Rows24) && g.Nf % 64 != 0) return hipErrorInvalidValue;
  if (gate_up && (!g.bias0 || !g.bias1)) return hipErrorInvalidValue;
  const bool odd = (kind == kI8F32 || kind == kI8Bf16) && (g.Nf % 8 != 0 || g.ldo % 8 != 0 || ((uintptr_t)g.out & 15) != 0);
  auto with = [&](auto k, auto o) {
    constexpr int kK = decltype(k)::value;
    constexpr bool kO = decltype(o)::value;
    auto stream = [&](auto mt) {
      constexpr int MT = decltype(mt)::value;
      const int tiles = g.counts ? g.N / (32 * MT) + std::min(E, g.N) : (g.N + 32 * MT - 1) / (32 * MT);
      const int fbs = (g.Nf + 32 * kStreamFB - 1) / (32 * kStreamFB);
      // enough waves to have memory's latency covered: 16 a CU
      int ks = 1;
      while (ks < 8 && 2 * ks <= g.KT && (long)fbs * tiles * ks < 16L * num_cus) ks *= 2;
      auto go = [&](auto kernel) {
        const int F = kStreamWaves / ks;
        hipLaunchKernelGGL(kernel, dim3((fbs + F - 1) / F, tiles), dim3(kStreamWaves * kWave), 0, st, g);
      };
      if (ks == 1) go(i8_stream_kernel<kK, kO, MT, 1>);
      else if (ks == 2) go(i8_stream_kernel<kK, kO, MT, 2>);
      else if (ks == 4) go(i8_stream_kernel<kK, kO, MT, 4>);
      else go(i8_stream_kernel<kK, kO, MT, 8>);
    };
    auto ring = [&](auto bm, auto bn, auto nw) {
      constexpr int BM = decltype(bm)::value, BN = decltype(bn)::value, NW = decltype(nw)::value;
      const long tiles = ((long)g.N / BM + std::min(E, g.N)) * ((g.Nf + BN - 1) / BN);
      const int per = NW == 8 ? 1 : 2;
      const int groups = (E + kMaxExperts - 1) / kMaxExperts;
      const int grid = (int)std::min<long>(tiles, (long)num_cus * per);
      hipLaunchKernelGGL((i8_ring_kernel<kK, kO, BM, BN, NW>), dim3(grid, groups), dim3(NW * kWave), 0, st, g,
                         (E + groups - 1) / groups);
    };
    // The stream kernel for few rows a segment, or little work in all, `units` waves' of it: up to two a CU it takes 15 us
    // where the ring of 128 x 128 tiles has 18 (1024 x 2048 x 1024), from four on 25 against 19 (2048 rows).  A wave takes 64
    // rows where 32 would make many units (16384 outputs of 64 rows: 14.6 us against 15.5; 4096: 12.5 against 11.3), unless
    // they are short (512 columns, 1024 x 1024: 9.8 us against 11.4).
    const long units = (g.counts ? (long)g.N / 32 + std::min(E, g.N) : ((long)g.N + 31) / 32) * ((g.Nf + 63) / 64);
    if ((long)g.N <= 32L * E || units <= num_cus || (units <= 2L * num_cus && g.KT < 16)) stream(IntC<1>{});
    else if ((long)g.N <= 64L * E || units <= 2L * num_cus) stream(IntC<2>{});
    else if (((long)g.N / 256 + E) * ((g.Nf + 255) / 256) < num_cus) ring(IntC<128>{}, IntC<128>{}, IntC<4>{});
    else ring(IntC<256>{}, IntC<256>{}, IntC<8>{});
  };
  if (kind == kI8GateUp) with(IntC<kI8GateUp>{}, std::false_type{});
  else if (kind == kI8GateUpF32) with(IntC<kI8GateUpF32>{}, std::false_type{});
  else if (kind == kI8Rows24) with(IntC<kI8Rows24>{}, std::false_type{});
  else if (kind == kI8F32) odd ? with(IntC<kI8F32>{}, std::true_type{}) : with(IntC<kI8F32>{}, std::false_type{});
  else odd ? with(IntC<kI8Bf16>{}, std::true_type{}) : with(IntC<kI8Bf16>{}, std::false_type{});
  return hipGetLastError();
}

}  // namespace mgpt

using namespace mgpt;

namespace {

int check_i8(const mgpt_i8_config* cfg, int N) {
  if (!cfg) return fail(MGPT_ERR_INVALID_ARGUMENT, "config is null");
  if (N < 0) return fail(MGPT_ERR_INVALID_ARGUMENT, "negative num_tokens");
  if (N > 1 << 21) return fail(MGPT_ERR_UNSUPPORTED, "num_tokens %d > 2^21", N);
  if (cfg->in_features < 1 || cfg->out_features < 1)
    return fail(MGPT_ERR_INVALID_ARGUMENT, "invalid in_features=%d out_features=%d", cfg->in_features,
                cfg->out_features);
  if (cfg->in_features > 1 << 17)   // 127^2 times as many fit 32 bits
    return fail(MGPT_ERR_UNSUPPORTED, "in_features %d > 2^17", cfg->in_features);
  if (cfg->out_features > 1 << 24) return fail(MGPT_ERR_UNSUPPORTED, "out_features %d > 2^24", cfg->out_features);
  if (cfg->dtype != MGPT_DTYPE_F32 && cfg->dtype != MGPT_DTYPE_BF16)
    return fail(MGPT_ERR_UNSUPPORTED, "unsupported dtype %d", cfg->dtype);
  return MGPT_OK;
}

size_t row_blocks(int rows) { return ((size_t)rows + kI8Rows - 1) / kI8Rows; }

// Workspace of a forward: the rows' tiles and scales.
struct I8Layout {
  size_t scale, total;
};
I8Layout i8_layout(const mgpt_i8_config* cfg, int N) {
  I8Layout l;
  l.scale = row_blocks(N) * i8_row_block_bytes(cfg->in_features);   // (a multiple of 4 KB)
  l.total = l.scale + (row_blocks(N) * kI8Rows * 4 + 255) / 256 * 256;
  return l;
}

QuantizeArgs dense_rows(const void* x, int N, int K, char* q, float* scale) {
  QuantizeArgs a{};
  a.src = x;
  a.ld = K;
  a.N = N;
  a.K = K;
  a.q = q;
  a.scale = scale;
  return a;
}

}  // namespace

extern "C" {

int mgpt_i8_weight_bytes(const mgpt_i8_config* cfg, size_t* bytes) {
  if (int rc = check_i8(cfg, 0)) return rc;
  if (!bytes) return fail(MGPT_ERR_INVALID_ARGUMENT, "null bytes");
  *bytes = row_blocks(cfg->out_features) * i8_row_block_bytes(cfg->in_features);
  return MGPT_OK;
}

int mgpt_i8_pack_weight(const mgpt_i8_config* cfg, const void* weight, int weight_dtype, void* packed, float* scales,
                        void* stream) {
  if (int rc = check_i8(cfg, 0)) return rc;
  if (weight_dtype != MGPT_DTYPE_F32 && weight_dtype != MGPT_DTYPE_BF16)
    return fail(MGPT_ERR_UNSUPPORTED, "unsupported weight dtype %d", weight_dtype);
  if (!weight || !packed || !scales) return fail(MGPT_ERR_INVALID_ARGUMENT, "null weight, packed or scales");
  if ((uintptr_t)packed & 255) return fail(MGPT_ERR_INVALID_ARGUMENT, "packed must be 256-byte aligned");
  const QuantizeArgs a = dense_rows(weight, cfg->out_features, cfg->in_features, (char*)packed, scales);
  HIP_TRY(launch_i8_quantize(weight_dtype == MGPT_DTYPE_F32 ? kRowsF32 : kRowsBf16, a,
                             (int)row_blocks(cfg->out_features), (hipStream_t)stream));
  return MGPT_OK;
}

int mgpt_i8_pack_quantized(const mgpt_i8_config* cfg, const int8_t* weight, void* packed, void* stream) {
  if (int rc = check_i8(cfg, 0)) return rc;
  if (!weight || !packed) return fail(MGPT_ERR_INVALID_ARGUMENT, "null weight or packed");
  if ((uintptr_t)packed & 255) return fail(MGPT_ERR_INVALID_ARGUMENT, "packed must be 256-byte aligned");
  HIP_TRY(launch_i8_tile(weight, cfg->out_features, cfg->in_features, (char*)packed, (hipStream_t)stream));
  return MGPT_OK;
}

int mgpt_i8_linear_workspace_bytes(const mgpt_i8_config* cfg, int num_tokens, size_t* bytes) {
  if (int rc = check_i8(cfg, num_tokens)) return rc;
  if (!bytes) return fail(MGPT_ERR_INVALID_ARGUMENT, "null bytes");
  *bytes = i8_layout(cfg, num_tokens).total;
  return MGPT_OK;
}

int mgpt_i8_linear_forward(const mgpt_i8_config* cfg, const void* x, const void* packed, const float* scales,
                           const float* bias, void* y, int num_tokens, void* workspace, size_t workspace_bytes,
                           void* stream) {
  if (int rc = check_i8(cfg, num_tokens)) return rc;
  if (num_tokens == 0) return MGPT_OK;
  if (!x || !packed || !scales || !y || !workspace)
    return fail(MGPT_ERR_INVALID_ARGUMENT, "null x, packed, scales, y or workspace");
  if (((uintptr_t)packed | (uintptr_t)workspace) & 255)
    return fail(MGPT_ERR_INVALID_ARGUMENT, "packed and workspace must be 256-byte aligned");
  const int K = cfg->in_features, M = cfg->out_features, N = num_tokens;
  const I8Layout l = i8_layout(cfg, N);
  if (workspace_bytes < l.total)
    return fail(MGPT_ERR_WORKSPACE_TOO_SMALL, "workspace needs %zu bytes, got %zu", l.total, workspace_bytes);
  const bool f32 = cfg->dtype == MGPT_DTYPE_F32;
  char* q = (char*)workspace;
  float* sa = (float*)(q + l.scale);
  HIP_TRY(launch_i8_quantize(f32 ? kRowsF32 : kRowsBf16, dense_rows(x, N, K, q, sa), (int)row_blocks(N),
                             (hipStream_t)stream));
  I8Args g{};
  g.A = q;
  g.sa = sa;
  g.B = (const char*)packed;
  g.sb = scales;
  g.ldsb = M;
  g.KT = (K + kI8Slab - 1) / kI8Slab;
  g.Nf = M;
  g.b_blocks = (int)row_blocks(M);
  g.bias0 = bias;
  g.bias_ld = M;
  g.E = 1;
  g.N = N;
  g.out = y;
  g.ldo = M;
  HIP_TRY(launch_i8_gemm(f32 ? kI8F32 : kI8Bf16, g, compute_units(), (hipStream_t)stream));
  return MGPT_OK;
}

}  // extern "C"
