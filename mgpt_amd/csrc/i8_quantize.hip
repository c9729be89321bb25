// i8_quantize.hip -- rows in 8-bit integers with a scale each: s = max|x| / 127, q = rint(x
// 127 / max|x|), in the layout of i8.hpp.
//
// A block takes a row block; lane l of a wave has 16 neighbouring columns of row l % 32, which are an
// operand tile's 16 bytes of that lane, so that rows are read as 64-byte pieces and tiles
// written as whole kilobytes.  One pass finds the maxima, a second one, from
// registers where the row block fits them, rounds.  x 127 / max|x| is formed in 64 bits: fp32 would put
// every hundred-thousandth value on the wrong side of a border between two integers, and values on a border
// (bf16 has many: max|x| / 2 is 63.5) have to be seen there.  A row that holds an infinity or a NaN has
// the scale NaN, and so have its outputs.
#include <algorithm>
#include <type_traits>

#include "i8.hpp"

namespace mgpt {
namespace {

// 16 values of a row as they are in memory.
template <QuantizeSource SRC>
struct Raw {
  uint4 w[SRC == kRowsF32 ? 4 : 2];
  int e;   // kRowsHidden: their exponent
};

template <QuantizeSource SRC, bool VEC>
__device__ __forceinline__ Raw<SRC> load_raw(const QuantizeArgs& g, size_t row, int c, bool live) {
  Raw<SRC> r{};
  if (!live) return r;
  if constexpr (SRC == kRowsHidden) {
    const uint4* p = reinterpret_cast<const uint4*>(g.h.q + row * g.h.Hp + c);
    r.w[0] = p[0];
    r.w[1] = p[1];
    r.e = g.h.e[row * (g.h.Hp / 32) + c / 32];
  } else {
    typedef std::conditional_t<SRC == kRowsF32, uint32_t, uint16_t> T;
    const T* p = reinterpret_cast<const T*>(g.src) + row * g.ld + c;
    constexpr int kV = sizeof(r.w) / 16, kPer = 16 / sizeof(T);
    if constexpr (VEC) {   // K is a multiple of a vector's values
#pragma unroll
      for (int i = 0; i < kV; ++i)
        if (c + i * kPer < g.K) r.w[i] = reinterpret_cast<const uint4*>(p)[i];
    } else {
      T v[16];
#pragma unroll
      for (int i = 0; i < 16; ++i) v[i] = c + i < g.K ? p[i] : (T)0;
      __builtin_memcpy(r.w, v, sizeof(r.w));
    }
  }
  return r;
}

template <QuantizeSource SRC>
__device__ __forceinline__ void values(const QuantizeArgs& g, const Raw<SRC>& r, int c, float rs, float (&x)[16]) {
  const uint32_t* w = reinterpret_cast<const uint32_t*>(r.w);
  if constexpr (SRC == kRowsF32) {
#pragma unroll
    for (int i = 0; i < 16; ++i) x[i] = __uint_as_float(w[i]);
  } else if constexpr (SRC == kRowsBf16) {
#pragma unroll
    for (int i = 0; i < 16; ++i) x[i] = __uint_as_float(i & 1 ? w[i / 2] & 0xFFFF0000u : w[i / 2] << 16);
  } else {
    // (e 255: not finite)
    const float unit = r.e == 255 ? __uint_as_float(0x7FC00000u) : __uint_as_float((uint32_t)max(r.e - 14, 1) << 23);
#pragma unroll
    for (int i = 0; i < 16; ++i) x[i] = (float)(int16_t)(i & 1 ? w[i / 2] >> 16 : w[i / 2] & 0xFFFF) * unit;
  }
  if constexpr (SRC != kRowsHidden)
    if (g.gamma) {
#pragma unroll
      for (int i = 0; i < 16; ++i) x[i] = c + i < g.K ? (x[i] * rs) * g.gamma[c + i] : 0.0f;
    }
}

template <QuantizeSource SRC, bool VEC, int NW>
__global__ __launch_bounds__(NW * kWave) void i8_quantize_kernel(QuantizeArgs g) {
  constexpr int kHold = 4;   // tiles of a wave that stay in registers
  __shared__ uint32_t s_top[NW][kI8Rows];
  const int block = blockIdx.x;
  int row0, rows;
  if (g.counts) {
    TileInfo t;
    if (!find_tile<kI8Rows>(g.counts, g.E, block, &t)) return;
    row0 = t.row0;
    rows = t.row_end - t.row0;
  } else {
    row0 = block * kI8Rows;
    rows = g.N - row0;
  }
  const int w = threadIdx.x / kWave, lane = lane_id(), r = lane & 31, half = lane >> 5;
  const bool live = r < rows;
  size_t row = 0;
  float rs = 1.0f;
  if (live) {
    row = row0 + r;
    if (g.perm) row = g.perm[row] / g.k;
    if (g.gamma) rs = g.rstd[row];
  }
  const int tiles = (g.K + kI8Slab - 1) / kI8Slab * (kI8Slab / 32);
  // neighbouring tiles to a wave, so that it has whole lines of the rows
  const int per = (tiles + NW - 1) / NW, t0 = w * per, t1 = min(tiles, t0 + per);
  Raw<SRC> held[kHold];
  uint32_t top = 0;
  auto look = [&](const Raw<SRC>& raw, int c) {
    float x[16];
    values<SRC>(g, raw, c, rs, x);
#pragma unroll
    for (int i = 0; i < 16; ++i) top = max(top, __float_as_uint(x[i]) & 0x7FFFFFFFu);
  };
  auto column = [&](int t) { return t * 32 + half * 16; };
#pragma unroll
  for (int u = 0; u < kHold; ++u)
    if (t0 + u < t1) held[u] = load_raw<SRC, VEC>(g, row, column(t0 + u), live && column(t0 + u) < g.K);
#pragma unroll
  for (int u = 0; u < kHold; ++u)
    if (t0 + u < t1) look(held[u], column(t0 + u));
  for (int t = t0 + kHold; t < t1; ++t) look(load_raw<SRC, VEC>(g, row, column(t), live && column(t) < g.K), column(t));
  {
    const auto o = __builtin_amdgcn_permlane32_swap(top, top, false, false);
    top = max(o[0], o[1]);
  }
  if (half == 0) s_top[w][r] = top;
  __syncthreads();
  top = 0;
#pragma unroll
  for (int i = 0; i < NW; ++i) top = max(top, s_top[i][r]);
  const bool finite = top < 0x7F800000u;
  const float most = __uint_as_float(top);
  if (w == 0 && half == 0 && live)
    g.scale[(size_t)block * kI8Rows + r] = finite ? most / 127.0f : __uint_as_float(0x7FC00000u);
  const double f = finite && top ? 127.0 / (double)most : 0.0;
  char* out = g.q + (size_t)block * i8_row_block_bytes(g.K) + lane * 16;
  auto put = [&](const Raw<SRC>& raw, int t) {
    float x[16];
    values<SRC>(g, raw, column(t), rs, x);
    uint32_t q[4];
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      // To the nearest 2^-40 first: a quotient of two floats that is not between two integers is 2^-34
      // away from there (254 x - (2n + 1) max is a whole number of their units), the product's rounding 2^-45.
      // Then to the nearest integer, ties to even, in the low bits.
      double d = (double)(finite ? x[i] : 0.0f) * f;
      d = (d + 0x1.8p12) - 0x1.8p12;
      d += 0x1.8p52;
      const uint32_t b = (uint32_t)__double2loint(d) & 0xFF;
      q[i / 4] = i % 4 ? q[i / 4] | b << (8 * (i % 4)) : b;
    }
    *reinterpret_cast<uint4*>(out + (size_t)t * 1024) = make_uint4(q[0], q[1], q[2], q[3]);
  };
#pragma unroll
  for (int u = 0; u < kHold; ++u)
    if (t0 + u < t1) put(held[u], t0 + u);
  for (int t = t0 + kHold; t < t1; ++t) put(load_raw<SRC, VEC>(g, row, column(t), live && column(t) < g.K), t);
}

__global__ __launch_bounds__(256) void i8_tile_kernel(const int8_t* __restrict__ q, int M, int K,
                                                      char* __restrict__ out) {
  const size_t block = blockIdx.x;
  const int lane = lane_id(), r = lane & 31;
  const size_t row = block * kI8Rows + r;
  const int tiles = (K + kI8Slab - 1) / kI8Slab * (kI8Slab / 32);
  for (int t = blockIdx.y * 4 + threadIdx.x / kWave; t < tiles; t += gridDim.y * 4) {
    const int c = t * 32 + (lane >> 5) * 16;
    uint32_t w[4] = {0, 0, 0, 0};
    if (row < (size_t)M)
#pragma unroll
      for (int i = 0; i < 16; ++i)
        if (c + i < K) w[i / 4] |= (uint32_t)(uint8_t)q[row * K + c + i] << (8 * (i % 4));
    *reinterpret_cast<uint4*>(out + block * i8_row_block_bytes(K) + (size_t)t * 1024 + lane * 16) =
        make_uint4(w[0], w[1], w[2], w[3]);
  }
}

}  // namespace

hipError_t launch_i8_quantize(QuantizeSource src, const QuantizeArgs& g, int max_blocks, hipStream_t st) {
  if (max_blocks <= 0) return hipSuccess;
  if (src == kRowsHidden && (g.h.Hp != g.K || g.K % 32 != 0 || ((uintptr_t)g.h.q & 15) != 0)) return hipErrorInvalidValue;
  const size_t size = src == kRowsF32 ? 4 : 2;
  const bool vec = src == kRowsHidden || (g.K * size % 16 == 0 && g.ld * size % 16 == 0 && ((uintptr_t)g.src & 15) == 0);
  const int tiles = (g.K + 31) / 32;
  auto go = [&](auto s, auto v) {
    auto launch = [&](auto kernel, int nw) {
      hipLaunchKernelGGL(kernel, dim3(max_blocks), dim3(nw * kWave), 0, st, g);
    };
    constexpr QuantizeSource kS = decltype(s)::value;
    constexpr bool kV = decltype(v)::value;
    // a wave's tiles stay in its registers up to 64 of a row block
    if (tiles <= 16) launch(i8_quantize_kernel<kS, kV, 4>, 4);
    else if (tiles <= 32) launch(i8_quantize_kernel<kS, kV, 8>, 8);
    else launch(i8_quantize_kernel<kS, kV, 16>, 16);
  };
  auto with = [&](auto s) { vec ? go(s, std::true_type{}) : go(s, std::false_type{}); };
  if (src == kRowsF32) with(std::integral_constant<QuantizeSource, kRowsF32>{});
  else if (src == kRowsBf16) with(std::integral_constant<QuantizeSource, kRowsBf16>{});
  else go(std::integral_constant<QuantizeSource, kRowsHidden>{}, std::true_type{});
  return hipGetLastError();
}

hipError_t launch_i8_tile(const int8_t* q, int M, int K, char* out, hipStream_t st) {
  if (M <= 0) return hipSuccess;
  hipLaunchKernelGGL(i8_tile_kernel, dim3((M + kI8Rows - 1) / kI8Rows, std::min(8, (K + 127) / 128)), dim3(256), 0, st,
                     q, M, K, out);
  return hipGetLastError();
}

}  // namespace mgpt
