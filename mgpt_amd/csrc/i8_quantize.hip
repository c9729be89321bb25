// i8_quantize.hip -- rows in 8-bit integers with a scale each: s = max|x| / 127, q = rint(x r), r = 127 (1 / max|x|)
// and both products rounded to 64 bits, in the layout of i8.hpp.
//
// A block takes 8 rows of a row block, a wave of it 128 columns of them at a time: 16 neighbouring ones a lane, so
// that rows are read, and the tiles' parts written, as whole lines.  One pass finds the maxima, a second one, from
// registers up to 8192 columns, rounds.  In 64 bits, whose rate is that of 32 here: fp32 would
// put every hundred-thousandth value on the wrong side of a border between two integers.  (x = max|x| / 2, which a bf16
// row often has, is on the border of 63 and 64; r's rounding decides, in a program of 64-bit operations as here.)  A
// row that holds an infinity or a NaN has the scale NaN, and so have its outputs.
//
// Measured: 16384 x 2048 bf16 25 us (4.0 TB/s), one row 4 us; hidden units 32768 x 2816 70 us (4.6 TB/s).  Blocks of
// whole row blocks, 64 bytes of a row at a time, took 44 and 8 us, and 110 for hidden units of 16 bits.
#include <algorithm>
#include <type_traits>

#include "i8.hpp"

namespace mgpt {
namespace {

constexpr int kPart = 8;   // rows of a block

// 16 values of a row as they are in memory.
template <QuantizeSource SRC>
struct Raw {
  uint4 w[SRC == kRowsF32 ? 4 : 2];
  uint2 n;        // kRowsHidden: their lower bits,
  uint32_t top;   // and the largest magnitude of their 32
};

template <QuantizeSource SRC, bool VEC>
__device__ __forceinline__ Raw<SRC> load_raw(const QuantizeArgs& g, size_t row, int c, bool live) {
  Raw<SRC> r{};
  if (!live) return r;
  if constexpr (SRC == kRowsHidden) {
    const uint4* p = reinterpret_cast<const uint4*>(g.h.q + row * g.h.ld + c);
    r.w[0] = p[0];
    r.w[1] = p[1];
    r.n = *reinterpret_cast<const uint2*>(g.h.n + row * (g.h.ld / 2) + c / 2);
    r.top = g.h.top[row * (g.h.ld / 32) + c / 32];
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

// Hidden unit i of the 16, in 2^(e - 145).
__device__ __forceinline__ int hidden(const Raw<kRowsHidden>& r, int i) {
  const uint32_t w = reinterpret_cast<const uint32_t*>(r.w)[i / 2], n = i & 4 ? r.n.y : r.n.x;
  const int hi = i & 1 ? (int)w >> 16 : (int)(int16_t)w;
  return hi << 4 | (int)(n >> (8 * (i & 3) + (i & 8 ? 4 : 0)) & 15);
}

// The values, kRowsF32 or kRowsBf16.
template <QuantizeSource SRC>
__device__ __forceinline__ void values(const QuantizeArgs& g, const Raw<SRC>& r, int c, float rs, float (&x)[16]) {
  const uint32_t* w = reinterpret_cast<const uint32_t*>(r.w);
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    if constexpr (SRC == kRowsF32) x[i] = __uint_as_float(w[i]);
    else x[i] = __uint_as_float(i & 1 ? w[i / 2] & 0xFFFF0000u : w[i / 2] << 16);
  }
  if (g.gamma) {
#pragma unroll
    for (int i = 0; i < 16; ++i) x[i] = c + i < g.K ? (x[i] * rs) * g.gamma[c + i] : 0.0f;
  }
}

// The largest magnitude's bits as fp32 (infinity's or more: not finite).
template <QuantizeSource SRC>
__device__ __forceinline__ uint32_t largest(const QuantizeArgs& g, const Raw<SRC>& r, int c, float rs) {
  typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
  const uint32_t* w = reinterpret_cast<const uint32_t*>(r.w);
  uint32_t top = 0;
  if constexpr (SRC == kRowsHidden) {
    return r.top;
  } else if (SRC == kRowsBf16 && !g.gamma) {
    u16x2 most = {0, 0};
#pragma unroll
    for (int i = 0; i < 8; ++i) most = __builtin_elementwise_max(most, __builtin_bit_cast(u16x2, w[i] & 0x7FFF7FFFu));
    return (uint32_t)max(most[0], most[1]) << 16;
  } else {
    float x[16];
    values<SRC>(g, r, c, rs, x);
#pragma unroll
    for (int i = 0; i < 16; ++i) top = max(top, __float_as_uint(x[i]) & 0x7FFFFFFFu);
    return top;
  }
}

// Four values' integers, as bytes: the sum rounds the product to a whole number, ties to even, in its low bits.
__device__ __forceinline__ uint32_t round4(double a, double b, double c, double d, double r) {
  auto low = [&](double x) { return (uint32_t)__double2loint(x * r + 0x1.8p52); };
  const uint32_t ab = __builtin_amdgcn_perm(low(b), low(a), 0x0c0c0400), cd = __builtin_amdgcn_perm(low(d), low(c), 0x0c0c0400);
  return __builtin_amdgcn_perm(cd, ab, 0x05040100);
}

// HOLD: slabs of a wave that stay in registers
template <QuantizeSource SRC, bool VEC, int NW, int HOLD>
__global__ __launch_bounds__(NW * kWave) void i8_quantize_kernel(QuantizeArgs g) {
  __shared__ uint32_t s_top[NW][kPart];
  const int block = (int)blockIdx.x / (kI8Rows / kPart), part = (int)blockIdx.x % (kI8Rows / kPart);
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
  if (g.counts && part * kPart >= rows) return;   // (rows whose products nothing keeps)
  const int w = threadIdx.x / kWave, lane = lane_id(), chunk = lane / kPart, r = part * kPart + lane % kPart;
  const bool live = r < rows;
  size_t row = 0;
  float rs = 1.0f;
  if (live) {
    row = row0 + r;
    if (g.perm) row = g.perm[row] / g.k;
    if (g.gamma) rs = g.rstd[row];
  }
  const int slabs = (g.K + kI8Slab - 1) / kI8Slab;
  Raw<SRC> held[HOLD];
  uint32_t top = 0;
  auto look = [&](const Raw<SRC>& raw, int c) { top = max(top, largest<SRC>(g, raw, c, rs)); };
  auto column = [&](int t) { return t * kI8Slab + chunk * 16; };
  auto load = [&](int t) { return load_raw<SRC, VEC>(g, row, column(t), live && column(t) < g.K); };
#pragma unroll
  for (int u = 0; u < HOLD; ++u)
    if (w + u * NW < slabs) held[u] = load(w + u * NW);
#pragma unroll
  for (int u = 0; u < HOLD; ++u)
    if (w + u * NW < slabs) look(held[u], column(w + u * NW));
  for (int t = w + HOLD * NW; t < slabs; t += NW) look(load(t), column(t));
#pragma unroll
  for (int d = kPart; d < kWave; d *= 2) top = max(top, (uint32_t)__shfl_xor((int)top, d, kWave));
  if (chunk == 0) s_top[w][lane] = top;
  __syncthreads();
  top = 0;
#pragma unroll
  for (int i = 0; i < NW; ++i) top = max(top, s_top[i][lane % kPart]);
  const bool finite = top < 0x7F800000u;
  const float most = __uint_as_float(top);
  if (w == 0 && chunk == 0 && live)
    g.scale[(size_t)block * kI8Rows + r] =
        !finite ? __uint_as_float(0x7FC00000u) : g.by_product ? most * (1.0f / 127.0f) : most / 127.0f;
  const double f = finite && top ? 127.0 * (1.0 / (double)most) : 0.0;
  // (column c: tile c / 32 of the row block, its half c / 16)
  char* out = g.q + (size_t)block * i8_row_block_bytes(g.K) + (chunk / 2) * 1024 + (chunk % 2 * kI8Rows + r) * 16;
  auto put = [&](const Raw<SRC>& raw, int t) {
    uint32_t q[4];
    if constexpr (SRC == kRowsHidden) {
      const double fu = f * (double)__uint_as_float((uint32_t)(max((int)(raw.top >> 23), 20) - 18) << 23);
      auto x = [&](int i) { return (double)hidden(raw, i); };
#pragma unroll
      for (int i = 0; i < 4; ++i) q[i] = round4(x(4 * i), x(4 * i + 1), x(4 * i + 2), x(4 * i + 3), fu);
    } else {
      float x[16];
      values<SRC>(g, raw, column(t), rs, x);
#pragma unroll
      for (int i = 0; i < 4; ++i) q[i] = round4(x[4 * i], x[4 * i + 1], x[4 * i + 2], x[4 * i + 3], f);
    }
    *reinterpret_cast<uint4*>(out + (size_t)t * (kI8Slab * kI8Rows)) = make_uint4(q[0], q[1], q[2], q[3]);
  };
#pragma unroll
  for (int u = 0; u < HOLD; ++u)
    if (w + u * NW < slabs) put(held[u], w + u * NW);
  for (int t = w + HOLD * NW; t < slabs; t += NW) put(load(t), t);
}

// VEC: a lane's 16 columns are a vector or past K.
template <bool VEC>
__global__ __launch_bounds__(256) void i8_tile_kernel(const int8_t* __restrict__ q, int M, int K,
                                                      char* __restrict__ out) {
  const size_t block = blockIdx.x;
  const int lane = lane_id(), r = lane & 31;
  const size_t row = block * kI8Rows + r;
  const int tiles = (K + kI8Slab - 1) / kI8Slab * (kI8Slab / 32);
  for (int t = blockIdx.y * 4 + threadIdx.x / kWave; t < tiles; t += gridDim.y * 4) {
    const int c = t * 32 + (lane >> 5) * 16;
    uint4 w = make_uint4(0, 0, 0, 0);
    if (row < (size_t)M) {
      if constexpr (VEC) {
        if (c < K) w = *reinterpret_cast<const uint4*>(q + row * K + c);
      } else {
        uint32_t u[4] = {0, 0, 0, 0};
#pragma unroll
        for (int i = 0; i < 16; ++i)
          if (c + i < K) u[i / 4] |= (uint32_t)(uint8_t)q[row * K + c + i] << (8 * (i % 4));
        w = make_uint4(u[0], u[1], u[2], u[3]);
      }
    }
    *reinterpret_cast<uint4*>(out + block * i8_row_block_bytes(K) + (size_t)t * 1024 + lane * 16) = w;
  }
}

}  // namespace

hipError_t launch_i8_quantize(QuantizeSource src, const QuantizeArgs& g, int max_blocks, hipStream_t st) {
  if (max_blocks <= 0) return hipSuccess;
  if (src == kRowsHidden && (g.h.ld != g.K || g.K % 32 != 0 || ((uintptr_t)g.h.q & 15) != 0 || ((uintptr_t)g.h.n & 7) != 0)) return hipErrorInvalidValue;
  const size_t size = src == kRowsF32 ? 4 : 2;
  const bool vec = src == kRowsHidden || (g.K * size % 16 == 0 && g.ld * size % 16 == 0 && ((uintptr_t)g.src & 15) == 0);
  const int slabs = (g.K + kI8Slab - 1) / kI8Slab;
  if ((long)max_blocks * (kI8Rows / kPart) * (slabs <= 4 ? 2 : slabs <= 8 ? 4 : slabs <= 32 ? 8 : 16) * kWave >= 1L << 32)
    return hipErrorInvalidConfiguration;   // (more threads than a grid holds)
  auto go = [&](auto s, auto v) {
    auto launch = [&](auto kernel, int nw) {
      hipLaunchKernelGGL(kernel, dim3(max_blocks * (kI8Rows / kPart)), dim3(nw * kWave), 0, st, g);
    };
    constexpr QuantizeSource kS = decltype(s)::value;
    constexpr bool kV = decltype(v)::value;
    // Waves whose registers hold the rows: two slabs each, of long rows four (at 16 slabs 4 and 2 a wave take 28 and 25 us
    // for 16384 rows, at 22 of hidden units 72 and, on 16 waves, 84).
    if (slabs <= 4) launch(i8_quantize_kernel<kS, kV, 2, 2>, 2);
    else if (slabs <= 8) launch(i8_quantize_kernel<kS, kV, 4, 2>, 4);
    else if (slabs <= 16) launch(i8_quantize_kernel<kS, kV, 8, 2>, 8);
    else if (slabs <= 32) launch(i8_quantize_kernel<kS, kV, 8, 4>, 8);
    else launch(i8_quantize_kernel<kS, kV, 16, 4>, 16);
  };
  auto with = [&](auto s) { vec ? go(s, std::true_type{}) : go(s, std::false_type{}); };
  if (src == kRowsF32) with(std::integral_constant<QuantizeSource, kRowsF32>{});
  else if (src == kRowsBf16) with(std::integral_constant<QuantizeSource, kRowsBf16>{});
  else go(std::integral_constant<QuantizeSource, kRowsHidden>{}, std::true_type{});
  return hipGetLastError();
}

hipError_t launch_i8_tile(const int8_t* q, int M, int K, char* out, hipStream_t st) {
  if (M <= 0) return hipSuccess;
  auto go = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, dim3((M + kI8Rows - 1) / kI8Rows, std::min(8, (K + 127) / 128)), dim3(256), 0, st, q, M,
                       K, out);
  };
  K % 16 == 0 && ((uintptr_t)q & 15) == 0 ? go(i8_tile_kernel<true>) : go(i8_tile_kernel<false>);
  return hipGetLastError();
}

}  // namespace mgpt
