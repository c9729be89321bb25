// norm.hip -- the norms around a block, fused with its gate and the residual stream:
//   r_h = 1 / sqrt(mean(h^2) + eps),  n = h r_h           (h: the block's output)
//   o   = s x + gate * (n * gamma_post)                   (x: the residual stream)
//   r_o = 1 / sqrt(mean(o^2) + eps),  y = (o r_o) * gamma_pre
// o goes on as the residual stream and y into the next block; without gamma_post n is
// h itself, without gate it is 1, without gamma_pre there is no y.  gate has G rows, one
// for each N / G consecutive tokens (1: a learned scale; one per sequence or token: a
// conditioned one).  The reference has the pre-norm alone (layers/RMSNormLayer.cpp,
// utils/Tensor.cpp:785-800), which mgpt_moe_forward_block fuses into its router.
//
// Backward, for the gradients dout of o and dy of y, with z = o r_o (o formed again from
// x and h, not read):
//   q  = dy gamma_pre,  do = dout + r_o (q - z mean(q z))
//   dx = s do,  dn = do gate gamma_post,  dh = r_h (dn - n mean(dn n))
//   T_g = sum over group g's tokens of do n:  dgate_g = T_g gamma_post,
//   dgamma_post = sum_g T_g gate_g,  dgamma_pre = sum over tokens of dy z
//
// What bounds it: memory; forward x, h in, o, y out, backward x, h, dout, dy in, dx, dh
// out.  A row stays in the registers of its W waves (8 columns a lane and vector, NV
// vectors), so that everything is read once; the gains sit in registers (or LDS) across
// a stream's rows.  A stream is W waves that take rows in turn.  MI355X: forward 16384 x
// 1024 bf16 22 us (134 MB, 6.1 TB/s), 32768 x 2048 97 us (537 MB, 5.5 TB/s); stores past
// the caches 23 and 103.  Column sums are kept per lane over a stream's rows, added over a
// block's streams through LDS, and over the blocks by norm_reduce_kernel, in a fixed
// order: the same call gives the same bits.
// All arithmetic is fp32; out, y, dx and dh are rounded once.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <initializer_list>
#include <type_traits>

#include "../../include/mgpt_moe.h"
#include "capi_internal.hpp"
#include "common.hpp"

namespace mgpt {

hipError_t launch_fill_zero(float* p, size_t n, hipStream_t stream);   // wgrad.hip

namespace {

constexpr int kMaxC = 16384;

template <int CTRL, int ROWS>
__device__ __forceinline__ float dpp_fadd(float v) {
  return v + __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, ROWS, 0xf, false));
}
// Sum over the 64 lanes, in every lane.
__device__ __forceinline__ float wave_fsum(float v) {
  v = dpp_fadd<0x111, 0xf>(v);
  v = dpp_fadd<0x112, 0xf>(v);
  v = dpp_fadd<0x114, 0xf>(v);
  v = dpp_fadd<0x118, 0xf>(v);
  v = dpp_fadd<0x142, 0xa>(v);
  v = dpp_fadd<0x143, 0xc>(v);
  return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), kWave - 1));
}

// Sum over a stream's W waves.  `slot` alternates between calls, so one barrier
// suffices; every wave of the block calls it the same number of times.
template <int W>
__device__ __forceinline__ float stream_sum(float v, float (*red)[16], int w, int slot) {
  v = wave_fsum(v);
  if constexpr (W > 1) {
    if (lane_id() == 0) red[slot][w] = v;
    __syncthreads();
    const int w0 = w / W * W;
    v = red[slot][w0];
#pragma unroll
    for (int i = 1; i < W; ++i) v += red[slot][w0 + i];
  }
  return v;
}

// A lane's 8 columns of a row of C, from c on: neighbours where the row is 16-byte aligned
// and C a multiple of 8 (vec), else every 64th, so that a wave's are neighbours.  Columns
// past the row are zeros and not written.
__device__ __forceinline__ int first_column(int wave, int lane, bool vec) {
  return vec ? (wave * kWave + lane) * 8 : wave * 512 + lane;
}
__device__ __forceinline__ int column(int c, int q, bool vec) { return c + (vec ? q : q * kWave); }

template <typename T>
__device__ __forceinline__ void load8(const T* __restrict__ row, int c, int C, bool vec, float (&o)[8]) {
  if (vec) {
    if (c >= C) {
#pragma unroll
      for (int q = 0; q < 8; ++q) o[q] = 0.0f;
    } else if constexpr (sizeof(T) == 4) {
      const float4 a = *reinterpret_cast<const float4*>(row + c);
      const float4 b = *reinterpret_cast<const float4*>(row + c + 4);
      o[0] = a.x; o[1] = a.y; o[2] = a.z; o[3] = a.w;
      o[4] = b.x; o[5] = b.y; o[6] = b.z; o[7] = b.w;
    } else {
      const uint4 u = *reinterpret_cast<const uint4*>(row + c);
      const uint32_t wv[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        o[2 * q] = __uint_as_float(wv[q] << 16);
        o[2 * q + 1] = __uint_as_float(wv[q] & 0xFFFF0000u);
      }
    }
  } else {
#pragma unroll
    for (int q = 0; q < 8; ++q) o[q] = c + q * kWave < C ? to_f32(row[c + q * kWave]) : 0.0f;
  }
}

template <typename T>
__device__ __forceinline__ void store8(T* __restrict__ row, int c, int C, bool vec, const float (&o)[8],
                                       bool once = false) {
  if (vec) {
    if (c >= C) return;
    if constexpr (sizeof(T) == 4) {
      float4* p = reinterpret_cast<float4*>(row + c);
      const float4 a = make_float4(o[0], o[1], o[2], o[3]), b = make_float4(o[4], o[5], o[6], o[7]);
      if (once) {
        store_once(p, a);
        store_once(p + 1, b);
      } else {
        p[0] = a;
        p[1] = b;
      }
    } else {
      uint4* p = reinterpret_cast<uint4*>(row + c);
      const uint4 a = make_uint4(pack_bf16x2(o[0], o[1]), pack_bf16x2(o[2], o[3]), pack_bf16x2(o[4], o[5]),
                                 pack_bf16x2(o[6], o[7]));
      if (once) store_once(p, a);
      else *p = a;
    }
  } else {
#pragma unroll
    for (int q = 0; q < 8; ++q)
      if (c + q * kWave < C) store_act(row + c + q * kWave, o[q]);
  }
}

// A gain's 8 columns, 1 where there is none.
__device__ __forceinline__ void load_gain(const float* row, int c, int C, bool vec, float (&o)[8]) {
  if (row) {
    load8(row, c, C, vec, o);
  } else {
#pragma unroll
    for (int q = 0; q < 8; ++q) o[q] = 1.0f;
  }
}

struct NormArgs {
  int N, C, G;       // G: rows of the gate (N % G == 0)
  float scale, eps;
  int vec;           // rows as 16-byte vectors
  const float *post, *gate, *pre;
  float *rh, *ro;    // forward: written; backward: read
  // backward: which rows a block takes (see NormPlan), and whether dx and dh are stored
  // past the caches
  int parts, chunk, step, span, per_block, once;
};

// Rows to blocks.  Many rows a group (a gate's rows): `parts` blocks per group, each of
// which starts `chunk` rows after the one before, takes a row a stream and goes on `step`
// rows further, for `span` rows.  Few rows a group (parts = 0): whole groups, `per_block`
// consecutive ones a block, that its streams take in turn.
struct NormPlan {
  int blocks, parts, chunk, step, span, per_block, W, NV;
};

template <typename T, int W, int NV>
__global__ __launch_bounds__(W <= 4 ? 256 : W * 64) void norm_forward_kernel(
    NormArgs a, const T* __restrict__ x, const T* __restrict__ h, T* __restrict__ out, T* __restrict__ y) {
  __shared__ float red[2][16];
  constexpr int S = W <= 4 ? 4 / W : 1;   // streams of a block
  const int w = __builtin_amdgcn_readfirstlane((int)threadIdx.x / kWave), lane = lane_id();
  const int col = first_column(w % W, lane, a.vec);   // vector v: from col + v W 512 on
  float post[NV][8], gate[NV][8], pre[NV][8];
#pragma unroll
  for (int v = 0; v < NV; ++v) {
    load_gain(a.post, col + v * W * 512, a.C, a.vec, post[v]);
    load_gain(a.pre, col + v * W * 512, a.C, a.vec, pre[v]);
  }
  const int R = a.N / a.G;
  int g_of = -1;
  const float inv = 1.0f / (float)a.C;
  // (every wave of a block makes the same number of turns: the sums meet at barriers)
  for (int r0 = blockIdx.x * S; r0 < a.N; r0 += gridDim.x * S) {
    const int row = min(r0 + w / W, a.N - 1);
    const bool live = r0 + w / W < a.N;
    const T* xr = x + (size_t)row * a.C;
    const T* hr = h + (size_t)row * a.C;
    float xv[NV][8], hv[NV][8];
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      load8(hr, col + v * W * 512, a.C, a.vec, hv[v]);
      load8(xr, col + v * W * 512, a.C, a.vec, xv[v]);
    }
    const int g = row / R;
    if (g != g_of) {
      g_of = g;
#pragma unroll
      for (int v = 0; v < NV; ++v)
        load_gain(a.gate ? a.gate + (size_t)g * a.C : nullptr, col + v * W * 512, a.C, a.vec, gate[v]);
    }
    float rh = 1.0f;
    if (a.post) {
      float ss = 0.0f;
#pragma unroll
      for (int v = 0; v < NV; ++v)
#pragma unroll
        for (int q = 0; q < 8; ++q) ss += hv[v][q] * hv[v][q];
      rh = 1.0f / sqrtf(stream_sum<W>(ss, red, w, 0) * inv + a.eps);
    }
    float so = 0.0f;
#pragma unroll
    for (int v = 0; v < NV; ++v)
#pragma unroll
      for (int q = 0; q < 8; ++q) {
        const float o = a.scale * xv[v][q] + gate[v][q] * ((hv[v][q] * rh) * post[v][q]);
        xv[v][q] = o;
        so += o * o;
      }
    if (live) {
#pragma unroll
      for (int v = 0; v < NV; ++v) store8(out + (size_t)row * a.C, col + v * W * 512, a.C, a.vec, xv[v]);
    }
    if (a.pre) {
      const float ro = 1.0f / sqrtf(stream_sum<W>(so, red, w, 1) * inv + a.eps);
#pragma unroll
      for (int v = 0; v < NV; ++v)
#pragma unroll
        for (int q = 0; q < 8; ++q) xv[v][q] = (xv[v][q] * ro) * pre[v][q];
      if (live) {
#pragma unroll
        for (int v = 0; v < NV; ++v) store8(y + (size_t)row * a.C, col + v * W * 512, a.C, a.vec, xv[v]);
      }
      if (live && w % W == 0 && lane == 0) a.ro[row] = ro;
    }
    if (a.post && live && w % W == 0 && lane == 0) a.rh[row] = rh;
    // the next row's sums reuse the slots: with one of them missing, a slot is written
    // again after a single barrier, which its readers may not have passed
    if (W > 1 && !(a.post && a.pre)) __syncthreads();
  }
}

// Column sums of a block's streams added in stream order, written by the first.
template <int W, int NV>
__device__ __forceinline__ void block_columns(const float (&acc)[NV][8], float* lds, int w, int lane, int C,
                                              bool vec, float* __restrict__ dst) {
  constexpr int S = W <= 4 ? 4 / W : 1;
  const int col = first_column(w % W, lane, vec), s = w / W;
  float t[NV][8];
#pragma unroll
  for (int v = 0; v < NV; ++v)
#pragma unroll
    for (int q = 0; q < 8; ++q) t[v][q] = acc[v][q];
  if constexpr (S > 1) {
    __syncthreads();   // the last use of lds
#pragma unroll
    for (int v = 0; v < NV; ++v)
#pragma unroll
      for (int q = 0; q < 8; ++q)   // [stream][vector, column of 8][lane of the stream]
        lds[((s * NV + v) * 8 + q) * (W * kWave) + (w % W) * kWave + lane] = acc[v][q];
    __syncthreads();
    if (s == 0) {
#pragma unroll
      for (int o = 1; o < S; ++o)
#pragma unroll
        for (int v = 0; v < NV; ++v)
#pragma unroll
          for (int q = 0; q < 8; ++q)
            t[v][q] += lds[((o * NV + v) * 8 + q) * (W * kWave) + (w % W) * kWave + lane];
    }
  }
  if (s == 0) {
#pragma unroll
    for (int v = 0; v < NV; ++v)
#pragma unroll
      for (int q = 0; q < 8; ++q) {
        const int c = column(col + v * W * 512, q, vec);
        if (c < C) dst[c] = t[v][q];
      }
  }
}

// sum_part: a block's T_g (parts > 0) or its part of dgamma_post (whole groups); pre_part:
// its part of dgamma_pre, each [blocks][C].
template <typename T, int W, int NV, bool WHOLE>
__global__ __launch_bounds__(W <= 4 ? 256 : W * 64) void norm_backward_kernel(
    NormArgs a, const T* __restrict__ x, const T* __restrict__ h, const T* __restrict__ dout,
    const T* __restrict__ dy, T* __restrict__ dx, T* __restrict__ dh, float* __restrict__ dgate,
    float* __restrict__ sum_part, float* __restrict__ pre_part) {
  constexpr int S = W <= 4 ? 4 / W : 1;
  __shared__ float red[2][16];
  __shared__ float lds[S > 1 ? S * W * kWave * NV * 8 : 1];
  const int w = __builtin_amdgcn_readfirstlane((int)threadIdx.x / kWave), lane = lane_id();
  const int col = first_column(w % W, lane, a.vec), s = w / W;
  const int R = a.N / a.G;
  const float inv = 1.0f / (float)a.C;
  float post[NV][8], gate[NV][8], pre[NV][8], t_acc[NV][8], pre_acc[NV][8];
#pragma unroll
  for (int v = 0; v < NV; ++v) {
    load_gain(a.post, col + v * W * 512, a.C, a.vec, post[v]);
    load_gain(a.pre, col + v * W * 512, a.C, a.vec, pre[v]);
#pragma unroll
    for (int q = 0; q < 8; ++q) t_acc[v][q] = pre_acc[v][q] = 0.0f;
  }
  auto load_gate = [&](int g) __attribute__((always_inline)) {
#pragma unroll
    for (int v = 0; v < NV; ++v)
      load_gain(a.gate ? a.gate + (size_t)g * a.C : nullptr, col + v * W * 512, a.C, a.vec, gate[v]);
  };
  // one row; a row that is not live only keeps the barriers
  auto do_row = [&](int row, bool live) __attribute__((always_inline)) {
    const size_t at = (size_t)row * a.C;
    float o[NV][8], n[NV][8], d[NV][8], z[NV][8];
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      load8(x + at, col + v * W * 512, a.C, a.vec, o[v]);
      load8(h + at, col + v * W * 512, a.C, a.vec, n[v]);
      if (dout) {
        load8(dout + at, col + v * W * 512, a.C, a.vec, d[v]);
      } else {
#pragma unroll
        for (int q = 0; q < 8; ++q) d[v][q] = 0.0f;
      }
      if (a.pre) load8(dy + at, col + v * W * 512, a.C, a.vec, z[v]);
    }
    const float rh = a.post ? a.rh[row] : 1.0f;
#pragma unroll
    for (int v = 0; v < NV; ++v)
#pragma unroll
      for (int q = 0; q < 8; ++q) n[v][q] *= rh;
    if (a.pre) {
      const float ro = a.ro[row];
      float s1 = 0.0f;
#pragma unroll
      for (int v = 0; v < NV; ++v)
#pragma unroll
        for (int q = 0; q < 8; ++q) {
          o[v][q] = __builtin_fmaf(a.scale, o[v][q], gate[v][q] * (n[v][q] * post[v][q])) * ro;
          s1 = __builtin_fmaf(z[v][q] * pre[v][q], o[v][q], s1);
        }
      s1 = stream_sum<W>(s1, red, w, 0) * inv;
#pragma unroll
      for (int v = 0; v < NV; ++v)
#pragma unroll
        for (int q = 0; q < 8; ++q) {
          d[v][q] = __builtin_fmaf(ro, __builtin_fmaf(z[v][q], pre[v][q], -(o[v][q] * s1)), d[v][q]);
          if (live) pre_acc[v][q] = __builtin_fmaf(z[v][q], o[v][q], pre_acc[v][q]);
        }
    }
    float s2 = 0.0f;
#pragma unroll
    for (int v = 0; v < NV; ++v)
#pragma unroll
      for (int q = 0; q < 8; ++q) {
        if (live) t_acc[v][q] = __builtin_fmaf(d[v][q], n[v][q], t_acc[v][q]);
        z[v][q] = d[v][q] * gate[v][q] * post[v][q];
        s2 = __builtin_fmaf(z[v][q], n[v][q], s2);
        d[v][q] *= a.scale;
      }
    if (live) {
#pragma unroll
      for (int v = 0; v < NV; ++v) store8(dx + at, col + v * W * 512, a.C, a.vec, d[v], a.once);
    }
    if (a.post) {
      s2 = stream_sum<W>(s2, red, w, 1) * inv;
#pragma unroll
      for (int v = 0; v < NV; ++v)
#pragma unroll
        for (int q = 0; q < 8; ++q) z[v][q] = rh * __builtin_fmaf(-n[v][q], s2, z[v][q]);
    }
    if (live) {
#pragma unroll
      for (int v = 0; v < NV; ++v) store8(dh + at, col + v * W * 512, a.C, a.vec, z[v], a.once);
    }
    if (W > 1 && !(a.post && a.pre)) __syncthreads();   // (as in the forward)
  };
  if constexpr (!WHOLE) {
    const int g = blockIdx.x / a.parts, part = blockIdx.x % a.parts;
    const int r1 = g * R + min(R, part * a.chunk + a.span);
    load_gate(g);
    for (int r0 = g * R + part * a.chunk; r0 < r1; r0 += a.step) do_row(min(r0 + s, r1 - 1), r0 + s < r1);
    block_columns<W, NV>(t_acc, lds, w, lane, a.C, a.vec, sum_part + (size_t)blockIdx.x * a.C);
  } else {
    float post_acc[NV][8];
#pragma unroll
    for (int v = 0; v < NV; ++v)
#pragma unroll
      for (int q = 0; q < 8; ++q) post_acc[v][q] = 0.0f;
    const int g1 = min(a.G, ((int)blockIdx.x + 1) * a.per_block);
    for (int g0 = blockIdx.x * a.per_block; g0 < g1; g0 += S) {
      const int g = min(g0 + s, g1 - 1);
      const bool live = g0 + s < g1;
      load_gate(g);
      for (int r = 0; r < R; ++r) do_row(g * R + r, live);
#pragma unroll
      for (int v = 0; v < NV; ++v)
#pragma unroll
        for (int q = 0; q < 8; ++q) {
          const int c = column(col + v * W * 512, q, a.vec);
          if (dgate && live && c < a.C) dgate[(size_t)g * a.C + c] = t_acc[v][q] * post[v][q];
          post_acc[v][q] += t_acc[v][q] * gate[v][q];
          t_acc[v][q] = 0.0f;
        }
    }
    block_columns<W, NV>(post_acc, lds, w, lane, a.C, a.vec, sum_part + (size_t)blockIdx.x * a.C);
  }
  if (a.pre) block_columns<W, NV>(pre_acc, lds, w, lane, a.C, a.vec, pre_part + (size_t)blockIdx.x * a.C);
}

// 8 columns as they are in memory: a row that is requested while another is worked on.
// widen: as fp32, or zeros.
template <typename T> struct Raw;
template <> struct Raw<bf16_t> { uint4 u; };
template <> struct Raw<float> { float4 a, b; };
__device__ __forceinline__ void widen(const Raw<float>& r, bool in, float (&o)[8]) {
  const float v[8] = {r.a.x, r.a.y, r.a.z, r.a.w, r.b.x, r.b.y, r.b.z, r.b.w};
#pragma unroll
  for (int q = 0; q < 8; ++q) o[q] = in ? v[q] : 0.0f;
}
__device__ __forceinline__ void widen(const Raw<bf16_t>& r, bool in, float (&o)[8]) {
  const uint32_t wv[4] = {in ? r.u.x : 0u, in ? r.u.y : 0u, in ? r.u.z : 0u, in ? r.u.w : 0u};
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    o[2 * q] = __uint_as_float(wv[q] << 16);
    o[2 * q + 1] = __uint_as_float(wv[q] & 0xFFFF0000u);
  }
}

// norm_backward_kernel for the case that training has: both norms and dout there, rows of
// 16-byte vectors up to 512 W columns, groups split over blocks.  Nothing in a row's
// course depends on what is there, so that the compiler can count loads and stores: a
// row's stores need not have ended for the next row's values, which were requested
// before them, to be used (memory operations of a wave end in order).  The gains are in
// LDS, which leaves the registers to that second row.  A stream without a row of its own
// in a turn repeats the group's last one, whose results it stores once more, and adds
// nothing to the column sums.
// MI355X, us against norm_backward_kernel: 16384 x 1024 bf16 41.6 -> 36.4, 32768 x 2048 190
// -> 175 (805 MB, 4.6 TB/s), 20000 x 512 23.4 -> 22.3; 4096 x 4096 fp32 75 -> 78, 8000 x 8192
// 187 -> 190.  A gain or dout less keeps norm_backward_kernel: 16384 x 1024 38 with gamma_pre
// alone, 37 without dout, 32768 x 2048 182.  Memory bounds it: without the sums over a row it
// takes as long, without one of the two stores 30 us less at 32768 x 2048, without two of the
// four loads 60.
template <typename T, int W, bool ONCE>
__global__ __launch_bounds__(W <= 4 ? 256 : W * 64, 4) void norm_backward_full_kernel(
    NormArgs a, const T* __restrict__ x, const T* __restrict__ h, const T* __restrict__ dout,
    const T* __restrict__ dy, T* __restrict__ dx, T* __restrict__ dh, float* __restrict__ sum_part,
    float* __restrict__ pre_part) {
  constexpr int S = W <= 4 ? 4 / W : 1;
  __shared__ float red[2][16];
  __shared__ float lds[S > 1 ? S * W * kWave * 8 : 1];
  __shared__ __attribute__((aligned(16))) float gains[3][W * 512];
  const int w = __builtin_amdgcn_readfirstlane((int)threadIdx.x / kWave), lane = lane_id();
  const int col = first_column(w % W, lane, true), s = w / W;
  const int R = a.N / a.G, g = blockIdx.x / a.parts, part = blockIdx.x % a.parts;
  const float inv = 1.0f / (float)a.C;
  for (int c = threadIdx.x; c < W * 512; c += blockDim.x) {
    const bool in = c < a.C;
    gains[0][c] = in ? a.post[c] : 0.0f;
    gains[1][c] = in ? a.pre[c] : 0.0f;
    gains[2][c] = !in ? 0.0f : a.gate ? a.gate[(size_t)g * a.C + c] : 1.0f;
  }
  __syncthreads();
  auto gain = [&](int k, float (&o)[8]) __attribute__((always_inline)) {
    const float4* p = reinterpret_cast<const float4*>(&gains[k][col]);
    const float4 u = p[0], v = p[1];
    o[0] = u.x; o[1] = u.y; o[2] = u.z; o[3] = u.w;
    o[4] = v.x; o[5] = v.y; o[6] = v.z; o[7] = v.w;
  };
  // (lanes past the row read its first columns, take them as zeros, and store nothing)
  const bool in_row = col < a.C;
  const int from = in_row ? col : 0;
  Raw<T> nx, nh, nd, ny;
  float nrh, nro;
  auto request = [&](int row) __attribute__((always_inline)) {
    const size_t at = (size_t)row * a.C + from;
    nx = *reinterpret_cast<const Raw<T>*>(x + at);
    nh = *reinterpret_cast<const Raw<T>*>(h + at);
    nd = *reinterpret_cast<const Raw<T>*>(dout + at);
    ny = *reinterpret_cast<const Raw<T>*>(dy + at);
    nrh = a.rh[row];
    nro = a.ro[row];
  };
  float t_acc[8], pre_acc[8];
#pragma unroll
  for (int q = 0; q < 8; ++q) t_acc[q] = pre_acc[q] = 0.0f;
  const int r1 = g * R + min(R, part * a.chunk + a.span);
  int r0 = g * R + part * a.chunk;
  request(min(r0 + s, r1 - 1));
  for (; r0 < r1; r0 += a.step) {
    const int row = min(r0 + s, r1 - 1);
    const bool live = r0 + s < r1;
    float o[8], n[8], d[8], z[8];
    widen(nx, in_row, o);
    widen(nh, in_row, n);
    widen(nd, in_row, d);
    widen(ny, in_row, z);
    const float rh = nrh, ro = nro;
    request(min(r0 + a.step + s, r1 - 1));
    float s1 = 0.0f;
    {
      float post[8], gate[8], pre[8];
      gain(0, post);
      gain(2, gate);
      gain(1, pre);
#pragma unroll
      for (int q = 0; q < 8; ++q) {
        n[q] *= rh;
        o[q] = __builtin_fmaf(a.scale, o[q], gate[q] * (n[q] * post[q])) * ro;
        const float k = z[q] * pre[q];
        s1 = __builtin_fmaf(k, o[q], s1);
        pre_acc[q] = live ? __builtin_fmaf(z[q], o[q], pre_acc[q]) : pre_acc[q];
        z[q] = k;
      }
    }
    s1 = stream_sum<W>(s1, red, w, 0) * inv;
    float s2 = 0.0f;
    {
      float post[8], gate[8];
      gain(0, post);
      gain(2, gate);
#pragma unroll
      for (int q = 0; q < 8; ++q) {
        d[q] = __builtin_fmaf(ro, __builtin_fmaf(-o[q], s1, z[q]), d[q]);
        t_acc[q] = live ? __builtin_fmaf(d[q], n[q], t_acc[q]) : t_acc[q];
        z[q] = d[q] * gate[q] * post[q];
        s2 = __builtin_fmaf(z[q], n[q], s2);
        d[q] *= a.scale;
      }
    }
    s2 = stream_sum<W>(s2, red, w, 1) * inv;
#pragma unroll
    for (int q = 0; q < 8; ++q) z[q] = rh * __builtin_fmaf(-n[q], s2, z[q]);
    if (in_row) {
      store8(dx + (size_t)row * a.C, col, a.C, true, d, ONCE);
      store8(dh + (size_t)row * a.C, col, a.C, true, z, ONCE);
    }
  }
  float t[1][8], p[1][8];
#pragma unroll
  for (int q = 0; q < 8; ++q) {
    t[0][q] = t_acc[q];
    p[0][q] = pre_acc[q];
  }
  block_columns<W, 1>(t, lds, w, lane, a.C, true, sum_part + (size_t)blockIdx.x * a.C);
  block_columns<W, 1>(p, lds, w, lane, a.C, true, pre_part + (size_t)blockIdx.x * a.C);
}

// Sums rows r0 .. r1 - 1 of src [.][C] at 64 columns by 16 waves, in a fixed order; the
// first wave has them.
__device__ __forceinline__ float column_sum(const float* __restrict__ src, int r0, int r1, int C, int c,
                                            float (*lds)[kWave], int w, int lane) {
  float s0 = 0.0f, s1 = 0.0f, s2 = 0.0f, s3 = 0.0f;
  if (c < C) {
    int r = r0 + w;
    for (; r + 48 < r1; r += 64) {
      s0 += src[(size_t)r * C + c];
      s1 += src[(size_t)(r + 16) * C + c];
      s2 += src[(size_t)(r + 32) * C + c];
      s3 += src[(size_t)(r + 48) * C + c];
    }
    for (; r < r1; r += 16) s0 += src[(size_t)r * C + c];
  }
  lds[w][lane] = (s0 + s1) + (s2 + s3);
  __syncthreads();
  float t = 0.0f;
  if (w == 0)
    for (int i = 0; i < 16; ++i) t += lds[i][lane];
  __syncthreads();
  return t;
}

// Grid (columns / 64, rows): row 0 sums pre_part, row 1 + g group g's blocks of sum_part
// (parts > 0) or, where whole groups went to a block, row 1 all of them.
// One group: dgamma_post here; more: T_g gate_g to group_sums [G][C], added by a second launch
// (groups_only).
__global__ __launch_bounds__(1024) void norm_reduce_kernel(
    const float* __restrict__ sum_part, const float* __restrict__ pre_part, int blocks, int parts, int G, int C,
    const float* __restrict__ post, const float* __restrict__ gate, float* __restrict__ dpost,
    float* __restrict__ dgate, float* __restrict__ dpre, float* __restrict__ group_sums) {
  __shared__ float lds[16][kWave];
  const int w = threadIdx.x / kWave, lane = lane_id(), c = blockIdx.x * kWave + lane;
  if (blockIdx.y == 0) {
    if (!dpre) return;
    const float t = column_sum(pre_part, 0, blocks, C, c, lds, w, lane);
    if (w == 0 && c < C) dpre[c] = t;
    return;
  }
  const int g = blockIdx.y - 1;
  if (parts == 0) {
    if (!dpost) return;
    const float t = column_sum(sum_part, 0, blocks, C, c, lds, w, lane);
    if (w == 0 && c < C) dpost[c] = t;
    return;
  }
  const float t = column_sum(sum_part, g * parts, (g + 1) * parts, C, c, lds, w, lane);
  if (w != 0 || c >= C) return;
  if (dgate) dgate[(size_t)g * C + c] = t * (post ? post[c] : 1.0f);
  if (!dpost) return;
  const float u = t * (gate ? gate[(size_t)g * C + c] : 1.0f);
  if (G == 1) dpost[c] = u;
  else group_sums[(size_t)g * C + c] = u;
}

// Waves and vectors of a row.  Forward: 1024 columns a wave, whose gains then serve more
// of a row (16384 x 1024: 22.4 us, with 512 24.5; 32768 x 2048: 95 / 110).  Backward: 512,
// for twice the waves on a CU (norm_backward_kernel, us with 1024 / 512: 16384 x 1024 53 /
// 44, 32768 x 2048 259 / 199).
void row_layout(int C, bool backward, int* W, int* NV) {
  *NV = C <= (backward ? 8192 : 512) ? 1 : 2;
  int w = 1;
  while (w * *NV * 512 < C) w *= 2;
  *W = w;
}

NormPlan plan_backward(int N, int C, int G, bool full) {
  NormPlan p{};
  row_layout(C, true, &p.W, &p.NV);
  const int S = p.W <= 4 ? 4 / p.W : 1, R = N / G;
  // Enough blocks for the chip, few enough that their column sums cost little; half as many
  // where a wave has two rows in flight (us with 512 / 1024 blocks: 16384 x 1024 36.4 /
  // 41.8, 32768 x 2048 175 / 185; norm_backward_kernel, one row in flight, 59 / 44).
  const int target = p.W > 4 ? 256 : full ? 512 : 1024;
  if (R < 8 || G >= target * S) {
    const int per = (G + target - 1) / target;
    p.per_block = (per + S - 1) / S * S;
    p.blocks = (G + p.per_block - 1) / p.per_block;
  } else {
    // A block's own run of rows, or rows in turn with the group's other blocks, whose rows in
    // flight then are neighbours (us of norm_backward_kernel, run / in turn: 20000 x 512 23.8 /
    // 25.3, 32768 x 2048 198 / 191, 8000 x 8192 206 / 189).
    p.parts = std::max(1, std::min((target + G - 1) / G, (R + S - 1) / S));
    if (p.W == 1) {
      p.chunk = p.span = ((R + p.parts - 1) / p.parts + S - 1) / S * S;
      p.step = S;
      p.parts = (R + p.chunk - 1) / p.chunk;
    } else {
      p.chunk = S;
      p.step = p.parts * S;
      p.span = R;
    }
    p.blocks = G * p.parts;
  }
  return p;
}

struct NormLayout {
  size_t sum_part, pre_part, group_sums, total;
};
size_t align_up(size_t v) { return (v + 255) / 256 * 256; }
NormLayout norm_layout(const NormPlan& p, int C, int G) {
  NormLayout l{};
  l.pre_part = align_up((size_t)p.blocks * C * 4);
  l.group_sums = l.pre_part + align_up((size_t)p.blocks * C * 4);
  l.total = l.group_sums + (p.parts > 0 && G > 1 ? align_up((size_t)G * C * 4) : 0);
  return l;
}

// f(waves, vectors) of row_layout's rows: one vector, or two forward past 512 columns and
// backward past 8192, where it is 16 waves.
template <bool BACKWARD, typename F>
hipError_t for_layout(int W, int NV, F&& f) {
  constexpr std::integral_constant<int, 1> one;
  constexpr std::integral_constant<int, 2> two;
  constexpr std::integral_constant<int, 16> most;
  if (BACKWARD && NV == 2) {
    f(most, two);
  } else if (!BACKWARD && NV == 1) {
    f(one, one);
  } else {
    constexpr std::integral_constant<int, BACKWARD ? 1 : 2> nv;
    switch (W) {
      case 1: f(one, nv); break;
      case 2: f(two, nv); break;
      case 4: f(std::integral_constant<int, 4>{}, nv); break;
      case 8: f(std::integral_constant<int, 8>{}, nv); break;
      default: f(most, nv); break;
    }
  }
  return hipGetLastError();
}

int check_norm(const mgpt_norm_config* cfg, int N, bool gated) {
  if (!cfg) return fail(MGPT_ERR_INVALID_ARGUMENT, "config is null");
  if (N < 0) return fail(MGPT_ERR_INVALID_ARGUMENT, "negative num_tokens");
  if (N > 1 << 30) return fail(MGPT_ERR_UNSUPPORTED, "num_tokens %d > 2^30", N);
  if (cfg->embed_dim <= 0) return fail(MGPT_ERR_INVALID_ARGUMENT, "embed_dim %d", cfg->embed_dim);
  if (cfg->embed_dim > kMaxC)
    return fail(MGPT_ERR_UNSUPPORTED, "embed_dim %d > %d", cfg->embed_dim, kMaxC);
  if (cfg->dtype != MGPT_DTYPE_F32 && cfg->dtype != MGPT_DTYPE_BF16)
    return fail(MGPT_ERR_UNSUPPORTED, "unsupported dtype %d", cfg->dtype);
  if (!(cfg->eps >= 0.0f) || !std::isfinite(cfg->residual_scale))
    return fail(MGPT_ERR_INVALID_ARGUMENT, "eps must be >= 0 and residual_scale finite");
  if (cfg->gate_rows < 1 || (gated && N % cfg->gate_rows != 0))
    return fail(MGPT_ERR_INVALID_ARGUMENT, "gate_rows %d must divide num_tokens %d", cfg->gate_rows, N);
  return MGPT_OK;
}

NormArgs norm_args(const mgpt_norm_config* cfg, int N, const float* post, const float* gate, const float* pre,
                   float* rh, float* ro, std::initializer_list<const void*> rows) {
  NormArgs a{};
  a.N = N;
  a.C = cfg->embed_dim;
  // (without a gate its rows mean nothing: one group)
  a.G = gate ? cfg->gate_rows : 1;
  a.scale = cfg->residual_scale;
  a.eps = cfg->eps;
  a.post = post;
  a.gate = gate;
  a.pre = pre;
  a.rh = rh;
  a.ro = ro;
  uintptr_t bits = 0;
  for (const void* p : rows) bits |= (uintptr_t)p;
  a.vec = a.C % 8 == 0 && (bits & 15) == 0;
  return a;
}

}  // namespace
}  // namespace mgpt

using namespace mgpt;

extern "C" {

int mgpt_norm_forward(const mgpt_norm_config* cfg, const void* x, const void* h, const float* gamma_post,
                      const float* gate, const float* gamma_pre, void* out, void* y, float* rstd_post,
                      float* rstd_pre, int num_tokens, void* stream) {
  if (int rc = check_norm(cfg, num_tokens, gate != nullptr)) return rc;
  if (num_tokens == 0) return MGPT_OK;
  if (!x || !h || !out) return fail(MGPT_ERR_INVALID_ARGUMENT, "null x, h or out");
  if ((gamma_pre && (!y || !rstd_pre)) || (gamma_post && !rstd_post))
    return fail(MGPT_ERR_INVALID_ARGUMENT, "gamma_pre needs y and rstd_pre, gamma_post needs rstd_post");
  const NormArgs a = norm_args(cfg, num_tokens, gamma_post, gate, gamma_pre, rstd_post, rstd_pre,
                               {x, h, out, gamma_pre ? y : nullptr, gamma_post, gate, gamma_pre});
  int W, NV;
  row_layout(a.C, false, &W, &NV);
  const int S = W <= 4 ? 4 / W : 1, rows = (num_tokens + S - 1) / S;
  const int grid = std::min(rows, compute_units() * (W <= 4 ? 4 : 16 / W));
  auto go = [&](auto t) {
    using T = decltype(t);
    return for_layout<false>(W, NV, [&](auto w, auto nv) {
      constexpr int kW = decltype(w)::value, kNV = decltype(nv)::value;
      hipLaunchKernelGGL((norm_forward_kernel<T, kW, kNV>), dim3(grid), dim3(kW <= 4 ? 256 : kW * 64), 0,
                         (hipStream_t)stream, a, (const T*)x, (const T*)h, (T*)out, (T*)y);
    });
  };
  HIP_TRY(cfg->dtype == MGPT_DTYPE_F32 ? go(float{}) : go(bf16_t{}));
  return MGPT_OK;
}

int mgpt_norm_backward_workspace_bytes(const mgpt_norm_config* cfg, int num_tokens, size_t* bytes) {
  if (!bytes) return fail(MGPT_ERR_INVALID_ARGUMENT, "null bytes");
  if (int rc = check_norm(cfg, num_tokens, false)) return rc;
  *bytes = 0;
  if (num_tokens == 0) return MGPT_OK;
  // with and without a gate (whose rows decide the blocks)
  const int C = cfg->embed_dim, G = num_tokens % cfg->gate_rows == 0 ? cfg->gate_rows : 1;
  for (const int g : {G, 1})
    for (const bool full : {false, true})
      *bytes = std::max(*bytes, norm_layout(plan_backward(num_tokens, C, g, full), C, g).total);
  return MGPT_OK;
}

int mgpt_norm_backward(const mgpt_norm_config* cfg, const void* x, const void* h, const float* gamma_post,
                       const float* gate, const float* gamma_pre, const float* rstd_post,
                       const float* rstd_pre, const void* dout, const void* dy, void* dx, void* dh,
                       float* dgamma_post, float* dgate, float* dgamma_pre, int num_tokens, void* workspace,
                       size_t workspace_bytes, void* stream) {
  if (int rc = check_norm(cfg, num_tokens, gate != nullptr)) return rc;
  if ((dgamma_post && !gamma_post) || (dgate && !gate) || (dgamma_pre && !gamma_pre))
    return fail(MGPT_ERR_INVALID_ARGUMENT, "a gradient of a gain that is null");
  const int C = cfg->embed_dim;
  if (num_tokens == 0) {   // no token adds to the gains' gradients
    if (dgamma_post) HIP_TRY(launch_fill_zero(dgamma_post, C, (hipStream_t)stream));
    if (dgate) HIP_TRY(launch_fill_zero(dgate, (size_t)cfg->gate_rows * C, (hipStream_t)stream));
    if (dgamma_pre) HIP_TRY(launch_fill_zero(dgamma_pre, C, (hipStream_t)stream));
    return MGPT_OK;
  }
  if (!x || !h || !dx || !dh) return fail(MGPT_ERR_INVALID_ARGUMENT, "null x, h, dx or dh");
  if ((gamma_pre && (!dy || !rstd_pre)) || (gamma_post && !rstd_post))
    return fail(MGPT_ERR_INVALID_ARGUMENT, "gamma_pre needs dy and rstd_pre, gamma_post needs rstd_post");
  if (!gamma_pre && !dout) return fail(MGPT_ERR_INVALID_ARGUMENT, "null dout without gamma_pre");
  if (!workspace) return fail(MGPT_ERR_INVALID_ARGUMENT, "null workspace");
  if ((uintptr_t)workspace & 255) return fail(MGPT_ERR_INVALID_ARGUMENT, "workspace must be 256-byte aligned");
  NormArgs a = norm_args(cfg, num_tokens, gamma_post, gate, gamma_pre, const_cast<float*>(rstd_post),
                         const_cast<float*>(rstd_pre),
                         {x, h, dout, gamma_pre ? dy : nullptr, dx, dh, gamma_post, gate, gamma_pre});
  const bool all = a.vec && a.post && a.pre && dout && C <= 8192;   // what norm_backward_full_kernel takes
  const NormPlan p = plan_backward(a.N, C, a.G, all);
  const NormLayout l = norm_layout(p, C, a.G);
  if (workspace_bytes < l.total)
    return fail(MGPT_ERR_WORKSPACE_TOO_SMALL, "workspace needs %zu bytes, got %zu", l.total, workspace_bytes);
  a.parts = p.parts;
  a.chunk = p.chunk;
  a.step = p.step;
  a.span = p.span;
  a.per_block = p.per_block;
  // (us, cached / past the caches: 32768 x 2048 191 / 179, 8000 x 8192 189 / 176, but 20000 x
  // 512, whose outputs the last-level cache holds, 25.3 / 26.7)
  a.once = 2 * (size_t)a.N * C * (cfg->dtype == MGPT_DTYPE_F32 ? 4 : 2) >= (size_t)128 << 20;
  float* sums = (float*)workspace;
  float* pres = (float*)((char*)workspace + l.pre_part);
  float* groups = (float*)((char*)workspace + l.group_sums);
  hipStream_t st = (hipStream_t)stream;
  auto go = [&](auto t) {
    using T = decltype(t);
    return for_layout<true>(p.W, p.NV, [&](auto w, auto nv) {
      constexpr int kW = decltype(w)::value, kNV = decltype(nv)::value;
      auto launch = [&](auto kernel) {
        hipLaunchKernelGGL(kernel, dim3(p.blocks), dim3(kW <= 4 ? 256 : kW * 64), 0, st, a, (const T*)x,
                           (const T*)h, (const T*)dout, (const T*)dy, (T*)dx, (T*)dh, dgate, sums, pres);
      };
      if constexpr (kNV == 1) {
        if (p.parts > 0 && all) {
          auto full = [&](auto kernel) {
            hipLaunchKernelGGL(kernel, dim3(p.blocks), dim3(kW <= 4 ? 256 : kW * 64), 0, st, a, (const T*)x,
                               (const T*)h, (const T*)dout, (const T*)dy, (T*)dx, (T*)dh, sums, pres);
          };
          if (a.once) full(norm_backward_full_kernel<T, kW, true>);
          else full(norm_backward_full_kernel<T, kW, false>);
          return;
        }
      }
      if (p.parts > 0) launch(norm_backward_kernel<T, kW, kNV, false>);
      else launch(norm_backward_kernel<T, kW, kNV, true>);
    });
  };
  HIP_TRY(cfg->dtype == MGPT_DTYPE_F32 ? go(float{}) : go(bf16_t{}));
  const bool whole = p.parts == 0;
  if (!dgamma_post && !dgamma_pre && !(dgate && !whole)) return MGPT_OK;
  const dim3 tiles((C + kWave - 1) / kWave, 1 + (whole ? 1 : a.G));
  hipLaunchKernelGGL(norm_reduce_kernel, tiles, dim3(1024), 0, st, sums, pres, p.blocks, p.parts, a.G, C,
                     gamma_post, gate, dgamma_post, whole ? nullptr : dgate, dgamma_pre, groups);
  if (!whole && a.G > 1 && dgamma_post)   // the groups' sums: as whole groups' partial sums
    hipLaunchKernelGGL(norm_reduce_kernel, dim3(tiles.x, 2), dim3(1024), 0, st, groups, nullptr, a.G, 0, a.G, C,
                       nullptr, nullptr, dgamma_post, nullptr, nullptr, nullptr);
  HIP_TRY(hipGetLastError());
  return MGPT_OK;
}

}  // extern "C"
