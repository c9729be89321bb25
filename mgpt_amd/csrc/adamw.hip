// adamw.hip -- one AdamW step over many tensors, moments in 32 or in 8 bits.
//
// Reference: AdamWOptimizer::step (nn/optimisers/AdamWOptimiser.h:13-97), which runs
// Tensor::adamw_step (utils/Tensor.cpp:683-701) tensor by tensor.  Per element, with g
// the gradient times the caller's scale and t the step's number, every operation
// rounded to fp32 in this order:
//   m = b1 m + (1 - b1) g,  v = b2 v + ((1 - b2) g) g
//   p = p - (lr wd) p,      p = p - (lr (m c1)) / (sqrt(v c2) + eps)
// c1 = 1 / (1 - b1^t) and c2 likewise (formed in fp64, rounded once).
//
// 8-bit moments.  256 consecutive elements of a tensor, a wave's 4 per lane, share a
// biased power of two per moment, taken from the block's largest finite magnitude:
//  * m: e4m3 x 2^(e - 134), nearest even.  The block's largest value lands in
//    [128, 256), so nothing overflows and scaling is exact.
//  * v: unsigned, 5 bits of exponent and 3 of fraction (code c in 1 .. 254 is the fp32
//    with bits ((e - 31) << 23) + (c << 20)); the largest value's exponent is the 30th,
//    one is left for rounding up.  v moves by (1 - b2) = 0.001 a step, far less than
//    half of a code's step (6%), so rounding to nearest would hold it for good: it is
//    rounded up with the probability of what is cut off, 16 bits of a counter hash
//    (Wellons' lowbias32 over the element pair and the step: the same call gives the same
//    bits).  v > 0 is never held as 0, which m / (sqrt(0) + eps) would blow up.
//  * A moment that is not finite is held as NaN (e4m3's, code 255) and does not
//    enter the block's power of two, so it stays where it arose.
// Moments are decoded, updated and used in fp32; only what is held is rounded.
//
// What bounds it: memory.  Per element 28 bytes in 32 bits with fp32 gradients, 14 in 8
// bits with bf16 ones (+2 with a bf16 copy).  A block of threads takes 4096 elements of
// one tensor (found by a search of the tensors' table, which is a kernel argument: any
// set of tensors in one launch per 116), every load of a lane requested before the first
// use, all of it past the caches, which would hold none of it for the next step.  MI355X,
// 98 tensors of 139M elements: 665 to 684 us in 32 bits (5.7 to 5.9 TB/s; through the
// caches 741), 367 to 380 in 8 with bf16 gradients and copies (16 bytes an element, 5.9
// TB/s; the first sixty launches after a pause take up to 520).
#include <hip/hip_runtime.h>

#include <cmath>

#include "../../include/mgpt_moe.h"
#include "capi_internal.hpp"
#include "common.hpp"

namespace mgpt {
namespace {

constexpr int kBlock = 256;        // elements that share 8-bit exponents: one wave x 4
constexpr int kIters = 4;          // blocks per wave
constexpr int kTile = 4 * kIters * kBlock;   // elements per workgroup
constexpr uint64_t kMaxTiles = 1u << 23;     // per launch (2^31 threads)

struct AdamwTensors {
  static constexpr int kMax = 116;   // keeps the argument block under 4 KB
  float* p[kMax];
  const void* g[kMax];
  bf16_t* copy[kMax];
  uint32_t block0[kMax];      // first state block
  uint32_t tile0[kMax + 1];   // first workgroup; past the last tensor: all of them
  uint16_t tail[kMax];        // elements of the last workgroup's tile, 1 .. kTile
  int n;
};

struct AdamwArgs {
  float lr, b1, b2, a1, a2, eps, shrink, c1, c2;   // a = 1 - b, shrink = lr wd
  uint32_t step;
  const int32_t* step_device;
  const float* grad_scale;
  char *m, *v;
  uint8_t *me, *ve;
};

__host__ __device__ inline double int_power(double b, uint32_t n) {
  double r = 1.0;
  for (; n; n >>= 1, b *= b)
    if (n & 1) r *= b;
  return r;
}
__host__ __device__ inline float bias_correction(float b, uint32_t t) {
  return (float)(1.0 / (1.0 - int_power((double)b, t)));
}

// Largest of the 64 lanes' non-negative values, by DPP (as wave_incl_scan).
template <int CTRL, int ROWS>
__device__ __forceinline__ uint32_t dpp_max(uint32_t v) {
  const uint32_t o = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, ROWS, 0xf, false);
  return v > o ? v : o;
}
__device__ __forceinline__ uint32_t wave_max(uint32_t v) {
  v = dpp_max<0x111, 0xf>(v);
  v = dpp_max<0x112, 0xf>(v);
  v = dpp_max<0x114, 0xf>(v);
  v = dpp_max<0x118, 0xf>(v);
  v = dpp_max<0x142, 0xa>(v);
  v = dpp_max<0x143, 0xc>(v);
  return (uint32_t)__builtin_amdgcn_readlane((int)v, kWave - 1);
}

__device__ __forceinline__ uint32_t hash32(uint32_t x) {   // lowbias32
  x ^= x >> 16;
  x *= 0x7FEB352Du;
  x ^= x >> 15;
  x *= 0x846CA68Bu;
  return x ^ (x >> 16);
}

template <int V>
struct IntTag {};

// |x|'s bits, 0 for what is not finite
__device__ __forceinline__ uint32_t finite_bits(float x) {
  const uint32_t u = __float_as_uint(x) & 0x7FFFFFFFu;
  return u < 0x7F800000u ? u : 0u;
}

// Four moments of a lane, as they are held.
template <int BITS> struct Held;
template <> struct Held<32> { float4 m, v; };
template <> struct Held<8> { uint32_t m, v; int me, ve; };

__device__ __forceinline__ Held<32> load_held32(const AdamwArgs& a, size_t at) {
  return {load_once(reinterpret_cast<const float4*>(a.m + 4 * at)), load_once(reinterpret_cast<const float4*>(a.v + 4 * at))};
}
__device__ __forceinline__ Held<8> load_held8(const AdamwArgs& a, size_t at, size_t block) {
  return {load_once(reinterpret_cast<const uint32_t*>(a.m + at)), load_once(reinterpret_cast<const uint32_t*>(a.v + at)),
          a.me[block], a.ve[block]};
}
template <int BITS>
__device__ __forceinline__ Held<BITS> load_held(const AdamwArgs& a, size_t at, size_t block) {
  if constexpr (BITS == 32) return load_held32(a, at);
  else return load_held8(a, at, block);
}

__device__ __forceinline__ void decode(const Held<32>& h, float (&m)[4], float (&v)[4]) {
  m[0] = h.m.x; m[1] = h.m.y; m[2] = h.m.z; m[3] = h.m.w;
  v[0] = h.v.x; v[1] = h.v.y; v[2] = h.v.z; v[3] = h.v.w;
}
__device__ __forceinline__ void decode(const Held<8>& h, float (&m)[4], float (&v)[4]) {
  // exponents below the smallest that is written (a state of zero bytes) count as it
  const float s = __uint_as_float((uint32_t)(max(h.me, 16) - 7) << 23);
  const uint32_t base = (uint32_t)(max(h.ve, 32) - 31) << 23;
  const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)h.m, false);
  const auto hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)h.m, true);
  m[0] = lo[0] * s; m[1] = lo[1] * s; m[2] = hi[0] * s; m[3] = hi[1] * s;
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    const uint32_t c = (h.v >> (8 * q)) & 0xFFu;
    v[q] = __uint_as_float(c == 0 ? 0u : c == 255 ? 0x7FC00000u : base + (c << 20));
  }
}

__device__ __forceinline__ void store_held(const AdamwArgs& a, size_t at, size_t, uint32_t,
                                           const float (&m)[4], const float (&v)[4], IntTag<32>) {
  store_once(reinterpret_cast<float4*>(a.m + 4 * at), make_float4(m[0], m[1], m[2], m[3]));
  store_once(reinterpret_cast<float4*>(a.v + 4 * at), make_float4(v[0], v[1], v[2], v[3]));
}
__device__ __forceinline__ void store_held(const AdamwArgs& a, size_t at, size_t block, uint32_t step,
                                           const float (&m)[4], const float (&v)[4], IntTag<8>) {
  uint32_t um = 0, uv = 0;
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    um = max(um, finite_bits(m[q]));
    uv = max(uv, finite_bits(v[q]));
  }
  const uint32_t me = max(wave_max(um) >> 23, 16u), ve = max((wave_max(uv) >> 23) + 1, 32u);
  const float s = __uint_as_float((261u - me) << 23);   // 2^(134 - me)
  float t[4];
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    const float x = m[q] * s;
    t[q] = fabsf(x) <= 256.0f ? x : __uint_as_float(0x7FC00000u);
  }
  int cm = __builtin_amdgcn_cvt_pk_fp8_f32(t[0], t[1], 0, false);
  cm = __builtin_amdgcn_cvt_pk_fp8_f32(t[2], t[3], cm, true);
  // 16 random bits an element; `at` counts elements of the state modulo 2^32
  const uint32_t key = step * 0x9E3779B9u, pair = (uint32_t)(at >> 1);
  const uint32_t r[2] = {hash32(pair ^ key), hash32((pair + 1) ^ key)};
  uint32_t cv = 0;
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    const uint32_t u = __float_as_uint(v[q]);
    const uint32_t rnd = (q & 1) ? r[q / 2] >> 16 : r[q / 2] & 0xFFFFu;
    int c = (int)((u + (rnd << 4)) >> 20) - (int)((ve - 31) << 3);
    c = max(c, 1);   // (at most 248: ve is one above the block's largest exponent)
    c = u == 0 ? 0 : u < 0x7F800000u ? c : 255;
    cv |= (uint32_t)c << (8 * q);
  }
  store_once(reinterpret_cast<uint32_t*>(a.m + at), (uint32_t)cm);
  store_once(reinterpret_cast<uint32_t*>(a.v + at), cv);
  if (lane_id() == 0) {
    a.me[block] = (uint8_t)me;
    a.ve[block] = (uint8_t)ve;
  }
}

__device__ __forceinline__ void load_grad4(const float* g, float (&o)[4]) {
  const float4 x = load_once(reinterpret_cast<const float4*>(g));
  o[0] = x.x; o[1] = x.y; o[2] = x.z; o[3] = x.w;
}
__device__ __forceinline__ void load_grad4(const bf16_t* g, float (&o)[4]) {
  const uint2 x = load_once(reinterpret_cast<const uint2*>(g));
  o[0] = __uint_as_float(x.x << 16); o[1] = __uint_as_float(x.x & 0xFFFF0000u);
  o[2] = __uint_as_float(x.y << 16); o[3] = __uint_as_float(x.y & 0xFFFF0000u);
}

template <int BITS, typename GT>
__global__ __launch_bounds__(256) void adamw_kernel(AdamwTensors ts, AdamwArgs a) {
  // the tensor of this workgroup: the last whose first one is not after it
  int lo = 0, hi = ts.n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) / 2;
    if (ts.tile0[mid] <= blockIdx.x) lo = mid;
    else hi = mid;
  }
  float* __restrict__ p = ts.p[lo];
  const GT* __restrict__ g = static_cast<const GT*>(ts.g[lo]);
  bf16_t* __restrict__ copy = ts.copy[lo];
  const uint32_t tile = blockIdx.x - ts.tile0[lo];
  const int left = blockIdx.x + 1 == ts.tile0[lo + 1] ? ts.tail[lo] : kTile;   // elements of this tile
  uint32_t step = a.step;
  if (a.step_device) {
    step = (uint32_t)max(*a.step_device, 1);
    a.c1 = bias_correction(a.b1, step);
    a.c2 = bias_correction(a.b2, step);
  }
  const float gs = a.grad_scale ? *a.grad_scale : 1.0f;
  const int w = __builtin_amdgcn_readfirstlane((int)threadIdx.x / kWave), lane = lane_id();
  const int64_t first = (int64_t)tile * kTile;
  const size_t block0 = (size_t)ts.block0[lo] + (size_t)tile * (kTile / kBlock);
  auto update = [&](float& pv, float gv, float& m, float& v) __attribute__((always_inline)) {
    gv = gv * gs;
    m = m * a.b1 + gv * a.a1;
    v = v * a.b2 + (gv * a.a2) * gv;
    pv = pv - pv * a.shrink;
    pv = pv - ((m * a.c1) * a.lr) / (sqrtf(v * a.c2) + a.eps);
  };
  const bool aligned = ((reinterpret_cast<uintptr_t>(p) & 15) | (reinterpret_cast<uintptr_t>(g) & (4 * sizeof(GT) - 1)) |
                        (reinterpret_cast<uintptr_t>(copy) & 7)) == 0;
  if (aligned && left == kTile) {
    float4 pv[kIters];
    float gv[kIters][4];
    Held<BITS> held[kIters];
#pragma unroll
    for (int i = 0; i < kIters; ++i) {
      const int b = 4 * i + w;
      const int64_t e = first + b * kBlock + 4 * lane;
      pv[i] = load_once(reinterpret_cast<const float4*>(p + e));
      load_grad4(g + e, gv[i]);
      held[i] = load_held<BITS>(a, (block0 + b) * kBlock + 4 * lane, block0 + b);
    }
#pragma unroll
    for (int i = 0; i < kIters; ++i) {
      const int b = 4 * i + w;
      const int64_t e = first + b * kBlock + 4 * lane;
      float m[4], v[4], x[4] = {pv[i].x, pv[i].y, pv[i].z, pv[i].w};
      decode(held[i], m, v);
#pragma unroll
      for (int q = 0; q < 4; ++q) update(x[q], gv[i][q], m[q], v[q]);
      store_once(reinterpret_cast<float4*>(p + e), make_float4(x[0], x[1], x[2], x[3]));
      store_held(a, (block0 + b) * kBlock + 4 * lane, block0 + b, step, m, v, IntTag<BITS>{});
      if (copy)
        store_once(reinterpret_cast<uint2*>(copy + e), make_uint2(pack_bf16x2(x[0], x[1]), pack_bf16x2(x[2], x[3])));
    }
    return;
  }
  // a tensor's end, or one that is not aligned: element by element.  Elements past
  // the end are zeros throughout (the state has room for whole blocks).
  for (int i = 0; i < kIters; ++i) {
    const int b = 4 * i + w;
    if (b * kBlock >= left) return;
    const int64_t e = first + b * kBlock + 4 * lane;
    const size_t at = (block0 + b) * kBlock + 4 * lane;
    float m[4], v[4], x[4];
    decode(load_held<BITS>(a, at, block0 + b), m, v);
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      x[q] = 0.0f;
      if (b * kBlock + 4 * lane + q < left) {
        x[q] = p[e + q];
        update(x[q], to_f32(g[e + q]), m[q], v[q]);
        p[e + q] = x[q];
        if (copy) copy[e + q] = f32_to_bf16(x[q]);
      } else {
        m[q] = v[q] = 0.0f;
      }
    }
    store_held(a, at, block0 + b, step, m, v, IntTag<BITS>{});
  }
}

int64_t blocks_of(int64_t size) { return (size + kBlock - 1) / kBlock; }

int state_blocks(int n, const int64_t* sizes, int state_bits, size_t* blocks) {
  if (n < 0 || (n > 0 && !sizes)) return fail(MGPT_ERR_INVALID_ARGUMENT, "negative num_tensors or null sizes");
  if (state_bits != 32 && state_bits != 8)
    return fail(MGPT_ERR_UNSUPPORTED, "state_bits %d: 32 or 8", state_bits);
  size_t nb = 0;
  for (int i = 0; i < n; ++i) {
    if (sizes[i] < 0 || sizes[i] > (int64_t)1 << 34)
      return fail(MGPT_ERR_INVALID_ARGUMENT, "tensor %d has %lld elements", i, (long long)sizes[i]);
    nb += (size_t)blocks_of(sizes[i]);
  }
  if (nb > 0xFFFFFFFFu) return fail(MGPT_ERR_UNSUPPORTED, "%zu state blocks exceed 2^32", nb);
  *blocks = nb;
  return MGPT_OK;
}

}  // namespace
}  // namespace mgpt

using namespace mgpt;

extern "C" {

int mgpt_adamw_state_bytes(int num_tensors, const int64_t* sizes, int state_bits, size_t* bytes) {
  if (!bytes) return fail(MGPT_ERR_INVALID_ARGUMENT, "null bytes");
  size_t nb = 0;
  if (int rc = state_blocks(num_tensors, sizes, state_bits, &nb)) return rc;
  *bytes = nb * kBlock * 2 * (state_bits / 8) + (state_bits == 8 ? 2 * nb : 0);
  return MGPT_OK;
}

int mgpt_adamw_step(const mgpt_adamw_config* cfg, int num_tensors, const int64_t* sizes,
                    float* const* params, const void* const* grads, void* const* copies, void* state,
                    size_t state_bytes, int step, const int32_t* step_device, const float* grad_scale,
                    void* stream) {
  if (!cfg) return fail(MGPT_ERR_INVALID_ARGUMENT, "config is null");
  if (!(cfg->beta1 >= 0.0f && cfg->beta1 < 1.0f && cfg->beta2 >= 0.0f && cfg->beta2 < 1.0f))
    return fail(MGPT_ERR_INVALID_ARGUMENT, "betas must be in [0, 1)");
  if (!(cfg->eps >= 0.0f) || !std::isfinite(cfg->lr) || !std::isfinite(cfg->weight_decay))
    return fail(MGPT_ERR_INVALID_ARGUMENT, "eps must be >= 0, lr and weight_decay finite");
  if (cfg->grad_dtype != MGPT_DTYPE_F32 && cfg->grad_dtype != MGPT_DTYPE_BF16)
    return fail(MGPT_ERR_UNSUPPORTED, "unsupported gradient dtype %d", cfg->grad_dtype);
  size_t nb = 0, need = 0;
  if (int rc = state_blocks(num_tensors, sizes, cfg->state_bits, &nb)) return rc;
  if (nb == 0) return MGPT_OK;
  if (!params || !grads || !state) return fail(MGPT_ERR_INVALID_ARGUMENT, "null params, grads or state");
  if (!step_device && step < 1) return fail(MGPT_ERR_INVALID_ARGUMENT, "step %d: the first step is 1", step);
  (void)mgpt_adamw_state_bytes(num_tensors, sizes, cfg->state_bits, &need);
  if (state_bytes < need)
    return fail(MGPT_ERR_WORKSPACE_TOO_SMALL, "state needs %zu bytes, got %zu", need, state_bytes);
  const uintptr_t galign = cfg->grad_dtype == MGPT_DTYPE_F32 ? 3 : 1;
  if ((uintptr_t)state & 15) return fail(MGPT_ERR_INVALID_ARGUMENT, "state must be 16-byte aligned");
  for (int i = 0; i < num_tensors; ++i) {
    if (sizes[i] == 0 || !grads[i]) continue;
    if (!params[i]) return fail(MGPT_ERR_INVALID_ARGUMENT, "params[%d] is null", i);
    if (((uintptr_t)params[i] & 3) || ((uintptr_t)grads[i] & galign) || (copies && ((uintptr_t)copies[i] & 1)))
      return fail(MGPT_ERR_INVALID_ARGUMENT, "tensor %d is not aligned to its elements", i);
  }
  AdamwArgs a{};
  a.lr = cfg->lr;
  a.b1 = cfg->beta1;
  a.b2 = cfg->beta2;
  a.a1 = 1.0f - a.b1;
  a.a2 = 1.0f - a.b2;
  a.eps = cfg->eps;
  a.shrink = cfg->lr * cfg->weight_decay;
  a.step = (uint32_t)(step < 1 ? 1 : step);
  a.c1 = bias_correction(a.b1, a.step);
  a.c2 = bias_correction(a.b2, a.step);
  a.step_device = step_device;
  a.grad_scale = grad_scale;
  const size_t held = nb * kBlock * (cfg->state_bits / 8);
  a.m = (char*)state;
  a.v = a.m + held;
  a.me = (uint8_t*)(a.v + held);
  a.ve = a.me + nb;
  AdamwTensors ts;
  ts.n = 0;
  uint64_t tiles = 0;
  auto flush = [&]() -> hipError_t {
    if (ts.n == 0) return hipSuccess;
    auto go = [&](auto kernel) {
      ts.tile0[ts.n] = (uint32_t)tiles;
      hipLaunchKernelGGL(kernel, dim3((unsigned)tiles), dim3(256), 0, (hipStream_t)stream, ts, a);
    };
    const bool f32 = cfg->grad_dtype == MGPT_DTYPE_F32;
    if (cfg->state_bits == 32) {
      if (f32) go(adamw_kernel<32, float>);
      else go(adamw_kernel<32, bf16_t>);
    } else {
      if (f32) go(adamw_kernel<8, float>);
      else go(adamw_kernel<8, bf16_t>);
    }
    ts.n = 0;
    tiles = 0;
    return hipGetLastError();
  };
  size_t block = 0;
  for (int i = 0; i < num_tensors; ++i) {
    const int64_t size = sizes[i];
    if (size > 0 && grads[i]) {
      const uint64_t t = (uint64_t)((size + kTile - 1) / kTile);
      if (ts.n == AdamwTensors::kMax || tiles + t > kMaxTiles) HIP_TRY(flush());
      ts.p[ts.n] = params[i];
      ts.g[ts.n] = grads[i];
      ts.copy[ts.n] = copies ? (bf16_t*)copies[i] : nullptr;
      ts.tail[ts.n] = (uint16_t)(size - (int64_t)(t - 1) * kTile);
      ts.block0[ts.n] = (uint32_t)block;
      ts.tile0[ts.n] = (uint32_t)tiles;
      ++ts.n;
      tiles += t;
    }
    block += (size_t)blocks_of(size);
  }
  HIP_TRY(flush());
  return MGPT_OK;
}

}  // extern "C"
