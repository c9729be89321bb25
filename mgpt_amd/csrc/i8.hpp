// i8.hpp -- products in 8-bit integers: the layout of their operands and what the
// kernels that make and multiply them (i8_quantize.hip, i8_gemm.hip) share with the
// layer (moe_capi.hip).
//
// Rows lie in tiles of 32 rows x 32 columns, 1 KB each, as v_mfma_i32_32x32x32_i8 takes an
// operand: lane l of a wave has columns 16 (l / 32) .. + 15 of row l % 32.  A row block (32 rows) is
// its tiles in the order of the columns, padded with zeros to whole slabs of 128; an operand is its row blocks.
// So a wave's load, to registers or to LDS, is 1 KB in a row, and a fragment in LDS needs no swizzle.
// Rows of several experts: each expert's begin a row block.
#pragma once

#include "common.hpp"

namespace mgpt {

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x16 __attribute__((ext_vector_type(16)));

constexpr int kI8Slab = 128;   // columns of a slab
constexpr int kI8Rows = 32;    // rows of a row block

__host__ __device__ inline size_t i8_row_block_bytes(int K) {
  return (size_t)((K + kI8Slab - 1) / kI8Slab) * kI8Slab * kI8Rows;
}

// Hidden units of a bf16 caller between the two products of an expert: 20 bits each, with a power of two for every 32:
// v 2^(e - 145), e the exponent byte (20 at least) of the largest magnitude of the 32, which is held as it was.  They are
// rounded to a step of max|h| / 127 of the whole row next, of which these bits are 2^-12 at most; in bf16 one value in
// eight would end a step off in the integers that follow (its rounding is 0.03 of their steps, rms), in 16 bits one in
// four hundred, here one in six thousand.  The largest magnitudes give a row's without its values.
struct HiddenRows {
  int16_t* q;      // [rows][ld]: v's upper 16 bits
  uint32_t* top;   // [rows][ld / 32]: |x|'s bits as fp32, infinity's or more: one of the 32 is not finite
  int ld;
  // [rows][ld / 2]: column 32 i + 16 b + 8 a + 4 h + c's lower bits in byte 16 i + 8 b + 4 h + c, its lower half where
  // a is 0 (a lane's accumulators and the quantiser's lane both have them in two words)
  uint8_t* n;
};

// Expert outputs of a bf16 caller between the down product and the combine: the upper 24 bits of the fp32 number, so
// that each is off by 2^-16 of itself at most, whatever its neighbours (outputs that share an exponent lose their bits
// beside a channel that is hundreds of times as large, as models have them), against the 2^-8 that y is rounded to.
struct Rows24 {
  uint16_t* hi;    // [rows][ld]
  uint8_t* low;    // [rows][ld]
  int ld;
};

// Rows to quantise.  Dense: rows 0 .. N - 1 of src.  By experts (counts): slot s of a segment is row
// perm[s] / k of src, or row s where perm is null.  rstd / gamma: (x rstd) gamma instead of x.
struct QuantizeArgs {
  const void* src;
  size_t ld;               // elements
  HiddenRows h;            // instead of src
  int N, K;
  const int32_t *counts, *perm;
  int E, k;
  const float *rstd, *gamma;
  int by_product;          // scales are max|x| (1 / 127), both factors of 32 bits, instead of the quotient
  char* q;                 // row blocks
  float* scale;            // [row blocks][32]
};
enum QuantizeSource { kRowsF32, kRowsBf16, kRowsHidden };
// max_blocks: of the row blocks there can be.
hipError_t launch_i8_quantize(QuantizeSource src, const QuantizeArgs& g, int max_blocks, hipStream_t st);
// q: [M][K] int8, row-major, as row blocks.
hipError_t launch_i8_tile(const int8_t* q, int M, int K, char* out, hipStream_t st);

// One product y = (A B^T) sa sb + bias, or by experts.
struct I8Args {
  const char* A;           // row blocks of the segments' rows
  const float* sa;         // [row blocks][32]
  const char* B;           // [E] row blocks of the outputs
  const float* sb;         // [E][ldsb]
  size_t b_expert;         // bytes of an expert's B
  int ldsb;
  int KT;                  // slabs
  int Nf;                  // outputs (gate/up: packed rows), of which the kernel stores only these
  int b_blocks;            // row blocks of an expert's B
  const float *bias0, *bias1;   // [E][bias_ld] or null (gate/up: of gate and up)
  int bias_ld;
  const int32_t* counts;   // rows of each expert, or null: one segment of N rows
  int E, N;                // N: rows in all
  void* out;               // [rows][ldo]
  size_t ldo;
  HiddenRows h;            // kI8GateUp: instead
  Rows24 o;                // kI8Rows24: instead
  int rowsfirst;           // set by the launcher: a lane has an output column
  int e_base;
};
enum I8Out { kI8F32, kI8Bf16, kI8GateUp, kI8Rows24, kI8GateUpF32 };
// kI8GateUp, kI8GateUpF32, kI8Rows24: Nf is a multiple of 64.
hipError_t launch_i8_gemm(I8Out kind, const I8Args& g, int num_cus, hipStream_t st);

}  // namespace mgpt
