// Float32 products on the 16-bit matrix cores, and operands read down the
// columns of LDS (mlp8.hip, rows8.hip).
//
// Products of float32 factors on the 16-bit matrix cores (a 32 x 32 x 16
// instruction takes 32 cycles, eight float32 ones of 32 x 32 x 2 take 512): a
// factor is split into three bfloat16 pieces, which hold its 24 bits at
// float32's range, and the six largest products of pieces are summed in float32
// (the other three are at most 2^-26 of |a b| together).  A value's pieces depend on nothing else, so
// each product is as exact whatever stands beside it in its row or matrix.
// (Two float16 halves and three products are faster, but halves need a power of
// two shared by a row or matrix: what is 2^-18 of the largest value there loses
// bits, what is 2^-40 of it vanishes.)  Factors below 2^-110 lose their last
// pieces to bfloat16's subnormal numbers.  A code is exact in bfloat16, so its
// products need one factor split and three products.  A factor that is not
// finite makes its products NaN.
//
// The sums of these instructions are rounded toward minus infinity (measured:
// the errors of sums of either sign are negative), which long sums over rows
// that cancel add up: 2^20 rows of 83 -> 128 -> 19, db1 6.5e-6 off.  Where
// gradients are summed in chunks of rows, every second chunk is computed with
// the upstream's sign changed, and the chunks' errors cancel.
#pragma once

#include "sphops_internal.hpp"
#include "sphops_device.hpp"

namespace sphops {

namespace {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef float f32x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

__device__ __forceinline__ f32x16 mma(bf16x8 a, bf16x8 b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}

struct Thirds {
  bf16x8 v[3];
};
// Two values at a time: a pair's pieces back in float32 are its word's halves.
__device__ __forceinline__ uint32_t bf16_pair(float& a, float& b) {
  typedef float f32x2 __attribute__((ext_vector_type(2)));
  typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
  const uint32_t w = __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2{a, b}), bf16x2));
  a -= __builtin_bit_cast(float, w << 16);
  b -= __builtin_bit_cast(float, w & 0xffff0000u);
  return w;
}
// The first piece at most the largest bfloat16, past which float32's largest
// values (from 3.396e38 on) would round up to infinity.
__device__ __forceinline__ uint32_t bf16_pair_top(float& a, float& b) {
  constexpr float kTop = 0x1.fep127f;
  float p = __builtin_amdgcn_fmed3f(a, -kTop, kTop), q = __builtin_amdgcn_fmed3f(b, -kTop, kTop);
  const uint32_t w = bf16_pair(p, q);
  a -= __builtin_bit_cast(float, w << 16);
  b -= __builtin_bit_cast(float, w & 0xffff0000u);
  return w;
}
// TOP: values may be that large.
template <bool TOP = true>
__device__ __forceinline__ Thirds split3(f32x8 v) {
  Thirds r;
#pragma unroll
  for (int i = 0; i < 3; ++i) {
    u32x4 w;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      float x = v[2 * j], y = v[2 * j + 1];
      w[j] = TOP && i == 0 ? bf16_pair_top(x, y) : bf16_pair(x, y);
      v[2 * j] = x;
      v[2 * j + 1] = y;
    }
    r.v[i] = __builtin_bit_cast(bf16x8, w);
  }
  return r;
}
__device__ __forceinline__ f32x16 mma(const Thirds& a, const Thirds& b, f32x16 c) {
  c = mma(a.v[1], b.v[1], mma(a.v[2], b.v[0], mma(a.v[0], b.v[2], c)));
  return mma(a.v[0], b.v[0], mma(a.v[1], b.v[0], mma(a.v[0], b.v[1], c)));
}

// The same with the product of the first pieces in a sum of its own: it is
// rounded once a step at the sum's size, not six times.
__device__ __forceinline__ void mma(const Thirds& a, const Thirds& b, f32x16& c, f32x16& low) {
  low = mma(a.v[1], b.v[1], mma(a.v[2], b.v[0], mma(a.v[0], b.v[2], low)));
  low = mma(a.v[1], b.v[0], mma(a.v[0], b.v[1], low));
  c = mma(a.v[0], b.v[0], c);
}

// Four codes, which bfloat16 holds exactly.
__device__ __forceinline__ bf16x4 codes_bf16(uint32_t w) {
  const uint32_t u = w ^ 0x80808080u;
  f32x4 v = {(float)(u & 0xffu), (float)((u >> 8) & 0xffu), (float)((u >> 16) & 0xffu), (float)(u >> 24)};
  return __builtin_convertvector(v - 128.0f, bf16x4);
}

// Four 16-bit values down a column: of each 16 lanes, lane i gives the address
// of four values of row i / 4 of a block of 4 rows by 16 columns, columns 4 (i %
// 4) .. + 3, and receives column i.  (A plain LDS read moves rows.)
__device__ __forceinline__ s16x4 read_column(const void* p) {
  return __builtin_amdgcn_ds_read_tr16_b64_v4i16(
      (__attribute__((address_space(3))) s16x4*)const_cast<void*>(p));
}
__device__ __forceinline__ s16x8 join(s16x4 a, s16x4 b) {
  return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
}

}  // namespace

}  // namespace sphops
