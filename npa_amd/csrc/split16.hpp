// Float32 products on the 16-bit matrix cores, and operands read down the
// columns of LDS (mlp8.hip, rows8.hip).
//
// Products of float32 factors on the 16-bit matrix cores (a 32 x 32 x 16
// instruction takes 32 cycles, eight float32 ones of 32 x 32 x 2 take 512):
// * a factor is scaled by a power of two and split into two halves, hi = v to
//   11 bits and lo = v - hi to 11 more, and a product is hi hi + hi lo + lo hi
//   with float32 sums (the splitting that H. Ootomo and R. Yokota published,
//   2022).  What it leaves out is at most 2^-22 of |a b|, and half the smallest
//   subnormal of a factor, 2^-40 of the largest value that shares its scale;
// * where no scale serves (sums over rows of any size) three bfloat16 pieces
//   hold all 24 bits at float32's range, and six products are taken;
// * a code is exact in either type, so its products need one factor split.
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
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef float f32x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

__device__ __forceinline__ f32x16 mma(f16x8 a, f16x8 b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x16 mma(bf16x8 a, bf16x8 b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}

// A power of two p with m p in [2^14, 2^15) for the largest magnitude m (as
// bits), kept where p and 1 / p are normal, and 1 / p.
struct Pow2 {
  float p, ip;
};
__device__ __forceinline__ Pow2 pow2_for(uint32_t max_bits) {
  const int e = min(268 - (int)(max_bits >> 23), 253);
  return {__builtin_bit_cast(float, (uint32_t)e << 23), __builtin_bit_cast(float, (uint32_t)(254 - e) << 23)};
}

struct Halves {
  f16x8 hi, lo;
};
__device__ __forceinline__ Halves split(f32x8 v) {
  Halves r;
  r.hi = __builtin_convertvector(v, f16x8);
  f32x8 rest;
  float minus = -1.0f;
  asm("" : "+v"(minus));  // keeps the subtraction one mixed-precision multiply-add
#pragma unroll
  for (int j = 0; j < 8; ++j) rest[j] = __builtin_fmaf((float)r.hi[j], minus, v[j]);
  r.lo = __builtin_convertvector(rest, f16x8);
  return r;
}
// + a b for factors in halves, the small products first
__device__ __forceinline__ f32x16 mma(const Halves& a, const Halves& b, f32x16 c) {
  return mma(a.hi, b.hi, mma(a.hi, b.lo, mma(a.lo, b.hi, c)));
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
__device__ __forceinline__ Thirds split3(f32x8 v) {
  Thirds r;
#pragma unroll
  for (int i = 0; i < 3; ++i) {
    u32x4 w;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      float x = v[2 * j], y = v[2 * j + 1];
      w[j] = bf16_pair(x, y);
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

// Eight codes as halves: as unsigned numbers code + 128 they are the low bits
// of the halves 1024 + code + 128.
__device__ __forceinline__ f16x8 codes_f16(u32x2 w) {
  u32x4 r;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const uint32_t u = w[i] ^ 0x80808080u;
    r[2 * i] = __builtin_amdgcn_perm(0x64646464u, u, 0x04010400u);
    r[2 * i + 1] = __builtin_amdgcn_perm(0x64646464u, u, 0x04030402u);
  }
  return __builtin_bit_cast(f16x8, r) - (_Float16)1152.0f;
}
__device__ __forceinline__ f16x4 codes_f16(uint32_t w) {
  const uint32_t u = w ^ 0x80808080u;
  const u32x2 r = {__builtin_amdgcn_perm(0x64646464u, u, 0x04010400u),
                   __builtin_amdgcn_perm(0x64646464u, u, 0x04030402u)};
  return __builtin_bit_cast(f16x4, r) - (_Float16)1152.0f;
}
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
