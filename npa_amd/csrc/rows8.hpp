// Rows in 8 bits: one float32 scale and one int8 code a value (see rows8.hip).
#pragma once

#include "sphops_internal.hpp"
#include "sphops_device.hpp"

#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>

#include <type_traits>

namespace sphops {

// Rows whose largest value is smaller are held against this one: 127 / m and
// m / 127 stay normal numbers, and a row of zeros needs no case of its own.
constexpr float kRowFloor = 0x1p-100f;

struct RowScale {
  float inv;    // 127 / m: code = rint(x * inv)
  float scale;  // m / 127: value = code * scale; NaN for a row that is not finite
  bool finite;
};

// From the largest |x| of a row as the bits of the float: as unsigned integers
// they order like the values, with infinity and then NaN above all of them, so
// a maximum of bits keeps what a maximum of floats may drop.
__device__ __forceinline__ RowScale row_scale(uint32_t max_bits) {
#pragma clang fp contract(off)
  RowScale r;
  r.finite = max_bits < 0x7f800000u;
  const float m = fmaxf(__builtin_bit_cast(float, r.finite ? max_bits : 0u), kRowFloor);
  r.inv = r.finite ? 127.0f / m : 0.0f;
  r.scale = r.finite ? m / 127.0f : __builtin_nanf("");
  return r;
}

__device__ __forceinline__ uint32_t abs_bits(float v) { return __builtin_bit_cast(uint32_t, v) & 0x7fffffffu; }

// A code in the low byte of a word: added to 1.5 * 2^23, whose last place is 1,
// the product is rounded to the nearest whole number, ties to the even one, and
// stands in the low bits.  Codes of finite rows lie in [-127, 127]: |x| * fl(127
// / m) < 127.5.
__device__ __forceinline__ uint32_t row_code(float v, float inv) {
#pragma clang fp contract(off)
  const float p = v * inv;
  return __builtin_bit_cast(uint32_t, p + 12582912.0f);
}

// The low bytes of four words, first value lowest.
__device__ __forceinline__ uint32_t pack4(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  return __builtin_amdgcn_perm(__builtin_amdgcn_perm(d, c, 0x0c0c0400u), __builtin_amdgcn_perm(b, a, 0x0c0c0400u),
                               0x05040100u);
}

// Four codes of a row: zeros in a row that is not finite.
__device__ __forceinline__ uint32_t row_codes4(float a, float b, float c, float d, const RowScale& q) {
  const uint32_t w = pack4(row_code(a, q.inv), row_code(b, q.inv), row_code(c, q.inv), row_code(d, q.inv));
  return q.finite ? w : 0u;
}

// code * scale.  127 times m / 127 rounds past float32's largest number for that
// one m alone, which stands in masks: it stays that number.
__device__ __forceinline__ float row_value(int code, float scale) {
  const float v = (float)code * scale;
  return fabsf(v) > 0x1.fffffep127f ? copysignf(0x1.fffffep127f, v) : v;  // NaN stays
}

// Element types of the rows (SPHOPS_F32, SPHOPS_BF16, SPHOPS_F16).
__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__hip_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
template <class T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ __hip_bfloat16 from_f32<__hip_bfloat16>(float v) { return __float2bfloat16(v); }
// The empty asm keeps a product before it a float: the compiler else takes both
// in one mixed-precision instruction, which rounds once where the definition
// rounds to float32 first.
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) {
  asm("" : "+v"(v));
  return __float2half(v);
}

// 16 bytes of a row: V values, at any alignment a row can start at.
template <class T>
struct Piece {
  static constexpr int V = 16 / sizeof(T);
  struct __attribute__((packed, aligned(alignof(T)))) Raw {
    uint32_t w[4];
  };
  Raw raw;
  __device__ __forceinline__ float get(int j) const {
    if constexpr (sizeof(T) == 4) return __builtin_bit_cast(float, raw.w[j]);
    else return to_f32(__builtin_bit_cast(T, (uint16_t)(raw.w[j / 2] >> (16 * (j % 2)))));
  }
  __device__ __forceinline__ void set(int j, T v) {
    if constexpr (sizeof(T) == 4) raw.w[j] = __builtin_bit_cast(uint32_t, v);
    else raw.w[j / 2] = (raw.w[j / 2] & (0xffffu << (16 - 16 * (j % 2)))) |
                        ((uint32_t)__builtin_bit_cast(uint16_t, v) << (16 * (j % 2)));
  }
  // values k .. k + V - 1 of a row of `cols`, zeros past it
  __device__ __forceinline__ void load(const T* __restrict__ row, int k, int cols) {
    if (k + V <= cols) {
      raw = *reinterpret_cast<const Raw*>(row + k);
    } else {
      raw = Raw{};
#pragma unroll
      for (int j = 0; j < V; ++j)
        if (k + j < cols) set(j, row[k + j]);
    }
  }
  __device__ __forceinline__ void store(T* __restrict__ row, int k, int cols) const {
    if (k + V <= cols) {
      *reinterpret_cast<Raw*>(row + k) = raw;
    } else {
#pragma unroll
      for (int j = 0; j < V; ++j) {
        if (k + j < cols) {
          if constexpr (sizeof(T) == 4) row[k + j] = __builtin_bit_cast(T, raw.w[j]);
          else row[k + j] = __builtin_bit_cast(T, (uint16_t)(raw.w[j / 2] >> (16 * (j % 2))));
        }
      }
    }
  }
};

// Floats as a piece, each rounded once to the nearest, two at a time.
template <class T>
__device__ __forceinline__ Piece<T> piece_of(const float (&v)[Piece<T>::V]) {
  Piece<T> p;
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int j = 0; j < 4; ++j) p.raw.w[j] = __builtin_bit_cast(uint32_t, v[j]);
  } else {
    using E = std::conditional_t<std::is_same_v<T, __half>, _Float16, __bf16>;
    typedef float f32x2 __attribute__((ext_vector_type(2)));
    typedef E e16x2 __attribute__((ext_vector_type(2)));
#pragma unroll
    for (int j = 0; j < 4; ++j)
      p.raw.w[j] = __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2{v[2 * j], v[2 * j + 1]}), e16x2));
  }
  return p;
}

template <bool RELU>
__device__ __forceinline__ uint32_t top_of(uint32_t top, float v) {
  return RELU && v <= 0.0f ? top : max(top, abs_bits(v));
}

// One value of an integer layer: each step rounds by itself, so every kernel
// gives the same bits, whatever its tiles.
__device__ __forceinline__ float linear8_value(int sum, float row_scale, float channel_scale, float bias) {
#pragma clang fp contract(off)
  const float unit = row_scale * channel_scale;
  const float v = (float)sum * unit;
  return v + bias;
}

// f(T{}) for a type code; the caller has checked the code.
template <class F>
void with_type(int type, F&& f) {
  if (type == SPHOPS_F32) f(float{});
  else if (type == SPHOPS_BF16) f(__hip_bfloat16{});
  else f(__half{});
}

}  // namespace sphops
