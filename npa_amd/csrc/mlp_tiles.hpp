// What the MLP kernels share (mlp_rows.hip, mlp8.hip): row tiles of 32 through
// range-checked buffer loads and stores, operand images in LDS, launch shapes.
#pragma once

#include "sphops_internal.hpp"
#include "sphops_device.hpp"

#include <type_traits>
#include <utility>

namespace sphops {

namespace {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

constexpr int kT = 32;            // matrix-core tile side
constexpr int kHid = kMlpHidden;  // 128
constexpr int kHT = kHid / kT;    // hidden tiles

// Buffer resource over `bytes` from base: loads past it return 0, stores past
// it are dropped; kPast is an offset past any of them.
constexpr uint32_t kPast = 0x80000000u;
__device__ __forceinline__ __amdgpu_buffer_rsrc_t rows_rsrc(const float* base, int64_t bytes) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<float*>(base), (short)0, (int)bytes, 0x00020000);
}
__device__ __forceinline__ float load1(__amdgpu_buffer_rsrc_t r, uint32_t off) {
  return __builtin_bit_cast(float, __builtin_amdgcn_raw_buffer_load_b32(r, off, 0, 0));
}
__device__ __forceinline__ f32x4 load4(__amdgpu_buffer_rsrc_t r, uint32_t off) {
  return __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(r, off, 0, 0));
}
__device__ __forceinline__ void store1(__amdgpu_buffer_rsrc_t r, uint32_t off, float v) {
  __builtin_amdgcn_raw_buffer_store_b32(__builtin_bit_cast(uint32_t, v), r, off, 0, 0);
}
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
__device__ __forceinline__ void store4(__amdgpu_buffer_rsrc_t r, uint32_t off, f32x4 v) {
  __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, v), r, off, 0, 0);
}

__device__ __forceinline__ f32x16 mma(float a, float b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x2f32(a, b, c, 0, 0, 0);
}

// relu as torch computes it: NaN stays NaN
__device__ __forceinline__ float relu(float v) { return v <= 0.0f ? 0.0f : v; }

// Four columns loaded `shift` before their place, moved up and zero-filled
// (4 or more: none of them exist).
__device__ __forceinline__ f32x4 move_up(f32x4 t, int shift) {
  if (shift & 1) t = f32x4{t[1], t[2], t[3], 0.0f};
  if (shift & 2) t = f32x4{t[2], t[3], 0.0f, 0.0f};
  if (shift >= 4) t = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  return t;
}

// A lane's share of row c of a row tile of `width` >= 4 columns, G = ceil(width
// / 8): columns 8 g + 4 h .. + 3 (h the lane's half) for each group g, in
// 16-byte loads (dword-aligned).  The last group's load is moved back to end
// with the row, so that it stays inside it, and its values moved up and
// zero-filled.
template <int G>
struct RowLoad {
  uint32_t off, off_last;  // bytes
  int shift;               // columns the last load was moved back by; 4 or more: none of them exist
  __device__ __forceinline__ RowLoad(int width, int c, int h) {
    const int k = 8 * (G - 1) + 4 * h, at = min(k, width - 4);
    off = (uint32_t)(c * width + 4 * h) * 4u;
    off_last = (uint32_t)(c * width + at) * 4u;
    shift = k - at;
  }
  __device__ __forceinline__ void load(__amdgpu_buffer_rsrc_t r, f32x4 (&v)[G]) const {
#pragma unroll
    for (int g = 0; g < G - 1; ++g) v[g] = load4(r, off + 32u * g);
    v[G - 1] = load4(r, off_last);
  }
  // after the loads, before the first use
  __device__ __forceinline__ void settle(f32x4 (&v)[G]) const { v[G - 1] = move_up(v[G - 1], shift); }
};

// Result columns of a transposed tile back to row c: registers 4 q .. 4 q + 3
// are columns col0 + 8 q + 4 h .. + 3.
__device__ __forceinline__ void store_row(__amdgpu_buffer_rsrc_t r, int width, int col0, int c, int h, f32x16 acc) {
  const uint32_t row = (uint32_t)(c * width);
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    const int k = col0 + 8 * q + 4 * h;
    const f32x4 v = {acc[4 * q], acc[4 * q + 1], acc[4 * q + 2], acc[4 * q + 3]};
    if (col0 + 8 * q + 8 <= width) {  // uniform
      store4(r, (row + (uint32_t)k) * 4u, v);
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) store1(r, k + j < width ? (row + (uint32_t)(k + j)) * 4u : kPast, v[j]);
    }
  }
}

// Fills an operand image of N entries (entry i = load(i)) by T threads, kBatch
// entries a thread in flight: a workgroup builds its images before its first
// row tile, and one entry at a time that took longer than the tiles of few
// rows (see k_mlp_forward and k_mlp_input_grad).
template <int N, int T, class Load>
__device__ __forceinline__ void build_image(f32x4* image, Load load) {
  constexpr int kBatch = 8;
#pragma unroll 1
  for (int i0 = 0; i0 < N; i0 += kBatch * T) {
    f32x4 v[kBatch];
#pragma unroll
    for (int u = 0; u < kBatch; ++u) v[u] = load(min(i0 + u * T + (int)threadIdx.x, N - 1));
#pragma unroll
    for (int u = 0; u < kBatch; ++u) {
      const int i = i0 + u * T + (int)threadIdx.x;
      if (i < N) image[i] = v[u];
    }
  }
}

// Workgroups of the tile kernels: two waves a SIMD over the 256 CUs (what
// registers allow), fewer for fewer tiles.
inline dim3 tile_grid(int64_t tiles, int threads) {
  const int waves = threads / 64;
  return dim3((uint32_t)std::min<int64_t>(2048 / waves, (tiles + waves - 1) / waves));
}

// f(integral_constant n) for a run-time 1 <= n <= N.
template <int N, class F>
void with_groups(int n, F&& f) {
  if constexpr (N > 1) {
    if (n < N) return with_groups<N - 1>(n, std::forward<F>(f));
  }
  f(std::integral_constant<int, N>{});
}

}  // namespace

}  // namespace sphops
