// Operand images of the MLP's weights as three bfloat16 pieces a value, and rows
// in and out of the products with them (mlp8.hip, expert_mlp.hip).
#pragma once

#include "mlp_tiles.hpp"
#include "split16.hpp"

namespace sphops {

namespace {

__device__ __forceinline__ __amdgpu_buffer_rsrc_t bytes_rsrc(const int8_t* base, int64_t bytes) {
  return rows_rsrc(reinterpret_cast<const float*>(base), bytes);
}

// Eight values of a row of n from column k (zeros past it), through a resource
// over all rows.
__device__ __forceinline__ f32x8 load8(__amdgpu_buffer_rsrc_t r, int row, int n, int k) {
  const uint32_t at = (uint32_t)(row * n + k) * 4u;
  f32x8 v = __builtin_shufflevector(load4(r, at), load4(r, at + 16u), 0, 1, 2, 3, 4, 5, 6, 7);
#pragma unroll
  for (int j = 0; j < 8; ++j) v[j] = k + j < n ? v[j] : 0.0f;  // the next row's
  return v;
}

// Result columns 32 t + lane % 32 of a tile whose registers are rows 8 (r / 4) +
// 4 (lane / 32) + r % 4: a store writes two runs of 128 bytes.  The empty asm
// keeps the 16 offsets of every tile from being held all along.
__device__ __forceinline__ void store_columns(__amdgpu_buffer_rsrc_t r, int width, int col, int h, f32x16 v) {
  uint32_t line = (uint32_t)width * 4u;
  asm volatile("" : "+s"(line));
  const uint32_t at = col < width ? 4u * (uint32_t)h * line + 4u * (uint32_t)col : kPast;
#pragma unroll
  for (int i = 0; i < 16; ++i) store1(r, at + (uint32_t)(8 * (i / 4) + i % 4) * line, v[i]);
}

// The columns that a lane of half h holds of step s of a product over a row: two
// steps take 16 neighbouring ones, so that a lane's loads of a row are whole
// 64-byte pieces.
__device__ __forceinline__ constexpr int step_column(int s, int h) { return 32 * (s / 2) + 16 * h + 8 * (s % 2); }

// W1 in pieces as an operand image: lane l's 16 bytes of entry (s, t), at
// image_lane(s, l), are W1[32 t + l % 32][step_column(s, l / 32) .. + 7].  All
// threads; the caller's barrier ends it.
//
// image_lane exchanges hidden rows so that the 32 lanes of half a column read
// (read_column: 4 rows by 32 columns, 8 bytes a lane) lie in different banks;
// as the rows stand, four of them meet in each.
__device__ __forceinline__ int image_lane(int s, int l) { return l ^ ((l >> 5) << 3) ^ ((s & 1) << 2); }

template <int KS, int kThreads>
__device__ __forceinline__ void w1_image(const float* __restrict__ w1, int nin, bf16x8 (&image)[3][KS][kHT][64]) {
  constexpr int kEntries = KS * kHT * 64, kOwn = (kEntries + kThreads - 1) / kThreads;
  const __amdgpu_buffer_rsrc_t r = rows_rsrc(w1, kHid * nin * 4);
  f32x8 v[kOwn];
#pragma unroll
  for (int u = 0; u < kOwn; ++u) {
    const int i = u * kThreads + (int)threadIdx.x, l = i & 63, t = (i >> 6) % kHT, s = (i >> 6) / kHT;
    v[u] = f32x8{};
    if (i < kEntries) v[u] = load8(r, kT * t + (l & 31), nin, step_column(s, l >> 5));
  }
#pragma unroll
  for (int u = 0; u < kOwn; ++u) {
    const int i = u * kThreads + (int)threadIdx.x, l = i & 63, t = (i >> 6) % kHT, s = (i >> 6) / kHT;
    if (i >= kEntries) continue;
    const Thirds x = split3(v[u]);
#pragma unroll
    for (int p = 0; p < 3; ++p) image[p][s][t][image_lane(s, l)] = x.v[p];
  }
}

// Steps of 16 columns of an input of up to 32 CT: of the widest, 168, the
// twelfth step's columns are all past the end.
constexpr int image_steps(int ct) { return 32 * ct > kMaxMlpIn + 23 ? 2 * ct - 1 : 2 * ct; }
static_assert(step_column(11, 0) >= kMaxMlpIn && image_steps(6) == 11 && image_steps(5) == 10, "nothing left out");

// Pieces of W2 that stand in LDS beside W1's image (12 KB a step; W2 24 KB a
// tile of outputs): all three, or the first one, and every wave keeps the other
// two in registers.
constexpr int lds_pieces(int ct, int ot) { return 12288 * image_steps(ct) + 24576 * ot + 2048 <= 163840 ? 3 : 1; }

constexpr int kMaxKS = (kMaxMlpIn + 15) / 16, kMaxOS = kMaxMlpOut / 16, kMaxCT = (kMaxMlpIn + kT - 1) / kT;

}  // namespace

}  // namespace sphops
