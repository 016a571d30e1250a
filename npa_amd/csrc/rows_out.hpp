// Rows in and out of a wave's registers (norm.hip, experts.hip).
#pragma once

#include "rows8.hpp"

namespace sphops {

namespace {

// Values k .. of a row, the caller's word that they are whole; else as far as it reaches.
template <class T>
__device__ __forceinline__ void load_piece(Piece<T>& p, bool whole, const T* __restrict__ row, int k, int cols) {
  if (whole) p.raw = *reinterpret_cast<const typename Piece<T>::Raw*>(row + k);
  else if (k < cols) p.load(row, k, cols);
  else p.raw = typename Piece<T>::Raw{};
}

// A wave's rows on their way out, which stand one after another in memory: short
// ones (up to 16 lanes each) go through LDS of the wave's own and leave in whole
// runs of 1024 bytes, whatever the row's length.
template <class T, int L, int N>
struct RowsOut {
  static constexpr bool kStaged = L <= 16;
  static constexpr int V = Piece<T>::V;
  uint32_t words[kStaged ? N * 256 : 1];
  // o: the lane's pieces of row `first` + lane / L of y; rows from `rows` on are not written
  __device__ __forceinline__ void operator()(const Piece<T> (&o)[N], T* __restrict__ y, int64_t first, int64_t rows,
                                             int cols) {
    const int lane = threadIdx.x & 63, l = threadIdx.x % L;
    if (kStaged && (sizeof(T) == 4 || cols % 2 == 0)) {  // words of LDS stay whole
      T* const own = reinterpret_cast<T*>(words);
      __builtin_amdgcn_wave_barrier();
#pragma unroll
      for (int n = 0; n < N; ++n) {
        const int k = (n * L + l) * V, at = ((lane / L) * cols + k) * (int)sizeof(T) / 4;
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (n < N - 1 || k + j * V / 4 < cols) words[at + j] = o[n].raw.w[j];
      }
      __builtin_amdgcn_wave_barrier();
      const int64_t left = rows - first;
      const int all = (int)(left < 0 ? 0 : left < 64 / L ? left : 64 / L) * cols;
      T* const to = y + first * cols;
#pragma unroll
      for (int n = 0; n < N; ++n) {
        const int k = (n * 64 + lane) * V;
        if (k >= all) continue;
        Piece<T> p;
        __builtin_memcpy(&p.raw, own + k, 16);
        p.store(to, k, all);
      }
    } else {
      const int64_t r = first + lane / L;
#pragma unroll
      for (int n = 0; n < N; ++n) {
        const int k = (n * L + l) * V;
        if (r >= rows) continue;
        if (n < N - 1) *reinterpret_cast<typename Piece<T>::Raw*>(y + r * cols + k) = o[n].raw;
        else if (k < cols) o[n].store(y + r * cols, k, cols);
      }
    }
  }
};

}  // namespace

}  // namespace sphops
