// Rows in 8 bits, for gfx950: activations kept between forward and backward,
// and the operands of the integer products (linear8.hip, mlp8.hip).
//
//   m = max(max |x|, 2^-100)    scale = m / 127
//   code = rint(x * (127 / m))  value = code * scale
//
// in float32 steps, ties to the even code.  A row that holds a NaN or an
// infinity has a NaN scale and zero codes: whatever is computed from it is NaN.
#include "rows8.hpp"

#include <type_traits>

namespace sphops {

namespace {

constexpr int kRowThreads = 256;

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

template <bool RELU>
__device__ __forceinline__ uint32_t top_of(uint32_t top, float v) {
  return RELU && v <= 0.0f ? top : max(top, abs_bits(v));
}

// The codes of one piece, written up to ld (a multiple of 4).
template <class T, bool RELU>
__device__ __forceinline__ void write_codes(int8_t* __restrict__ row, const Piece<T>& p, int k, int ld,
                                            const RowScale& q) {
#pragma unroll
  for (int i = 0; i < Piece<T>::V / 4; ++i) {
    if (k + 4 * i >= ld) continue;
    uint32_t w;
    if constexpr (RELU) {
      uint32_t c[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float v = p.get(4 * i + j);
        c[j] = v > 0.0f ? max(1u, row_code(v, q.inv) & 0xffu) : 0u;
      }
      w = q.finite ? pack4(c[0], c[1], c[2], c[3]) : 0u;
    } else {
      w = row_codes4(p.get(4 * i), p.get(4 * i + 1), p.get(4 * i + 2), p.get(4 * i + 3), q);
    }
    *reinterpret_cast<uint32_t*>(row + k + 4 * i) = w;
  }
}

// L lanes a row, which they hold in N pieces each: the row is read once.  With
// RELU the row kept is relu(x), and no positive value has the code 0: a code is
// positive exactly where x is.  L = 256: the workgroup's four waves share a
// row.
template <class T, bool RELU, int L, int N>
__global__ __launch_bounds__(kRowThreads) void k_quantize_rows(const T* __restrict__ x, int64_t stride,
                                                               int8_t* __restrict__ codes, int64_t ld,
                                                               float* __restrict__ scale, int64_t rows, int cols) {
  constexpr int V = Piece<T>::V, kRows = kRowThreads / L;
  __shared__ uint32_t tops[2][4];
  const int l = threadIdx.x % L;
  int turn = 0;
  for (int64_t r0 = (int64_t)blockIdx.x * kRows; r0 < rows; r0 += (int64_t)gridDim.x * kRows, turn ^= 1) {
    const int64_t r = min<int64_t>(r0 + threadIdx.x / L, rows - 1);  // lanes past the last row do it again
    const T* __restrict__ row = x + r * stride;
    Piece<T> p[N];
#pragma unroll
    for (int n = 0; n < N; ++n) p[n].load(row, (n * L + l) * V, cols);
    uint32_t top = 0;
#pragma unroll
    for (int n = 0; n < N; ++n) {
#pragma unroll
      for (int j = 0; j < V; ++j) top = top_of<RELU>(top, p[n].get(j));
    }
#pragma unroll
    for (int s = 1; s < (L < 64 ? L : 64); s *= 2) top = max(top, (uint32_t)__shfl_xor((int)top, s));
    if constexpr (L > 64) {
      // two sets in turn: a wave writes a set again only after the other turn's barrier
      if (threadIdx.x % 64 == 0) tops[turn][threadIdx.x / 64] = top;
      __syncthreads();
      top = max(max(tops[turn][0], tops[turn][1]), max(tops[turn][2], tops[turn][3]));
    }
    const RowScale q = row_scale(top);
#pragma unroll
    for (int n = 0; n < N; ++n) write_codes<T, RELU>(codes + r * ld, p[n], (n * L + l) * V, (int)ld, q);
    if (l == 0) scale[r] = q.scale;
    // padding past the pieces (ld up to the next multiple of a wide alignment)
    for (int k = (N * L * V) + 4 * l; k < (int)ld; k += 4 * L) *reinterpret_cast<uint32_t*>(codes + r * ld + k) = 0;
  }
}

// Rows of any length: a workgroup a row, which is read twice (the second time
// from cache).
template <class T, bool RELU>
__global__ __launch_bounds__(kRowThreads) void k_quantize_long_rows(const T* __restrict__ x, int64_t stride,
                                                                    int8_t* __restrict__ codes, int64_t ld,
                                                                    float* __restrict__ scale, int64_t rows,
                                                                    int cols) {
  constexpr int V = Piece<T>::V;
  __shared__ uint32_t tops[2][4];
  int turn = 0;
  for (int64_t r = blockIdx.x; r < rows; r += gridDim.x, turn ^= 1) {
    const T* __restrict__ row = x + r * stride;
    uint32_t top = 0;
    for (int k = threadIdx.x * V; k < cols; k += kRowThreads * V) {
      Piece<T> p;
      p.load(row, k, cols);
#pragma unroll
      for (int j = 0; j < V; ++j) top = top_of<RELU>(top, p.get(j));
    }
#pragma unroll
    for (int s = 1; s < 64; s *= 2) top = max(top, (uint32_t)__shfl_xor((int)top, s));
    if (threadIdx.x % 64 == 0) tops[turn][threadIdx.x / 64] = top;
    __syncthreads();
    top = max(max(tops[turn][0], tops[turn][1]), max(tops[turn][2], tops[turn][3]));
    const RowScale q = row_scale(top);
    for (int k = threadIdx.x * V; k < (int)ld; k += kRowThreads * V) {
      Piece<T> p;
      p.load(row, k, cols);
      write_codes<T, RELU>(codes + r * ld, p, k, (int)ld, q);
    }
    if (threadIdx.x == 0) scale[r] = q.scale;
  }
}

// L lanes a row (256 / L rows a workgroup's turn), 16 bytes of the result a lane.
template <class T, int L>
__global__ __launch_bounds__(kRowThreads) void k_restore_rows(const int8_t* __restrict__ codes, int64_t ld,
                                                              const float* __restrict__ scale, T* __restrict__ out,
                                                              int64_t rows, int cols) {
  constexpr int V = Piece<T>::V, kRows = kRowThreads / L;
  const int l = threadIdx.x % L;
  for (int64_t r = (int64_t)blockIdx.x * kRows + threadIdx.x / L; r < rows; r += (int64_t)gridDim.x * kRows) {
    const float s = scale[r];
    const int8_t* __restrict__ row = codes + r * ld;
    for (int k = l * V; k < cols; k += L * V) {
      Piece<T> p;
#pragma unroll
      for (int i = 0; i < V / 4; ++i) {
        const uint32_t w = k + 4 * i < (int)ld ? *reinterpret_cast<const uint32_t*>(row + k + 4 * i) : 0;
#pragma unroll
        for (int j = 0; j < 4; ++j) p.set(4 * i + j, from_f32<T>((float)(int8_t)(w >> (8 * j)) * s));
      }
      p.store(out + r * cols, k, cols);
    }
  }
}

dim3 row_grid(int64_t rows, int rows_a_turn) {
  return dim3((uint32_t)std::min<int64_t>((rows + rows_a_turn - 1) / rows_a_turn, 16384));
}

// f(integral_constant L, integral_constant N) for rows of `pieces` 16-byte pieces; false: longer than all of them
template <class F>
bool with_lanes(int64_t pieces, F&& f) {
  auto at = [&](auto l, auto n) {
    if (pieces > decltype(l)::value * decltype(n)::value) return false;
    f(l, n);
    return true;
  };
#define SPHOPS_LANES(L, N) at(std::integral_constant<int, L>{}, std::integral_constant<int, N>{})
  return SPHOPS_LANES(4, 1) || SPHOPS_LANES(8, 1) || SPHOPS_LANES(8, 2) || SPHOPS_LANES(8, 3) ||
         SPHOPS_LANES(16, 2) || SPHOPS_LANES(16, 3) || SPHOPS_LANES(16, 4) || SPHOPS_LANES(32, 3) ||
         SPHOPS_LANES(32, 4) || SPHOPS_LANES(64, 3) || SPHOPS_LANES(64, 4) || SPHOPS_LANES(64, 6) ||
         SPHOPS_LANES(64, 8) || SPHOPS_LANES(64, 12) || SPHOPS_LANES(256, 4) || SPHOPS_LANES(256, 8);
#undef SPHOPS_LANES
}

template <class T, bool RELU>
void launch_quantize(const T* x, int64_t stride, int8_t* codes, int64_t ld, float* scale, int64_t rows, int cols,
                     hipStream_t st) {
  const int64_t pieces = (cols + Piece<T>::V - 1) / Piece<T>::V;
  const bool held = with_lanes(pieces, [&](auto l, auto n) {
    constexpr int L = decltype(l)::value;
    hipLaunchKernelGGL((k_quantize_rows<T, RELU, L, decltype(n)::value>), row_grid(rows, kRowThreads / L),
                       dim3(kRowThreads), 0, st, x, stride, codes, ld, scale, rows, cols);
  });
  if (!held)
    hipLaunchKernelGGL((k_quantize_long_rows<T, RELU>), row_grid(rows, 1), dim3(kRowThreads), 0, st, x, stride, codes,
                       ld, scale, rows, cols);
}

}  // namespace

void run_quantize_rows(const void* x, int type, int64_t stride, int8_t* codes, int64_t ld, float* scale, int64_t rows,
                       int64_t cols, bool relu, hipStream_t st) {
  if (rows == 0) return;
  with_type(type, [&](auto t) {
    using T = decltype(t);
    if (relu) launch_quantize<T, true>(static_cast<const T*>(x), stride, codes, ld, scale, rows, (int)cols, st);
    else launch_quantize<T, false>(static_cast<const T*>(x), stride, codes, ld, scale, rows, (int)cols, st);
  });
  SPHOPS_LAUNCHED();
}

void run_restore_rows(const int8_t* codes, int64_t ld, const float* scale, void* out, int type, int64_t rows,
                      int64_t cols, hipStream_t st) {
  if (rows == 0) return;
  with_type(type, [&](auto t) {
    using T = decltype(t);
    const int64_t pieces = (cols + Piece<T>::V - 1) / Piece<T>::V;
    auto launch = [&](auto l) {
      constexpr int L = decltype(l)::value;
      hipLaunchKernelGGL((k_restore_rows<T, L>), row_grid(rows, kRowThreads / L), dim3(kRowThreads), 0, st, codes, ld,
                         scale, static_cast<T*>(out), rows, (int)cols);
    };
    if (pieces <= 8) launch(std::integral_constant<int, 8>{});
    else if (pieces <= 16) launch(std::integral_constant<int, 16>{});
    else if (pieces <= 32) launch(std::integral_constant<int, 32>{});
    else if (pieces <= 256) launch(std::integral_constant<int, 64>{});
    else launch(std::integral_constant<int, 256>{});
  });
  SPHOPS_LAUNCHED();
}

// The rows again in 32 bits, then the weight gradient of linear_grad.hip.
int64_t rows8_weight_grad_floats(int64_t rows, int nin, int nout) {
  return rows * nin + linear_grad_chunks(rows, nin, nout) * ((int64_t)nin * nout + nout);
}

void run_rows8_weight_grad(const int8_t* codes, int64_t ld, const float* scale, const float* dy, float* dw, float* db,
                           int64_t rows, int nin, int nout, float* work, hipStream_t st) {
  run_restore_rows(codes, ld, scale, work, SPHOPS_F32, rows, nin, st);
  run_linear_weight_grad(work, dy, dw, db, rows, nin, nout, work + rows * nin, false, st);
}

}  // namespace sphops
