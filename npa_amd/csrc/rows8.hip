// Rows in 8 bits, for gfx950: activations kept between forward and backward,
// and the operands of the integer products (linear8.hip, mlp8.hip).
//
//   m = max(max |x|, 2^-100)    scale = m / 127
//   code = rint(x * (127 / m))  value = code * scale
//
// in float32 steps, ties to the even code.  A row that holds a NaN or an
// infinity has a NaN scale and zero codes: whatever is computed from it is NaN.
#include "rows8.hpp"

namespace sphops {

namespace {

// One wave a row, the row read twice (the second time from cache).  With RELU
// the row is relu(x), and no positive value has the code 0: a code is positive
// exactly where x is.
template <class T, bool RELU>
__global__ __launch_bounds__(256) void k_quantize_rows(const T* __restrict__ x, int64_t stride,
                                                       int8_t* __restrict__ codes, int64_t ld,
                                                       float* __restrict__ scale, int64_t rows, int64_t cols) {
  const int lane = threadIdx.x & 63;
  for (int64_t r = (int64_t)blockIdx.x * 4 + threadIdx.x / 64; r < rows; r += (int64_t)gridDim.x * 4) {
    const T* __restrict__ row = x + r * stride;
    uint32_t top = 0;
    for (int64_t k = lane; k < cols; k += 64) {
      const float v = to_f32(row[k]);
      if (!RELU || !(v <= 0.0f)) top = max(top, abs_bits(v));
    }
#pragma unroll
    for (int s = 1; s < 64; s *= 2) top = max(top, (uint32_t)__shfl_xor((int)top, s));
    const RowScale q = row_scale(top);
    for (int64_t k = lane; k < ld; k += 64) {
      int c = 0;
      if (k < cols && q.finite) {
        const float v = to_f32(row[k]);
        c = RELU ? (v > 0.0f ? max(1, row_code(v, q.inv)) : 0) : row_code(v, q.inv);
      }
      codes[r * ld + k] = (int8_t)c;
    }
    if (lane == 0) scale[r] = q.scale;
  }
}

template <class T>
__global__ __launch_bounds__(256) void k_restore_rows(const int8_t* __restrict__ codes, int64_t ld,
                                                      const float* __restrict__ scale, T* __restrict__ out,
                                                      int64_t rows, int64_t cols) {
  const int lane = threadIdx.x & 63;
  for (int64_t r = (int64_t)blockIdx.x * 4 + threadIdx.x / 64; r < rows; r += (int64_t)gridDim.x * 4) {
    const float s = scale[r];
    for (int64_t k = lane; k < cols; k += 64) out[r * cols + k] = from_f32<T>((float)codes[r * ld + k] * s);
  }
}

dim3 row_grid(int64_t rows) { return dim3((uint32_t)std::min<int64_t>((rows + 3) / 4, 8192)); }

}  // namespace

void run_quantize_rows(const void* x, int type, int64_t stride, int8_t* codes, int64_t ld, float* scale, int64_t rows,
                       int64_t cols, bool relu, hipStream_t st) {
  if (rows == 0) return;
  with_type(type, [&](auto t) {
    using T = decltype(t);
    if (relu)
      hipLaunchKernelGGL((k_quantize_rows<T, true>), row_grid(rows), dim3(256), 0, st, static_cast<const T*>(x),
                         stride, codes, ld, scale, rows, cols);
    else
      hipLaunchKernelGGL((k_quantize_rows<T, false>), row_grid(rows), dim3(256), 0, st, static_cast<const T*>(x),
                         stride, codes, ld, scale, rows, cols);
  });
  SPHOPS_LAUNCHED();
}

void run_restore_rows(const int8_t* codes, int64_t ld, const float* scale, void* out, int type, int64_t rows,
                      int64_t cols, hipStream_t st) {
  if (rows == 0) return;
  with_type(type, [&](auto t) {
    using T = decltype(t);
    hipLaunchKernelGGL((k_restore_rows<T>), row_grid(rows), dim3(256), 0, st, codes, ld, scale, static_cast<T*>(out),
                       rows, cols);
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
