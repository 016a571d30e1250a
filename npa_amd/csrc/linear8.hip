// A linear layer in 8-bit integers, for gfx950: y = (cx cw^T) * (sx sw) + b
// with a scale for each row of the input and each output channel, the sums in
// int32 on the integer matrix cores (v_mfma_i32_32x32x32_i8).
#include "rows8.hpp"

namespace sphops {

namespace {

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x16 __attribute__((ext_vector_type(16)));

// One wave a tile of 32 rows and 32 channels.  Lane l supplies 16 codes of
// input row l % 32 and 16 of channel l % 32, at k = 16 (l / 32) of a step of
// 32; result register r of lane l is row 8 (r / 4) + 4 (l / 32) + r % 4,
// channel l % 32.  xq's rows end in zeros up to a multiple of 32, so what a
// channel's last step reads past its row (the next channel's codes) counts
// nothing; the last channel's is not read past the end.
template <class T>
__global__ __launch_bounds__(256) void k_linear8(const int8_t* __restrict__ xq, int64_t xld,
                                                 const float* __restrict__ xs, const int8_t* __restrict__ wq,
                                                 int64_t wld, const float* __restrict__ ws,
                                                 const float* __restrict__ b, T* __restrict__ y, int64_t rows,
                                                 int outs, int row_tiles, int out_tiles) {
  const int lane = threadIdx.x & 63, c = lane & 31, h = lane >> 5;
  const int64_t job = (int64_t)blockIdx.x * 4 + threadIdx.x / 64;
  if (job >= (int64_t)row_tiles * out_tiles) return;
  const int64_t r0 = job / out_tiles * 32;
  const int o0 = (int)(job % out_tiles) * 32;
  const int64_t row = min<int64_t>(r0 + c, rows - 1);
  const int out = min(o0 + c, outs - 1);
  const int8_t* __restrict__ xp = xq + row * xld + 16 * h;
  const int8_t* __restrict__ wp = wq + (int64_t)out * wld + 16 * h;
  i32x16 acc = i32x16{};
  for (int64_t k = 0; k < xld; k += 32) {
    const i32x4 a = *reinterpret_cast<const i32x4*>(xp + k);
    const i32x4 w = k + 16 * h < wld ? *reinterpret_cast<const i32x4*>(wp + k) : i32x4{};
    acc = __builtin_amdgcn_mfma_i32_32x32x32_i8(a, w, acc, 0, 0, 0);
  }
  if (o0 + c >= outs) return;
  const float s = ws[out], bias = b != nullptr ? b[out] : 0.0f;
#pragma unroll
  for (int r = 0; r < 16; ++r) {
    const int64_t at = r0 + 8 * (r / 4) + 4 * h + r % 4;
    if (at < rows) y[at * outs + out] = from_f32<T>(linear8_value(acc[r], xs[at], s, bias));
  }
}

int64_t padded_cols(int64_t cols) { return (cols + 31) / 32 * 32; }

}  // namespace

// Codes (rows of padded_cols bytes), then the scales.
int64_t linear8_workspace_bytes(int64_t rows, int64_t cols, int) { return rows * (padded_cols(cols) + 4); }

void run_linear8(const void* x, int type, int64_t stride, const int8_t* wq, int64_t wld, const float* ws,
                 const float* b, void* y, int64_t rows, int64_t cols, int outs, void* work, hipStream_t st) {
  if (rows == 0) return;
  const int64_t xld = padded_cols(cols);
  int8_t* xq = static_cast<int8_t*>(work);
  float* xs = reinterpret_cast<float*>(xq + rows * xld);
  run_quantize_rows(x, type, stride, xq, xld, xs, rows, cols, false, st);
  const int row_tiles = (int)((rows + 31) / 32), out_tiles = (outs + 31) / 32;
  const int64_t jobs = (int64_t)row_tiles * out_tiles;
  with_type(type, [&](auto t) {
    using T = decltype(t);
    hipLaunchKernelGGL((k_linear8<T>), dim3((uint32_t)((jobs + 3) / 4)), dim3(256), 0, st, xq, xld, xs, wq, wld, ws,
                       b, static_cast<T*>(y), rows, outs, row_tiles, out_tiles);
  });
  SPHOPS_LAUNCHED();
}

}  // namespace sphops
