// The NPA MLP (Linear, ReLU, Linear with 128 hidden units over one row per
// particle, models/npa.py:63-78 of the reference) on rows in 8 bits, for
// gfx950: in inference with both layers as integer products, and its backward
// in training from an input kept in 8 bits.
#include "mlp_tiles.hpp"
#include "rows8.hpp"

namespace sphops {

namespace {

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x16 __attribute__((ext_vector_type(16)));

constexpr int kServeThreads = 256;

// One wave a tile of 32 rows (rows as the columns n of the products, as in
// mlp_rows.hip).  For a step of 32 columns lane l holds 16 codes of row l % 32,
// columns 32 s + 16 (l / 32) + 0..15, and of channel l % 32 in the weights'
// image.  The hidden tile's result registers 4 q .. 4 q + 3 of lane l are hidden
// units 8 q + 4 (l / 32) + 0..3 of its row: packed to one word each they are
// the second product's operand, with W2's image in the same order, so hidden
// codes never leave registers.  KS: steps of 32 input columns; OT: output tiles.
template <int KS, int OT>
__global__ __launch_bounds__(kServeThreads, 2) void k_mlp8(
    const float* __restrict__ z, const int8_t* __restrict__ w1, int64_t ld1, const float* __restrict__ s1,
    const float* __restrict__ b1, const int8_t* __restrict__ w2, int64_t ld2, const float* __restrict__ s2,
    const float* __restrict__ b2, float* __restrict__ y, int64_t rows, int nin, int nout, int64_t tiles) {
  __shared__ i32x4 w1img[KS][kHT][64];
  __shared__ i32x4 w2img[kHT][OT][64];
  __shared__ f32x4 s1s[kHid / 4], b1s[kHid / 4], s2s[OT * kT / 4], b2s[OT * kT / 4];
  const int lane = threadIdx.x & 63, c = lane & 31, h = lane >> 5;
  for (int i = threadIdx.x; i < KS * kHT * 64; i += kServeThreads) {
    const int l = i & 63, t = (i >> 6) % kHT, s = (i >> 6) / kHT, k = 32 * s + 16 * (l >> 5);
    i32x4 v = i32x4{};
    if (k < ld1) v = *reinterpret_cast<const i32x4*>(w1 + (int64_t)(kT * t + (l & 31)) * ld1 + k);
    w1img[s][t][l] = v;
  }
  for (int i = threadIdx.x; i < kHT * OT * 64; i += kServeThreads) {
    const int l = i & 63, o = (i >> 6) % OT, t = (i >> 6) / OT, n = kT * o + (l & 31);
    i32x4 v = i32x4{};
    if (n < nout) {
      const int8_t* p = w2 + (int64_t)n * ld2 + kT * t + 4 * (l >> 5);
#pragma unroll
      for (int q = 0; q < 4; ++q) v[q] = *reinterpret_cast<const int*>(p + 8 * q);
    }
    w2img[t][o][l] = v;
  }
  if (threadIdx.x < kHid) {
    reinterpret_cast<float*>(s1s)[threadIdx.x] = s1[threadIdx.x];
    reinterpret_cast<float*>(b1s)[threadIdx.x] = b1 != nullptr ? b1[threadIdx.x] : 0.0f;
  }
  if (threadIdx.x < OT * kT) {
    const bool on = (int)threadIdx.x < nout;
    reinterpret_cast<float*>(s2s)[threadIdx.x] = on ? s2[threadIdx.x] : 0.0f;
    reinterpret_cast<float*>(b2s)[threadIdx.x] = on && b2 != nullptr ? b2[threadIdx.x] : 0.0f;
  }
  __syncthreads();

  const int64_t step = (int64_t)gridDim.x * (kServeThreads / 64);
  int64_t tile = (int64_t)__builtin_amdgcn_readfirstlane((int)(blockIdx.x * (kServeThreads / 64) + threadIdx.x / 64));
  for (; tile < tiles; tile += step) {
    const int64_t r0 = tile * kT, nr = min<int64_t>(kT, rows - r0);
    const __amdgpu_buffer_rsrc_t rz = rows_rsrc(z + r0 * nin, nr * nin * 4);
    f32x4 zv[KS][4];
    uint32_t top = 0;
#pragma unroll
    for (int s = 0; s < KS; ++s) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int k = 32 * s + 16 * h + 4 * i;
        zv[s][i] = load4(rz, (uint32_t)(c * nin + k) * 4u);
      }
    }
#pragma unroll
    for (int s = 0; s < KS; ++s) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          // past the row's end lies the next row
          if (s == KS - 1 && 32 * s + 16 * h + 4 * i + j >= nin) zv[s][i][j] = 0.0f;
          top = max(top, abs_bits(zv[s][i][j]));
        }
      }
    }
    top = max(top, (uint32_t)__shfl_xor((int)top, 32));
    const RowScale qz = row_scale(top);
    i32x16 acc[kHT];
#pragma unroll
    for (int t = 0; t < kHT; ++t) acc[t] = i32x16{};
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      i32x4 cz;
#pragma unroll
      for (int i = 0; i < 4; ++i)
        cz[i] = (int)row_codes4(zv[s][i][0], zv[s][i][1], zv[s][i][2], zv[s][i][3], qz);
#pragma unroll
      for (int t = 0; t < kHT; ++t)
        acc[t] = __builtin_amdgcn_mfma_i32_32x32x32_i8(w1img[s][t][lane], cz, acc[t], 0, 0, 0);
    }
    f32x16 hv[kHT];
    top = 0;
#pragma unroll
    for (int t = 0; t < kHT; ++t) {
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const f32x4 sv = s1s[8 * t + 2 * q + h], bv = b1s[8 * t + 2 * q + h];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float v = relu(linear8_value(acc[t][4 * q + j], qz.scale, sv[j], bv[j]));
          hv[t][4 * q + j] = v;
          top = max(top, abs_bits(v));
        }
      }
    }
    top = max(top, (uint32_t)__shfl_xor((int)top, 32));
    const RowScale qh = row_scale(top);
    i32x16 out[OT];
#pragma unroll
    for (int o = 0; o < OT; ++o) out[o] = i32x16{};
#pragma unroll
    for (int t = 0; t < kHT; ++t) {
      i32x4 ch;
#pragma unroll
      for (int q = 0; q < 4; ++q)
        ch[q] = (int)row_codes4(hv[t][4 * q], hv[t][4 * q + 1], hv[t][4 * q + 2], hv[t][4 * q + 3], qh);
#pragma unroll
      for (int o = 0; o < OT; ++o)
        out[o] = __builtin_amdgcn_mfma_i32_32x32x32_i8(w2img[t][o][lane], ch, out[o], 0, 0, 0);
    }
    const __amdgpu_buffer_rsrc_t ry = rows_rsrc(y + r0 * nout, nr * nout * 4);
#pragma unroll
    for (int o = 0; o < OT; ++o) {
      f32x16 v;
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const f32x4 sv = s2s[8 * o + 2 * q + h], bv = b2s[8 * o + 2 * q + h];
#pragma unroll
        for (int j = 0; j < 4; ++j) v[4 * q + j] = linear8_value(out[o][4 * q + j], qh.scale, sv[j], bv[j]);
      }
      store_row(ry, nout, kT * o, c, h, v);
    }
  }
}

}  // namespace

void run_mlp8(const float* z, const int8_t* w1, int64_t ld1, const float* s1, const float* b1, const int8_t* w2,
              int64_t ld2, const float* s2, const float* b2, float* y, int64_t rows, int nin, int nout,
              hipStream_t st) {
  if (rows == 0) return;
  const int64_t tiles = (rows + kT - 1) / kT;
  with_groups<(kMaxMlpIn + 31) / 32>((nin + 31) / 32, [&](auto ks) {
    with_groups<2>(nout <= kT ? 1 : 2, [&](auto ot) {
      hipLaunchKernelGGL((k_mlp8<decltype(ks)::value, decltype(ot)::value>), tile_grid(tiles, kServeThreads),
                         dim3(kServeThreads), 0, st, z, w1, ld1, s1, b1, w2, ld2, s2, b2, y, rows, nin, nout, tiles);
    });
  });
  SPHOPS_LAUNCHED();
}

// The backward from codes: the rows and the hidden values again in 32 bits,
// then the gradients of mlp_rows.hip.
int64_t mlp_rows8_floats(int64_t rows, int nin, int nout) {
  return rows * (nin + kHid + nout) + mlp_weight_grad_floats(rows, nin, nout);
}

void run_mlp_rows8_backward(const int8_t* codes, int64_t ld, const float* scale, const float* dy, const float* w1,
                            const float* b1, const float* w2, float* dz, float* dw1, float* db1, float* dw2,
                            float* db2, int64_t rows, int nin, int nout, float* work, hipStream_t st) {
  float *zr = work, *a = zr + rows * nin, *y = a + rows * kHid, *part = y + rows * nout;
  run_restore_rows(codes, ld, scale, zr, SPHOPS_F32, rows, nin, st);
  run_mlp_forward(zr, w1, b1, w2, nullptr, a, y, rows, nin, nout, st);
  if (dz != nullptr) run_mlp_input_grad(dy, w1, w2, a, dz, rows, nin, nout, st);
  if (dw1 != nullptr || db1 != nullptr || dw2 != nullptr || db2 != nullptr)
    run_mlp_weight_grad(zr, a, dy, w2, dw1, db1, dw2, db2, rows, nin, nout, part, st);
}

}  // namespace sphops
