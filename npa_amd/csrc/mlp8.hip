// The NPA MLP (Linear, ReLU, Linear with 128 hidden units over one row per
// particle, models/npa.py:63-78 of the reference) on rows in 8 bits, for
// gfx950: in inference with both layers as integer products, and its backward
// in training from an input kept in 8 bits.
#include "mlp_tiles.hpp"
#include "rows8.hpp"
#include "split16.hpp"

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
//
// Bound: HBM, 4 (nin + nout) bytes a row: 2^20 x 83 -> 19 in 93 us (4.6 TB/s); 4096
// rows 7 us, the weights' images and one row tile's latency.
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
    asm volatile("" ::: "memory");  // the images stay in LDS: read ahead of the loop they spill
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

namespace {

// ---------------------------------------------------------------- training

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

// ------------------------------------------------------ training: forward

// y = relu(z W1^T + b1) W2^T + b2 and z in 8 bits.  One wave a tile of 32 rows
// (rows as the columns n): z's rows, both weights and the hidden values are
// split into three bfloat16 pieces (split16.hpp).  Every value keeps its 24
// bits whatever else is in its row or matrix: with halves that shared a power of
// two a row, a hidden unit or a matrix, a column 2^24 larger than the rest cost
// y 13 of its bits and a hidden unit with a bias of -1e30 all of them.
// The hidden tile's result registers 8 j .. 8 j + 7 of lane l are hidden units
// 16 j + 4 (l / 32) + 0..3 and 8 more of its row: as they stand they are an
// operand with W2's image in the same order, and as the first operand they leave
// y's rows in registers and its columns in lanes, whose stores are whole.
// The largest of a product's six parts have sums of their own: they are rounded
// as often as there are steps, not six times as often.
//
// Bound: matrix and vector work, which add up; 2^20 rows, 83 -> 19 in 208 us (a
// SIMD's 192 matrix instructions of 32 cycles and 1340 vector ones of 4 a row
// tile make 197 + 171 thousand cycles, counted 360 to 400 in all; 0.52 GB, 101 us
// at the rate of a copy).  With shared powers of two and halves, half the matrix
// work: 146 us.
template <int CT, int OT, int kThreads>
__global__ __launch_bounds__(kThreads, kThreads / 256) void k_mlp_forward8(
    const float* __restrict__ z, const float* __restrict__ w1, const float* __restrict__ b1,
    const float* __restrict__ w2, const float* __restrict__ b2, int8_t* __restrict__ codes, int64_t ld,
    float* __restrict__ scale, float* __restrict__ y, int64_t rows, int nin, int nout, int64_t tiles) {
  constexpr int KS = image_steps(CT), P = lds_pieces(CT, OT), kHeld = P < 3 ? OT : 0;
  __shared__ bf16x8 w1img[3][KS][kHT][64];
  __shared__ bf16x8 w2img[P][kHT][2][OT][64];
  __shared__ __attribute__((aligned(16))) float b1s[kHid], b2s[OT * kT];
  const int lane = threadIdx.x & 63, c = lane & 31, h = lane >> 5;
  const int lane0 = image_lane(0, lane), lane1 = image_lane(1, lane);
  w1_image<KS, kThreads>(w1, nin, w1img);
  // entry (t, p, o) of W2: W2[32 o + l % 32][32 t + 16 p + 4 (l / 32) + 0..3, and 8 more]
  const __amdgpu_buffer_rsrc_t r2 = rows_rsrc(w2, nout * kHid * 4);
  auto w2_entry = [&](int tp, int o, int l) {
    const int n = kT * o + (l & 31);
    const uint32_t at = n < nout ? (uint32_t)(n * kHid + 16 * tp + 4 * (l >> 5)) * 4u : kPast;
    return split3(__builtin_shufflevector(load4(r2, at), load4(r2, at + 32u), 0, 1, 2, 3, 4, 5, 6, 7));
  };
  bf16x8 w2r[kHT][2][kHeld + 1][2];
  if constexpr (P == 3) {
    constexpr int kEntries = kHT * 2 * OT * 64;
    static_assert(kEntries % kThreads == 0, "whole turns");
#pragma unroll
    for (int u = 0; u < kEntries / kThreads; ++u) {
      const int i = u * kThreads + (int)threadIdx.x, l = i & 63, o = (i >> 6) % OT, tp = (i >> 6) / OT;
      const Thirds x = w2_entry(tp, o, l);
#pragma unroll
      for (int q = 0; q < 3; ++q) w2img[q][tp / 2][tp % 2][o][l] = x.v[q];
    }
  } else {
#pragma unroll
    for (int t = 0; t < kHT; ++t) {
#pragma unroll
      for (int p = 0; p < 2; ++p) {
#pragma unroll
        for (int o = 0; o < OT; ++o) {
          const Thirds x = w2_entry(2 * t + p, o, lane);
          if (threadIdx.x < 64) w2img[0][t][p][o][lane] = x.v[0];
          w2r[t][p][o][0] = x.v[1];
          w2r[t][p][o][1] = x.v[2];
        }
      }
    }
  }
  if (threadIdx.x < kHid) b1s[threadIdx.x] = b1 != nullptr ? b1[threadIdx.x] : 0.0f;
  if (threadIdx.x < OT * kT) b2s[threadIdx.x] = b2 != nullptr && (int)threadIdx.x < nout ? b2[threadIdx.x] : 0.0f;
  __syncthreads();

  const int64_t step = (int64_t)gridDim.x * (kThreads / 64);
  int64_t tile = (int64_t)__builtin_amdgcn_readfirstlane((int)(threadIdx.x / 64 * gridDim.x + blockIdx.x));
  f32x4 zn[CT][4];
  auto load = [&](int64_t t) {
    const int64_t r0 = t * kT, nr = t < tiles ? min<int64_t>(kT, rows - r0) : 0;
    const __amdgpu_buffer_rsrc_t rz = rows_rsrc(z + (nr > 0 ? r0 * nin : 0), nr * nin * 4);
#pragma unroll
    for (int s = 0; s < CT; ++s) {
#pragma unroll
      for (int i = 0; i < 4; ++i) zn[s][i] = load4(rz, (uint32_t)(c * nin + 32 * s + 16 * h + 4 * i) * 4u);
    }
  };
  load(tile);
  for (; tile < tiles; tile += step) {
    asm volatile("" ::: "memory");  // the images stay in LDS: read ahead of the loop they spill
    const int64_t r0 = tile * kT, nr = min<int64_t>(kT, rows - r0);
    uint32_t zt = 0;
#pragma unroll
    for (int s = 0; s < CT; ++s) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          if (s == CT - 1 && 32 * s + 16 * h + 4 * i + j >= nin) zn[s][i][j] = 0.0f;  // the next row's
          zt = max(zt, abs_bits(zn[s][i][j]));
        }
      }
    }
    zt = max(zt, (uint32_t)__shfl_xor((int)zt, 32));
    const RowScale q = row_scale(zt);
    const __amdgpu_buffer_rsrc_t rc = bytes_rsrc(codes + r0 * ld, nr * ld);
#pragma unroll
    for (int s = 0; s < CT; ++s) {
      const int k = 32 * s + 16 * h;
      u32x4 w;
#pragma unroll
      for (int i = 0; i < 4; ++i) w[i] = row_codes4(zn[s][i][0], zn[s][i][1], zn[s][i][2], zn[s][i][3], q);
      if (s < CT - 1) {
        __builtin_amdgcn_raw_buffer_store_b128(w, rc, (uint32_t)(c * (int)ld + k), 0, 0);
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
          __builtin_amdgcn_raw_buffer_store_b32(
              w[i], rc, k + 4 * i < (int)ld ? (uint32_t)(c * (int)ld + k + 4 * i) : kPast, 0, 0);
      }
    }
    if (h == 0 && c < nr) scale[r0 + c] = q.scale;
    Thirds zs[KS];
#pragma unroll
    for (int s = 0; s < KS; ++s)
      zs[s] = split3(__builtin_shufflevector(zn[s / 2][s % 2 * 2], zn[s / 2][s % 2 * 2 + 1], 0, 1, 2, 3, 4, 5, 6, 7));
    __builtin_amdgcn_sched_barrier(0);
    load(tile + step);  // in flight until the next row tile
    __builtin_amdgcn_sched_barrier(0);
    f32x16 out[OT], rest[OT];
#pragma unroll
    for (int o = 0; o < OT; ++o) out[o] = rest[o] = f32x16{};
#pragma unroll
    for (int t = 0; t < kHT; ++t) {
      f32x16 acc = f32x16{}, low = f32x16{};
#pragma unroll
      for (int k = 0; k < KS; ++k) {
        const int l = k % 2 == 0 ? lane0 : lane1;
        mma(Thirds{w1img[0][k][t][l], w1img[1][k][t][l], w1img[2][k][t][l]}, zs[k], acc, low);
      }
#pragma unroll
      for (int p = 0; p < 2; ++p) {
        f32x8 v;
#pragma unroll
        for (int g = 2 * p; g < 2 * p + 2; ++g) {
          const f32x4 bv = *reinterpret_cast<const f32x4*>(b1s + kT * t + 8 * g + 4 * h);
#pragma unroll
          for (int j = 0; j < 4; ++j) v[4 * (g - 2 * p) + j] = relu(acc[4 * g + j] + low[4 * g + j] + bv[j]);
        }
        const Thirds hs = split3(v);
#pragma unroll
        for (int o = 0; o < OT; ++o) {
          Thirds w;
          w.v[0] = w2img[0][t][p][o][lane];
          if constexpr (P == 3) {
            w.v[1] = w2img[1][t][p][o][lane];
            w.v[2] = w2img[2][t][p][o][lane];
          } else {
            w.v[1] = w2r[t][p][o][0];
            w.v[2] = w2r[t][p][o][1];
          }
          mma(hs, w, out[o], rest[o]);
        }
      }
    }
    const __amdgpu_buffer_rsrc_t ry = rows_rsrc(y + r0 * nout, nr * nout * 4);
#pragma unroll
    for (int o = 0; o < OT; ++o) {
      const float bv = b2s[kT * o + c];
#pragma unroll
      for (int r = 0; r < 16; ++r) out[o][r] = out[o][r] + rest[o][r] + bv;
      store_columns(ry, nout, kT * o + c, h, out[o]);
    }
  }
}

// ------------------------------------------------- training: input gradient

// dz from codes and dy.  One wave a tile of 32 rows, rows as the columns n:
// hidden tile by hidden tile, a (for its sign) from the codes and dh = W2^T dy
// masked by it; then dz += dh W1 with W1's image read down its columns, dh's
// result registers as they stand being the first operand.  All float32 factors
// in three bfloat16 pieces, as in the forward.  dz's stores are whole lines
// because rows are registers in its product.
//
// Bound: as the forward's; 2^20 rows, 83 -> 19 in 240 us (270 + 154 thousand
// cycles of 410 to 456; 168 us with halves).
template <int CT, int OT, int kThreads>
__global__ __launch_bounds__(kThreads, kThreads / 256) void k_mlp_input_grad8(
    const int8_t* __restrict__ codes, int64_t ld, const float* __restrict__ scale, const float* __restrict__ dy,
    const float* __restrict__ w1, const float* __restrict__ b1, const float* __restrict__ w2, float* __restrict__ dz,
    int64_t rows, int nin, int nout, int64_t tiles) {
  constexpr int KS = image_steps(CT), OS = 2 * OT, P = lds_pieces(CT, OT), kHeld = P < 3 ? OS : 0;
  __shared__ bf16x8 w1img[3][KS][kHT][64];
  __shared__ bf16x8 w2img[P][OS][kHT][64];
  __shared__ __attribute__((aligned(16))) float b1s[kHid];
  const int lane = threadIdx.x & 63, c = lane & 31, h = lane >> 5;
  w1_image<KS, kThreads>(w1, nin, w1img);
  // entry (s, t) of W2: W2[step_column(s, l / 32) + 0..7][32 t + l % 32]
  const __amdgpu_buffer_rsrc_t r2 = rows_rsrc(w2, nout * kHid * 4);
  auto w2_entry = [&](int s, int t, int l) {
    const int k = step_column(s, l >> 5), n = kT * t + (l & 31);
    f32x8 v;
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = load1(r2, k + j < nout ? (uint32_t)((k + j) * kHid + n) * 4u : kPast);
    return split3(v);
  };
  bf16x8 w2r[kHeld + 1][kHT][2];
  if constexpr (P == 3) {
    constexpr int kEntries = OS * kHT * 64;
    static_assert(kEntries % kThreads == 0, "whole turns");
#pragma unroll
    for (int u = 0; u < kEntries / kThreads; ++u) {
      const int i = u * kThreads + (int)threadIdx.x, l = i & 63, t = (i >> 6) % kHT, s = (i >> 6) / kHT;
      const Thirds x = w2_entry(s, t, l);
#pragma unroll
      for (int q = 0; q < 3; ++q) w2img[q][s][t][l] = x.v[q];
    }
  } else {
#pragma unroll
    for (int s = 0; s < OS; ++s) {
#pragma unroll
      for (int t = 0; t < kHT; ++t) {
        const Thirds x = w2_entry(s, t, lane);
        if (threadIdx.x < 64) w2img[0][s][t][lane] = x.v[0];
        w2r[s][t][0] = x.v[1];
        w2r[s][t][1] = x.v[2];
      }
    }
  }
  if (threadIdx.x < kHid) b1s[threadIdx.x] = b1 != nullptr ? b1[threadIdx.x] : 0.0f;
  __syncthreads();

  // a column read of W1's image: columns 16 (lane / 16 % 2) + 4 (lane % 4) ..
  // + 3 of a tile's 32, hidden rows 4 h + lane % 16 / 4 from a multiple of 8
  const int i16 = lane & 15, half = (lane >> 4) & 1, odd = (i16 >> 1) & 1;
  const int even = (half * 32 + 4 * h + (i16 >> 2)) * 16 + (i16 & 1) * 8;
  const int wcol = odd ? (kHT * 64 + half * 32 + ((4 * h + (i16 >> 2)) ^ 4)) * 16 + (i16 & 1) * 8 : even;
  const int first8 = 8 * 16 * half, second8 = 8 * 16 * (1 - half);  // the first and second eight rows
  const int lane0 = image_lane(0, lane), lane1 = image_lane(1, lane);
  const int64_t step = (int64_t)gridDim.x * (kThreads / 64);
  int64_t tile = (int64_t)__builtin_amdgcn_readfirstlane((int)(threadIdx.x / 64 * gridDim.x + blockIdx.x));
  u32x4 cn[CT];
  f32x4 dn[OT][4];
  float sn;
  auto load = [&](int64_t t) {
    const int64_t r0 = t < tiles ? t * kT : 0, nr = t < tiles ? min<int64_t>(kT, rows - r0) : 0;
    const __amdgpu_buffer_rsrc_t rc = bytes_rsrc(codes + r0 * ld, nr * ld), rs = rows_rsrc(scale + r0, nr * 4);
    const __amdgpu_buffer_rsrc_t rd = rows_rsrc(dy + r0 * nout, nr * nout * 4);
#pragma unroll
    for (int s = 0; s < CT; ++s)
      cn[s] = __builtin_amdgcn_raw_buffer_load_b128(rc, (uint32_t)(c * (int)ld + 32 * s + 16 * h), 0, 0);
#pragma unroll
    for (int s = 0; s < OT; ++s) {
#pragma unroll
      for (int i = 0; i < 4; ++i) dn[s][i] = load4(rd, (uint32_t)(c * nout + 32 * s + 16 * h + 4 * i) * 4u);
    }
    sn = load1(rs, (uint32_t)c * 4u);
  };
  load(tile);
  auto column = [&](int t, int p, int ct, int q) {
    // the step that the widest input leaves out: its columns, which are not
    // stored, read the one before it
    const int at = 2 * ct + 1 < KS ? wcol : even;
    const char* s = reinterpret_cast<const char*>(&w1img[q][2 * ct][t][16 * p]) + at;
    return __builtin_bit_cast(bf16x8, join(read_column(s + first8), read_column(s + second8)));
  };
  for (; tile < tiles; tile += step) {
    asm volatile("" ::: "memory");  // the images stay in LDS: read ahead of the loop they spill
    const int64_t r0 = tile * kT, nr = min<int64_t>(kT, rows - r0);
    // codes past the row's end meet zeros in W1's image
    bf16x8 cz[KS];
#pragma unroll
    for (int s = 0; s < KS; ++s)
      cz[s] = __builtin_shufflevector(codes_bf16(cn[s / 2][s % 2 * 2]), codes_bf16(cn[s / 2][s % 2 * 2 + 1]), 0, 1, 2,
                                      3, 4, 5, 6, 7);
    const float sc = sn;
    Thirds ds[OS];
#pragma unroll
    for (int s = 0; s < OS; ++s) {
      f32x8 v = __builtin_shufflevector(dn[s / 2][s % 2 * 2], dn[s / 2][s % 2 * 2 + 1], 0, 1, 2, 3, 4, 5, 6, 7);
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (s / 2 == OT - 1 && step_column(s, h) + j >= nout) v[j] = 0.0f;  // the next row's
      ds[s] = split3(v);
    }
    f32x16 out[CT];
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) out[ct] = f32x16{};
#pragma unroll
    for (int t = 0; t < kHT; ++t) {
      f32x16 a = f32x16{}, dh = f32x16{}, low = f32x16{};
#pragma unroll
      for (int q = 2; q >= 0; --q) {
#pragma unroll
        for (int k = 0; k < KS; ++k) a = mma(w1img[q][k][t][k % 2 == 0 ? lane0 : lane1], cz[k], a);
      }
#pragma unroll
      for (int k = 0; k < OS; ++k) {
        Thirds w;
        w.v[0] = w2img[0][k][t][lane];
        if constexpr (P == 3) {
          w.v[1] = w2img[1][k][t][lane];
          w.v[2] = w2img[2][k][t][lane];
        } else {
          w.v[1] = w2r[k][t][0];
          w.v[2] = w2r[k][t][1];
        }
        mma(w, ds[k], dh, low);
      }
      if (t == kHT - 1) {  // into the registers that this tile's codes and dy leave
        __builtin_amdgcn_sched_barrier(0);
        load(tile + step);
        __builtin_amdgcn_sched_barrier(0);
      }
      Thirds hs[2];
#pragma unroll
      for (int p = 0; p < 2; ++p) {
        f32x8 v;
#pragma unroll
        for (int g = 2 * p; g < 2 * p + 2; ++g) {
          const f32x4 bv = *reinterpret_cast<const f32x4*>(b1s + kT * t + 8 * g + 4 * h);
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            // as torch: 0 where relu(a) <= 0, so a NaN lets the upstream pass
            const float d = dh[4 * g + j] + low[4 * g + j];
            v[4 * (g - 2 * p) + j] = a[4 * g + j] * sc + bv[j] <= 0.0f ? 0.0f : d;
          }
        }
        hs[p] = split3(v);
      }
      // the tile's part is summed by itself, small products first, and added
      // with a rounding to nearest
#pragma unroll
      for (int ct = 0; ct < CT; ++ct) {
        f32x16 part = f32x16{};
#pragma unroll
        for (int n = 0; n < 12; ++n) {
          // pieces (dh, W1) in the order of their products' sizes
          constexpr int kD[6] = {1, 2, 0, 1, 0, 0}, kW[6] = {1, 0, 2, 0, 1, 0};
          part = mma(hs[n % 2].v[kD[n / 2]], column(t, n % 2, ct, kW[n / 2]), part);
        }
        out[ct] += part;
        __builtin_amdgcn_sched_barrier(0);  // one tile's columns at a time: read ahead of their turn they spill
      }
    }
    const __amdgpu_buffer_rsrc_t rz = rows_rsrc(dz + r0 * nin, nr * nin * 4);
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) store_columns(rz, nin, kT * ct + c, h, out[ct]);
  }
}

// ------------------------------------------------ training: weight gradients

constexpr int kGradThreads = 256;
// Waves a SIMD: two where they do not spill.  us with one and two: 2^20 rows, 83 ->
// 19 247 and 210; 2^18, 96 -> 30 73 and 68, 112 -> 19 83 and 87, 83 -> 35 83 and 91.
constexpr int weight_grad8_waves(int ks, int os) { return ks > 6 || os > 2 ? 1 : 2; }

// Workgroup = one chunk of rows, wave t the hidden units 32 t .. 32 t + 31 with
// their weights' pieces in registers.  A row tile's codes (as bfloat16) and
// dy's pieces stand in LDS by rows: read along rows they are the operands of a
// = z W1^T and dh = dy W2, read down columns those of dW1 = (dh s)^T codes and
// dW2 = dy^T relu(a), whose other operands come in a's and dh's result layout.
// The next tile is loaded under this one's products.  The chunk's partial sums:
// dW1 (128 x nin), db1 (128), dW2 (nout x 128), db2 (nout).
//
// Six products of bfloat16 pieces, three against codes.  Hidden values and
// upstreams above the largest bfloat16, 3.39e38, count as infinite here.
// Bound: matrix and vector work, which add up (246 + 196 thousand cycles of a SIMD,
// counted 412 to 445 in all); 2^20 rows, 83 -> 19 in 208 us, in a profile 256.
template <int KS, int OS>
__global__ __launch_bounds__(kGradThreads, weight_grad8_waves(KS, OS)) void k_mlp_weight_grad8(
    const int8_t* __restrict__ codes, int64_t ld, const float* __restrict__ scale, const float* __restrict__ dy,
    const float* __restrict__ w1, const float* __restrict__ b1, const float* __restrict__ w2,
    float* __restrict__ part, int64_t rows, int nin, int nout, int64_t chunk_rows) {
  constexpr int CT = (KS + 1) / 2, OT = (OS + 1) / 2;
  // 16-bit values a row of LDS: an odd number of 64 bytes, and each 16 bytes of
  // rows 4 to 7 of eight exchanged with its neighbour (at), so that neither the
  // reads along rows nor those down columns meet in a bank
  constexpr int kZ = (CT | 1) * kT, kD = (OT | 1) * kT;
  constexpr int kZG = CT * 8, kDG = OT * 8;              // groups of 4 columns a row
  constexpr int kLZ = kT * kZG / kGradThreads, kLD = kT * kDG / kGradThreads;
  __shared__ __attribute__((aligned(16))) __bf16 zs[2][kT][kZ], ds[2][3][kT][kD];
  __shared__ __attribute__((aligned(16))) float ss[2][kT];
  __shared__ bf16x8 w2img[OS][3][4][64];
  __shared__ f32x4 sums[kGradThreads];
  auto at = [](int row, int k) { return k ^ (row & 4 ? 8 : 0); };
  const int lane = threadIdx.x & 63, c = lane & 31, h = lane >> 5;
  const int band = __builtin_amdgcn_readfirstlane((int)threadIdx.x / 64) * kT;
  const int64_t r0 = (int64_t)blockIdx.x * chunk_rows, nr = min<int64_t>(chunk_rows, rows - r0);
  // Every second chunk takes -dy, and its sums change sign at the end: see split16.hpp
  const float sign = blockIdx.x & 1 ? -1.0f : 1.0f;

  Thirds w1v[KS];  // W1[band + c][16 s + 8 h ..]; W2[16 s + 8 h + j][band + c] in LDS, each wave its own
  {
    const __amdgpu_buffer_rsrc_t rw1 = rows_rsrc(w1, kHid * nin * 4), rw2 = rows_rsrc(w2, nout * kHid * 4);
#pragma unroll
    for (int s = 0; s < KS; ++s) w1v[s] = split3(load8(rw1, band + c, nin, 16 * s + 8 * h));
#pragma unroll
    for (int s = 0; s < OS; ++s) {
      f32x8 v;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int k = 16 * s + 8 * h + j;
        v[j] = load1(rw2, k < nout ? (uint32_t)(k * kHid + band + c) * 4u : kPast);
      }
      const Thirds x = split3(v);
#pragma unroll
      for (int p = 0; p < 3; ++p) w2img[s][p][threadIdx.x / 64][lane] = x.v[p];
    }
  }
  const float bias = b1 != nullptr ? b1[band + c] : 0.0f;
  f32x16 acc1[CT], acc2[OT];
#pragma unroll
  for (int ct = 0; ct < CT; ++ct) acc1[ct] = f32x16{};
#pragma unroll
  for (int o = 0; o < OT; ++o) acc2[o] = f32x16{};
  float sb1 = 0.0f;
  f32x4 sb2[kLD];
#pragma unroll
  for (int u = 0; u < kLD; ++u) sb2[u] = f32x4{};

  // rows past the chunk load zeros: dy's add nothing
  uint32_t zst[kLZ];
  f32x4 dst[kLD];
  float sst;
  auto load = [&](int64_t t0) {
    const int64_t left = t0 < nr ? nr - t0 : 0, at = left > 0 ? r0 + t0 : 0, n = left < kT ? left : (int64_t)kT;
    const __amdgpu_buffer_rsrc_t rz = bytes_rsrc(codes + at * ld, n * ld);
    const __amdgpu_buffer_rsrc_t rs = rows_rsrc(scale + at, n * 4);
    const __amdgpu_buffer_rsrc_t rd = rows_rsrc(dy + at * nout, n * nout * 4);
#pragma unroll
    for (int u = 0; u < kLZ; ++u) {
      const int i = u * kGradThreads + (int)threadIdx.x, row = i / kZG, k = 4 * (i % kZG);
      zst[u] = __builtin_amdgcn_raw_buffer_load_b32(rz, k < (int)ld ? (uint32_t)(row * (int)ld + k) : kPast, 0, 0);
    }
#pragma unroll
    for (int u = 0; u < kLD; ++u) {
      const int i = u * kGradThreads + (int)threadIdx.x, row = i / kDG, k = 4 * (i % kDG);
      dst[u] = load4(rd, k < nout ? (uint32_t)(row * nout + k) * 4u : kPast);
    }
    sst = load1(rs, threadIdx.x < kT ? threadIdx.x * 4u : kPast);
  };
  // column reads of a tile's rows: lane i of 16 gives row 4 h + i / 4 and columns 16 (lane / 16 % 2) + 4 (i % 4)
  const int i16 = lane & 15, rrow = 4 * h + (i16 >> 2);
  const int rcol = at(rrow, 16 * ((lane >> 4) & 1) + 4 * (i16 & 3));
  load(0);
  int buf = 0;
  for (int64_t t0 = 0; t0 < nr; t0 += kT, buf ^= 1) {
#pragma unroll
    for (int u = 0; u < kLZ; ++u) {
      const int i = u * kGradThreads + (int)threadIdx.x;
      *reinterpret_cast<bf16x4*>(&zs[buf][i / kZG][at(i / kZG, 4 * (i % kZG))]) = codes_bf16(zst[u]);
    }
#pragma unroll
    for (int u = 0; u < kLD; ++u) {
      const int i = u * kGradThreads + (int)threadIdx.x, row = i / kDG, k = 4 * (i % kDG);
      f32x4 v = dst[u];
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (k + j >= nout) v[j] = 0.0f;  // the next row's
      sb2[u] += v;
      v *= sign;
#pragma unroll
      for (int p = 0; p < 3; ++p) {
        float x0 = v[0], x1 = v[1], x2 = v[2], x3 = v[3];
        const u32x2 x = {bf16_pair(x0, x1), bf16_pair(x2, x3)};
        v = f32x4{x0, x1, x2, x3};
        *reinterpret_cast<u32x2*>(&ds[buf][p][row][at(row, k)]) = x;
      }
    }
    if (threadIdx.x < kT) ss[buf][threadIdx.x] = sst;
    // one barrier a tile: a wave writes a buffer again only after the next
    // barrier, which every wave reaches after its reads of this one
    __syncthreads();
    __builtin_amdgcn_sched_barrier(0);
    load(t0 + kT);
    __builtin_amdgcn_sched_barrier(0);
    f32x16 a = f32x16{}, dh = f32x16{};
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      const bf16x8 z8 = *reinterpret_cast<const bf16x8*>(&zs[buf][c][at(c, 16 * s + 8 * h)]);
      a = mma(z8, w1v[s].v[0], mma(z8, w1v[s].v[1], mma(z8, w1v[s].v[2], a)));
    }
#pragma unroll
    for (int s = 0; s < OS; ++s) {
      Thirds d, w;
#pragma unroll
      for (int p = 0; p < 3; ++p) {
        d.v[p] = *reinterpret_cast<const bf16x8*>(&ds[buf][p][c][at(c, 16 * s + 8 * h)]);
        w.v[p] = w2img[s][p][threadIdx.x / 64][lane];
      }
      dh = mma(d, w, dh);
    }
    f32x8 hv[2], gv[2];
    float tb1 = 0.0f;  // a row tile's: one long chain of sums had twice the error (2^20 rows 6.1e-7, plain float32 3.6e-7)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const f32x4 sv = *reinterpret_cast<const f32x4*>(&ss[buf][8 * g + 4 * h]);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float av = a[4 * g + j] * sv[j] + bias;
        const float d = av <= 0.0f ? 0.0f : dh[4 * g + j];
        tb1 += d;
        hv[g / 2][4 * (g % 2) + j] = relu(av);
        gv[g / 2][4 * (g % 2) + j] = d * sv[j];
      }
    }
    sb1 += tb1;
#pragma unroll
    for (int p = 0; p < 2; ++p) {
      const Thirds hs = split3<false>(hv[p]), gs = split3<false>(gv[p]);
#pragma unroll
      for (int o = 0; o < OT; ++o) {
        Thirds d;
#pragma unroll
        for (int q = 0; q < 3; ++q)
          d.v[q] = __builtin_bit_cast(bf16x8, join(read_column(&ds[buf][q][16 * p + rrow][kT * o + rcol]),
                                                   read_column(&ds[buf][q][16 * p + 8 + rrow][kT * o + rcol])));
        acc2[o] = mma(d, hs, acc2[o]);
      }
#pragma unroll
      for (int ct = 0; ct < CT; ++ct) {
        const bf16x8 z8 = __builtin_bit_cast(bf16x8, join(read_column(&zs[buf][16 * p + rrow][kT * ct + rcol]),
                                                          read_column(&zs[buf][16 * p + 8 + rrow][kT * ct + rcol])));
        acc1[ct] = mma(gs.v[0], z8, mma(gs.v[1], z8, mma(gs.v[2], z8, acc1[ct])));
      }
    }
  }

  const int64_t n1 = (int64_t)kHid * nin, n2 = (int64_t)nout * kHid;
  float* __restrict__ p = part + (int64_t)blockIdx.x * (n1 + kHid + n2 + nout);
#pragma unroll
  for (int ct = 0; ct < CT; ++ct) {
    const int col = kT * ct + c;
    if (col < nin) {
#pragma unroll
      for (int r = 0; r < 16; ++r) p[(int64_t)(band + 8 * (r / 4) + 4 * h + r % 4) * nin + col] = acc1[ct][r] * sign;
    }
  }
  sb1 += __shfl_xor(sb1, 32);
  if (h == 0) p[n1 + band + c] = sb1 * sign;
#pragma unroll
  for (int o = 0; o < OT; ++o) {
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      const int m = kT * o + 8 * (r / 4) + 4 * h + r % 4;
      if (m < nout) p[n1 + kHid + (int64_t)m * kHid + band + c] = acc2[o][r] * sign;
    }
  }
  // db2: thread i has summed rows i / kDG (and, with several pieces a thread,
  // that many more rows) of columns 4 (i % kDG) ..
#pragma unroll
  for (int u = 1; u < kLD; ++u) sb2[0] += sb2[u];
  sums[threadIdx.x] = sb2[0];
  __syncthreads();
  if ((int)threadIdx.x < nout) {
    float t = 0.0f;
    for (int i = 0; i < kGradThreads / kDG; ++i) t += sums[i * kDG + threadIdx.x / 4][threadIdx.x % 4];
    p[n1 + kHid + n2 + threadIdx.x] = t;
  }
}

// A chunk for every workgroup the chip holds at once, at least two row tiles
// and at most kMaxChunkRows.
int64_t grad8_chunk_rows(int64_t rows, int nin, int nout) {
  const int64_t want = 256 * weight_grad8_waves((nin + 15) / 16, (nout + 15) / 16);
  const int64_t c = (rows + want - 1) / want;
  return std::min<int64_t>(kMaxChunkRows, std::max<int64_t>(64, (c + kT - 1) / kT * kT));
}
int64_t grad8_chunks(int64_t rows, int nin, int nout) {
  const int64_t c = grad8_chunk_rows(rows, nin, nout);
  return rows > 0 ? (rows + c - 1) / c : 0;
}

constexpr int kMaxKS = (kMaxMlpIn + 15) / 16, kMaxOS = kMaxMlpOut / 16, kMaxCT = (kMaxMlpIn + kT - 1) / kT;

// Workgroups of the row tile kernels: one a CU, a row tile for each where there
// are fewer than the waves.
// Their threads: two waves a SIMD where 256 registers hold a row tile, else one.
// At 2^18 rows, us with two and one (the last below the bounds and the first
// past them): forward 83 -> 35 65 and 71, 128 -> 30 69 and 76, 112 -> 35 88 and 82,
// 150 -> 19 99 and 87; input gradient 83 -> 35 68 and 83, 128 -> 30 97 and 93, 112
// -> 35 127 and 103.
constexpr int tile_threads(bool two) { return two ? 512 : 256; }
inline dim3 spread_grid(int64_t tiles) { return dim3((uint32_t)std::min<int64_t>(256, tiles)); }

}  // namespace

void run_mlp_rows8_forward(const float* z, const float* w1, const float* b1, const float* w2, const float* b2,
                           int8_t* codes, int64_t ld, float* scale, float* y, int64_t rows, int nin, int nout,
                           hipStream_t st) {
  if (rows == 0) return;
  const int64_t tiles = (rows + kT - 1) / kT;
  with_groups<kMaxCT>((nin + kT - 1) / kT, [&](auto ct) {
    with_groups<2>(nout <= kT ? 1 : 2, [&](auto ot) {
      constexpr int CT = decltype(ct)::value, OT = decltype(ot)::value, T = tile_threads(CT + OT <= 5);
      hipLaunchKernelGGL((k_mlp_forward8<CT, OT, T>), spread_grid(tiles), dim3(T), 0, st, z, w1, b1, w2, b2, codes,
                         ld, scale, y, rows, nin, nout, tiles);
    });
  });
  SPHOPS_LAUNCHED();
}

int64_t mlp_rows8_floats(int64_t rows, int nin, int nout) {
  return grad8_chunks(rows, nin, nout) * ((int64_t)kHid * nin + kHid + (int64_t)nout * kHid + nout);
}

void run_mlp_rows8_backward(const int8_t* codes, int64_t ld, const float* scale, const float* dy, const float* w1,
                            const float* b1, const float* w2, float* dz, float* dw1, float* db1, float* dw2,
                            float* db2, int64_t rows, int nin, int nout, float* work, hipStream_t st) {
  const int64_t tiles = (rows + kT - 1) / kT;
  if (dz != nullptr && rows > 0) {
    with_groups<kMaxCT>((nin + kT - 1) / kT, [&](auto ct) {
      with_groups<2>(nout <= kT ? 1 : 2, [&](auto ot) {
        constexpr int CT = decltype(ct)::value, OT = decltype(ot)::value, T = tile_threads(CT <= 3);
        hipLaunchKernelGGL((k_mlp_input_grad8<CT, OT, T>), spread_grid(tiles), dim3(T), 0, st,
                           codes, ld, scale, dy, w1, b1, w2, dz, rows, nin, nout, tiles);
      });
    });
    SPHOPS_LAUNCHED();
  }
  if (dw1 == nullptr && db1 == nullptr && dw2 == nullptr && db2 == nullptr) return;
  const int64_t chunks = grad8_chunks(rows, nin, nout);
  if (chunks > 0) {
    with_groups<kMaxKS>((nin + 15) / 16, [&](auto ks) {
      with_groups<kMaxOS>((nout + 15) / 16, [&](auto os) {
        hipLaunchKernelGGL((k_mlp_weight_grad8<decltype(ks)::value, decltype(os)::value>), dim3((uint32_t)chunks),
                           dim3(kGradThreads), 0, st, codes, ld, scale, dy, w1, b1, w2, work, rows, nin, nout,
                           grad8_chunk_rows(rows, nin, nout));
      });
    });
    SPHOPS_LAUNCHED();
  }
  run_mlp_chunk_sum(work, dw1, db1, dw2, db2, nin, nout, chunks, st);
}

}  // namespace sphops
