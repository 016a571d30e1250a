// The NPA MLP (Linear, ReLU, Linear with 128 hidden units over one row per
// particle, models/npa.py:63-78 of the reference) of several experts over rows
// sorted by expert, float32, for gfx950: one kernel forward, one for the input
// gradient and one for the weights'.
//
//   a = z W1_e^T + b1_e   y = relu(a) W2_e^T + b2_e   dh = (dy W2_e) (a > 0)   dz = dh W1_e
//   dW1_e = dh^T z   db1_e = sum dh   dW2_e = dy^T relu(a)   db2_e = sum dy
//
// Float32 factors are three bfloat16 pieces each and a product six matrix
// instructions (split16.hpp).  Hidden values never leave registers: the forward
// keeps one bit of each for the input gradient, and the weight gradients compute
// them again.
//
// The rows' tiles of 32, expert after expert, are shared out evenly among the
// workgroups (part_of).
#include "grouped.hpp"
#include "mlp_images.hpp"

namespace sphops {

namespace {

__device__ __forceinline__ int64_t uniform(int64_t v) {
  return (int64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)v) |
         (int64_t)__builtin_amdgcn_readfirstlane((int)(v >> 32)) << 32;
}

// The row tiles, expert after expert (the rows behind the last expert's a group
// of their own where they count), are cut into `shares` equal ones, and those
// again where one expert's end and the next one's begin.  Workgroup i < shares has
// the first part of share i, workgroup shares + e the part that begins with group
// e's first tile inside a share.
struct Part {
  int group;       // -1: none
  int64_t lo, hi;  // rows
};
__device__ __forceinline__ Part part_of(const int32_t* __restrict__ offsets, int experts, int64_t slots, int shares,
                                        bool behind) {
  Part p{-1, 0, 0};
  const int64_t tiles = uniform(group_tiles(offsets, experts, slots, kT, behind));
  const int64_t cut = min<int64_t>(shares, tiles);  // no share is empty
  int64_t first, last;
  if ((int)blockIdx.x < shares) {
    if (blockIdx.x >= cut) return p;
    first = tiles * blockIdx.x / cut;
    last = tiles * (blockIdx.x + 1) / cut;
  } else {
    const int e = (int)blockIdx.x - shares;
    first = e > 0 ? uniform(group_tiles(offsets, e, slots, kT, false)) : 0;
    if (first >= tiles) return p;
    const int64_t share = ((first + 1) * cut - 1) / tiles;  // that holds the tile
    last = tiles * (share + 1) / cut;
    if (first == tiles * share / cut) return p;  // the share's first part
  }
  const GroupTile g = group_tile(offsets, experts, slots, first, kT, behind);
  if (g.group < 0 || ((int)blockIdx.x >= shares && g.group != (int)blockIdx.x - shares)) return p;  // an empty group
  p.group = g.group;
  p.lo = uniform(g.lo + g.tile * kT);
  p.hi = uniform(min<int64_t>(g.hi, p.lo + (last - first) * kT));
  return p;
}

__device__ __forceinline__ void zero_part(float* __restrict__ to, int64_t lo, int64_t hi, int width) {
  for (int64_t i = lo * width + threadIdx.x; i < hi * width; i += blockDim.x) to[i] = 0.0f;
}

// ---------------------------------------------------------------- forward

// One wave a tile of 32 rows (rows as the columns n).  The hidden tile's result
// registers 8 j .. 8 j + 7 of lane l are hidden units 16 j + 4 (l / 32) + 0..3 and
// 8 more of its row: as they stand they are an operand with W2's image in the
// same order, and as the first operand they leave y's rows in registers and its
// columns in lanes, whose stores are whole.  The largest of a product's six
// parts have sums of their own, rounded once a step.
// mask (slots x 4 words, or null): the lane's bit 16 t + r of its half's two words
// says that register r of hidden tile t is above 0 (or NaN).
// Bound: matrix and vector work, which add up: 2^20 rows of 8 experts, 83 -> 19, in 239
// us (193 + 188 thousand cycles of a SIMD; a CU counts 389 busy of 468).
template <int CT, int OT, int kThreads>
__global__ __launch_bounds__(kThreads, kThreads / 256) void k_expert_mlp_forward(
    const float* __restrict__ z, const float* __restrict__ w1, const float* __restrict__ b1,
    const float* __restrict__ w2, const float* __restrict__ b2, const int32_t* __restrict__ offsets,
    float* __restrict__ y, uint2* __restrict__ mask, int64_t slots, int experts, int nin, int nout, int shares) {
  constexpr int KS = image_steps(CT), P = lds_pieces(CT, OT), kHeld = P < 3 ? OT : 0;
  __shared__ bf16x8 w1img[3][KS][kHT][64];
  __shared__ bf16x8 w2img[P][kHT][2][OT][64];
  __shared__ __attribute__((aligned(16))) float b1s[kHid], b2s[OT * kT];
  const int lane = threadIdx.x & 63, c = lane & 31, h = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x / 64);
  const int lane0 = image_lane(0, lane), lane1 = image_lane(1, lane);
  const Part share = part_of(offsets, experts, slots, shares, true);
  if (share.group < 0) return;
  const int e = share.group;
  if (e == experts) {
    zero_part(y, share.lo, share.hi, nout);
    return;
  }
  w1_image<KS, kThreads>(w1 + (int64_t)e * kHid * nin, nin, w1img);
  // entry (t, p, o) of W2: W2[32 o + l % 32][32 t + 16 p + 4 (l / 32) + 0..3, and 8 more]
  const __amdgpu_buffer_rsrc_t r2 = rows_rsrc(w2 + (int64_t)e * nout * kHid, nout * kHid * 4);
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
  if (threadIdx.x < kHid) b1s[threadIdx.x] = b1 != nullptr ? b1[e * kHid + threadIdx.x] : 0.0f;
  if (threadIdx.x < OT * kT)
    b2s[threadIdx.x] = b2 != nullptr && (int)threadIdx.x < nout ? b2[e * nout + threadIdx.x] : 0.0f;
  __syncthreads();

  f32x4 zn[CT][4];
  auto load = [&](int64_t r0) {
    const int64_t nr = r0 < share.hi ? min<int64_t>(kT, share.hi - r0) : 0;
    const __amdgpu_buffer_rsrc_t rz = rows_rsrc(z + (nr > 0 ? r0 * nin : 0), nr * nin * 4);
#pragma unroll
    for (int s = 0; s < CT; ++s) {
#pragma unroll
      for (int i = 0; i < 4; ++i) zn[s][i] = load4(rz, (uint32_t)(c * nin + 32 * s + 16 * h + 4 * i) * 4u);
    }
  };
  int64_t r0 = share.lo + wave * kT;
  load(r0);
  for (; r0 < share.hi; r0 += kThreads / 64 * kT) {
    asm volatile("" ::: "memory");  // the images stay in LDS: read ahead of the loop they spill
    const int64_t nr = min<int64_t>(kT, share.hi - r0);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (32 * (CT - 1) + 16 * h + 4 * i + j >= nin) zn[CT - 1][i][j] = 0.0f;  // the next row's
    }
    Thirds zs[KS];
#pragma unroll
    for (int s = 0; s < KS; ++s)
      zs[s] = split3(__builtin_shufflevector(zn[s / 2][s % 2 * 2], zn[s / 2][s % 2 * 2 + 1], 0, 1, 2, 3, 4, 5, 6, 7));
    __builtin_amdgcn_sched_barrier(0);
    load(r0 + kThreads / 64 * kT);  // in flight until the next row tile
    __builtin_amdgcn_sched_barrier(0);
    f32x16 out[OT], rest[OT];
#pragma unroll
    for (int o = 0; o < OT; ++o) out[o] = rest[o] = f32x16{};
    uint32_t bits[2] = {0, 0};
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
          for (int j = 0; j < 4; ++j) {
            const float a = acc[4 * g + j] + low[4 * g + j] + bv[j];
            v[4 * (g - 2 * p) + j] = relu(a);
            bits[t / 2] |= a <= 0.0f ? 0u : 1u << (16 * (t % 2) + 4 * g + j);
          }
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
      __builtin_amdgcn_sched_barrier(0);  // one hidden tile's images at a time
    }
    if (mask != nullptr && c < nr) mask[(r0 + c) * 2 + h] = uint2{bits[0], bits[1]};
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

// --------------------------------------------------------- input gradient

// One wave a tile of 32 rows, rows as the columns n: hidden tile by hidden tile
// dh = W2^T dy masked by the forward's bits; then dz += dh W1 with W1's image read
// down its columns, dh's result registers as they stand being the first operand.
// Bound: as the forward's; 205 us (193 + 160 thousand cycles, 318 busy of 388).
template <int CT, int OT, int kThreads>
__global__ __launch_bounds__(kThreads, kThreads / 256) void k_expert_mlp_input_grad(
    const float* __restrict__ dy, const float* __restrict__ w1, const float* __restrict__ w2,
    const uint2* __restrict__ mask, const int32_t* __restrict__ offsets, float* __restrict__ dz, int64_t slots,
    int experts, int nin, int nout, int shares) {
  constexpr int KS = image_steps(CT), OS = 2 * OT, P = lds_pieces(CT, OT), kHeld = P < 3 ? OS : 0;
  __shared__ bf16x8 w1img[3][KS][kHT][64];
  __shared__ bf16x8 w2img[P][OS][kHT][64];
  const int lane = threadIdx.x & 63, c = lane & 31, h = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x / 64);
  // a column read of W1's image: columns 16 (lane / 16 % 2) + 4 (lane % 4) ..
  // + 3 of a tile's 32, hidden rows 4 h + lane % 16 / 4 from a multiple of 8
  const int i16 = lane & 15, half = (lane >> 4) & 1, odd = (i16 >> 1) & 1;
  const int even = (half * 32 + 4 * h + (i16 >> 2)) * 16 + (i16 & 1) * 8;
  const int wcol = odd ? (kHT * 64 + half * 32 + ((4 * h + (i16 >> 2)) ^ 4)) * 16 + (i16 & 1) * 8 : even;
  const int first8 = 8 * 16 * half, second8 = 8 * 16 * (1 - half);  // the first and second eight rows
  auto column = [&](int t, int p, int ct, int q) {
    // the step that the widest input leaves out: its columns, which are not
    // stored, read the one before it
    const int at = 2 * ct + 1 < KS ? wcol : even;
    const char* s = reinterpret_cast<const char*>(&w1img[q][2 * ct][t][16 * p]) + at;
    return __builtin_bit_cast(bf16x8, join(read_column(s + first8), read_column(s + second8)));
  };
  const Part share = part_of(offsets, experts, slots, shares, true);
  if (share.group < 0) return;
  const int e = share.group;
  if (e == experts) {
    zero_part(dz, share.lo, share.hi, nin);
    return;
  }
  w1_image<KS, kThreads>(w1 + (int64_t)e * kHid * nin, nin, w1img);
  // entry (s, t) of W2: W2[step_column(s, l / 32) + 0..7][32 t + l % 32]
  const __amdgpu_buffer_rsrc_t r2 = rows_rsrc(w2 + (int64_t)e * nout * kHid, nout * kHid * 4);
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
  __syncthreads();

  f32x4 dn[OT][4];
  uint2 mn;
  auto load = [&](int64_t r0) {
    const int64_t nr = r0 < share.hi ? min<int64_t>(kT, share.hi - r0) : 0, at = nr > 0 ? r0 : 0;
    const __amdgpu_buffer_rsrc_t rd = rows_rsrc(dy + at * nout, nr * nout * 4);
    const __amdgpu_buffer_rsrc_t rm = rows_rsrc(reinterpret_cast<const float*>(mask + at * 2), nr * 16);
#pragma unroll
    for (int s = 0; s < OT; ++s) {
#pragma unroll
      for (int i = 0; i < 4; ++i) dn[s][i] = load4(rd, (uint32_t)(c * nout + 32 * s + 16 * h + 4 * i) * 4u);
    }
    mn.x = __builtin_amdgcn_raw_buffer_load_b32(rm, (uint32_t)(16 * c + 8 * h), 0, 0);
    mn.y = __builtin_amdgcn_raw_buffer_load_b32(rm, (uint32_t)(16 * c + 8 * h + 4), 0, 0);
  };
  int64_t r0 = share.lo + wave * kT;
  load(r0);
  for (; r0 < share.hi; r0 += kThreads / 64 * kT) {
    asm volatile("" ::: "memory");  // the images stay in LDS: read ahead of the loop they spill
    const int64_t nr = min<int64_t>(kT, share.hi - r0);
    const uint32_t bits[2] = {mn.x, mn.y};
    Thirds ds[OS];
#pragma unroll
    for (int s = 0; s < OS; ++s) {
      f32x8 v = __builtin_shufflevector(dn[s / 2][s % 2 * 2], dn[s / 2][s % 2 * 2 + 1], 0, 1, 2, 3, 4, 5, 6, 7);
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (s / 2 == OT - 1 && step_column(s, h) + j >= nout) v[j] = 0.0f;  // the next row's
      ds[s] = split3(v);
    }
    __builtin_amdgcn_sched_barrier(0);
    load(r0 + kThreads / 64 * kT);  // in flight until the next row tile
    __builtin_amdgcn_sched_barrier(0);
    f32x16 out[CT];
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) out[ct] = f32x16{};
#pragma unroll
    for (int t = 0; t < kHT; ++t) {
      f32x16 dh = f32x16{}, low = f32x16{};
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
      Thirds hs[2];
#pragma unroll
      for (int p = 0; p < 2; ++p) {
        f32x8 v;
#pragma unroll
        for (int r = 8 * p; r < 8 * p + 8; ++r)
          v[r - 8 * p] = bits[t / 2] >> (16 * (t % 2) + r) & 1 ? dh[r] + low[r] : 0.0f;
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

// -------------------------------------------------------- weight gradients

constexpr int kGradThreads = 256;
// Waves a SIMD: two where they do not spill.
constexpr int grad_waves(int ks, int os) { return ks > 6 || os > 2 ? 1 : 2; }

// One expert's part of the workgroup's share at a time, wave t the hidden units
// 32 t .. 32 t + 31 with W1's pieces in registers.  A row tile's z and dy stand in
// LDS by rows, in pieces: read along rows they are the operands of a = z W1^T and
// dh = dy W2, read down columns those of dW1 = dh^T z and dW2 = dy^T relu(a),
// whose other operands come in a's and dh's result layout.  The next tile is
// loaded under this one's products.  The sums of workgroup i stand at
// place i of `part`: dW1 (128 x nin), db1 (128), dW2 (nout x 128), db2 (nout).
// Bound: as the forward's; 354 us (385 + 272 thousand cycles, 589 busy of 650), more than a
// third of the products for hidden values that the forward had.
//
// The ReLU's side is taken from these values, which are summed in another order than
// the forward's: where one lies within its rounding of 0, they may be on either side,
// and so may dz and the weights' gradients, each of which is then right by itself.
template <int KS, int OS>
__global__ __launch_bounds__(kGradThreads, grad_waves(KS, OS)) void k_expert_mlp_weight_grad(
    const float* __restrict__ z, const float* __restrict__ dy, const float* __restrict__ w1,
    const float* __restrict__ b1, const float* __restrict__ w2, const int32_t* __restrict__ offsets,
    float* __restrict__ part, int64_t slots, int experts, int nin, int nout, int shares) {
  constexpr int CT = (KS + 1) / 2, OT = (OS + 1) / 2;
  // 16-bit values a row of LDS: an odd number of 64 bytes, and each 16 bytes of
  // rows 4 to 7 of eight exchanged with its neighbour (at), so that neither the
  // reads along rows nor those down columns meet in a bank
  constexpr int kZ = (CT | 1) * kT, kD = (OT | 1) * kT;
  constexpr int kZG = CT * 8, kDG = OT * 8;  // groups of 4 columns a row
  constexpr int kLZ = kT * kZG / kGradThreads, kLD = kT * kDG / kGradThreads;
  // one buffer where two do not leave room for a second workgroup
  __shared__ __attribute__((aligned(16))) __bf16 zs[3][kT][kZ], ds[3][kT][kD];
  __shared__ bf16x8 w2img[OS][3][4][64];
  __shared__ f32x4 sums[kGradThreads];
  auto at = [](int row, int k) { return k ^ (row & 4 ? 8 : 0); };
  const int lane = threadIdx.x & 63, c = lane & 31, h = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x / 64), band = wave * kT;
  // column reads of a tile's rows: lane i of 16 gives row 4 h + i / 4 and columns 16 (lane / 16 % 2) + 4 (i % 4)
  const int i16 = lane & 15, rrow = 4 * h + (i16 >> 2);
  const int rcol = at(rrow, 16 * ((lane >> 4) & 1) + 4 * (i16 & 3));
  const Part share = part_of(offsets, experts, slots, shares, false);
  if (share.group < 0) return;
  const int e = share.group;
  const int64_t n1 = (int64_t)kHid * nin, n2 = (int64_t)nout * kHid;
  const int64_t place = blockIdx.x;
  // Every second part takes -dy, and its sums change sign at the end: see split16.hpp
  const float sign = place & 1 ? -1.0f : 1.0f;
  Thirds w1v[KS];  // W1[band + c][16 s + 8 h ..]; W2[16 s + 8 h + j][band + c] in LDS, each wave its own
  {
    const __amdgpu_buffer_rsrc_t rw1 = rows_rsrc(w1 + e * n1, n1 * 4), rw2 = rows_rsrc(w2 + e * n2, n2 * 4);
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
      for (int p = 0; p < 3; ++p) w2img[s][p][wave][lane] = x.v[p];
    }
  }
  const float bias = b1 != nullptr ? b1[e * kHid + band + c] : 0.0f;
  f32x16 acc1[CT], acc2[OT];
#pragma unroll
  for (int ct = 0; ct < CT; ++ct) acc1[ct] = f32x16{};
#pragma unroll
  for (int o = 0; o < OT; ++o) acc2[o] = f32x16{};
  float sb1 = 0.0f;
  f32x4 sb2[kLD];
#pragma unroll
  for (int u = 0; u < kLD; ++u) sb2[u] = f32x4{};

  // rows past the part load zeros: dy's add nothing
  f32x4 zst[kLZ], dst[kLD];
  auto load = [&](int64_t r0) {
    const int64_t left = r0 < share.hi ? share.hi - r0 : 0, from = left > 0 ? r0 : 0, n = left < kT ? left : (int64_t)kT;
    const __amdgpu_buffer_rsrc_t rz = rows_rsrc(z + from * nin, n * nin * 4);
    const __amdgpu_buffer_rsrc_t rd = rows_rsrc(dy + from * nout, n * nout * 4);
#pragma unroll
    for (int u = 0; u < kLZ; ++u) {
      const int i = u * kGradThreads + (int)threadIdx.x, row = i / kZG, k = 4 * (i % kZG);
      zst[u] = load4(rz, k < nin ? (uint32_t)(row * nin + k) * 4u : kPast);
    }
#pragma unroll
    for (int u = 0; u < kLD; ++u) {
      const int i = u * kGradThreads + (int)threadIdx.x, row = i / kDG, k = 4 * (i % kDG);
      dst[u] = load4(rd, k < nout ? (uint32_t)(row * nout + k) * 4u : kPast);
    }
  };
  auto put = [&](f32x4 v, auto& image, int row, int k, int width) {
#pragma unroll
    for (int p = 0; p < 3; ++p) {
      float x0 = v[0], x1 = v[1], x2 = v[2], x3 = v[3];
      const u32x2 x = p == 0 ? u32x2{bf16_pair_top(x0, x1), bf16_pair_top(x2, x3)} : u32x2{bf16_pair(x0, x1), bf16_pair(x2, x3)};
      v = f32x4{x0, x1, x2, x3};
      *reinterpret_cast<u32x2*>(&image[p][row][at(row, k)]) = x;
    }
  };
  load(share.lo);
  for (int64_t r0 = share.lo; r0 < share.hi; r0 += kT) {
    __syncthreads();  // the tile before has been read
#pragma unroll
    for (int u = 0; u < kLZ; ++u) {
      const int i = u * kGradThreads + (int)threadIdx.x, row = i / kZG, k = 4 * (i % kZG);
      f32x4 v = zst[u];
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (k + j >= nin) v[j] = 0.0f;  // the next row's
      put(v, zs, row, k, nin);
    }
#pragma unroll
    for (int u = 0; u < kLD; ++u) {
      const int i = u * kGradThreads + (int)threadIdx.x, row = i / kDG, k = 4 * (i % kDG);
      f32x4 v = dst[u];
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (k + j >= nout) v[j] = 0.0f;
      sb2[u] += v;
      put(v * sign, ds, row, k, nout);
    }
    __syncthreads();
    __builtin_amdgcn_sched_barrier(0);
    load(r0 + kT);
    __builtin_amdgcn_sched_barrier(0);
    f32x16 a = f32x16{}, dh = f32x16{};
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      Thirds x;
#pragma unroll
      for (int p = 0; p < 3; ++p) x.v[p] = *reinterpret_cast<const bf16x8*>(&zs[p][c][at(c, 16 * s + 8 * h)]);
      a = mma(x, w1v[s], a);
    }
#pragma unroll
    for (int s = 0; s < OS; ++s) {
      Thirds d, w;
#pragma unroll
      for (int p = 0; p < 3; ++p) {
        d.v[p] = *reinterpret_cast<const bf16x8*>(&ds[p][c][at(c, 16 * s + 8 * h)]);
        w.v[p] = w2img[s][p][wave][lane];
      }
      dh = mma(d, w, dh);
    }
    f32x8 hv[2], gv[2];
    float tb1 = 0.0f;  // a row tile's: one long chain of sums has twice the error
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      const float av = a[r] + bias, d = av <= 0.0f ? 0.0f : dh[r];
      tb1 += d;
      hv[r / 8][r % 8] = relu(av);
      gv[r / 8][r % 8] = d;
    }
    sb1 += tb1;
#pragma unroll
    for (int p = 0; p < 2; ++p) {
      const Thirds hs = split3(hv[p]), gs = split3(gv[p]);
      auto columns = [&](auto& image, int col) {
        Thirds d;
#pragma unroll
        for (int q = 0; q < 3; ++q)
          d.v[q] = __builtin_bit_cast(bf16x8, join(read_column(&image[q][16 * p + rrow][col + rcol]),
                                                   read_column(&image[q][16 * p + 8 + rrow][col + rcol])));
        return d;
      };
#pragma unroll
      for (int o = 0; o < OT; ++o) acc2[o] = mma(columns(ds, kT * o), hs, acc2[o]);
#pragma unroll
      for (int ct = 0; ct < CT; ++ct) acc1[ct] = mma(gs, columns(zs, kT * ct), acc1[ct]);
    }
  }

  float* __restrict__ p = part + place * (n1 + kHid + n2 + nout);
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

// The gradients of expert blockIdx.y: its parts' sums, in a fixed order: wave q
// of the workgroup adds every 16th of them, four neighbouring values a lane.
// `shares`: as the parts were cut.
constexpr int kSumWaves = 16;
__global__ __launch_bounds__(64 * kSumWaves) void k_expert_mlp_sum(const float* __restrict__ part,
                                                                   const int32_t* __restrict__ offsets,
                                                                   float* __restrict__ dw1, float* __restrict__ db1,
                                                                   float* __restrict__ dw2, float* __restrict__ db2,
                                                                   int64_t slots, int experts, int n1, int n2, int nout,
                                                                   int shares) {
  __shared__ f32x4 red[kSumWaves][64];
  const int lane = threadIdx.x & 63, q = threadIdx.x >> 6, e = (int)blockIdx.y, n = n1 + kHid + n2 + nout;
  const GroupSpan g = group_span(offsets, experts, slots, kT, e);
  f32x4 t = f32x4{};
  const int at = (int)blockIdx.x * 256 + 4 * lane;
  if (g.tiles > 0 && at < n) {
    // the first share's part is the expert's own where it begins inside the share
    const int64_t cut = min<int64_t>(shares, g.all);
    const int first = (int)(((g.before + 1) * cut - 1) / g.all), last = (int)(((g.before + g.tiles) * cut - 1) / g.all);
    const bool inside = g.before != g.all * first / cut;
    auto add = [&](int i) {
      const float* __restrict__ p = part + (int64_t)(i == first && inside ? shares + e : i) * n + at;
      if (at + 4 <= n) {
        Piece<float> v;
        v.load(p, 0, 4);
        t += f32x4{v.get(0), v.get(1), v.get(2), v.get(3)};
      } else {
#pragma unroll
        for (int j = 0; j < 3; ++j)
          if (at + j < n) t[j] += p[j];
      }
    };
    int i = first + q;
    if (i <= last) add(i);
#pragma unroll 4
    for (i += kSumWaves; i <= last; i += kSumWaves) add(i);
  }
  red[q][lane] = t;
  __syncthreads();
  // thread i: value i of the workgroup's 256
  const int to = (int)blockIdx.x * 256 + (int)threadIdx.x;
  if (threadIdx.x >= 256 || to >= n) return;
  float v = 0.0f;
#pragma unroll
  for (int k = 0; k < kSumWaves; ++k) v += red[k][threadIdx.x / 4][threadIdx.x % 4];
  auto put = [&](float* out, int first, int count) {
    if (out != nullptr && to >= first && to < first + count) out[(int64_t)e * count + to - first] = v;
  };
  put(dw1, 0, n1);
  put(db1, n1, kHid);
  put(dw2, n1 + kHid, n2);
  put(db2, n1 + kHid + n2, nout);
}

int64_t most_row_tiles(int64_t slots, int64_t groups) { return slots / kT + std::min(groups, slots); }

// Shares of the rows where the card holds `room` workgroups at once: their parts
// should all fit, or those that come last wait for one of the others on their own
// XCD (2^20 rows of 83 -> 19, 8 experts: forward 347 us with 256 shares, 265 with
// 247, in a profile).  Many experts give up no more than half of the room for that.
int64_t shares_of(int64_t room, int64_t parts) { return room - std::min(parts, room / 2); }
int64_t row_shares(int64_t slots, int experts) {
  return std::min(shares_of(256, experts + 1), most_row_tiles(slots, experts + 1));
}
// For the weight gradients also enough that none sums more than kMaxChunkRows rows.
int64_t grad_shares(int64_t slots, int experts, int nin, int nout) {
  const int64_t most = most_row_tiles(slots, experts);
  const int64_t want = shares_of(256 * grad_waves((nin + 15) / 16, (nout + 15) / 16), experts);
  return std::min(most, std::max(want, (most * kT + kMaxChunkRows - 1) / kMaxChunkRows));
}
constexpr int share_threads(bool two) { return two ? 512 : 256; }

}  // namespace

bool expert_mlp_fits(int64_t slots, int experts, int nin, int hidden, int nout) {
  return mlp_fits(slots, nin, hidden, nout) && experts >= 1 && experts <= kMaxExperts;
}

void run_expert_mlp_forward(const float* z, const float* w1, const float* b1, const float* w2, const float* b2,
                            const int32_t* offsets, float* y, uint32_t* mask, int64_t slots, int experts, int nin,
                            int nout, hipStream_t st) {
  if (slots == 0) return;
  const int64_t shares = row_shares(slots, experts);
  with_groups<kMaxCT>((nin + kT - 1) / kT, [&](auto ct) {
    with_groups<2>(nout <= kT ? 1 : 2, [&](auto ot) {
      constexpr int CT = decltype(ct)::value, OT = decltype(ot)::value, T = share_threads(CT + OT <= 5);
      hipLaunchKernelGGL((k_expert_mlp_forward<CT, OT, T>), dim3((uint32_t)(shares + experts + 1)), dim3(T), 0, st, z, w1, b1, w2,
                         b2, offsets, y, reinterpret_cast<uint2*>(mask), slots, experts, nin, nout, (int)shares);
    });
  });
  SPHOPS_LAUNCHED();
}

void run_expert_mlp_input_grad(const float* dy, const float* w1, const float* w2, const uint32_t* mask,
                               const int32_t* offsets, float* dz, int64_t slots, int experts, int nin, int nout,
                               hipStream_t st) {
  if (slots == 0) return;
  const int64_t shares = row_shares(slots, experts);
  with_groups<kMaxCT>((nin + kT - 1) / kT, [&](auto ct) {
    with_groups<2>(nout <= kT ? 1 : 2, [&](auto ot) {
      constexpr int CT = decltype(ct)::value, OT = decltype(ot)::value, T = share_threads(CT <= 3);
      hipLaunchKernelGGL((k_expert_mlp_input_grad<CT, OT, T>), dim3((uint32_t)(shares + experts + 1)), dim3(T), 0, st, dy, w1, w2,
                         reinterpret_cast<const uint2*>(mask), offsets, dz, slots, experts, nin, nout, (int)shares);
    });
  });
  SPHOPS_LAUNCHED();
}

int64_t expert_mlp_floats(int64_t slots, int experts, int nin, int nout) {
  if (slots == 0) return 0;
  return (grad_shares(slots, experts, nin, nout) + experts) * ((int64_t)kHid * nin + kHid + (int64_t)nout * kHid + nout);
}

void run_expert_mlp_weight_grad(const float* z, const float* dy, const float* w1, const float* b1, const float* w2,
                                const int32_t* offsets, float* dw1, float* db1, float* dw2, float* db2, int64_t slots,
                                int experts, int nin, int nout, float* work, hipStream_t st) {
  const int64_t shares = slots > 0 ? grad_shares(slots, experts, nin, nout) : 0;
  if (shares > 0) {
    with_groups<kMaxKS>((nin + 15) / 16, [&](auto ks) {
      with_groups<kMaxOS>((nout + 15) / 16, [&](auto os) {
        hipLaunchKernelGGL((k_expert_mlp_weight_grad<decltype(ks)::value, decltype(os)::value>),
                           dim3((uint32_t)(shares + experts)), dim3(kGradThreads), 0, st, z, dy, w1, b1, w2, offsets,
                           work, slots, experts, nin, nout, (int)shares);
      });
    });
    SPHOPS_LAUNCHED();
  }
  const int n1 = kHid * nin, n2 = nout * kHid, n = n1 + kHid + n2 + nout;
  hipLaunchKernelGGL(k_expert_mlp_sum, dim3((uint32_t)((n + 255) / 256), (uint32_t)experts), dim3(64 * kSumWaves), 0, st,
                     work, offsets, dw1, db1, dw2, db2, slots, experts, n1, n2, nout, (int)shares);
  SPHOPS_LAUNCHED();
}

}  // namespace sphops
