// A linear layer in 8-bit integers, for gfx950: y = (cx cw^T) * (sx sw) + b
// with a scale for each row of the input and each output channel, the sums in
// int32 on the integer matrix cores.  The sums are exact and each later step
// rounds by itself, so every kernel here gives the same bits.
#include "rows8.hpp"

#include <type_traits>

namespace sphops {

namespace {

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x16 __attribute__((ext_vector_type(16)));

constexpr int kStep = 128;  // bytes of a row a step of the tile kernel takes

__device__ __forceinline__ i32x16 mma8(i32x4 a, i32x4 b, i32x16 c) {
  return __builtin_amdgcn_mfma_i32_32x32x32_i8(a, b, c, 0, 0, 0);
}

// 64 lanes' 16 bytes from memory to LDS, lane l's to lds + 16 l, past the
// registers; done once the wave's vector memory count says so.
__device__ __forceinline__ void load_to_lds(const int8_t* src, int8_t* lds) {
  __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)src,
                                   (__attribute__((address_space(3))) void*)lds, 16, 0, 0);
}

// Output tiles in an order that keeps the tiles an XCD works on at a time in a
// block of 8 row tiles by a few column tiles, whose panels its L2 holds.
__device__ __forceinline__ void tile_of(uint32_t id, int mt, int nt, int& m, int& n) {
  constexpr uint32_t kGroup = 8;
  const uint32_t per = kGroup * (uint32_t)nt, g = id / per, first = g * kGroup;
  const uint32_t size = min(kGroup, (uint32_t)mt - first), at = id - g * per;
  m = (int)(first + at % size);
  n = (int)(at / size);
}

// Workgroup = a tile of BM rows by BN channels, WM x WN waves of BM / WM by BN
// / WN each.  A step of 128 bytes of both panels goes from memory straight to
// LDS, S - 1 steps ahead of its products.  In LDS a row's eight 16-byte
// pieces are exchanged by the row's low bits (piece p stands at p ^ (row % 8)):
// the 8 rows that a quarter of a wave's operand read takes then lie in
// different banks.  For 32 x 32 x 32, lane l supplies 16 bytes of row l % 32 at
// k = 16 (l / 32).
//
// Bound: the matrix cores and the loads' latency under them: 8192 x 4096 -> 8192
// in 270 us for a call among others, 20 of them to put x into 8 bits (2.2 POP/s; the
// library's int8 product alone 255; kernels profiled by themselves 292 + 20), 4096^3
// 80.  The 256 and 128 tiles take 2 stages (4 for the 128: 1024 x 4096 -> 4096 34 us
// for 35, but 2048 rows 60 for 53), the 64 tile, whose workgroups are few and wait on
// memory, 4 (128 x 4096 -> 4096 15 us, 2 stages 21).
//
// xq's rows end in zeros up to a multiple of the step, so what a channel's last
// step holds past its codes counts nothing; its address is kept inside the row.
template <class T, int BM, int BN, int WM, int WN, int S>
__global__ __launch_bounds__(64 * WM * WN) void k_linear8_tile(const int8_t* __restrict__ xq, int64_t xld,
                                                               const float* __restrict__ xs,
                                                               const int8_t* __restrict__ wq, int64_t wld,
                                                               const float* __restrict__ ws,
                                                               const float* __restrict__ b, T* __restrict__ y,
                                                               int64_t rows, int outs, int mt, int nt) {
  constexpr int kWaves = WM * WN, TM = BM / WM / 32, TN = BN / WN / 32;
  constexpr int kLoadsA = BM / 8 / kWaves, kLoadsB = BN / 8 / kWaves;  // a wave's loads of 8 rows a step
  static_assert(kLoadsA * 8 * kWaves == BM && kLoadsB * 8 * kWaves == BN, "whole loads");
  static_assert(S == 2 || S == 4, "stages");
  // separate arrays: a load into one is no reason to wait before a read of the other
  constexpr int kStage = (BM + BN) * kStep;  // the rows' panel, then the channels'
  __shared__ __attribute__((aligned(16))) int8_t s0[kStage], s1[kStage], s2[S > 2 ? kStage : 16], s3[S > 2 ? kStage : 16];
  auto stage = [&](int i) { return i == 0 ? s0 : i == 1 ? s1 : i == 2 ? s2 : s3; };
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x / 64);
  const int c = lane & 31, h = lane >> 5;
  int mi, ni;
  tile_of(xcd_block_id(), mt, nt, mi, ni);
  const int64_t m0 = (int64_t)mi * BM;
  const int n0 = ni * BN;

  const int piece = 16 * ((lane & 7) ^ (lane >> 3));  // of the step's 128 bytes
  // 32-bit offsets from the panels' first rows
  const int8_t* __restrict__ ap = xq + m0 * xld;
  const int8_t* __restrict__ bp = wq + (int64_t)n0 * wld;
  const int rows_here = (int)min<int64_t>(BM, rows - m0), outs_here = min(BN, outs - n0);
  uint32_t oa[kLoadsA], ob[kLoadsB];
#pragma unroll
  for (int i = 0; i < kLoadsA; ++i)
    oa[i] = (uint32_t)min((i * kWaves + wave) * 8 + (lane >> 3), rows_here - 1) * (uint32_t)xld + (uint32_t)piece;
#pragma unroll
  for (int i = 0; i < kLoadsB; ++i)
    ob[i] = (uint32_t)min((i * kWaves + wave) * 8 + (lane >> 3), outs_here - 1) * (uint32_t)wld;
  const int last = (int)wld - 16, end = (int)xld;
  // past the last step: the last one again, which nothing reads
  auto load = [&](int k, int8_t* as) {
    int8_t* const bs = as + BM * kStep;
    k = min(k, end - kStep);
    const int8_t* __restrict__ ak = ap + k;
#pragma unroll
    for (int i = 0; i < kLoadsA; ++i) load_to_lds(ak + oa[i], as + (i * kWaves + wave) * 1024);
    const uint32_t kb = (uint32_t)min(k + piece, last);
#pragma unroll
    for (int i = 0; i < kLoadsB; ++i) load_to_lds(bp + (ob[i] + kb), bs + (i * kWaves + wave) * 1024);
    __builtin_amdgcn_sched_barrier(0);  // the loads go out before the products, not after them
  };
  const int wm = wave / WN * (BM / WM), wn = wave % WN * (BN / WN);
  i32x16 acc[TM][TN];
#pragma unroll
  for (int i = 0; i < TM; ++i) {
#pragma unroll
    for (int j = 0; j < TN; ++j) acc[i][j] = i32x16{};
  }
  auto compute = [&](const int8_t* as) {
    const int8_t* const bs = as + BM * kStep;
#pragma unroll
    for (int s = 0; s < kStep / 32; ++s) {
      const int at = c * kStep + 16 * ((2 * s + h) ^ (c & 7));
      i32x4 a[TM], w[TN];
#pragma unroll
      for (int i = 0; i < TM; ++i) a[i] = *reinterpret_cast<const i32x4*>(as + (wm + 32 * i) * kStep + at);
#pragma unroll
      for (int j = 0; j < TN; ++j) w[j] = *reinterpret_cast<const i32x4*>(bs + (wn + 32 * j) * kStep + at);
#pragma unroll
      for (int i = 0; i < TM; ++i) {
#pragma unroll
        for (int j = 0; j < TN; ++j) acc[i][j] = mma8(w[j], a[i], acc[i][j]);
      }
    }
  };
#pragma unroll
  for (int i = 0; i < S - 1; ++i) load(i * kStep, stage(i));
  // every wave's loads of a step have landed (vmcnt: `later` may be in flight),
  // and every wave has read the step before (lgkmcnt(0)), whose place the next
  // load takes
#define SPHOPS_TURN(later)                           \
  asm volatile("" ::: "memory");                     \
  __builtin_amdgcn_s_waitcnt(0x0070 | (later));      \
  __builtin_amdgcn_s_barrier();                      \
  asm volatile("" ::: "memory")
  const int steps = end / kStep;
  int k = 0;
  for (int g = 0; g < steps / S; ++g) {
#pragma unroll
    for (int i = 0; i < S; ++i, k += kStep) {
      SPHOPS_TURN((S - 2) * (kLoadsA + kLoadsB));
      load(k + (S - 1) * kStep, stage((i + S - 1) % S));
      compute(stage(i));
    }
  }
  // the steps that are left, and no load in flight where LDS is used again below
  SPHOPS_TURN(0);
#undef SPHOPS_TURN
#pragma unroll
  for (int i = 0; i < S - 1; ++i) {
    if (i < steps % S) compute(stage(i));
  }
  // Result register r of lane l is channel 8 (r / 4) + 4 (l / 32) + r % 4 of row l
  // % 32: four neighbours at a time go to the wave's own 4 KB of LDS, 32 rows of
  // UC channels (16-byte pieces exchanged as above), and leave as whole lines.
  // Stored from the registers, 64 bytes a row, they took 56 us of 370 at 8192 x
  // 4096 -> 8192.
  constexpr int V = Piece<T>::V, UC = 32 * TN < 128 / (int)sizeof(T) ? 32 * TN : 128 / (int)sizeof(T);
  constexpr int kPieces = UC / V, kStores = 32 * kPieces / 64;
  __syncthreads();  // the last step's panels have been read
  typedef float f32x4 __attribute__((ext_vector_type(4)));
  f32x4* const units = reinterpret_cast<f32x4*>(s1);  // the channels' scales, then their biases
  for (int n = threadIdx.x; n < BN; n += 64 * kWaves) {
    const int out = min(n0 + n, outs - 1);
    reinterpret_cast<float*>(units)[n] = ws[out];
    reinterpret_cast<float*>(units)[BN + n] = b != nullptr ? b[out] : 0.0f;
  }
  __syncthreads();
  static_assert(kWaves * 4096 <= kStage && 8 * BN <= kStage, "room");
  int8_t* const own = s0 + wave * 4096;
#pragma unroll
  for (int i = 0; i < TM; ++i) {
    asm volatile("" ::: "memory");  // the channels' scales stay in LDS
    const float xscale = xs[min<int64_t>(m0 + wm + 32 * i + c, rows - 1)];
#pragma unroll
    for (int u = 0; u < 32 * TN / UC; ++u) {
      const int col0 = n0 + wn + UC * u;
#pragma unroll
      for (int t = 0; t < UC / 32; ++t) {
        const int j = u * UC / 32 + t;
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const int at = 32 * t + 8 * q + 4 * h;
          const f32x4 s = units[(wn + UC * u + at) / 4], bias = units[(BN + wn + UC * u + at) / 4];
          T v[4];
#pragma unroll
          for (int e = 0; e < 4; ++e)
            v[e] = from_f32<T>(linear8_value(acc[i][j][4 * q + e], xscale, s[e], bias[e]));
          __builtin_memcpy(own + c * UC * sizeof(T) + 16 * ((at / V) ^ (c % kPieces)) + at % V * sizeof(T), v,
                           sizeof(v));
        }
      }
      __builtin_amdgcn_wave_barrier();
#pragma unroll
      for (int n = 0; n < kStores; ++n) {
        const int row = (64 * n + lane) / kPieces, piece16 = (64 * n + lane) % kPieces;
        Piece<T> p;
        __builtin_memcpy(&p.raw, own + row * UC * sizeof(T) + 16 * (piece16 ^ (row % kPieces)), 16);
        const int64_t to = m0 + wm + 32 * i + row;
        if (to < rows) p.store(y + to * outs, col0 + V * piece16, outs);
      }
      __builtin_amdgcn_wave_barrier();
    }
  }
}

// A few short rows (single tokens) in one launch: workgroup = 16 channels, its
// eight waves a share of the length each, with 16 x 16 x 64 instructions.  Every
// workgroup puts the rows into 8 bits for itself, into LDS (they come from L2;
// a launch of their own costs more), while its first weights are on their way.
// Bound: latency, then the weights' bytes: 1 x 4096 -> 4096 in 4.7 us (a launch
// takes 4.2), 1 x 8192 -> 8192 in 13.5 (5.0 TB/s).
// R: rows rounded up to a power of two; N: 16-byte pieces of x a thread holds.
constexpr int kTokenThreads = 512, kTokenWaves = 8, kTokenRows = 16, kTokenCodes = 32768;
template <class T, int R, int N>
__global__ __launch_bounds__(kTokenThreads) void k_linear8_token(const T* __restrict__ x, int64_t stride, int cols,
                                                                 const int8_t* __restrict__ wq, int64_t wld,
                                                                 const float* __restrict__ ws,
                                                                 const float* __restrict__ b, T* __restrict__ y,
                                                                 int rows, int outs, int xld, int share) {
  constexpr int V = Piece<T>::V, L = kTokenThreads / R;  // threads a row
  __shared__ __attribute__((aligned(16))) int8_t codes[kTokenCodes + 16 * R];
  __shared__ uint32_t tops[kTokenWaves];
  __shared__ float scales[R];
  __shared__ i32x4 sums[kTokenWaves][64];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x / 64);
  const int l = threadIdx.x % L, row = threadIdx.x / L, ld = xld + 16;  // rows of LDS in different banks
  const T* __restrict__ from = x + (int64_t)min(row, rows - 1) * stride;
  Piece<T> p[N];
#pragma unroll
  for (int n = 0; n < N; ++n) p[n].load(from, (n * L + l) * V, cols);
  const int c = lane & 15, h = lane >> 4, out = (int)blockIdx.x * 16 + c, last = (int)wld - 16;
  const int8_t* __restrict__ wp = wq + (int64_t)min(out, outs - 1) * wld;
  const int k0 = wave * share, k1 = min(k0 + share, xld);
  constexpr int kAhead = 8;  // steps of 64 bytes in flight
  i32x4 w[kAhead];
  auto load = [&](int k) {
#pragma unroll
    for (int u = 0; u < kAhead; ++u) w[u] = *reinterpret_cast<const i32x4*>(wp + min(k + 64 * u + 16 * h, last));
  };
  __builtin_amdgcn_sched_barrier(0);
  load(k0);
  __builtin_amdgcn_sched_barrier(0);
  uint32_t top = 0;
#pragma unroll
  for (int n = 0; n < N; ++n) {
#pragma unroll
    for (int j = 0; j < V; ++j) top = top_of<false>(top, p[n].get(j));
  }
#pragma unroll
  for (int s = 1; s < (L < 64 ? L : 64); s *= 2) top = max(top, (uint32_t)__shfl_xor((int)top, s));
  if constexpr (L > 64) {
    if (lane == 0) tops[wave] = top;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < L / 64; ++i) top = max(top, tops[row * (L / 64) + i]);
  }
  const RowScale q = row_scale(top);
#pragma unroll
  for (int n = 0; n < N; ++n) {
    const int k = (n * L + l) * V;
#pragma unroll
    for (int i = 0; i < V / 4; ++i)
      if (k + 4 * i < xld)
        *reinterpret_cast<uint32_t*>(codes + row * ld + k + 4 * i) =
            row_codes4(p[n].get(4 * i), p[n].get(4 * i + 1), p[n].get(4 * i + 2), p[n].get(4 * i + 3), q);
  }
  if (l == 0) scales[row] = q.scale;
  __syncthreads();
  const int8_t* __restrict__ xp = codes + (c & (R - 1)) * ld + 16 * h;  // rows past R again: their sums are not kept
  i32x4 acc = i32x4{};
  for (int k = k0; k < k1; k += 64 * kAhead) {
    if (k != k0) load(k);
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      if (k + 64 * u >= k1) break;
      acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(*reinterpret_cast<const i32x4*>(xp + k + 64 * u), w[u], acc, 0, 0, 0);
    }
  }
  sums[wave][lane] = acc;
  __syncthreads();
  // result register r of lane l is row 4 (l / 16) + r, channel l % 16
  if (threadIdx.x >= 16 * R) return;
  const int at = threadIdx.x / 16, n = threadIdx.x % 16, channel = (int)blockIdx.x * 16 + n;
  if (at >= rows || channel >= outs) return;
  int total = 0;
#pragma unroll
  for (int i = 0; i < kTokenWaves; ++i) total += sums[i][16 * (at / 4) + n][at % 4];
  y[(int64_t)at * outs + channel] =
      from_f32<T>(linear8_value(total, scales[at], ws[channel], b != nullptr ? b[channel] : 0.0f));
}

// f(integral_constants R, N) if the rows suit k_linear8_token: their codes fit 32
// KB.  Against two launches with the 64 tile: 1 x 4096 -> 4096 4.7 and 13.4 us, 16 x
// 2048 -> 2048 float32 5.8 and 9.5, 16 x 2048 -> 8192 8.7 and 9.8, 8 x 4096 -> 16384
// 17.2 and 17.6: every workgroup's own work on the rows has used up the gain there.
template <class T, class F>
bool with_token(int64_t rows, int64_t cols, int64_t xld, F&& f) {
  if (rows > kTokenRows) return false;
  auto at = [&](auto r) {
    constexpr int R = decltype(r)::value, L = kTokenThreads / R, V = Piece<T>::V, kMost = kTokenCodes / R / L / V;
    if (rows > R || R * xld > kTokenCodes) return false;
    const int64_t n = (xld / V + L - 1) / L;  // every code up to xld has a thread
    if constexpr (kMost >= 16) {
      if (n > 8) return f(r, std::integral_constant<int, 16>{}), true;
    }
    if (n > 4) f(r, std::integral_constant<int, 8>{});
    else if (n > 2) f(r, std::integral_constant<int, 4>{});
    else if (n > 1) f(r, std::integral_constant<int, 2>{});
    else f(r, std::integral_constant<int, 1>{});
    return true;
  };
  return at(std::integral_constant<int, 1>{}) || at(std::integral_constant<int, 2>{}) ||
         at(std::integral_constant<int, 4>{}) || at(std::integral_constant<int, 8>{}) ||
         at(std::integral_constant<int, 16>{});
}

int64_t padded_cols(int64_t cols) { return (cols + kStep - 1) / kStep * kStep; }
int64_t tiles_of(int64_t n, int tile) { return (n + tile - 1) / tile; }

}  // namespace

// Codes (rows of padded_cols bytes), then the scales.
int64_t linear8_workspace_bytes(int64_t rows, int64_t cols, int) { return rows * (padded_cols(cols) + 4); }

void run_linear8(const void* x, int type, int64_t stride, const int8_t* wq, int64_t wld, const float* ws,
                 const float* b, void* y, int64_t rows, int64_t cols, int outs, void* work, hipStream_t st) {
  if (rows == 0) return;
  const int64_t xld = padded_cols(cols);
  bool done = false;
  with_type(type, [&](auto t) {
    using T = decltype(t);
    done = with_token<T>(rows, cols, xld, [&](auto r, auto n) {
      const int share = (int)((xld / kTokenWaves + 63) / 64 * 64);
      hipLaunchKernelGGL((k_linear8_token<T, decltype(r)::value, decltype(n)::value>),
                         dim3((uint32_t)tiles_of(outs, 16)), dim3(kTokenThreads), 0, st, static_cast<const T*>(x),
                         stride, (int)cols, wq, wld, ws, b, static_cast<T*>(y), (int)rows, outs, (int)xld, share);
    });
  });
  if (done) {
    SPHOPS_LAUNCHED();
    return;
  }
  int8_t* xq = static_cast<int8_t*>(work);
  float* xs = reinterpret_cast<float*>(xq + rows * xld);
  run_quantize_rows(x, type, stride, xq, xld, xs, rows, cols, false, st);
  with_type(type, [&](auto t) {
    using T = decltype(t);
    T* out = static_cast<T*>(y);
    auto tile = [&](auto bm, auto bn, auto wm, auto wn, auto stages) {
      constexpr int BM = decltype(bm)::value, BN = decltype(bn)::value, WM = decltype(wm)::value,
                    WN = decltype(wn)::value;
      const int64_t mt = tiles_of(rows, BM), nt = tiles_of(outs, BN);
      hipLaunchKernelGGL((k_linear8_tile<T, BM, BN, WM, WN, decltype(stages)::value>), dim3((uint32_t)(mt * nt)), dim3(64 * WM * WN), 0, st,
                         xq, xld, xs, wq, wld, ws, b, out, rows, outs, (int)mt, (int)nt);
    };
#define SPHOPS_N(n) std::integral_constant<int, n>{}
    // the largest tile of which there are three for every four CUs; us with tiles of
    // 256, 128 and 64: 4096 x 4096 -> 4096 (256 of the first) 79, 89, 118; 2048 x 4096 ->
    // 4096 (128; 512 of the second) 64, 51, 70; 512 x 4096 -> 4096 (32; 128) 58, 31, 24.
    // Up to 128 channels half of a 256 tile counts for nothing: 65536 x 1024 -> 100 56,
    // 48, 55; 2^20 x 83 -> 128 float32 320, 268, 387; -> 160 56, 59, 63.
    if (outs > 128 && tiles_of(rows, 256) * tiles_of(outs, 256) >= 192)
      tile(SPHOPS_N(256), SPHOPS_N(256), SPHOPS_N(2), SPHOPS_N(4), SPHOPS_N(2));
    else if (tiles_of(rows, 128) * tiles_of(outs, 128) >= 192)
      tile(SPHOPS_N(128), SPHOPS_N(128), SPHOPS_N(2), SPHOPS_N(2), SPHOPS_N(2));
    else tile(SPHOPS_N(64), SPHOPS_N(64), SPHOPS_N(2), SPHOPS_N(2), SPHOPS_N(4));
#undef SPHOPS_N
  });
  SPHOPS_LAUNCHED();
}

}  // namespace sphops
