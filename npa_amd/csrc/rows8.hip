// Rows in 8 bits, for gfx950: activations kept between forward and backward,
// and the operands of the integer products (linear8.hip, mlp8.hip).
//
//   m = max(max |x|, 2^-100)    scale = m / 127
//   code = rint(x * (127 / m))  value = code * scale
//
// in float32 steps, ties to the even code.  A row that holds a NaN or an
// infinity has a NaN scale and zero codes: whatever is computed from it is NaN.
#include "rows8.hpp"
#include "split16.hpp"

#include <type_traits>

namespace sphops {

namespace {

constexpr int kRowThreads = 256;

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
// positive exactly where x is (in finite rows).  Values below half a scale are
// raised to a whole one for that, so what is computed from such codes leans
// upward where most of a row is small beside its largest.  L = 256: the workgroup's four waves share a
// row.
//
// Bound: HBM, x read once and a quarter of it written: 2^20 x 83 float32 in 91
// us (4.8 TB/s), 65536 x 163 in 11.  Rows of 2-byte values that start at odd
// places lose a quarter where they come from memory: 8191 x 4097 bfloat16 23 us,
// 8192 x 4096 19.  (Loads moved to even places, with the codes shifted between
// lanes, took 20.6 there and 10% longer where x is in cache.)
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

// Rows longer than a workgroup's registers hold: a workgroup a row, which is
// read twice (the second time from cache).  4096 x 8192 float32: 44 us, 26 with
// the row in registers.
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
// Bound: HBM, mostly the result's stores: 65536 x 163 float32 in 13.5 us (4.0
// TB/s), 8191 x 4097 bfloat16, at odd places, in 17.4 (5.8 TB/s).
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
        for (int j = 0; j < 4; ++j) p.set(4 * i + j, from_f32<T>(row_value((int)(int8_t)(w >> (8 * j)), s)));
      }
      p.store(out + r * cols, k, cols);
    }
  }
}

dim3 row_grid(int64_t rows, int rows_a_turn) {
  return dim3((uint32_t)std::min<int64_t>((rows + rows_a_turn - 1) / rows_a_turn, 16384));
}

// f(integral_constant L, integral_constant N) for rows of `pieces` 16-byte pieces;
// false: longer than all of them.  Few lanes with about four pieces
// each: with 64 lanes for every row of up to 192 pieces 65536 rows of 16, 83,
// 163, 200 and 600 float32 take 14, 16, 16, 15 and 28 us instead of 3, 5, 11, 11 and
// 28.  Long rows in steps of a lane's piece: 8191 x 4097 bfloat16, 513 pieces, 23 us
// with nine a lane and 32 with twelve.
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
         SPHOPS_LANES(32, 4) || SPHOPS_LANES(64, 3) || SPHOPS_LANES(64, 4) || SPHOPS_LANES(64, 5) ||
         SPHOPS_LANES(64, 6) || SPHOPS_LANES(64, 7) || SPHOPS_LANES(64, 8) || SPHOPS_LANES(64, 9) ||
         SPHOPS_LANES(64, 10) || SPHOPS_LANES(64, 12) || SPHOPS_LANES(256, 4) || SPHOPS_LANES(256, 8);
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
    // 65536 rows of 16 and of 83 float32: 3.4 and 8.5 us, with 64 lanes 7.2 and 10.6
    if (pieces <= 8) launch(std::integral_constant<int, 8>{});
    else if (pieces <= 16) launch(std::integral_constant<int, 16>{});
    else if (pieces <= 32) launch(std::integral_constant<int, 32>{});
    else if (pieces <= 256) launch(std::integral_constant<int, 64>{});
    else launch(std::integral_constant<int, 256>{});
  });
  SPHOPS_LAUNCHED();
}

namespace {

// Weight gradient from rows in 8 bits: dW = dy^T (codes * scale), db = column
// sums of dy.  A row's scale is put into dy, whose three bfloat16 pieces hold
// 24 bits at float32's range; a code is exact in bfloat16, so three matrix
// instructions of 32 x 32 x 16 (96 cycles) do what float32 ones take 512 for.
//
// Workgroup = a chunk of rows and a block of dW, WO x WI waves of 32 outputs by
// NI tiles of 32 inputs each.  32 rows a step stand in LDS by rows, dy's pieces
// and the codes as bfloat16, and both operands (whose k are the rows) are read
// down their columns.  A row of LDS is an odd number of 64 bytes: the four rows
// of a column read then lie in different banks.  The next step's rows are
// loaded under this one's products.
//
// Bound: HBM where blocks are few (2^20 rows, 83 -> 128: 136 us, 4.7 TB/s of codes
// and dy), the matrix cores where dW is wide (8192 rows, 2048 -> 2048: 190..220 us
// with its sum, three products at 1.0 PFLOP/s; the library's float32 product 505).
struct Grad8Plan {
  int wo, wi, ni, o_blocks, i_blocks;
  int64_t chunk_rows, chunks;
};

template <int WO, int WI, int NI>
__global__ __launch_bounds__(64 * WO * WI, 2) void k_rows8_weight_grad(
    const int8_t* __restrict__ codes, int64_t ld, const float* __restrict__ scale, const float* __restrict__ dy,
    float* __restrict__ part, int64_t rows, int nin, int nout, int i_blocks, int64_t chunk_rows, int64_t part_stride) {
  constexpr int kThreads = 64 * WO * WI, kStepRows = 32, kIT = WI * NI;
  constexpr int kC = (kIT | 1) * 32, kD = (WO | 1) * 32;          // 16-bit values a row of LDS
  constexpr int kCG = kIT * 8, kDG = WO * 8;                      // groups of 4 columns a row
  constexpr int kLC = (kStepRows * kCG + kThreads - 1) / kThreads, kLD = (kStepRows * kDG + kThreads - 1) / kThreads;
  static_assert(kThreads % kDG == 0, "a thread keeps its columns of dy");
  __shared__ __attribute__((aligned(16))) __bf16 cs[2][kStepRows][kC], ds[2][3][kStepRows][kD];
  __shared__ f32x4 sums[kThreads];
  const int lane = threadIdx.x & 63, c = lane & 31, h = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x / 64), wo = wave % WO, wi = wave / WO;
  const int block = (int)blockIdx.y, o0 = block / i_blocks * WO * 32, i0 = block % i_blocks * kIT * 32;
  const int64_t r0 = (int64_t)blockIdx.x * chunk_rows, left = rows - r0, nr = left < chunk_rows ? left : chunk_rows;
  // every second chunk takes -dy, and its sums change sign at the end: see split16.hpp
  const float sign = blockIdx.x & 1 ? -1.0f : 1.0f;
  uint32_t cst[kLC];
  f32x4 dst[kLD];
  float sst[kLD];
  f32x4 sb[kLD];
#pragma unroll
  for (int u = 0; u < kLD; ++u) sb[u] = f32x4{};
  f32x16 acc[NI];
#pragma unroll
  for (int t = 0; t < NI; ++t) acc[t] = f32x16{};

  auto buffer = [](const void* base, int64_t bytes) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(base), (short)0, (int)bytes, 0x00020000);
  };
  constexpr uint32_t kPast = 0x80000000u;
  // rows past the chunk load zeros, which add nothing
  auto load = [&](int64_t t0) {
    const int64_t rest = t0 < nr ? nr - t0 : 0, at = rest > 0 ? r0 + t0 : 0, n = rest < kStepRows ? rest : (int64_t)kStepRows;
    const __amdgpu_buffer_rsrc_t rc = buffer(codes + at * ld, n * ld), rs = buffer(scale + at, n * 4);
    const __amdgpu_buffer_rsrc_t rd = buffer(dy + at * nout, n * nout * 4);
#pragma unroll
    for (int u = 0; u < kLC; ++u) {
      const int i = u * kThreads + (int)threadIdx.x, row = i / kCG, k = i0 + 4 * (i % kCG);
      cst[u] = __builtin_amdgcn_raw_buffer_load_b32(
          rc, row < kStepRows && k < (int)ld ? (uint32_t)(row * (int)ld + k) : kPast, 0, 0);
    }
#pragma unroll
    for (int u = 0; u < kLD; ++u) {
      const int i = u * kThreads + (int)threadIdx.x, row = i / kDG, k = o0 + 4 * (i % kDG);
      dst[u] = __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(
          rd, row < kStepRows && k < nout ? (uint32_t)(row * nout + k) * 4u : kPast, 0, 0));
      sst[u] = __builtin_bit_cast(float, __builtin_amdgcn_raw_buffer_load_b32(
          rs, row < kStepRows ? (uint32_t)row * 4u : kPast, 0, 0));
    }
  };
  const int i16 = lane & 15, rrow = 4 * h + (i16 >> 2), rcol = 16 * ((lane >> 4) & 1) + 4 * (i16 & 3);
  load(0);
  int buf = 0;
  for (int64_t t0 = 0; t0 < nr; t0 += kStepRows, buf ^= 1) {
#pragma unroll
    for (int u = 0; u < kLC; ++u) {
      const int i = u * kThreads + (int)threadIdx.x;
      if (kStepRows * kCG % kThreads == 0 || i < kStepRows * kCG)
        *reinterpret_cast<bf16x4*>(&cs[buf][i / kCG][4 * (i % kCG)]) = codes_bf16(cst[u]);
    }
#pragma unroll
    for (int u = 0; u < kLD; ++u) {
      const int i = u * kThreads + (int)threadIdx.x, row = i / kDG, k = 4 * (i % kDG);
      if (kStepRows * kDG % kThreads != 0 && i >= kStepRows * kDG) continue;
      f32x4 v = dst[u];
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (o0 + k + j >= nout) v[j] = 0.0f;  // the next row's
      sb[u] += v;
      v *= sst[u] * sign;
#pragma unroll
      for (int p = 0; p < 3; ++p) {
        float x0 = v[0], x1 = v[1], x2 = v[2], x3 = v[3];
        const u32x2 x = {bf16_pair(x0, x1), bf16_pair(x2, x3)};
        v = f32x4{x0, x1, x2, x3};
        *reinterpret_cast<u32x2*>(&ds[buf][p][row][k]) = x;
      }
    }
    // one barrier a step: a wave writes a buffer again only after the next
    // barrier, which every wave reaches after its reads of this one
    __syncthreads();
    __builtin_amdgcn_sched_barrier(0);
    load(t0 + kStepRows);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int p = 0; p < kStepRows / 16; ++p) {
      Thirds d;
#pragma unroll
      for (int q = 0; q < 3; ++q)
        d.v[q] = __builtin_bit_cast(bf16x8, join(read_column(&ds[buf][q][16 * p + rrow][32 * wo + rcol]),
                                                 read_column(&ds[buf][q][16 * p + 8 + rrow][32 * wo + rcol])));
#pragma unroll
      for (int t = 0; t < NI; ++t) {
        const int col = 32 * (wi * NI + t) + rcol;
        const bf16x8 z = __builtin_bit_cast(
            bf16x8, join(read_column(&cs[buf][16 * p + rrow][col]), read_column(&cs[buf][16 * p + 8 + rrow][col])));
        acc[t] = mma(d.v[0], z, mma(d.v[1], z, mma(d.v[2], z, acc[t])));
      }
    }
  }
  float* __restrict__ p = part + (int64_t)blockIdx.x * part_stride;
#pragma unroll
  for (int t = 0; t < NI; ++t) {
    const int col = i0 + 32 * (wi * NI + t) + c;
    if (col >= nin) continue;
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      const int m = o0 + 32 * wo + 8 * (r / 4) + 4 * h + r % 4;
      if (m < nout) p[(int64_t)m * nin + col] = acc[t][r] * sign;
    }
  }
  if (i0 != 0) return;
#pragma unroll
  for (int u = 1; u < kLD; ++u) sb[0] += sb[u];
  sums[threadIdx.x] = sb[0];
  __syncthreads();
  for (int k = threadIdx.x; k < WO * 32; k += kThreads) {
    if (o0 + k >= nout) continue;
    float t = 0.0f;
    for (int i = 0; i < kThreads / kDG; ++i) t += sums[i * kDG + k / 4][k % 4];
    p[(int64_t)nout * nin + o0 + k] = t;
  }
}

// The chunks' sums of element e, dW then db, in the chunks' order.
__global__ __launch_bounds__(256) void k_rows8_sum(const float* __restrict__ part, float* __restrict__ dw,
                                                   float* __restrict__ db, int64_t nw, int nout, int64_t chunks) {
  const int64_t n = nw + nout, e = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (e >= n) return;
  float t = 0.0f;
#pragma unroll 4
  for (int64_t k = 0; k < chunks; ++k) t += part[k * n + e];
  if (e < nw) dw[e] = t;
  else if (db != nullptr) db[e - nw] = t;
}

// f(integral_constants WO, WI, NI) of a plan
template <class F>
void with_block(const Grad8Plan& p, F&& f) {
  auto ni = [&](auto wo, auto wi) {
    switch (p.ni) {
      case 1: return f(wo, wi, std::integral_constant<int, 1>{});
      case 2: return f(wo, wi, std::integral_constant<int, 2>{});
      case 3: return f(wo, wi, std::integral_constant<int, 3>{});
      default: return f(wo, wi, std::integral_constant<int, 4>{});
    }
  };
  const std::integral_constant<int, 1> c1{};
  const std::integral_constant<int, 2> c2{};
  const std::integral_constant<int, 4> c4{};
  if (p.wo == 1) ni(c1, c4);
  else if (p.wo == 2) ni(c2, c2);
  else if (p.wi == 1) ni(c4, c1);
  else ni(c4, c2);
}

// Waves: as many along the outputs as there are tiles, the rest along the inputs;
// eight where both are many, which halves what a block reads (262144 rows, 256 ->
// 256 123 us, four 182; 65536 rows, 163 -> 128 22 and 26).  Chunks: two for every
// CU, or one of eight waves, which is what the card holds at once (2^20 rows, 83
// -> 128 136 us, half as many chunks 179, twice 147; 8192 rows, 2048 -> 2048 191,
// 332 and 198), of at least two steps.  Four input tiles a wave in one row or
// column of waves (97 to 128 inputs and more than 64 outputs, 385 to 512 and up to
// 32) take 84 KB of LDS, one workgroup a CU, and run these chunks in two turns: 2^20
// rows, 128 -> 128 215 us beside 131 of 96 -> 128, 512 -> 32 204 beside 123 of 384.
Grad8Plan grad8_plan(int64_t rows, int nin, int nout) {
  Grad8Plan p;
  const int ot = (nout + 31) / 32, it = (nin + 31) / 32;
  p.wo = ot >= 3 ? 4 : ot;
  p.wi = p.wo == 1 ? 4 : p.wo == 2 ? 2 : it > 4 ? 2 : 1;
  p.o_blocks = (ot + p.wo - 1) / p.wo;
  p.i_blocks = (it + 4 * p.wi - 1) / (4 * p.wi);
  p.ni = (it + p.i_blocks * p.wi - 1) / (p.i_blocks * p.wi);
  const int64_t blocks = (int64_t)p.o_blocks * p.i_blocks, want = (p.wo * p.wi == 8 ? 256 : 512) / blocks;
  const int64_t c = (rows + std::max<int64_t>(1, want) - 1) / std::max<int64_t>(1, want);
  p.chunk_rows = std::min<int64_t>(kMaxChunkRows, std::max<int64_t>(64, (c + 31) / 32 * 32));
  p.chunks = rows > 0 ? (rows + p.chunk_rows - 1) / p.chunk_rows : 0;
  return p;
}

}  // namespace

bool rows8_weight_grad_fits(int64_t rows, int nin, int nout) {
  const Grad8Plan p = grad8_plan(rows, nin, nout);
  return (int64_t)p.o_blocks * p.i_blocks <= 65535 && p.chunks < (int64_t(1) << 31);
}

int64_t rows8_weight_grad_floats(int64_t rows, int nin, int nout) {
  const int64_t chunks = grad8_plan(rows, nin, nout).chunks;
  return chunks * ((int64_t)nin * nout + nout);
}

void run_rows8_weight_grad(const int8_t* codes, int64_t ld, const float* scale, const float* dy, float* dw, float* db,
                           int64_t rows, int nin, int nout, float* work, hipStream_t st) {
  const Grad8Plan p = grad8_plan(rows, nin, nout);
  const int64_t nw = (int64_t)nin * nout, n = nw + nout;
  if (p.chunks > 0) {
    with_block(p, [&](auto wo, auto wi, auto ni) {
      constexpr int WO = decltype(wo)::value, WI = decltype(wi)::value;
      hipLaunchKernelGGL((k_rows8_weight_grad<WO, WI, decltype(ni)::value>),
                         dim3((uint32_t)p.chunks, (uint32_t)(p.o_blocks * p.i_blocks)), dim3(64 * WO * WI), 0, st,
                         codes, ld, scale, dy, work, rows, nin, nout, p.i_blocks, p.chunk_rows, n);
    });
    SPHOPS_LAUNCHED();
  }
  // few chunks, or enough elements to fill the card: a thread an element; else the
  // workgroups of linear_grad.hip share an element's chunks out.  Whole gradient:
  // 512 rows, 2048 -> 2048 (2 chunks) 35 and 144 us; 4096, 1024 -> 1024 (8) 41 and
  // 67; 8192, 512 -> 512 (32) 28 and 35; 65536, 256 -> 256 (128 chunks, 65792
  // elements) 45 and 39; 2048, 64 -> 64 (32 chunks, 4160 elements) 8.4 and 7.0.
  if (p.chunks <= 16 || (p.chunks <= 64 && n >= 131072))
    hipLaunchKernelGGL(k_rows8_sum, dim3((uint32_t)((n + 255) / 256)), dim3(256), 0, st, work, dw, db, nw, nout,
                       p.chunks);
  else
    run_linear_chunk_sum(work, dw, db, nw, nout, p.chunks, st);
  SPHOPS_LAUNCHED();
}

}  // namespace sphops
