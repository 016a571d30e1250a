// Linear layers of experts over rows sorted by expert, for gfx950:
//
//   y[s] = x[s] W_e^T + b_e   dx[s] = dy[s] W_e   dW_e = sum of dy[s]^T x[s]   db_e = sum of dy[s]
//
// over the rows s of expert e, offsets[e] <= s < offsets[e + 1]; rows behind the
// last expert's are zeros.  Sums are float32, and so are products of float32 rows.
#include "grouped.hpp"

namespace sphops {

namespace {

// Output tiles of a block of 8 row tiles by all column tiles one after another,
// so that the tiles an XCD works on at a time share their panels in its L2.
__device__ __forceinline__ void tile_of(uint32_t id, int64_t mt, int nt, int64_t& m, int& n) {
  constexpr uint32_t kGroup = 8;
  const uint32_t per = kGroup * (uint32_t)nt, g = id / per, first = g * kGroup;
  const uint32_t size = (uint32_t)min<int64_t>(kGroup, mt - first), at = id - g * per;
  m = first + at % size;
  n = (int)(at / size);
}

// What the matrix cores are given of a type: itself, or three bfloat16 pieces.
template <class T>
using Piece16 = std::conditional_t<std::is_same_v<T, float>, __hip_bfloat16, T>;
template <class T>
constexpr int kPieces = std::is_same_v<T, float> ? 3 : 1;

__host__ __device__ __forceinline__ constexpr int64_t whole8(int64_t n) { return (n + 7) / 8 * 8; }

// Rows laid out for the kernels that load whole 16-byte pieces (HBM: 8192 x 2048
// float32 in 28 us, 6.0 TB/s, part of them in cache): out (rows x ld, ld a multiple
// of 8, zeros past cols) as they are, or as three planes of bfloat16 pieces.
constexpr int kLayThreads = 256;
template <class T>
__global__ __launch_bounds__(kLayThreads) void k_lay_out(const T* __restrict__ x, int64_t stride,
                                                         uint16_t* __restrict__ out, int64_t rows, int cols, int ld) {
  const int pieces = ld / 8;
  const int64_t n = rows * pieces;
  for (int64_t i = (int64_t)blockIdx.x * kLayThreads + threadIdx.x; i < n; i += (int64_t)gridDim.x * kLayThreads) {
    const int64_t row = i / pieces;
    const int k = (int)(i - row * pieces) * 8;
    uint16_t* const to = out + row * ld + k;
    if constexpr (std::is_same_v<T, float>) {
      Piece<float> p[2];
      p[0].load(x + row * stride, k, cols);
      p[1].load(x + row * stride, k + 4, cols);
      f32x8 v;
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = p[j / 4].get(j % 4);
      const Thirds t = split3(v);
#pragma unroll
      for (int q = 0; q < 3; ++q) *reinterpret_cast<bf16x8*>(to + q * rows * ld) = t.v[q];
    } else {
      Piece<T> p;
      p.load(x + row * stride, k, cols);
      *reinterpret_cast<u32x4*>(to) = __builtin_bit_cast(u32x4, p.raw);
    }
  }
}

// A workgroup's part of a product over rows: a tile, or a slice of one.  The
// launch covers the most that there can be.
struct RowsJob {
  GroupTile g;
  int n;                // column tile
  int slice, slices;    // of the sum
  int64_t place;        // of a slice's sums
  // steps first .. last - 1 of `steps`
  __device__ __forceinline__ int first(int steps) const { return (int)((int64_t)steps * slice / slices); }
  __device__ __forceinline__ int last(int steps) const { return (int)((int64_t)steps * (slice + 1) / slices); }
};
__device__ __forceinline__ bool rows_job(const int32_t* __restrict__ offsets, int experts, int64_t slots, int size,
                                         int nt, int room, int places, int depth, RowsJob& j) {
  const int64_t mt = group_tiles(offsets, experts, slots, size, true);
  const Turns t = turns_of((uint32_t)(mt * nt), (uint32_t)room, (uint32_t)places, depth);
  uint32_t id = blockIdx.x;
  j.slice = 0;
  j.slices = 1;
  j.place = 0;
  if (id < t.whole) {
    id = (id & 7u) * (t.whole >> 3) + (id >> 3);  // contiguous eighths to the XCDs (room is a multiple of 8)
  } else {
    const uint32_t at = id - t.whole;
    if (at >= t.left * t.slices) return false;
    j.slices = (int)t.slices;
    j.place = at;
    id = t.whole + at / t.slices;
    j.slice = __builtin_amdgcn_readfirstlane((int)(at % t.slices));
  }
  int64_t m;
  tile_of((uint32_t)__builtin_amdgcn_readfirstlane((int)id), mt, nt, m, j.n);
  j.g = group_tile(offsets, experts, slots, m, size, true);
  return j.g.group >= 0;
}

// A slice's sums as they stand in registers, `threads` lanes beside each other.
template <int TILES>
__device__ __forceinline__ void put_slice(f32x4* __restrict__ to, int threads, const f32x16 (&acc)[TILES]) {
#pragma unroll
  for (int i = 0; i < TILES; ++i) {
#pragma unroll
    for (int q = 0; q < 4; ++q)
      to[(i * 4 + q) * threads + threadIdx.x] =
          f32x4{acc[i][4 * q], acc[i][4 * q + 1], acc[i][4 * q + 2], acc[i][4 * q + 3]};
  }
}

// Rows behind the last expert's: zeros.
template <class T>
__device__ __forceinline__ void zero_rows(T* __restrict__ y, int64_t m0, int rows, int n0, int side, int outs) {
  constexpr int V = Piece<T>::V;
  for (int i = threadIdx.x; i < rows * (side / V); i += blockDim.x) {
    Piece<T> o;
    o.raw = typename Piece<T>::Raw{};
    o.store(y + (m0 + i / (side / V)) * outs, n0 + i % (side / V) * V, outs);
  }
}

// A piece of results on its way out: bias, then ReLU, then the mask.
template <class T>
__device__ __forceinline__ void finish(float (&v)[Piece<T>::V], const T* __restrict__ bias,
                                       const T* __restrict__ mask, bool relu, T* __restrict__ y, int at, int outs) {
  constexpr int V = Piece<T>::V;
  Piece<T> o, t;
  if (bias != nullptr) {
    t.load(bias, at, outs);
#pragma unroll
    for (int j = 0; j < V; ++j) v[j] += t.get(j);
  }
  if (mask != nullptr) t.load(mask, at, outs);
  o.raw = typename Piece<T>::Raw{};
#pragma unroll
  for (int j = 0; j < V; ++j) {
    if (relu) v[j] = v[j] <= 0.0f ? 0.0f : v[j];  // NaN stays
    if (mask != nullptr && t.get(j) <= 0.0f) v[j] = 0.0f;
    o.set(j, from_f32<T>(v[j]));
  }
  o.store(y, at, outs);
}

// Results of a wave's 32 x 32 on their way out, bias, ReLU and mask applied.
template <class T>
__device__ __forceinline__ void put_rows(const f32x16& acc, float* __restrict__ own, int row0, int col0, int64_t m0,
                                         int here, const T* __restrict__ bias, const T* __restrict__ mask, bool relu,
                                         T* __restrict__ y, int outs) {
  rows_of_tile<T>(acc, own, [&](int r, int c, float (&v)[Piece<T>::V]) {
    const int row = row0 + r, at = col0 + c;
    if (row >= here || at >= outs) return;
    finish<T>(v, bias, mask != nullptr ? mask + (m0 + row) * outs : nullptr, relu, y + (m0 + row) * outs, at, outs);
  });
}

// y (slots x outs) = x (slots x cols) W_e^T + b_e, W_e (outs x cols); BACK: y = x
// W_e with W_e (cols x outs), which is the input gradient.  relu: y = max(y, 0).
// mask (slots x outs): y = 0 where it is not above 0.
// A slice's sums go to `slices` (null: no tile is cut).
// 16-bit rows of any length at any place, through registers into LDS, the next
// step's loads under this one's products.  Bound: their latency, two barriers a
// step: 1023 rows of 7 experts, 2049 -> 1030 float16, in 25 us and 9 for the join.
template <class T, bool BACK>
__global__ __launch_bounds__(kGroupThreads) void k_group_rows(const T* __restrict__ x, int64_t xs,
                                                              const T* __restrict__ w, const T* __restrict__ b,
                                                              const T* __restrict__ mask,
                                                              const int32_t* __restrict__ offsets, T* __restrict__ y,
                                                              int64_t slots, int experts, int cols, int outs,
                                                              bool relu, int nt, int room, int places,
                                                              f32x4* __restrict__ slices) {
  using IA = PanelImage<T, true>;
  using IB = PanelImage<T, !BACK>;
  __shared__ __attribute__((aligned(16))) uint16_t lds[std::max(IA::kPlane + IB::kPlane, kOutbox)];
  uint16_t *const as = lds, *const bs = lds + IA::kPlane;
  RowsJob j;
  if (!rows_job(offsets, experts, slots, kSide, nt, room, places, cols, j)) return;
  const int64_t m0 = j.g.lo + j.g.tile * kSide;
  const int n0 = j.n * kSide, here = (int)min<int64_t>(kSide, j.g.hi - m0), outs_here = min(kSide, outs - n0);
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x / 64);
  const int row0 = wave / 4 * 64, col0 = wave % 4 * 32;
  if (j.g.group == experts) {
    if (j.slice == 0) zero_rows(y, m0, here, n0, kSide, outs);
    return;
  }
  const T* const we = w + (int64_t)j.g.group * cols * outs;
  const Panel<T> pa{x + m0 * xs, xs, here, cols};
  const Panel<T> pb = BACK ? Panel<T>{we + n0, outs, cols, outs_here} : Panel<T>{we + (int64_t)n0 * cols, cols, outs_here, cols};
  const int steps = (cols + kStepK - 1) / kStepK, first = j.first(steps), last = j.last(steps);
  Piece<T> ra[IA::kLoads], rb[IB::kLoads];
  TileSums<T> sums;
  sums.clear();
  IA::load(pa, first * kStepK, ra);
  IB::load(pb, first * kStepK, rb);
  for (int n = first; n < last; ++n) {
    IA::store(ra, as);
    IB::store(rb, bs);
    __syncthreads();
    if (n + 1 < last) {
      IA::load(pa, (n + 1) * kStepK, ra);
      IB::load(pb, (n + 1) * kStepK, rb);
    }
    sums.template step<IA, IB>(as, bs, row0, col0);
    __syncthreads();
  }
  if (j.slices > 1) {
    put_slice<2>(slices + j.place * (kSide * kSide / 4), kGroupThreads, sums.acc);
    return;
  }
  float* const own = reinterpret_cast<float*>(lds) + 1024 * wave;  // every wave is done with the panels
#pragma unroll
  for (int i = 0; i < 2; ++i)
    put_rows<T>(sums.acc[i], own, row0 + 32 * i, n0 + col0, m0, here,
                b != nullptr ? b + (int64_t)j.g.group * outs : nullptr, mask, relu, y, outs);
}

// The same for 16-bit rows in whole 16-byte pieces, or for float32 rows laid out
// as three bfloat16 pieces a value (xp and wp elements apart): panels straight
// from memory to LDS.  A slice's sums go to `slices` (null: no tile is cut) as
// they stand in registers.
// Bound: the matrix cores and what stands between two steps (one barrier, then the
// operands' first reads): 16384 rows of 8 experts, 2048 -> 4096 bfloat16 in 339 us
// (0.81 PFLOP/s; the library's one product of that size without experts 242), 41% of
// the cycles matrix-busy; 8192 rows of 4, 1024 -> 2048 float32 in 227 us (152
// TFLOP/s, the library's float32 135), 46%.  Reading the operands of the next 16 of
// the sum under the products of these changed nothing.
template <class T, bool BACK, int BM, int BN, int WM, int WN>
__global__ __launch_bounds__(64 * WM * WN) void k_group_rows_fast(
    const Piece16<T>* __restrict__ x, int64_t xs, int64_t xp, const Piece16<T>* __restrict__ w, int64_t ws, int64_t wp,
    const T* __restrict__ b, const T* __restrict__ mask, const int32_t* __restrict__ offsets, T* __restrict__ y,
    int64_t slots, int experts, int cols, int outs, bool relu, int nt, int room, int places, f32x4* __restrict__ slices) {
  using E = Piece16<T>;
  using Tile = FastTile<E, kPieces<T>, true, !BACK, BM, BN, WM, WN, false>;
  __shared__ __attribute__((aligned(16))) uint16_t s0[Tile::kStage], s1[Tile::kStage];
  RowsJob j;
  if (!rows_job(offsets, experts, slots, BM, nt, room, places, cols, j)) return;
  const GroupTile& g = j.g;
  const int64_t m0 = g.lo + g.tile * BM;
  const int n0 = j.n * BN, here = (int)min<int64_t>(BM, g.hi - m0), outs_here = min(BN, outs - n0);
  if (g.group == experts) {
    if (j.slice == 0) zero_rows(y, m0, here, n0, BN, outs);
    return;
  }
  // W_e has a row for each output, or (BACK) for each input
  const E* const we = w + (int64_t)g.group * (BACK ? cols : outs) * ws;
  typename Tile::A pa(Panel<E>{x + m0 * xs, xs, here, cols}, xp);
  typename Tile::B pb(BACK ? Panel<E>{we + n0, ws, cols, min(BN, (int)ws - n0)}
                           : Panel<E>{we + (int64_t)n0 * ws, ws, outs_here, cols}, wp);
  const int steps = (cols + Tile::KS - 1) / Tile::KS, first = j.first(steps), last = j.last(steps);
  pa.base += first * pa.step;
  pb.base += first * pb.step;
  Tile t;
  t.run(pa, pb, min(cols, last * Tile::KS) - first * Tile::KS, false, s0, s1);
  if (j.slices > 1) {
#pragma unroll
    for (int i = 0; i < Tile::TM; ++i)
      put_slice<Tile::TN>(slices + j.place * (BM * BN / 4) + i * Tile::TN * 4 * (64 * Tile::kWaves), 64 * Tile::kWaves, t.acc[i]);
    return;
  }
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x / 64);
  float* const own = reinterpret_cast<float*>(s0) + 1024 * wave;
  static_assert(Tile::kWaves * 2048 <= Tile::kStage, "room");
#pragma unroll
  for (int i = 0; i < Tile::TM; ++i) {
#pragma unroll
    for (int k = 0; k < Tile::TN; ++k)
      put_rows<T>(t.acc[i][k], own, wave / WN * (BM / WM) + 32 * i, n0 + wave % WN * (BN / WN) + 32 * k, m0, here,
                  b != nullptr ? b + (int64_t)g.group * outs : nullptr, mask, relu, y, outs);
  }
}

// The cut tiles: slices added in their order.  Workgroup (tile, one 32 x 32 of each of its waves').
template <class T, int BM, int BN, int WM, int WN>
__global__ __launch_bounds__(64 * WM * WN) void k_group_rows_join(const T* __restrict__ b, const T* __restrict__ mask,
                                                                  const int32_t* __restrict__ offsets,
                                                                  T* __restrict__ y, int64_t slots, int experts,
                                                                  int depth, int outs, bool relu, int nt, int room, int places,
                                                                  const f32x4* __restrict__ slices) {
  constexpr int kWaves = WM * WN, TN = BN / WN / 32;
  __shared__ __attribute__((aligned(16))) float room_of[kWaves][1024];
  const int64_t mt = group_tiles(offsets, experts, slots, BM, true);
  const Turns turns = turns_of((uint32_t)(mt * nt), (uint32_t)room, (uint32_t)places, depth);
  if (turns.slices == 1 || blockIdx.x >= turns.left) return;
  int64_t m;
  int n;
  tile_of(turns.whole + blockIdx.x, mt, nt, m, n);
  const GroupTile g = group_tile(offsets, experts, slots, m, BM, true);
  if (g.group < 0 || g.group == experts) return;
  const int64_t m0 = g.lo + g.tile * BM;
  const int n0 = n * BN, here = (int)min<int64_t>(BM, g.hi - m0), ij = (int)blockIdx.y;
  const f32x4* from = slices + (int64_t)blockIdx.x * turns.slices * (BM * BN / 4) + (int64_t)ij * 4 * (64 * kWaves) + threadIdx.x;
  f32x16 acc = f32x16{};
#pragma unroll 4
  for (uint32_t s = 0; s < turns.slices; ++s, from += BM * BN / 4) {
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const f32x4 v = from[q * (64 * kWaves)];
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[4 * q + e] += v[e];
    }
  }
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x / 64);
  put_rows<T>(acc, room_of[wave], wave / WN * (BM / WM) + 32 * (ij / TN), n0 + wave % WN * (BN / WN) + 32 * (ij % TN), m0,
              here, b != nullptr ? b + (int64_t)g.group * outs : nullptr, mask, relu, y, outs);
}

// The same for float32 rows as they are, on the float32 matrix cores, which bound
// it (a product of 32 x 32 x 2 takes 64 cycles): the whole call for 8191 rows of 4
// experts, 2049 -> 1030, takes 355 us, laid out in pieces first 291.
template <bool BACK, int BM, int BN, int WM, int WN>
__global__ __launch_bounds__(kWideThreads) void k_group_rows_wide(const float* __restrict__ x, int64_t xs,
                                                                  const float* __restrict__ w,
                                                                  const float* __restrict__ b,
                                                                  const float* __restrict__ mask,
                                                                  const int32_t* __restrict__ offsets,
                                                                  float* __restrict__ y, int64_t slots, int experts,
                                                                  int cols, int outs, bool relu, int nt, int room, int places,
                                                                  f32x4* __restrict__ slices) {
  using Tile = WideTile<true, !BACK, BM, BN, WM, WN>;
  __shared__ __attribute__((aligned(16))) float lds[Tile::kRoom];
  RowsJob j;
  if (!rows_job(offsets, experts, slots, BM, nt, room, places, cols, j)) return;
  const GroupTile& g = j.g;
  const int64_t m0 = g.lo + g.tile * BM;
  const int n0 = j.n * BN, here = (int)min<int64_t>(BM, g.hi - m0), outs_here = min(BN, outs - n0);
  if (g.group == experts) {
    if (j.slice == 0) zero_rows(y, m0, here, n0, BN, outs);
    return;
  }
  const float* const we = w + (int64_t)g.group * cols * outs;
  const int steps = (cols + kStepK - 1) / kStepK;
  Tile t;
  t.run(Panel<float>{x + m0 * xs, xs, here, cols},
        BACK ? Panel<float>{we + n0, outs, cols, outs_here} : Panel<float>{we + (int64_t)n0 * cols, cols, outs_here, cols},
        j.first(steps) * kStepK, min(cols, j.last(steps) * kStepK), lds, [](auto&) {});
  if (j.slices > 1) {
#pragma unroll
    for (int i = 0; i < Tile::TM; ++i)
      put_slice<Tile::TN>(slices + j.place * (BM * BN / 4) + i * Tile::TN * 4 * kWideThreads, kWideThreads, t.acc[i]);
    return;
  }
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x / 64);
#pragma unroll
  for (int i = 0; i < Tile::TM; ++i) {
#pragma unroll
    for (int k = 0; k < Tile::TN; ++k)
      put_rows<float>(t.acc[i][k], lds + 1024 * wave, wave / WN * (BM / WM) + 32 * i, n0 + wave % WN * (BN / WN) + 32 * k,
                      m0, here, b != nullptr ? b + (int64_t)g.group * outs : nullptr, mask, relu, y, outs);
  }
}

// A few rows an expert (single tokens): workgroup = 16 outputs of an expert and 64
// of its rows, the sum shared out over its waves, whose loads go to registers, eight
// lines of 128 bytes a row of W in flight: nothing waits for anything but memory.
// Bound: HBM, the weights of the experts that have rows.
constexpr int kTokenThreads = 256, kTokenWaves = 4, kTokenRows = 64;
template <class T>
struct Tokens {
  static constexpr int V = Piece<T>::V, kLine = 128 / (int)sizeof(T), kAhead = 8;  // values of a line; lines in flight
  f32x4 sums[kTokenWaves][4][64];

  // The lane's two pieces of a line from k on: 32 bytes at 32 (l / 16).
  __device__ __forceinline__ static void load(Piece<T> (&p)[2], const T* __restrict__ row, int k, int cols, bool whole) {
    const int at = k + 2 * V * ((int)(threadIdx.x & 63) >> 4);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      if (whole) p[i].raw = *reinterpret_cast<const typename Piece<T>::Raw*>(row + at + V * i);
      else if (at + V * i < cols) p[i].load(row, at + V * i, cols);
      else p[i].raw = typename Piece<T>::Raw{};
    }
  }
  __device__ __forceinline__ static f32x4 product(const Piece<T>& x, const Piece<T>& w, f32x4 c) {
    if constexpr (std::is_same_v<T, float>) {
#pragma unroll
      for (int j = 0; j < 4; ++j) c = __builtin_amdgcn_mfma_f32_16x16x4f32(x.get(j), w.get(j), c, 0, 0, 0);
      return c;
    } else {
      return mma16<T>(__builtin_bit_cast(s16x8, x.raw), __builtin_bit_cast(s16x8, w.raw), c);
    }
  }
  // Rows 0 .. here - 1 of x, up to 16 MT of them, times outputs n0 .. of W.
  template <int MT>
  __device__ __forceinline__ void run(const T* __restrict__ x, int64_t xs, int here, const T* __restrict__ w,
                                      const T* __restrict__ bias, T* __restrict__ y, int n0, int cols, int outs,
                                      bool relu) {
    const int lane = threadIdx.x & 63, c = lane & 15, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x / 64);
    const T* __restrict__ wr = w + (int64_t)min(n0 + c, outs - 1) * cols;
    const T* __restrict__ xr[MT];
    f32x4 acc[MT];
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      xr[m] = x + (int64_t)min(16 * m + c, here - 1) * xs;
      acc[m] = f32x4{};
    }
    const int lines = (cols + kLine - 1) / kLine, first = lines * wave / kTokenWaves, last = lines * (wave + 1) / kTokenWaves;
    for (int n = first; n < last; n += kAhead) {
      Piece<T> p[kAhead][2];
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        if (n + u < last) load(p[u], wr, (n + u) * kLine, cols, (n + u + 1) * kLine <= cols);
      }
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        if (n + u >= last) break;
#pragma unroll
        for (int m = 0; m < MT; ++m) {
          Piece<T> q[2];
          load(q, xr[m], (n + u) * kLine, cols, (n + u + 1) * kLine <= cols);
#pragma unroll
          for (int i = 0; i < 2; ++i) acc[m] = product(q[i], p[u][i], acc[m]);
        }
      }
    }
#pragma unroll
    for (int m = 0; m < MT; ++m) sums[wave][m][lane] = acc[m];
    __syncthreads();
    // result register r of lane l is row 4 (l / 16) + r, output l % 16
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      const int row = (int)threadIdx.x / 16, n = (int)threadIdx.x % 16, at = n0 + n;
      if (16 * m + row >= here || at >= outs) continue;
      float v = 0.0f;
#pragma unroll
      for (int i = 0; i < kTokenWaves; ++i) v += sums[i][m][16 * (row / 4) + n][row % 4];
      if (bias != nullptr) v += to_f32(bias[at]);
      if (relu) v = v <= 0.0f ? 0.0f : v;  // NaN stays
      y[(int64_t)(16 * m + row) * outs + at] = from_f32<T>(v);
    }
  }
};
template <class T>
__global__ __launch_bounds__(kTokenThreads) void k_group_tokens(const T* __restrict__ x, int64_t xs,
                                                                const T* __restrict__ w, const T* __restrict__ b,
                                                                const int32_t* __restrict__ offsets,
                                                                T* __restrict__ y, int64_t slots, int experts, int cols,
                                                                int outs, bool relu) {
  __shared__ Tokens<T> tokens;
  const int e = (int)blockIdx.y, n0 = (int)blockIdx.x * 16;
  const GroupRows g = group_rows(offsets, experts, slots, e);
  const int64_t m0 = g.lo + (int64_t)blockIdx.z * kTokenRows;
  if (m0 >= g.hi) return;
  const int here = (int)min<int64_t>(kTokenRows, g.hi - m0);
  if (e == experts) {
    zero_rows(y, m0, here, n0, 16, outs);
    return;
  }
  const T* const we = w + (int64_t)e * cols * outs;
  const T* const be = b != nullptr ? b + (int64_t)e * outs : nullptr;
  if (here <= 16) tokens.template run<1>(x + m0 * xs, xs, here, we, be, y + m0 * outs, n0, cols, outs, relu);
  else tokens.template run<4>(x + m0 * xs, xs, here, we, be, y + m0 * outs, n0, cols, outs, relu);
}

// A weight gradient's workgroup: which piece (chunk of rows, or expert) and which
// tile of dW.  A piece's tiles are dealt to the XCDs in contiguous shares, so that
// each XCD works on every piece (experts differ in rows) and tiles that share
// panels meet in its L2.
struct GradTile {
  int64_t piece;
  int m, n;
};
__device__ __forceinline__ GradTile grad_tile(int mt, int nt) {
  const uint32_t tiles = (uint32_t)(mt * nt), x = blockIdx.x % tiles;
  const uint32_t xcd = x & 7u, q = tiles >> 3, rem = tiles & 7u, at = xcd * q + min(xcd, rem) + (x >> 3);
  return GradTile{blockIdx.x / tiles, (int)(at / (uint32_t)nt), (int)(at % (uint32_t)nt)};
}
// Its rows.  Pieces that are whole experts come in the order of their rows, most
// first (up to 64 experts): what starts last is short.
__device__ __forceinline__ GroupTile grad_rows(const int32_t* __restrict__ offsets, int experts, int64_t slots,
                                               int64_t piece, int64_t chunk, bool chunks) {
  if (chunks) return group_tile(offsets, experts, slots, piece, chunk, false);
  GroupTile g;
  g.group = (int)piece;
  g.tile = 0;
  if (experts <= 64) {
    const int e = (int)(threadIdx.x & 63);
    int mine = -1;
    if (e < experts) {
      const GroupRows r = group_rows(offsets, experts, slots, e);
      mine = (int)(r.hi - r.lo);
    }
    int before = 0;
    for (int i = 0; i < experts; ++i) {
      const int other = __builtin_amdgcn_readlane(mine, i);
      before += other > mine || (other == mine && i < e) ? 1 : 0;
    }
    const uint64_t at = __ballot(e < experts && before == (int)piece);
    g.group = __ffsll((unsigned long long)at) - 1;
  }
  const GroupRows r = group_rows(offsets, experts, slots, g.group);
  g.lo = r.lo;
  g.hi = r.hi;
  return g;
}

// dW_e (outs x cols) and db_e of a chunk of the expert's rows.  part null: the
// chunk is all of them and the sums go out rounded to T; else they are float32
// in the chunk's place.
template <class T>
__global__ __launch_bounds__(kGroupThreads) void k_group_weight_grad(const T* __restrict__ dy, int64_t dys,
                                                                     const T* __restrict__ x, int64_t xs,
                                                                     const int32_t* __restrict__ offsets,
                                                                     T* __restrict__ dw, T* __restrict__ db,
                                                                     float* __restrict__ part, int64_t slots,
                                                                     int experts, int cols, int outs, int64_t chunk,
                                                                     int mt, int nt) {
  using I = PanelImage<T, false>;
  constexpr int V = Piece<T>::V;
  __shared__ __attribute__((aligned(16))) uint16_t room[std::max(2 * I::kPlane, kOutbox)];
  uint16_t *const as = room, *const bs = room + I::kPlane;
  const GradTile at = grad_tile(mt, nt);
  const int64_t piece = at.piece;
  const int m0 = at.m * kSide, n0 = at.n * kSide;
  const GroupTile g = grad_rows(offsets, experts, slots, piece, chunk, part != nullptr);
  if (g.group < 0) return;
  const int64_t lo = g.lo + g.tile * chunk;
  const int rows = (int)min<int64_t>(chunk, g.hi - lo);
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x / 64);
  const int row0 = wave / 4 * 64, col0 = wave % 4 * 32;
  const Panel<T> pa{dy + lo * dys + m0, dys, rows, min(kSide, outs - m0)};
  const Panel<T> pb{x + lo * xs + n0, xs, rows, min(kSide, cols - n0)};
  Piece<T> ra[I::kLoads], rb[I::kLoads];
  TileSums<T> sums;
  sums.clear();
  float bias[V];
#pragma unroll
  for (int j = 0; j < V; ++j) bias[j] = 0.0f;
  if (rows > 0) {
    I::load(pa, 0, ra);
    I::load(pb, 0, rb);
  }
  for (int k = 0; k < rows; k += kStepK) {
    I::store(ra, as);
    I::store(rb, bs);
    if (n0 == 0) {
#pragma unroll
      for (int i = 0; i < I::kLoads; ++i) {
#pragma unroll
        for (int j = 0; j < V; ++j) bias[j] += ra[i].get(j);
      }
    }
    __syncthreads();
    if (k + kStepK < rows) {
      I::load(pa, k + kStepK, ra);
      I::load(pb, k + kStepK, rb);
    }
    sums.template step<I, I>(as, bs, row0, col0);
    __syncthreads();
  }
  const int64_t nw = (int64_t)outs * cols;
  float* const own = reinterpret_cast<float*>(room) + 1024 * wave;  // every wave is done with the panels
  float* const mine = part != nullptr ? part + piece * (nw + outs) : nullptr;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    auto put = [&](auto type, auto* to) {
      using O = decltype(type);
      rows_of_tile<O>(sums.acc[i], own, [&](int r, int c, float (&v)[Piece<O>::V]) {
        const int row = m0 + row0 + 32 * i + r, col = n0 + col0 + c;
        if (row >= outs || col >= cols) return;
        Piece<O> o;
        o.raw = typename Piece<O>::Raw{};
#pragma unroll
        for (int j = 0; j < Piece<O>::V; ++j) o.set(j, from_f32<O>(v[j]));
        o.store(to + (int64_t)row * cols, col, cols);
      });
    };
    if (mine != nullptr) put(float{}, mine);
    else if (dw != nullptr) put(T{}, dw + g.group * nw);
  }
  if (n0 != 0 || (mine == nullptr && db == nullptr)) return;
  // a thread's columns again every kRowPieces threads
  float* const meet = reinterpret_cast<float*>(room);
  static_assert(kGroupThreads * V * 2 <= kOutbox, "room");
  __syncthreads();
#pragma unroll
  for (int j = 0; j < V; ++j) meet[threadIdx.x * V + j] = bias[j];
  __syncthreads();
  for (int c = threadIdx.x; c < kSide; c += kGroupThreads) {
    if (m0 + c >= outs) continue;
    float t = 0.0f;
#pragma unroll
    for (int i = 0; i < kGroupThreads / I::kRowPieces; ++i) t += meet[i * kSide + c];
    if (mine != nullptr) mine[nw + m0 + c] = t;
    else db[(int64_t)g.group * outs + m0 + c] = from_f32<T>(t);
  }
}

// The same for 16-bit rows in whole 16-byte pieces, or float32 rows laid out in
// bfloat16 pieces, straight from memory to LDS; db from products with ones.
// Bound: as k_group_rows_fast; 16384 rows of 8 experts, 2048 and 4096 wide, bfloat16
// in 308 us (0.89 PFLOP/s), 8192 rows of 4, 1024 and 2048, float32 in 262.
template <class T, int BM, int BN, int WM, int WN>
__global__ __launch_bounds__(64 * WM * WN) void k_group_weight_grad_fast(
    const Piece16<T>* __restrict__ dy, int64_t dys, int64_t dyp, const Piece16<T>* __restrict__ x, int64_t xs, int64_t xp,
    const int32_t* __restrict__ offsets, T* __restrict__ dw, T* __restrict__ db, float* __restrict__ part,
    int64_t slots, int experts, int cols, int outs, int64_t chunk, int mt, int nt) {
  using E = Piece16<T>;
  using Tile = FastTile<E, kPieces<T>, false, false, BM, BN, WM, WN, true>;
  static_assert(Tile::TM <= WN, "a wave of the row for each tile of rows");
  __shared__ __attribute__((aligned(16))) uint16_t s0[Tile::kStage], s1[Tile::kStage];
  static_assert(Tile::kWaves * 2048 <= Tile::kStage, "room");
  const GradTile at = grad_tile(mt, nt);
  const int64_t piece = at.piece;
  const int m0 = at.m * BM, n0 = at.n * BN;
  const GroupTile g = grad_rows(offsets, experts, slots, piece, chunk, part != nullptr);
  if (g.group < 0) return;
  const int64_t lo = g.lo + g.tile * chunk;
  const int rows = (int)min<int64_t>(chunk, g.hi - lo);
  const typename Tile::A pa(Panel<E>{dy + lo * dys + m0, dys, rows, (int)min<int64_t>(BM, whole8(outs) - m0)}, dyp);
  const typename Tile::B pb(Panel<E>{x + lo * xs + n0, xs, rows, (int)min<int64_t>(BN, whole8(cols) - n0)}, xp);
  Tile t;
  t.run(pa, pb, rows, n0 == 0, s0, s1);
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x / 64), wn = wave % WN;
  const int row0 = wave / WN * (BM / WM), col0 = wn * (BN / WN);
  const int64_t nw = (int64_t)outs * cols;
  float* const own = reinterpret_cast<float*>(s0) + 1024 * wave;
  float* const mine = part != nullptr ? part + piece * (nw + outs) : nullptr;
#pragma unroll
  for (int i = 0; i < Tile::TM; ++i) {
#pragma unroll
    for (int j = 0; j < Tile::TN; ++j) {
      auto put = [&](auto type, auto* to) {
        using O = decltype(type);
        rows_of_tile<O>(t.acc[i][j], own, [&](int r, int c, float (&v)[Piece<O>::V]) {
          const int row = m0 + row0 + 32 * i + r, col = n0 + col0 + 32 * j + c;
          if (row >= outs || col >= cols) return;
          Piece<O> o;
          o.raw = typename Piece<O>::Raw{};
#pragma unroll
          for (int e = 0; e < Piece<O>::V; ++e) o.set(e, from_f32<O>(v[e]));
          o.store(to + (int64_t)row * cols, col, cols);
        });
      };
      if (mine != nullptr) put(float{}, mine);
      else if (dw != nullptr) put(T{}, dw + g.group * nw);
    }
  }
  const int row = m0 + row0 + 32 * wn + (int)(threadIdx.x & 31);
  if (n0 != 0 || wn >= Tile::TM || (threadIdx.x & 63) >= 32 || row >= outs) return;
  if (mine != nullptr) mine[nw + row] = t.ones;
  else if (db != nullptr) db[(int64_t)g.group * outs + row] = from_f32<T>(t.ones);
}

// The same for float32 rows.
template <int BM, int BN, int WM, int WN>
__global__ __launch_bounds__(kWideThreads) void k_group_weight_grad_wide(
    const float* __restrict__ dy, int64_t dys, const float* __restrict__ x, int64_t xs,
    const int32_t* __restrict__ offsets, float* __restrict__ dw, float* __restrict__ db, float* __restrict__ part,
    int64_t slots, int experts, int cols, int outs, int64_t chunk, int mt, int nt) {
  using Tile = WideTile<false, false, BM, BN, WM, WN>;
  __shared__ __attribute__((aligned(16))) float room[Tile::kRoom];
  const GradTile at = grad_tile(mt, nt);
  const int64_t piece = at.piece;
  const int m0 = at.m * BM, n0 = at.n * BN;
  const GroupTile g = grad_rows(offsets, experts, slots, piece, chunk, part != nullptr);
  if (g.group < 0) return;
  const int64_t lo = g.lo + g.tile * chunk;
  const int rows = (int)min<int64_t>(chunk, g.hi - lo);
  f32x4 bias = f32x4{};
  Tile t;
  t.run(Panel<float>{dy + lo * dys + m0, dys, rows, min(BM, outs - m0)},
        Panel<float>{x + lo * xs + n0, xs, rows, min(BN, cols - n0)}, 0, rows, room, [&](auto& pieces) {
          if (n0 != 0) return;
          for (auto& p : pieces) bias += f32x4{p.get(0), p.get(1), p.get(2), p.get(3)};
        });
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x / 64);
  const int row0 = wave / WN * (BM / WM), col0 = wave % WN * (BN / WN);
  const int64_t nw = (int64_t)outs * cols;
  float* const mine = part != nullptr ? part + piece * (nw + outs) : nullptr;
  float* const to = mine != nullptr ? mine : dw != nullptr ? dw + g.group * nw : nullptr;
#pragma unroll
  for (int i = 0; i < Tile::TM; ++i) {
#pragma unroll
    for (int j = 0; j < Tile::TN; ++j) {
      rows_of_tile<float>(t.acc[i][j], room + 1024 * wave, [&](int r, int c, float (&v)[4]) {
        const int row = m0 + row0 + 32 * i + r, col = n0 + col0 + 32 * j + c;
        if (to == nullptr || row >= outs || col >= cols) return;
        Piece<float> o;
#pragma unroll
        for (int e = 0; e < 4; ++e) o.set(e, v[e]);
        o.store(to + (int64_t)row * cols, col, cols);
      });
    }
  }
  if (n0 != 0 || (mine == nullptr && db == nullptr)) return;
  // a thread's columns again every kRowPieces threads
  __syncthreads();
  *reinterpret_cast<f32x4*>(room + 4 * threadIdx.x) = bias;
  __syncthreads();
  if ((int)threadIdx.x >= BM || m0 + (int)threadIdx.x >= outs) return;
  float sum = 0.0f;
#pragma unroll
  for (int i = 0; i < kWideThreads / Tile::A::kRowPieces; ++i) sum += room[i * BM + threadIdx.x];
  if (mine != nullptr) mine[nw + m0 + threadIdx.x] = sum;
  else db[(int64_t)g.group * outs + m0 + threadIdx.x] = sum;
}

// dW and db of expert blockIdx.y: its chunks' sums in the chunks' order.
template <class T>
__global__ __launch_bounds__(256) void k_group_chunk_sum(const float* __restrict__ part,
                                                         const int32_t* __restrict__ offsets, T* __restrict__ dw,
                                                         T* __restrict__ db, int64_t slots, int experts, int64_t nw,
                                                         int outs, int64_t chunk, int64_t chunks) {
  const int e = (int)blockIdx.y;
  const GroupSpan g = group_span(offsets, experts, slots, chunk, e);
  const int64_t before = g.before, mine = g.tiles;
  const int64_t n = nw + outs, at = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (at >= n) return;
  float t = 0.0f;
#pragma unroll 8
  for (int64_t k = before; k < min<int64_t>(before + mine, chunks); ++k) t += part[k * n + at];
  if (at < nw) {
    if (dw != nullptr) dw[e * nw + at] = from_f32<T>(t);
  } else if (db != nullptr) {
    db[(int64_t)e * outs + (at - nw)] = from_f32<T>(t);
  }
}

int64_t tiles_of(int64_t n, int64_t tile) { return (n + tile - 1) / tile; }

// Rows of a weight gradient's chunk: as many chunks as fill the card, of 256
// rows at least and of kMaxGroupChunk at most.
//
// None where the experts' tiles fill the card: the chunks' float32 sums go to memory
// and back.  But up to kMaxWhole places only, which one expert may have all of: its
// sum is then that long, and its few workgroups work alone.  us with gradients, whole
// and in chunks (in brackets all places of one expert): bfloat16, 2048 -> 4096, 16384 of
// 8 909 and 1269 (1017, 1057), 32768 of 8 1703 and 2083 (1959, 1824), 65536 of 8 3290 and
// 3648 (4070, 3572); 1024 -> 1024, 16384 of 64 268 and 650 (548, 407), 65536 of 64 709 and
// 995 (2145, 796); 2048 -> 2048, 32768 of 64 1182 and 2557 (1535, 1667), 131072 of 8 4504
// and 3751; float32, 1024 -> 1024, 32768 of 64 1887 and 2204 (2976, 1997); on the wrong
// side 32768 of 16, 1536 -> 1536 bfloat16, 937 and 847.
constexpr int64_t kMaxGroupChunk = 8192, kMaxWhole = 32768;
struct GradPlan {
  int bm, bn, mt, nt;     // tiles of dW
  int64_t chunk, chunks;  // chunks 0: a workgroup takes all of an expert's rows
};
GradPlan grad_plan(int64_t slots, int experts, int64_t cols, int64_t outs, int bm, int bn) {
  GradPlan p;
  p.bm = bm;
  p.bn = bn;
  p.mt = (int)tiles_of(outs, bm);
  p.nt = (int)tiles_of(cols, bn);
  const int64_t tiles = (int64_t)p.mt * p.nt;
  const int64_t want = std::max<int64_t>(1, 512 / tiles);  // chunks in all
  p.chunk = std::min(kMaxGroupChunk, std::max<int64_t>(256, tiles_of(tiles_of(slots, want), 64) * 64));
  p.chunks = most_tiles(slots, experts, p.chunk);
  if (slots <= p.chunk || (tiles * experts >= 512 && slots <= kMaxWhole)) {
    p.chunk = std::max<int64_t>(slots, 1);
    p.chunks = 0;
  }
  return p;
}

// 16-bit rows of whole 16-byte pieces at multiples of 16 bytes, a panel's within 32
// bits of its first: those the fast kernels take as they are.
bool whole_pieces(const void* p, int64_t stride) {
  return reinterpret_cast<uintptr_t>(p) % 16 == 0 && stride % 8 == 0 && stride <= (1 << 22);
}

// 16-bit tiles: 256 where there are enough of them, else 128.  us, bfloat16, tiles of
// 256 and 128.  Over rows, 128 tiles of 256 (8192 rows of 4 experts, 2048 -> 1024) 73 and
// 59, 192 (8192 of 4, 2048 -> 1536; 12288 of 8, 4096 -> 1024) 74 and 83, 122 and 142, 1024
// (16384 of 8, 2048 -> 4096) 310 and 345; between them whole turns of the card decide:
// 256 (8192 of 8, 2048 -> 2048; 16384 of 8, 2048 -> 1024) 103 and 103, 97 and 87, 512 (16384
// of 8, 2048 -> 2048) 168 and 162.  Weight gradients, whole or in chunks, with the rest of
// the pass: 256 tiles (4096 of 4, 2048 -> 2048) 293 and 180, 512 (16384 of 8, 2048 -> 2048;
// 8192 of 32, 1024 -> 1024; 8192 of 8, 2048 -> 2048) 586 and 517, 156 and 148, 302 and 311,
// 640 (16384 of 10, 2048 -> 2048) 556 and 528, 768 (16384 of 16, 1536 -> 2048; of 12, 2048 ->
// 2048) 420 and 441, 563 and 548, 1024 (16384 of 8, 2048 -> 4096; of 64, 1024 -> 1024) 916
// and 949, 266 and 282; in chunks (65536 of 8, 2048 -> 4096; of 64, 1024 -> 1024) 3662 and
// 3901, 994 and 1014.
int rows_side(int64_t slots, int64_t outs) {
  return outs > 128 && slots / 256 * tiles_of(outs, 256) >= 192 ? 256 : 128;
}
int grad_side(int experts, int64_t cols, int64_t outs) {
  return outs > 128 && cols > 128 && tiles_of(outs, 256) * tiles_of(cols, 256) * experts >= 768 ? 256 : 128;
}
// Float32 tiles: 32, 64 or 128 outputs, as few as hold them; 32 rows where an expert
// has no more on average (2048 rows of 128 experts, 512 -> 512, 48 us, with 128 91).
int wide_side(int64_t n) { return n <= 32 ? 32 : n <= 64 ? 64 : 128; }
int wide_rows(int64_t slots, int experts) { return slots <= 32 * (int64_t)experts ? 32 : 128; }

// The plan of a weight gradient for its type (wide: float32) and alignment (fast: whole pieces).
GradPlan chosen_plan(int64_t slots, int experts, int64_t cols, int64_t outs, bool wide, bool fast) {
  if (!wide) {
    const int side = fast ? grad_side(experts, cols, outs) : kSide;
    return grad_plan(slots, experts, cols, outs, side, side);
  }
  int bm = wide_side(outs), bn = wide_side(cols);
  if (bm < 128 && bn < 128) bm = bn = 64;
  return grad_plan(slots, experts, cols, outs, bm, bn);
}

// That of float32 rows laid out in pieces: 256 x 128 where such tiles fill the chip
// without chunks and an expert has rows for a long sum, else 128 x 128.  us with
// gradients, 256 x 128 and 128 x 128: 16384 rows of 8 experts, 2048 -> 2048, 2689 and
// 2790; 16384 of 4, 2048 -> 4096, 4922 and 5150; short sums: 16384 of 16, 1024 ->
// 1024, 1009 and 859; 8192 of 8, 1024 -> 2048, 871 and 806; few tiles: 16384 of 8, 1024
// -> 1024, 861 and 797; 8192 of 4, 1024 -> 2048, 805 and 779; but 16384 of 2, 1024 ->
// 1024, 732 and 747.
GradPlan laid_plan(int64_t slots, int experts, int64_t cols, int64_t outs) {
  const bool tall = tiles_of(outs, 256) * tiles_of(cols, 128) * experts >= 512 && slots >= 2048 * (int64_t)experts;
  return grad_plan(slots, experts, cols, outs, tall ? 256 : 128, 128);
}

// A matrix as the fast kernels read it.
struct Laid {
  const void* base;
  int64_t stride, plane;
};

// Takes places for laid out rows off a workspace; without one it counts bytes.
struct Layouts {
  char* work;
  int64_t used = 0;
  int64_t take(int64_t bytes) {
    const int64_t at = used;
    used += (bytes + 15) / 16 * 16;
    return at;
  }
  static int64_t bytes_of(int type, int64_t rows, int64_t cols) {
    return (type == SPHOPS_F32 ? 3 : 1) * rows * whole8(cols) * 2;
  }
};

template <class T>
Laid lay_out(Layouts& l, const T* x, int64_t stride, int64_t rows, int64_t cols, hipStream_t st) {
  const int64_t ld = whole8(cols);
  uint16_t* const to = reinterpret_cast<uint16_t*>(
      l.work + l.take(Layouts::bytes_of(std::is_same_v<T, float> ? SPHOPS_F32 : SPHOPS_BF16, rows, cols)));
  const int64_t groups = std::min<int64_t>(tiles_of(rows * ld / 8, kLayThreads), 16384);
  if (groups > 0) {
    hipLaunchKernelGGL((k_lay_out<T>), dim3((uint32_t)groups), dim3(kLayThreads), 0, st, x, stride, to, rows, (int)cols,
                       (int)ld);
    SPHOPS_LAUNCHED();
  }
  return Laid{to, ld, rows * ld};
}

// Whether a layer's products have their operands laid out first: float32, and
// 16-bit rows that are not whole pieces.  The copies pay where experts have rows
// enough for their weights' and each value meets enough others, and not where they
// take more than 16 GB.  us so, and as they are: float16 8191 rows of 4 experts, 2049
// -> 1030, 98 and 104, with gradients 302 and 494; 1023 rows of 7 60 and 51, 200 and
// 149; float32 291 and 355, 951 and 1567; 4000 rows of 16 305 and 286.
bool lays_out(int type, int64_t slots, int experts, int64_t cols, int64_t outs, bool back) {
  if (cols < 256 || outs < 256 || slots < 512 * (int64_t)experts) return false;
  if (Layouts::bytes_of(type, slots, cols + outs) + Layouts::bytes_of(type, experts * outs, cols) > int64_t(1) << 34) return false;
  return slots * cols * outs >= (int64_t(1) << (type != SPHOPS_F32 && !back ? 35 : 32));
}

// A product over rows: its tiles, how many of their workgroups the card holds, and
// whether tiles may be cut: sums of two slices' depth.
struct RowsPlan {
  int bm, bn, room;
  bool cut;
  int64_t tiles = 0;  // the most that there can be
  int places() const { return cut ? (int)slice_places(tiles, room) : 0; }
  int64_t slices_bytes() const { return (int64_t)places() * bm * bn * 4; }
};
RowsPlan rows_plan(int type, bool fast, int64_t slots, int experts, int64_t cols, int64_t outs) {
  RowsPlan p{128, 128, 512, cols >= 2 * kSliceDepth, 0};
  if (type != SPHOPS_F32) {
    if (fast && rows_side(slots, outs) == 256) p.bm = p.bn = p.room = 256;
  } else if (fast) {
    p.bm = slots / 256 * tiles_of(outs, 128) >= 192 ? 256 : 128;
    p.room = 256;
  } else if (wide_rows(slots, experts) == 32) {
    p.bm = 32;
  } else {
    p.bn = wide_side(outs);
  }
  p.tiles = most_tiles(slots, experts + 1, p.bm) * tiles_of(outs, p.bn);
  return p;
}

// Launches kernel(...) for the plan's tiles and the join of cut ones.
template <class T, int BM, int BN, int WM, int WN, class Kernel>
void launch_rows(const RowsPlan& p, Layouts& l, const T* b, const T* mask, const int32_t* offsets, T* y, int64_t slots,
                 int experts, int64_t cols, int64_t outs, bool relu, hipStream_t st, Kernel&& kernel) {
  f32x4* const slices = p.cut ? reinterpret_cast<f32x4*>(l.work + l.take(p.slices_bytes())) : nullptr;
  const int nt = (int)tiles_of(outs, BN);
  kernel(dim3((uint32_t)(p.tiles + (p.cut ? p.room : 0))), dim3(64 * WM * WN), nt, slices);
  SPHOPS_LAUNCHED();
  if (!p.cut) return;
  hipLaunchKernelGGL((k_group_rows_join<T, BM, BN, WM, WN>),
                     dim3((uint32_t)std::min<int64_t>(p.room / 2, p.tiles), BM / WM / 32 * (BN / WN / 32)),
                     dim3(64 * WM * WN), 0, st, b, mask, offsets, y, slots, experts, (int)cols, (int)outs, relu, nt,
                     p.room, p.places(), slices);
  SPHOPS_LAUNCHED();
}

template <class T, bool BACK>
void rows_fast(Layouts& l, const Laid& x, const Laid& w, const T* b, const T* mask, const int32_t* offsets, T* y,
               int64_t slots, int experts, int64_t cols, int64_t outs, bool relu, hipStream_t st) {
  using E = Piece16<T>;
  const RowsPlan p = rows_plan(std::is_same_v<T, float> ? SPHOPS_F32 : SPHOPS_BF16, true, slots, experts, cols, outs);
  const auto with = [&](auto bm, auto bn, auto wm, auto wn) {
    constexpr int BM = decltype(bm)::value, BN = decltype(bn)::value, WM = decltype(wm)::value, WN = decltype(wn)::value;
    launch_rows<T, BM, BN, WM, WN>(p, l, b, mask, offsets, y, slots, experts, cols, outs, relu, st,
                                   [&](dim3 grid, dim3 block, int nt, f32x4* slices) {
      hipLaunchKernelGGL((k_group_rows_fast<T, BACK, BM, BN, WM, WN>), grid, block, 0, st, static_cast<const E*>(x.base),
                         x.stride, x.plane, static_cast<const E*>(w.base), w.stride, w.plane, b, mask, offsets, y, slots,
                         experts, (int)cols, (int)outs, relu, nt, p.room, p.places(), slices);
    });
  };
#define SPHOPS_N(n) std::integral_constant<int, n>{}
  if constexpr (std::is_same_v<T, float>) {
    if (p.bm == 256) with(SPHOPS_N(256), SPHOPS_N(128), SPHOPS_N(4), SPHOPS_N(2));
    else with(SPHOPS_N(128), SPHOPS_N(128), SPHOPS_N(2), SPHOPS_N(2));
  } else {
    if (p.bm == 256) with(SPHOPS_N(256), SPHOPS_N(256), SPHOPS_N(2), SPHOPS_N(4));
    else with(SPHOPS_N(128), SPHOPS_N(128), SPHOPS_N(2), SPHOPS_N(2));
  }
}

// As they are.
template <class T, bool BACK>
void rows_plain(Layouts& l, const T* x, int64_t xs, const T* w, const T* b, const T* mask, const int32_t* offsets, T* y,
                int64_t slots, int experts, int64_t cols, int64_t outs, bool relu, hipStream_t st) {
  const RowsPlan p = rows_plan(std::is_same_v<T, float> ? SPHOPS_F32 : SPHOPS_BF16, false, slots, experts, cols, outs);
  const auto with = [&](auto bm, auto bn, auto wm, auto wn) {
    constexpr int BM = decltype(bm)::value, BN = decltype(bn)::value, WM = decltype(wm)::value, WN = decltype(wn)::value;
    launch_rows<T, BM, BN, WM, WN>(p, l, b, mask, offsets, y, slots, experts, cols, outs, relu, st,
                                   [&](dim3 grid, dim3 block, int nt, f32x4* slices) {
      if constexpr (std::is_same_v<T, float>)
        hipLaunchKernelGGL((k_group_rows_wide<BACK, BM, BN, WM, WN>), grid, block, 0, st, x, xs, w, b, mask, offsets, y,
                           slots, experts, (int)cols, (int)outs, relu, nt, p.room, p.places(), slices);
      else
        hipLaunchKernelGGL((k_group_rows<T, BACK>), grid, block, 0, st, x, xs, w, b, mask, offsets, y, slots, experts,
                           (int)cols, (int)outs, relu, nt, p.room, p.places(), slices);
    });
  };
  if constexpr (std::is_same_v<T, float>) {
    if (p.bm == 32) with(SPHOPS_N(32), SPHOPS_N(128), SPHOPS_N(1), SPHOPS_N(4));
    else if (p.bn == 32) with(SPHOPS_N(128), SPHOPS_N(32), SPHOPS_N(4), SPHOPS_N(1));
    else if (p.bn == 64) with(SPHOPS_N(128), SPHOPS_N(64), SPHOPS_N(4), SPHOPS_N(1));
    else with(SPHOPS_N(128), SPHOPS_N(128), SPHOPS_N(2), SPHOPS_N(2));
  } else {
    with(SPHOPS_N(128), SPHOPS_N(128), SPHOPS_N(2), SPHOPS_N(4));
  }
#undef SPHOPS_N
}

// Bytes of slices: as the product runs, or (16-bit rows) as either alignment does.
int64_t rows_bytes(int type, int64_t slots, int experts, int64_t cols, int64_t outs, bool laid) {
  if (type == SPHOPS_F32) return rows_plan(type, laid, slots, experts, cols, outs).slices_bytes();
  return std::max(rows_plan(type, true, slots, experts, cols, outs).slices_bytes(),
                  rows_plan(type, false, slots, experts, cols, outs).slices_bytes());
}

// Few rows an expert: k_group_tokens, which reads x again for every 16 outputs and has a
// workgroup for each expert, its rows or not: as long as the products are few (for
// float32, whose matrix cores are slower, a quarter), and the workgroups.  us on the
// GPU, it and the tiles.  bfloat16, 4096 -> 2048: 32 rows of 16 experts 36 and 44, 64
// 50 and 46, 256 82 and 59; 1024 -> 1024: 256 of 16 16 and 24, 128 of 64 23 and 26,
// 512 of 64 37 and 28; 83 -> 128: 1024 of 64 6 and 9, of 256 19 and 11.  float32, 1024 ->
// 1024: 64 of 16 23 and 23, 256 of 16 35 and 28, 64 of 64 34 and 51.
constexpr int64_t kTokenSlots = 1024, kTokenProducts = int64_t(5) << 26, kTokenGroups = 1 << 15;
bool few_rows(int type, int64_t slots, int experts, int64_t cols, int64_t outs) {
  return slots <= kTokenSlots && slots <= 16 * (int64_t)experts &&
         slots * cols * outs <= (type == SPHOPS_F32 ? kTokenProducts / 4 : kTokenProducts) &&
         tiles_of(outs, 16) * (experts + 1) * tiles_of(slots, kTokenRows) <= kTokenGroups;
}

template <class T>
bool fast_as_is(const void* x, int64_t xs, int64_t cols, const void* w, int64_t ws) {
  return !std::is_same_v<T, float> && whole_pieces(x, xs) && cols % 8 == 0 && whole_pieces(w, ws);
}

}  // namespace

// Whether every launch of a layer, forward and backward and at either alignment, stays
// below the 2^32 threads that one can have along x.
bool group_linear_fits(int type, int64_t slots, int experts, int64_t cols, int64_t outs) {
  const auto threads = [](int64_t groups, int size) { return groups < (int64_t(1) << 32) / size; };
  const bool wide = type == SPHOPS_F32;
  for (const bool fast : {false, true}) {
    for (const bool back : {false, true}) {
      const RowsPlan p = rows_plan(type, fast, slots, experts, back ? outs : cols, back ? cols : outs);
      const int size = wide ? (p.bm == 256 ? 512 : 256) : fast && p.bm == 128 ? 256 : 512;
      if (!threads(p.tiles + p.room, size)) return false;
    }
    const GradPlan p = wide && fast ? laid_plan(slots, experts, cols, outs) : chosen_plan(slots, experts, cols, outs, wide, fast);
    if (!threads(std::max<int64_t>(p.chunks, experts) * p.mt * p.nt, wide && !fast ? kWideThreads : kGroupThreads)) return false;
  }
  return threads(tiles_of(cols * outs + outs, 256), 256);
}

int64_t group_linear_workspace_bytes(int type, int64_t slots, int experts, int64_t cols, int64_t outs) {
  Layouts l{nullptr};
  const bool laid = lays_out(type, slots, experts, cols, outs, false);
  if (laid) {
    l.take(Layouts::bytes_of(type, slots, cols));
    l.take(Layouts::bytes_of(type, experts * outs, cols));
  }
  if (!few_rows(type, slots, experts, cols, outs)) l.take(rows_bytes(type, slots, experts, cols, outs, laid));
  return l.used;
}

void run_group_linear(const void* x, int type, int64_t xs, const void* w, const void* b, const int32_t* offsets,
                      void* y, int64_t slots, int experts, int64_t cols, int64_t outs, bool relu, void* work,
                      hipStream_t st) {
  if (slots == 0) return;
  with_type(type, [&](auto t) {
    using T = decltype(t);
    const T *px = static_cast<const T*>(x), *pw = static_cast<const T*>(w), *pb = static_cast<const T*>(b);
    T* const py = static_cast<T*>(y);
    const bool as_is = fast_as_is<T>(x, xs, cols, w, cols);
    Layouts l{static_cast<char*>(work)};
    if (few_rows(type, slots, experts, cols, outs)) {
      const dim3 grid((uint32_t)tiles_of(outs, 16), (uint32_t)(experts + 1), (uint32_t)tiles_of(slots, kTokenRows));
      hipLaunchKernelGGL((k_group_tokens<T>), grid, dim3(kTokenThreads), 0, st, px, xs, pw, pb, offsets, py, slots,
                         experts, (int)cols, (int)outs, relu);
    } else if (as_is || lays_out(type, slots, experts, cols, outs, false)) {
      const Laid lx = as_is ? Laid{x, xs, 0} : lay_out(l, px, xs, slots, cols, st);
      const Laid lw = as_is ? Laid{w, cols, 0} : lay_out(l, pw, cols, experts * outs, cols, st);
      rows_fast<T, false>(l, lx, lw, pb, nullptr, offsets, py, slots, experts, cols, outs, relu, st);
    } else {
      rows_plain<T, false>(l, px, xs, pw, pb, nullptr, offsets, py, slots, experts, cols, outs, relu, st);
    }
  });
  SPHOPS_LAUNCHED();
}

// The chunks of any of the kernels, and the laid out operands of both products.
int64_t group_backward_workspace_bytes(int type, int64_t slots, int experts, int64_t cols, int64_t outs) {
  int64_t chunks = 0;
  for (const bool fast : {false, true})
    chunks = std::max(chunks, chosen_plan(slots, experts, cols, outs, type == SPHOPS_F32, fast).chunks);
  if (type == SPHOPS_F32)
    chunks = std::max(chunks, laid_plan(slots, experts, cols, outs).chunks);
  Layouts l{nullptr};
  l.take(chunks * (cols * outs + outs) * (int64_t)sizeof(float));
  const bool laid = lays_out(type, slots, experts, cols, outs, true);
  if (laid) {
    l.take(Layouts::bytes_of(type, slots, outs));
    l.take(Layouts::bytes_of(type, experts * outs, cols));
    l.take(Layouts::bytes_of(type, slots, cols));
  }
  l.take(rows_bytes(type, slots, experts, outs, cols, laid));
  return l.used;
}

void run_group_backward(const void* dy, int64_t dys, const void* x, int type, int64_t xs, const void* w,
                        const void* mask, const int32_t* offsets, void* dx, void* dw, void* db, int64_t slots,
                        int experts, int64_t cols, int64_t outs, void* work, hipStream_t st) {
  const int64_t nw = cols * outs;
  const bool sums = dw != nullptr || db != nullptr;
  with_type(type, [&](auto t) {
    using T = decltype(t);
    constexpr bool wide = std::is_same_v<T, float>;
    const T *pdy = static_cast<const T*>(dy), *px = static_cast<const T*>(x), *pw = static_cast<const T*>(w);
    const T* const pm = static_cast<const T*>(mask);
    const bool laid = lays_out(type, slots, experts, cols, outs, true);
    const bool rows_as_is = fast_as_is<T>(dy, dys, outs, w, cols) && cols % 8 == 0;
    const bool grad_as_is = fast_as_is<T>(dy, dys, outs, x, xs) && cols % 8 == 0;
    Layouts l{static_cast<char*>(work)};
    int64_t chunks = 0;
    for (const bool fast : {false, true}) chunks = std::max(chunks, chosen_plan(slots, experts, cols, outs, wide, fast).chunks);
    if (wide) chunks = std::max(chunks, laid_plan(slots, experts, cols, outs).chunks);
    float* const part = reinterpret_cast<float*>(l.work + l.take(chunks * (nw + outs) * (int64_t)sizeof(float)));
    Laid ldy{dy, dys, 0};
    const bool lay_dy = slots > 0 && laid && ((dx != nullptr && !rows_as_is) || (sums && !grad_as_is));
    if (lay_dy) ldy = lay_out(l, pdy, dys, slots, outs, st);
    if (dx != nullptr && slots > 0) {
      if (rows_as_is || laid) {
        const Laid lw = rows_as_is ? Laid{w, cols, 0} : lay_out(l, pw, cols, experts * outs, cols, st);
        rows_fast<T, true>(l, ldy, lw, nullptr, pm, offsets, static_cast<T*>(dx), slots, experts, outs, cols, false, st);
      } else {
        rows_plain<T, true>(l, pdy, dys, pw, nullptr, pm, offsets, static_cast<T*>(dx), slots, experts, outs, cols, false, st);
      }
      SPHOPS_LAUNCHED();
    }
    if (!sums) return;
    const bool fast = grad_as_is || (laid && slots > 0);
    const GradPlan p = wide && fast ? laid_plan(slots, experts, cols, outs)
                                    : chosen_plan(slots, experts, cols, outs, wide, fast);
    float* const to = p.chunks > 0 ? part : nullptr;
    const dim3 grid((uint32_t)((p.chunks > 0 ? p.chunks : experts) * p.mt * p.nt));
    T *const pdw = static_cast<T*>(dw), *const pdb = static_cast<T*>(db);
    if (fast) {
      using E = Piece16<T>;
      const Laid lx = grad_as_is ? Laid{x, xs, 0} : lay_out(l, px, xs, slots, cols, st);
      const auto with = [&](auto kernel, int threads) {
        hipLaunchKernelGGL(kernel, grid, dim3(threads), 0, st, static_cast<const E*>(ldy.base), ldy.stride, ldy.plane,
                           static_cast<const E*>(lx.base), lx.stride, lx.plane, offsets, pdw, pdb, to, slots, experts,
                           (int)cols, (int)outs, p.chunk, p.mt, p.nt);
      };
      if constexpr (wide) {
        if (p.bm == 256) with(k_group_weight_grad_fast<T, 256, 128, 4, 2>, 512);
        else with(k_group_weight_grad_fast<T, 128, 128, 2, 2>, 256);
      }
      else if (p.bm == 256) with(k_group_weight_grad_fast<T, 256, 256, 2, 4>, 512);
      else with(k_group_weight_grad_fast<T, 128, 128, 2, 2>, 256);
    } else {
      const auto with = [&](auto kernel, int threads) {
        hipLaunchKernelGGL(kernel, grid, dim3(threads), 0, st, pdy, dys, px, xs, offsets, pdw, pdb, to, slots, experts,
                           (int)cols, (int)outs, p.chunk, p.mt, p.nt);
      };
      if constexpr (wide) {
        if (p.bm == 128 && p.bn == 128) with(k_group_weight_grad_wide<128, 128, 2, 2>, kWideThreads);
        else if (p.bm == 128 && p.bn == 64) with(k_group_weight_grad_wide<128, 64, 4, 1>, kWideThreads);
        else if (p.bm == 64 && p.bn == 128) with(k_group_weight_grad_wide<64, 128, 1, 4>, kWideThreads);
        else if (p.bm == 128) with(k_group_weight_grad_wide<128, 32, 4, 1>, kWideThreads);
        else if (p.bn == 128) with(k_group_weight_grad_wide<32, 128, 1, 4>, kWideThreads);
        else with(k_group_weight_grad_wide<64, 64, 2, 2>, kWideThreads);
      } else {
        with(k_group_weight_grad<T>, kGroupThreads);
      }
    }
    SPHOPS_LAUNCHED();
    if (p.chunks > 0)
      hipLaunchKernelGGL((k_group_chunk_sum<T>), dim3((uint32_t)tiles_of(nw + outs, 256), (uint32_t)experts), dim3(256),
                         0, st, part, offsets, pdw, pdb, slots, experts, nw, (int)outs, p.chunk, p.chunks);
    SPHOPS_LAUNCHED();
  });
}

}  // namespace sphops
