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

// The workgroup's row tile and column tile among those that there are (the
// launch covers the most that there can be); false: neither.
__device__ __forceinline__ bool rows_tile(const int32_t* __restrict__ offsets, int experts, int64_t slots, int size,
                                          int nt, GroupTile& g, int& n) {
  const int64_t mt = group_tiles(offsets, experts, slots, size, true);
  const uint32_t id = xcd_block_id((uint32_t)(mt * nt));
  if (id == 0xFFFFFFFFu) return false;
  int64_t m;
  tile_of(id, mt, nt, m, n);
  g = group_tile(offsets, experts, slots, m, size, true);
  return g.group >= 0;
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

// y (slots x outs) = x (slots x cols) W_e^T + b_e, W_e (outs x cols); BACK: y = x
// W_e with W_e (cols x outs), which is the input gradient.  relu: y = max(y, 0).
// mask (slots x outs): y = 0 where it is not above 0.
template <class T, bool BACK>
__global__ __launch_bounds__(kGroupThreads) void k_group_rows(const T* __restrict__ x, int64_t xs,
                                                              const T* __restrict__ w, const T* __restrict__ b,
                                                              const T* __restrict__ mask,
                                                              const int32_t* __restrict__ offsets, T* __restrict__ y,
                                                              int64_t slots, int experts, int cols, int outs,
                                                              bool relu, int nt) {
  using IA = PanelImage<T, true>;
  using IB = PanelImage<T, !BACK>;
  constexpr int V = Piece<T>::V;
  __shared__ __attribute__((aligned(16))) uint16_t room[std::max(IA::kPlane + IB::kPlane, kOutbox)];
  uint16_t *const as = room, *const bs = room + IA::kPlane;
  GroupTile g;
  int n;
  if (!rows_tile(offsets, experts, slots, kSide, nt, g, n)) return;
  const int64_t m0 = g.lo + g.tile * kSide;
  const int n0 = n * kSide, here = (int)min<int64_t>(kSide, g.hi - m0), outs_here = min(kSide, outs - n0);
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x / 64);
  const int row0 = wave / 4 * 64, col0 = wave % 4 * 32;
  if (g.group == experts) {
    zero_rows(y, m0, here, n0, kSide, outs);
    return;
  }
  const T* const we = w + (int64_t)g.group * cols * outs;
  const Panel<T> pa{x + m0 * xs, xs, here, cols};
  const Panel<T> pb = BACK ? Panel<T>{we + n0, outs, cols, outs_here} : Panel<T>{we + (int64_t)n0 * cols, cols, outs_here, cols};
  Piece<T> ra[IA::kLoads], rb[IB::kLoads];
  TileSums<T> sums;
  sums.clear();
  IA::load(pa, 0, ra);
  IB::load(pb, 0, rb);
  for (int k = 0; k < cols; k += kStepK) {
    IA::store(ra, as);
    IB::store(rb, bs);
    __syncthreads();
    if (k + kStepK < cols) {
      IA::load(pa, k + kStepK, ra);
      IB::load(pb, k + kStepK, rb);
    }
    sums.template step<IA, IB>(as, bs, row0, col0);
    __syncthreads();
  }
  float* const own = reinterpret_cast<float*>(room) + 1024 * wave;  // every wave is done with the panels
  const T* const be = b != nullptr ? b + (int64_t)g.group * outs : nullptr;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    rows_of_tile<T>(sums.acc[i], own, [&](int r, int c, float (&v)[V]) {
      const int row = row0 + 32 * i + r, at = n0 + col0 + c;
      if (row >= here || at >= outs) return;
      finish<T>(v, be, mask != nullptr ? mask + (m0 + row) * outs : nullptr, relu, y + (m0 + row) * outs, at, outs);
    });
  }
}

// The same for 16-bit rows in whole 16-byte pieces: panels straight from memory
// to LDS.
template <class T, bool BACK, int BM, int BN, int WM, int WN>
__global__ __launch_bounds__(64 * WM * WN) void k_group_rows_fast(const T* __restrict__ x, int64_t xs,
                                                                  const T* __restrict__ w, const T* __restrict__ b,
                                                                  const T* __restrict__ mask,
                                                                  const int32_t* __restrict__ offsets,
                                                                  T* __restrict__ y, int64_t slots, int experts,
                                                                  int cols, int outs, bool relu, int nt) {
  using Tile = FastTile<T, true, !BACK, BM, BN, WM, WN, false>;
  constexpr int V = Piece<T>::V;
  __shared__ __attribute__((aligned(16))) uint16_t s0[Tile::kStage], s1[Tile::kStage];
  GroupTile g;
  int n;
  if (!rows_tile(offsets, experts, slots, BM, nt, g, n)) return;
  const int64_t m0 = g.lo + g.tile * BM;
  const int n0 = n * BN, here = (int)min<int64_t>(BM, g.hi - m0), outs_here = min(BN, outs - n0);
  if (g.group == experts) {
    zero_rows(y, m0, here, n0, BN, outs);
    return;
  }
  const T* const we = w + (int64_t)g.group * cols * outs;
  const typename Tile::A pa(Panel<T>{x + m0 * xs, xs, here, cols});
  const typename Tile::B pb(BACK ? Panel<T>{we + n0, outs, cols, outs_here}
                                 : Panel<T>{we + (int64_t)n0 * cols, cols, outs_here, cols});
  Tile t;
  t.run(pa, pb, cols, false, s0, s1);
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x / 64);
  const int row0 = wave / WN * (BM / WM), col0 = wave % WN * (BN / WN);
  float* const own = reinterpret_cast<float*>(s0) + 1024 * wave;
  static_assert(Tile::kWaves * 2048 <= Tile::kStage, "room");
  const T* const be = b != nullptr ? b + (int64_t)g.group * outs : nullptr;
#pragma unroll
  for (int i = 0; i < Tile::TM; ++i) {
#pragma unroll
    for (int j = 0; j < Tile::TN; ++j) {
      rows_of_tile<T>(t.acc[i][j], own, [&](int r, int c, float (&v)[V]) {
        const int row = row0 + 32 * i + r, at = n0 + col0 + 32 * j + c;
        if (row >= here || at >= outs) return;
        finish<T>(v, be, mask != nullptr ? mask + (m0 + row) * outs : nullptr, relu, y + (m0 + row) * outs, at, outs);
      });
    }
  }
}

// The same for float32 rows.  Three bfloat16 pieces of each factor and six products
// take three eighths of the matrix cores' time, but putting them into pieces takes
// vector work that does not overlap, and their sums registers: 8192 x 1024 -> 2048
// in 337 us that way.
template <bool BACK, int BM, int BN, int WM, int WN>
__global__ __launch_bounds__(kWideThreads) void k_group_rows_wide(const float* __restrict__ x, int64_t xs,
                                                                  const float* __restrict__ w,
                                                                  const float* __restrict__ b,
                                                                  const float* __restrict__ mask,
                                                                  const int32_t* __restrict__ offsets,
                                                                  float* __restrict__ y, int64_t slots, int experts,
                                                                  int cols, int outs, bool relu, int nt) {
  using Tile = WideTile<true, !BACK, BM, BN, WM, WN>;
  __shared__ __attribute__((aligned(16))) float room[Tile::kRoom];
  GroupTile g;
  int n;
  if (!rows_tile(offsets, experts, slots, BM, nt, g, n)) return;
  const int64_t m0 = g.lo + g.tile * BM;
  const int n0 = n * BN, here = (int)min<int64_t>(BM, g.hi - m0), outs_here = min(BN, outs - n0);
  if (g.group == experts) {
    zero_rows(y, m0, here, n0, BN, outs);
    return;
  }
  const float* const we = w + (int64_t)g.group * cols * outs;
  Tile t;
  t.run(Panel<float>{x + m0 * xs, xs, here, cols},
        BACK ? Panel<float>{we + n0, outs, cols, outs_here} : Panel<float>{we + (int64_t)n0 * cols, cols, outs_here, cols},
        cols, room, [](auto&) {});
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x / 64);
  const int row0 = wave / WN * (BM / WM), col0 = wave % WN * (BN / WN);
  const float* const be = b != nullptr ? b + (int64_t)g.group * outs : nullptr;
#pragma unroll
  for (int i = 0; i < Tile::TM; ++i) {
#pragma unroll
    for (int j = 0; j < Tile::TN; ++j) {
      rows_of_tile<float>(t.acc[i][j], room + 1024 * wave, [&](int r, int c, float (&v)[4]) {
        const int row = row0 + 32 * i + r, at = n0 + col0 + 32 * j + c;
        if (row >= here || at >= outs) return;
        finish<float>(v, be, mask != nullptr ? mask + (m0 + row) * outs : nullptr, relu, y + (m0 + row) * outs, at, outs);
      });
    }
  }
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
__device__ __forceinline__ GroupTile grad_rows(const int32_t* __restrict__ offsets, int experts, int64_t slots,
                                               int64_t piece, int64_t chunk, bool chunks) {
  if (chunks) return group_tile(offsets, experts, slots, piece, chunk, false);
  GroupTile g;
  g.group = (int)piece;
  g.tile = 0;
  g.lo = piece == 0 ? 0 : min<int64_t>(max(offsets[piece], 0), slots);
  g.hi = max<int64_t>(g.lo, min<int64_t>(offsets[piece + 1], slots));
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

// The same for 16-bit rows in whole 16-byte pieces, straight from memory to LDS;
// db from products with ones.
template <class T, int BM, int BN, int WM, int WN>
__global__ __launch_bounds__(64 * WM * WN) void k_group_weight_grad_fast(
    const T* __restrict__ dy, int64_t dys, const T* __restrict__ x, int64_t xs, const int32_t* __restrict__ offsets,
    T* __restrict__ dw, T* __restrict__ db, float* __restrict__ part, int64_t slots, int experts, int cols, int outs,
    int64_t chunk, int mt, int nt) {
  using Tile = FastTile<T, false, false, BM, BN, WM, WN, true>;
  static_assert(Tile::TM <= WN, "a wave of the row for each tile of rows");
  __shared__ __attribute__((aligned(16))) uint16_t s0[Tile::kStage], s1[Tile::kStage];
  const GradTile at = grad_tile(mt, nt);
  const int64_t piece = at.piece;
  const int m0 = at.m * BM, n0 = at.n * BN;
  const GroupTile g = grad_rows(offsets, experts, slots, piece, chunk, part != nullptr);
  if (g.group < 0) return;
  const int64_t lo = g.lo + g.tile * chunk;
  const int rows = (int)min<int64_t>(chunk, g.hi - lo);
  const typename Tile::A pa(Panel<T>{dy + lo * dys + m0, dys, rows, min(BM, outs - m0)});
  const typename Tile::B pb(Panel<T>{x + lo * xs + n0, xs, rows, min(BN, cols - n0)});
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
  // every column of `ones` holds the same sums: lane l has row l % 32
  const int row = m0 + row0 + 32 * wn + (int)(threadIdx.x & 31);
  if (n0 != 0 || wn >= Tile::TM || (threadIdx.x & 63) >= 32 || row >= outs) return;
  if (mine != nullptr) mine[nw + row] = t.ones[0];
  else if (db != nullptr) db[(int64_t)g.group * outs + row] = from_f32<T>(t.ones[0]);
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
        Panel<float>{x + lo * xs + n0, xs, rows, min(BN, cols - n0)}, rows, room, [&](auto& pieces) {
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

// Tiles of `size` rows that the groups can have between them.
int64_t most_tiles(int64_t slots, int64_t groups, int64_t size) {
  return slots / size + std::min(groups, slots);
}

// Rows of a weight gradient's chunk: as many chunks as fill the card, of 256
// rows at least and of kMaxGroupChunk at most.
constexpr int64_t kMaxGroupChunk = 8192;
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
  if (slots <= p.chunk || (tiles * experts >= 512 && slots <= 2 * kMaxGroupChunk)) {
    p.chunk = std::max<int64_t>(slots, 1);
    p.chunks = 0;
  }
  return p;
}

// 16-bit rows of whole 16-byte pieces at multiples of 16 bytes, a panel's within 32 bits of its first.
bool whole_pieces(const void* p, int64_t stride) {
  return reinterpret_cast<uintptr_t>(p) % 16 == 0 && stride % 8 == 0 && stride <= (1 << 22);
}

// 16-bit tiles: 256 where there are enough of them, else 128.
int rows_side(int64_t slots, int64_t outs) {
  return outs > 128 && slots / 256 * tiles_of(outs, 256) >= 192 ? 256 : 128;
}
int grad_side(int experts, int64_t cols, int64_t outs) {
  return outs > 128 && cols > 128 && tiles_of(outs, 256) * tiles_of(cols, 256) * experts >= 192 ? 256 : 128;
}
// Float32 tiles: 32, 64 or 128 outputs, as few as hold them; 32 rows where an expert has no more on average.
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

}  // namespace

bool group_linear_fits(int64_t slots, int experts, int64_t cols, int64_t outs) {
  const int64_t limit = (int64_t(1) << 32) / kGroupThreads - 8;  // threads a launch
  for (const int64_t n : {outs, cols}) {
    if (most_tiles(slots, experts + 1, kSide) * tiles_of(n, 32) >= limit) return false;
    if (slots <= 32 * (int64_t)experts && most_tiles(slots, experts + 1, 32) * tiles_of(n, kSide) >= limit) return false;
  }
  for (const bool wide : {false, true}) {
    const GradPlan p = chosen_plan(slots, experts, cols, outs, wide, false);
    if ((int64_t)p.mt * p.nt * std::max<int64_t>(p.chunks, experts) >= limit) return false;
  }
  return tiles_of(cols * outs + outs, 256) * experts < limit;
}

void run_group_linear(const void* x, int type, int64_t xs, const void* w, const void* b, const void* mask,
                      const int32_t* offsets, void* y, int64_t slots, int experts, int64_t cols, int64_t outs,
                      bool relu, bool back, hipStream_t st) {
  if (slots == 0) return;
  with_type(type, [&](auto t) {
    using T = decltype(t);
    auto launch = [&](auto bk) {
      constexpr bool BACK = decltype(bk)::value;
      const auto with = [&](auto kernel, int bm, int bn, int threads) {
        const int64_t tiles = most_tiles(slots, experts + 1, bm) * tiles_of(outs, bn);
        hipLaunchKernelGGL(kernel, dim3((uint32_t)(tiles_of(tiles, 8) * 8)) /* whole turns of the eight XCDs */,
                           dim3(threads), 0, st, static_cast<const T*>(x), xs, static_cast<const T*>(w),
                           static_cast<const T*>(b), static_cast<const T*>(mask), offsets, static_cast<T*>(y), slots,
                           experts, (int)cols, (int)outs, relu, (int)tiles_of(outs, bn));
      };
      if constexpr (std::is_same_v<T, float>) {
        if (wide_rows(slots, experts) == 32) with(k_group_rows_wide<BACK, 32, 128, 1, 4>, 32, 128, kWideThreads);
        else if (wide_side(outs) == 32) with(k_group_rows_wide<BACK, 128, 32, 4, 1>, 128, 32, kWideThreads);
        else if (wide_side(outs) == 64) with(k_group_rows_wide<BACK, 128, 64, 4, 1>, 128, 64, kWideThreads);
        else with(k_group_rows_wide<BACK, 128, 128, 2, 2>, 128, 128, kWideThreads);
      } else if (whole_pieces(x, xs) && whole_pieces(w, BACK ? outs : cols) && cols % 8 == 0 &&
                 (!BACK || outs % 8 == 0)) {
        if (rows_side(slots, outs) == 256) with(k_group_rows_fast<T, BACK, 256, 256, 2, 4>, 256, 256, 512);
        else with(k_group_rows_fast<T, BACK, 128, 128, 2, 2>, 128, 128, 256);
      } else {
        with(k_group_rows<T, BACK>, kSide, kSide, kGroupThreads);
      }
    };
    if (back) launch(std::true_type{});
    else launch(std::false_type{});
  });
  SPHOPS_LAUNCHED();
}

// The workspace holds the chunks of any of the kernels.
int64_t group_weight_grad_floats(int64_t slots, int experts, int64_t cols, int64_t outs) {
  int64_t chunks = 0;
  for (const bool wide : {false, true}) {
    for (const bool fast : {false, true}) chunks = std::max(chunks, chosen_plan(slots, experts, cols, outs, wide, fast).chunks);
  }
  return chunks * (cols * outs + outs);
}

void run_group_weight_grad(const void* dy, int64_t dys, const void* x, int type, int64_t xs, const int32_t* offsets,
                           void* dw, void* db, int64_t slots, int experts, int64_t cols, int64_t outs, float* work,
                           hipStream_t st) {
  const int64_t nw = cols * outs;
  with_type(type, [&](auto t) {
    using T = decltype(t);
    constexpr bool wide = std::is_same_v<T, float>;
    const bool fast = !wide && whole_pieces(dy, dys) && whole_pieces(x, xs) && cols % 8 == 0 && outs % 8 == 0;
    const GradPlan p = chosen_plan(slots, experts, cols, outs, wide, fast);
    const int64_t blocks = (p.chunks > 0 ? p.chunks : experts) * p.mt * p.nt;
    const auto with = [&](auto kernel, int threads) {
      hipLaunchKernelGGL(kernel, dim3((uint32_t)blocks), dim3(threads), 0, st, static_cast<const T*>(dy), dys,
                         static_cast<const T*>(x), xs, offsets, static_cast<T*>(dw), static_cast<T*>(db),
                         p.chunks > 0 ? work : nullptr, slots, experts, (int)cols, (int)outs, p.chunk, p.mt, p.nt);
    };
    if constexpr (wide) {
      if (p.bm == 128 && p.bn == 128) with(k_group_weight_grad_wide<128, 128, 2, 2>, kWideThreads);
      else if (p.bm == 128 && p.bn == 64) with(k_group_weight_grad_wide<128, 64, 4, 1>, kWideThreads);
      else if (p.bm == 64 && p.bn == 128) with(k_group_weight_grad_wide<64, 128, 1, 4>, kWideThreads);
      else if (p.bm == 128) with(k_group_weight_grad_wide<128, 32, 4, 1>, kWideThreads);
      else if (p.bn == 128) with(k_group_weight_grad_wide<32, 128, 1, 4>, kWideThreads);
      else with(k_group_weight_grad_wide<64, 64, 2, 2>, kWideThreads);
    } else if (!fast) {
      with(k_group_weight_grad<T>, kGroupThreads);
    } else if (p.bm == 256) {
      with(k_group_weight_grad_fast<T, 256, 256, 2, 4>, 512);
    } else {
      with(k_group_weight_grad_fast<T, 128, 128, 2, 2>, 256);
    }
    SPHOPS_LAUNCHED();
    if (p.chunks > 0)
      hipLaunchKernelGGL((k_group_chunk_sum<T>), dim3((uint32_t)tiles_of(nw + outs, 256), (uint32_t)experts), dim3(256),
                         0, st, work, offsets, static_cast<T*>(dw), static_cast<T*>(db), slots, experts, nw, (int)outs,
                         p.chunk, p.chunks);
  });
  SPHOPS_LAUNCHED();
}

}  // namespace sphops
