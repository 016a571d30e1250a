// Products over rows sorted by expert (grouped.hip): which rows a workgroup's
// tile holds, panels through LDS as 16-bit pieces, and the matrix products of a
// tile.
#pragma once

#include "rows8.hpp"
#include "split16.hpp"
#include "turns.hpp"

#include <algorithm>
#include <type_traits>

namespace sphops {

namespace {

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

// Tile `id` of the groups' rows (group_rows) in tiles of `size`.  No tile leaves
// the rows, whatever the offsets hold; how many there are is bounded by most_tiles
// only where offsets do not decrease.  Every wave finds it for itself.
struct GroupTile {
  int group;        // -1: no such tile
  int64_t tile;     // within the group
  int64_t lo, hi;   // the group's rows
};
__device__ __forceinline__ GroupTile group_tile(const int32_t* __restrict__ offsets, int experts, int64_t slots,
                                                int64_t id, int64_t size, bool behind) {
  const int lane = threadIdx.x & 63, groups = experts + (behind ? 1 : 0);
  GroupTile g{-1, 0, 0, 0};
  for (int base = 0; base < groups; base += 64) {
    const int e = base + lane;
    GroupRows r{0, 0};
    if (e < groups) r = group_rows(offsets, experts, slots, e);
    const int64_t mine = (r.hi - r.lo + size - 1) / size;
    int64_t upto = mine;
#pragma unroll
    for (int s = 1; s < 64; s *= 2) {
      const int64_t other = __shfl_up(upto, s);
      if (lane >= s) upto += other;
    }
    const uint64_t past = __ballot(upto > id);
    if (past != 0) {
      const int at = __ffsll((unsigned long long)past) - 1;
      g.group = base + at;
      g.tile = id - __shfl(upto - mine, at);
      g.lo = __shfl(r.lo, at);
      g.hi = __shfl(r.hi, at);
      break;
    }
    id -= __shfl(upto, 63);
  }
  g.group = __builtin_amdgcn_readfirstlane(g.group);
  return g;
}

// The tiles of all groups.
__device__ __forceinline__ int64_t group_tiles(const int32_t* __restrict__ offsets, int experts, int64_t slots,
                                               int64_t size, bool behind) {
  const int lane = threadIdx.x & 63, groups = experts + (behind ? 1 : 0);
  int64_t all = 0;
  for (int base = 0; base < groups; base += 64) {
    const int e = base + lane;
    if (e < groups) {
      const GroupRows r = group_rows(offsets, experts, slots, e);
      all += (r.hi - r.lo + size - 1) / size;
    }
  }
#pragma unroll
  for (int s = 1; s < 64; s *= 2) all += __shfl_xor(all, s);
  return all;
}

// Group e's tiles, those of the groups before it and those of all experts.
struct GroupSpan {
  int64_t before, tiles, all;
};
__device__ __forceinline__ GroupSpan group_span(const int32_t* __restrict__ offsets, int experts, int64_t slots,
                                                int64_t size, int e) {
  const int lane = threadIdx.x & 63;
  GroupSpan g{0, 0, 0};
  for (int base = 0; base < experts; base += 64) {
    const int i = base + lane;
    int64_t mine = 0;
    if (i < experts) {
      const GroupRows r = group_rows(offsets, experts, slots, i);
      mine = (r.hi - r.lo + size - 1) / size;
    }
    int64_t before = i < e ? mine : 0;
    if (e >= base && e < base + 64) g.tiles = __shfl(mine, e - base);
#pragma unroll
    for (int s = 1; s < 64; s *= 2) {
      mine += __shfl_xor(mine, s);
      before += __shfl_xor(before, s);
    }
    g.before += before;
    g.all += mine;
  }
  return g;
}

template <class T>
__device__ __forceinline__ f32x16 mma16(s16x8 a, s16x8 b, f32x16 c) {
  if constexpr (std::is_same_v<T, __half>)
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0,
                                                  0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0,
                                                   0, 0);
}
template <class T>
__device__ __forceinline__ f32x4 mma16(s16x8 a, s16x8 b, f32x4 c) {
  if constexpr (std::is_same_v<T, __half>)
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0,
                                                  0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0,
                                                   0, 0);
}

// A panel of a product's operand: `rows` rows of `cols` values in memory.  KMAJOR: a
// row holds the values along the summed dimension of one output row (or
// column); else a row is one step of the sum and its values are the outputs'.
// What lies past the rows and columns counts as zeros.
template <class T>
struct Panel {
  const T* base;
  int64_t stride;
  int rows, cols;
};

constexpr int kStepK = 32;  // of the sum a step
constexpr int kSide = 128;  // a tile's rows and columns
constexpr int kGroupThreads = 512;
constexpr int kOutbox = kGroupThreads / 64 * 2048;  // 16-bit words of LDS: 4 KB a wave for results on their way out

// The pieces of a panel's step from `k` on that a thread of THREADS holds: piece
// threadIdx.x % PIECES of rows threadIdx.x / PIECES and on.
template <class T, bool KMAJOR, int PIECES, int LOADS, int THREADS, int STEP, int SIDE>
__device__ __forceinline__ void load_panel(const Panel<T>& p, int64_t k, Piece<T> (&out)[LOADS]) {
  const int col = (int)threadIdx.x % PIECES * Piece<T>::V, row = (int)threadIdx.x / PIECES;
  const int at = KMAJOR ? (int)k + col : col;
  const int64_t down = KMAJOR ? 0 : k;
  const bool whole = (KMAJOR ? k + STEP : SIDE) <= p.cols;
#pragma unroll
  for (int i = 0; i < LOADS; ++i) {
    const int64_t r = down + row + i * (THREADS / PIECES), kept = min(r, (int64_t)p.rows - 1);
    if (whole) {
      out[i].raw = *reinterpret_cast<const typename Piece<T>::Raw*>(p.base + kept * p.stride + at);
      // a K-major panel's rows past the end give outputs that nobody stores
      if (!KMAJOR && r >= p.rows) out[i].raw = typename Piece<T>::Raw{};
    } else if (r < p.rows) {
      out[i].load(p.base + r * p.stride, at, p.cols);
    } else {
      out[i].raw = typename Piece<T>::Raw{};
    }
  }
}

// 16-bit rows of any length at any place.
template <class T, bool KMAJOR>
struct PanelImage {
  static constexpr int V = Piece<T>::V;
  static constexpr int kRowPieces = (KMAJOR ? kStepK : kSide) / V;
  static constexpr int kLoads = kSide * kStepK / V / kGroupThreads;
  // 16-bit values: rows of 64 bytes whose 16-byte pieces are exchanged by the
  // row's bits, or 32 rows of an odd number of 64 bytes (read down columns)
  static constexpr int kPitch = KMAJOR ? kStepK : (kSide / 32 | 1) * 32;
  static constexpr int kPlane = (KMAJOR ? kSide : kStepK) * kPitch;
  static_assert(kGroupThreads % kRowPieces == 0 && kLoads >= 1, "whole rows a turn");

  // The step from `k` on of the summed dimension.
  __device__ __forceinline__ static void load(const Panel<T>& p, int64_t k, Piece<T> (&out)[kLoads]) {
    load_panel<T, KMAJOR, kRowPieces, kLoads, kGroupThreads, kStepK, kSide>(p, k, out);
  }
  __device__ __forceinline__ static void store(const Piece<T> (&in)[kLoads], uint16_t* __restrict__ lds) {
    const int col = (int)threadIdx.x % kRowPieces * V, row0 = (int)threadIdx.x / kRowPieces;
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      const int row = row0 + i * (kGroupThreads / kRowPieces);
      *reinterpret_cast<u32x4*>(lds + row * kPitch + (KMAJOR ? 8 * ((col / 8) ^ (row >> 2 & 3)) : col)) =
          __builtin_bit_cast(u32x4, in[i].raw);
    }
  }
  // Operand of 32 rows from `first` on, steps 16 s .. + 15 of the sum: lane l's
  // eight values are row l % 32, k = 16 s + 8 (l / 32) + 0 .. 7.
  __device__ __forceinline__ static s16x8 read(const uint16_t* __restrict__ lds, int first, int s) {
    const int lane = threadIdx.x & 63, h = lane >> 5;
    if constexpr (KMAJOR) {
      const int row = first + (lane & 31);
      return *reinterpret_cast<const s16x8*>(lds + row * kPitch + 8 * ((2 * s + h) ^ (row >> 2 & 3)));
    } else {
      const int i = lane & 15, row = 16 * s + 8 * h + (i >> 2), col = first + 16 * (lane >> 4 & 1) + 4 * (i & 3);
      return join(read_column(lds + row * kPitch + col), read_column(lds + (row + 4) * kPitch + col));
    }
  }
};

// Sums of a tile of 128 x 128 in eight waves of 64 rows by 32 columns.
template <class T>
struct TileSums {
  f32x16 acc[2];
  __device__ __forceinline__ void clear() { acc[0] = acc[1] = f32x16{}; }
  // A's operand rows are the output's rows, B's its columns; result register r of
  // lane l is column 8 (r / 4) + 4 (l / 32) + r % 4 of row l % 32.
  template <class IA, class IB>
  __device__ __forceinline__ void step(const uint16_t* __restrict__ a, const uint16_t* __restrict__ b, int row0,
                                       int col0) {
#pragma unroll
    for (int s = 0; s < kStepK / 16; ++s) {
      const s16x8 y = IB::read(b, col0, s);
#pragma unroll
      for (int i = 0; i < 2; ++i) acc[i] = mma16<T>(y, IA::read(a, row0 + 32 * i, s), acc[i]);
    }
  }
};

// ---- float32 rows, on the float32 matrix cores

constexpr int kWideThreads = 256;

// SIDE outputs by kStepK of the sum.  KMAJOR: rows of 128 bytes whose eight
// 16-byte pieces are exchanged by the row's low bits; else 32 rows, four of which
// are 32 banks apart.
template <bool KMAJOR, int SIDE>
struct WidePanel {
  static constexpr int kRowPieces = (KMAJOR ? kStepK : SIDE) / 4;
  static constexpr int kLoads = SIDE * kStepK / 4 / kWideThreads;
  static constexpr int kPitch = KMAJOR ? kStepK : SIDE + 8;
  static constexpr int kFloats = (KMAJOR ? SIDE : kStepK) * kPitch;
  static_assert(kWideThreads % kRowPieces == 0 && kLoads >= 1, "whole rows a turn");

  __device__ __forceinline__ static void load(const Panel<float>& p, int64_t k, Piece<float> (&out)[kLoads]) {
    load_panel<float, KMAJOR, kRowPieces, kLoads, kWideThreads, kStepK, SIDE>(p, k, out);
  }
  __device__ __forceinline__ static void store(const Piece<float> (&in)[kLoads], float* __restrict__ lds) {
    const int piece = (int)threadIdx.x % kRowPieces, row0 = (int)threadIdx.x / kRowPieces;
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      const int row = row0 + i * (kWideThreads / kRowPieces);
      *reinterpret_cast<u32x4*>(lds + row * kPitch + 4 * (KMAJOR ? piece ^ (row >> 1 & 7) : piece)) =
          __builtin_bit_cast(u32x4, in[i].raw);
    }
  }
  // Operand of 32 outputs from `first` on, steps 8 s .. + 7 of the sum: lane l's four
  // values are output l % 32, k = 8 s + 4 (l / 32) + 0 .. 3.
  __device__ __forceinline__ static f32x4 read(const float* __restrict__ lds, int first, int s) {
    const int lane = threadIdx.x & 63, h = lane >> 5, c = lane & 31;
    if constexpr (KMAJOR) {
      return *reinterpret_cast<const f32x4*>(lds + (first + c) * kPitch + 4 * ((2 * s + h) ^ (c >> 1 & 7)));
    } else {
      const float* const at = lds + (8 * s + 4 * h) * kPitch + first + c;
      return f32x4{at[0], at[kPitch], at[2 * kPitch], at[3 * kPitch]};
    }
  }
};

// Sums of a tile of BM x BN in WM x WN waves over from .. to - 1 of the sum (from a
// multiple of a step); seen(pieces) is
// given A's pieces of each step (which of them a thread holds, does not change).
template <bool KA, bool KB, int BM, int BN, int WM, int WN>
struct WideTile {
  static constexpr int TM = BM / WM / 32, TN = BN / WN / 32;
  static_assert(WM * WN * 64 == kWideThreads && TM >= 1 && TN >= 1, "four waves");
  using A = WidePanel<KA, BM>;
  using B = WidePanel<KB, BN>;
  static constexpr int kRoom = std::max(A::kFloats + B::kFloats, kWideThreads / 64 * 1024);  // floats of LDS
  f32x16 acc[TM][TN];

  template <class F>
  __device__ __forceinline__ void run(const Panel<float>& pa, const Panel<float>& pb, int from, int to, float* room,
                                      F&& seen) {
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x / 64);
    const int row0 = wave / WN * (BM / WM), col0 = wave % WN * (BN / WN);
    float *const as = room, *const bs = room + A::kFloats;
#pragma unroll
    for (int i = 0; i < TM; ++i) {
#pragma unroll
      for (int j = 0; j < TN; ++j) acc[i][j] = f32x16{};
    }
    if (from >= to) return;
    Piece<float> ra[A::kLoads], rb[B::kLoads];
    A::load(pa, from, ra);
    B::load(pb, from, rb);
    for (int k = from; k < to; k += kStepK) {
      A::store(ra, as);
      B::store(rb, bs);
      seen(ra);
      __syncthreads();
      if (k + kStepK < to) {
        A::load(pa, k + kStepK, ra);
        B::load(pb, k + kStepK, rb);
      }
#pragma unroll
      for (int s = 0; s < kStepK / 8; ++s) {
        f32x4 x[TM], y[TN];
#pragma unroll
        for (int i = 0; i < TM; ++i) x[i] = A::read(as, row0 + 32 * i, s);
#pragma unroll
        for (int j = 0; j < TN; ++j) y[j] = B::read(bs, col0 + 32 * j, s);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
#pragma unroll
          for (int i = 0; i < TM; ++i) {
#pragma unroll
            for (int j = 0; j < TN; ++j)
              acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x2f32(y[j][e], x[i][e], acc[i][j], 0, 0, 0);
          }
        }
      }
      __syncthreads();
    }
  }
};

// A wave's 32 x 32 results through 4 KB of LDS of its own and out as rows:
// f(row, column, values) for pieces of V neighbouring columns.
template <class T, class F>
__device__ __forceinline__ void rows_of_tile(const f32x16& v, float* __restrict__ own, F&& f) {
  constexpr int V = Piece<T>::V, kPieces = 32 / V;
  const int lane = threadIdx.x & 63, c = lane & 31, h = lane >> 5;
  __builtin_amdgcn_wave_barrier();
#pragma unroll
  for (int q = 0; q < 4; ++q)
    *reinterpret_cast<f32x4*>(own + 32 * c + 4 * ((2 * q + h) ^ (c >> 1 & 7))) =
        f32x4{v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3]};
  __builtin_amdgcn_wave_barrier();
#pragma unroll
  for (int n = 0; n < kPieces / 2; ++n) {
    const int row = (64 * n + lane) / kPieces, at = (64 * n + lane) % kPieces;
    float o[V];
#pragma unroll
    for (int i = 0; i < V / 4; ++i) {
      const f32x4 t = *reinterpret_cast<const f32x4*>(own + 32 * row + 4 * ((at * (V / 4) + i) ^ (row >> 1 & 7)));
#pragma unroll
      for (int j = 0; j < 4; ++j) o[4 * i + j] = t[j];
    }
    f(row, V * at, o);
  }
}

// ---- 16-bit operands straight from memory to LDS

// 64 lanes' 16 bytes from memory to LDS, lane l's to lds + 16 l, past the
// registers; done once the wave's vector memory count says so.
__device__ __forceinline__ void load_to_lds(const void* src, void* lds) {
  __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)src,
                                   (__attribute__((address_space(3))) void*)lds, 16, 0, 0);
}
__device__ const uint4 kZeros16 = {0, 0, 0, 0};

// A panel of SIDE outputs by KS of the sum, 2 KS SIDE bytes of LDS for each of P
// pieces of its values, loaded by WAVES waves.  KMAJOR: rows of 2 KS bytes whose
// 16-byte pieces are exchanged by the row's low bits, read as they are.  Else KS
// rows of 2 SIDE bytes, read down their columns; the 64-byte quarters are
// exchanged by the row's low two bits, so that the four rows of a column read
// lie in different banks.
// Rows are whole 16-byte pieces at multiples of 16 bytes; the values' pieces are
// `plane` elements apart.
template <class T, int P, int KS, bool KMAJOR, int SIDE, int WAVES>
struct FastPanel {
  static constexpr int kLoads = SIDE * KS / 512 / WAVES, kPiece = SIDE * KS;  // 16-bit words
  static constexpr int kRowPieces = KS / 8;
  static_assert(kLoads * 512 * WAVES == SIDE * KS && SIDE >= 128, "whole loads, four quarters a row");
  const T* base;
  int64_t plane;
  int64_t step;         // elements from one step to the next
  uint32_t at[kLoads];  // of the lane's 16 bytes, from base
  int k[kLoads];        // where they stand in the sum's step

  // so that the 16 rows of a quarter wave's read lie in different 16 bytes of the 64 banks
  __device__ __forceinline__ static int exchange(int row) { return KS == 64 ? row >> 1 & 7 : row >> 2 & 3; }

  __device__ __forceinline__ FastPanel(const Panel<T>& p, int64_t plane) : base(p.base), plane(plane) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x / 64);
    step = KMAJOR ? KS : KS * p.stride;
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      const int word = (i * WAVES + wave) * 512 + 8 * lane;
      if constexpr (KMAJOR) {
        const int row = word / KS;
        k[i] = 8 * (word % KS / 8 ^ exchange(row));
        at[i] = (uint32_t)min(row, p.rows - 1) * (uint32_t)p.stride + (uint32_t)k[i];  // rows past the end: nobody stores them
      } else {
        const int row = word / SIDE, col = 8 * (word % SIDE / 8 ^ (row & 3) << 2);
        k[i] = row;
        at[i] = (uint32_t)row * (uint32_t)p.stride + (uint32_t)min(col, p.cols - 8);
      }
    }
  }
  // Step n into `lds`; `left`: what is left of the sum (zeros past it).
  __device__ __forceinline__ void load(int64_t n, int left, uint16_t* lds) const {
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x / 64);
#pragma unroll
    for (int p = 0; p < P; ++p) {
      const T* __restrict__ from = base + n * step + p * plane;
      uint16_t* const to = lds + p * kPiece;
      if (left >= KS) {
#pragma unroll
        for (int i = 0; i < kLoads; ++i) load_to_lds(from + at[i], to + (i * WAVES + wave) * 512);
      } else {
#pragma unroll
        for (int i = 0; i < kLoads; ++i)
          load_to_lds(k[i] < left ? (const void*)(from + at[i]) : (const void*)&kZeros16, to + (i * WAVES + wave) * 512);
      }
    }
  }
  // What a lane adds for the operand of 32 outputs from `first` on.
  __device__ __forceinline__ static int place(int first) {
    const int lane = threadIdx.x & 63, h = lane >> 5;
    if constexpr (KMAJOR) {
      return (first + (lane & 31)) * KS;
    } else {
      const int i = lane & 15, row = 8 * h + (i >> 2), col = first + 16 * (lane >> 4 & 1) + 4 * (i & 3);
      return row * SIDE + 8 * (col / 8 ^ (row & 3) << 2) + col % 8;
    }
  }
  // Steps 16 s .. + 15 of the sum: lane l's k = 16 s + 8 (l / 32) + 0 .. 7.
  __device__ __forceinline__ static s16x8 read(const uint16_t* lds, int place, int s) {
    if constexpr (KMAJOR) {
      const int lane = threadIdx.x & 63;
      return *reinterpret_cast<const s16x8*>(lds + place + 8 * ((2 * s + (lane >> 5)) ^ exchange(lane & 31)));
    } else {
      return join(read_column(lds + place + 16 * s * SIDE), read_column(lds + place + (16 * s + 4) * SIDE));
    }
  }
};

// Sums of a tile of BM x BN outputs over `len` of the sum, in WM x WN waves of
// BM / WM by BN / WN each.  Two stages of LDS: a step's panels are loaded under
// the products of the one before.
//
// P = 3: values as three bfloat16 pieces, largest first, and the six largest
// products.  A step's products have sums of their own, which are added to the
// total in float32 with a rounding to nearest: the matrix cores' own sums round
// down.
template <class T, int P, bool KA, bool KB, int BM, int BN, int WM, int WN, bool ONES>
struct FastTile {
  static constexpr int KS = P == 1 ? 64 : 32;
  static constexpr int kWaves = WM * WN, TM = BM / WM / 32, TN = BN / WN / 32;
  static constexpr int kPanelA = P * BM * KS, kStage = kPanelA + P * BN * KS;  // 16-bit words
  using A = FastPanel<T, P, KS, KA, BM, kWaves>;
  using B = FastPanel<T, P, KS, KB, BN, kWaves>;
  f32x16 acc[TM][TN];
  float ones;  // ONES: of A's rows alone: lane l's row l % 32 of the wave's tile wn

  __device__ __forceinline__ void run(const A& a, const B& b, int len, bool count, uint16_t* s0, uint16_t* s1) {
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x / 64), wn = wave % WN;
    int pa[TM], pb[TN];
#pragma unroll
    for (int i = 0; i < TM; ++i) {
      pa[i] = A::place(wave / WN * (BM / WM) + 32 * i);
#pragma unroll
      for (int j = 0; j < TN; ++j) acc[i][j] = f32x16{};
    }
#pragma unroll
    for (int j = 0; j < TN; ++j) pb[j] = B::place(wn * (BN / WN) + 32 * j);
    ones = 0.0f;
    s16x8 one;
#pragma unroll
    for (int j = 0; j < 8; ++j) one[j] = std::is_same_v<T, __half> ? 0x3c00 : 0x3f80;
    auto load = [&](int n, uint16_t* lds) {
      // past the last step: the last one again, which nothing reads
      const int at = min(n, (len - 1) / KS);
      a.load(at, len - at * KS, lds);
      b.load(at, len - at * KS, lds + kPanelA);
      __builtin_amdgcn_sched_barrier(0);  // the loads go out before the products, not after them
    };
    auto compute = [&](const uint16_t* lds) {
      f32x16 part[P == 3 ? TM : 1][P == 3 ? TN : 1];
      if constexpr (P == 3) {
#pragma unroll
        for (int i = 0; i < TM; ++i) {
#pragma unroll
          for (int j = 0; j < TN; ++j) part[i][j] = f32x16{};
        }
      }
#pragma unroll
      for (int s = 0; s < KS / 16; ++s) {
        s16x8 x[TM][P], y[TN][P];
#pragma unroll
        for (int p = 0; p < P; ++p) {
#pragma unroll
          for (int i = 0; i < TM; ++i) x[i][p] = A::read(lds + p * A::kPiece, pa[i], s);
#pragma unroll
          for (int j = 0; j < TN; ++j) y[j][p] = B::read(lds + kPanelA + p * B::kPiece, pb[j], s);
        }
        if constexpr (P == 1) {
#pragma unroll
          for (int i = 0; i < TM; ++i) {
#pragma unroll
            for (int j = 0; j < TN; ++j) acc[i][j] = mma16<T>(y[j][0], x[i][0], acc[i][j]);
          }
        } else {
          constexpr int kX[6] = {1, 2, 0, 1, 0, 0}, kY[6] = {1, 0, 2, 0, 1, 0};  // small products first
#pragma unroll
          for (int q = 0; q < 6; ++q) {
#pragma unroll
            for (int i = 0; i < TM; ++i) {
#pragma unroll
              for (int j = 0; j < TN; ++j) part[i][j] = mma16<T>(y[j][kY[q]], x[i][kX[q]], part[i][j]);
            }
          }
        }
      }
      if constexpr (P == 3) {
#pragma unroll
        for (int i = 0; i < TM; ++i) {
#pragma unroll
          for (int j = 0; j < TN; ++j) acc[i][j] += part[i][j];
        }
      }
      if constexpr (ONES) {
        if (count) {  // after the products, whose registers it would add to
          __builtin_amdgcn_sched_barrier(0);
          f32x16 sum = f32x16{};
#pragma unroll
          for (int i = 0; i < TM; ++i) {
            if (wn != i) continue;
#pragma unroll
            for (int s = 0; s < KS / 16; ++s) {
#pragma unroll
              for (int p = P - 1; p >= 0; --p) sum = mma16<T>(one, A::read(lds + p * A::kPiece, pa[i], s), sum);
            }
          }
          ones += sum[0];
        }
      }
    };
    if (len <= 0) return;
    const int steps = (len + KS - 1) / KS;
    load(0, s0);
    // every wave's loads of a step have landed, and every wave has read the step
    // before, whose place the next load takes
#define SPHOPS_TURN()                    \
  asm volatile("" ::: "memory");         \
  __builtin_amdgcn_s_waitcnt(0x0070);    \
  __builtin_amdgcn_s_barrier();          \
  asm volatile("" ::: "memory")
    int n = 0;
    for (; n + 1 < steps; n += 2) {
      SPHOPS_TURN();
      load(n + 1, s1);
      compute(s0);
      SPHOPS_TURN();
      load(n + 2, s0);
      compute(s1);
    }
    SPHOPS_TURN();  // no load in flight where LDS is used again
#undef SPHOPS_TURN
    if (n < steps) compute(s0);
    __syncthreads();
  }
};

}  // namespace

}  // namespace sphops
