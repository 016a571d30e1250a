// Rows sorted by expert and back, for gfx950.
//
// A row has k entries, each of which names an expert (or none: any number
// outside 0 .. experts - 1).  A stable counting sort gives every entry a place,
// expert after expert, the entries without one behind the last; rows are copied
// into their entries' places, and the experts' results come back as the sum
// over a row's entries of weight times result.  Nothing is added by atomics on
// floats: a row's entries are summed in their order.
#include "rows_out.hpp"

#include <type_traits>

namespace sphops {

namespace {

constexpr int kSortThreads = 512, kSortWaves = kSortThreads / 64;
// Entries a thread takes of a tile: few while tiles are few, whose steps follow one
// another (16384 entries, 64 experts: three launches of 9, 5 and 9 us with eight, of 4, 2
// and 5 with two).
constexpr int kFewItems = 2, kManyItems = 8;
constexpr int64_t kManyEntries = 1 << 18;

// An entry's key: its expert, `experts` for none.
__device__ __forceinline__ uint32_t key_of(const void* __restrict__ index, bool wide, int64_t i, int experts) {
  const int64_t e = wide ? static_cast<const int64_t*>(index)[i] : static_cast<const int32_t*>(index)[i];
  return e >= 0 && e < experts ? (uint32_t)e : (uint32_t)experts;
}

// The lanes of the wave whose key is this lane's (`bits` wide), among those
// that are live.
__device__ __forceinline__ uint64_t same_key(uint32_t key, bool live, int bits) {
  uint64_t m = __ballot(live);
  for (int b = 0; b < bits; ++b) {
    const uint64_t set = __ballot((key >> b) & 1);
    m &= (key >> b) & 1 ? set : ~set;
  }
  return m;
}

// A tile's entries: the wave's share in order, 64 at a time.  Each gets its key
// and its rank among the wave's entries of that key; counts[wave][key] holds
// their number.
template <int ITEMS>
__device__ __forceinline__ void rank_tile(const void* __restrict__ index, bool wide, int64_t first, int64_t n,
                                          int experts, int bits, uint32_t* __restrict__ counts, uint32_t (&key)[ITEMS],
                                          uint32_t (&rank)[ITEMS]) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
  for (int i = 0; i < ITEMS; ++i) {
    const int64_t at = first + (int64_t)(wave * ITEMS + i) * 64 + lane;
    key[i] = at < n ? key_of(index, wide, at, experts) : 0xffffffffu;
  }
  for (int i = threadIdx.x; i < kSortWaves * (experts + 1); i += kSortThreads) counts[i] = 0;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < ITEMS; ++i) {
    const bool live = key[i] != 0xffffffffu;
    const uint64_t same = same_key(key[i], live, bits);
    const int leader = live ? __ffsll((unsigned long long)same) - 1 : lane;
    uint32_t before = 0;
    if (live && lane == leader)
      before = atomicAdd(&counts[wave * (experts + 1) + key[i]], (uint32_t)__popcll(same));
    before = (uint32_t)__shfl((int)before, leader);
    rank[i] = before + (uint32_t)__popcll(same & ((1ull << lane) - 1));
  }
  __syncthreads();
}

// Exclusive sums of total[0 .. experts - 1] in place; total[experts] receives
// the sum of them all, which is where the entries without an expert start.
__device__ __forceinline__ void scan_experts(uint32_t* __restrict__ total, int experts) {
  __shared__ uint32_t waves[kSortWaves];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  uint32_t carry = 0;
  for (int base = 0; base < experts; base += kSortThreads) {
    const int e = base + threadIdx.x;
    const uint32_t mine = e < experts ? total[e] : 0;
    uint32_t v = mine;
#pragma unroll
    for (int s = 1; s < 64; s *= 2) {
      const uint32_t other = (uint32_t)__shfl_up((int)v, s);
      if (lane >= s) v += other;
    }
    if (lane == 63) waves[wave] = v;
    __syncthreads();
    uint32_t all = 0;
#pragma unroll
    for (int i = 0; i < kSortWaves; ++i) {
      if (i < wave) v += waves[i];
      all += waves[i];
    }
    if (e < experts) total[e] = carry + v - mine;
    carry += all;
    __syncthreads();
  }
  if (threadIdx.x == 0) total[experts] = carry;
  __syncthreads();
}

// hist[key * tiles + tile]: the tile's entries of each key.
// Bound (this, the scan and the places): latency; 2^20 entries of 4 experts in 8 + 5
// + 9 us, 16384 of 64 in 4 + 2 + 5, one launch of 3 for a few.
template <int ITEMS>
__global__ __launch_bounds__(kSortThreads) void k_sort_count(const void* __restrict__ index, bool wide, int64_t n,
                                                             int experts, int bits, uint32_t* __restrict__ hist) {
  extern __shared__ uint32_t counts[];
  uint32_t key[ITEMS], rank[ITEMS];
  rank_tile<ITEMS>(index, wide, (int64_t)blockIdx.x * kSortThreads * ITEMS, n, experts, bits, counts, key, rank);
  for (int e = threadIdx.x; e <= experts; e += kSortThreads) {
    uint32_t t = 0;
#pragma unroll
    for (int w = 0; w < kSortWaves; ++w) t += counts[w * (experts + 1) + e];
    hist[(int64_t)e * gridDim.x + blockIdx.x] = t;
  }
}

// Exclusive sums over a key's tiles, in place; total[key]: all of them.
__global__ __launch_bounds__(256) void k_sort_scan(uint32_t* __restrict__ hist, int tiles,
                                                   uint32_t* __restrict__ total) {
  __shared__ uint32_t waves[4];
  uint32_t* __restrict__ row = hist + (int64_t)blockIdx.x * tiles;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  uint32_t carry = 0;
  for (int base = 0; base < tiles; base += 256) {
    const int t = base + threadIdx.x;
    const uint32_t mine = t < tiles ? row[t] : 0;
    uint32_t v = mine;
#pragma unroll
    for (int s = 1; s < 64; s *= 2) {
      const uint32_t other = (uint32_t)__shfl_up((int)v, s);
      if (lane >= s) v += other;
    }
    if (lane == 63) waves[wave] = v;
    __syncthreads();
    uint32_t all = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (i < wave) v += waves[i];
      all += waves[i];
    }
    if (t < tiles) row[t] = carry + v - mine;
    carry += all;
    __syncthreads();
  }
  if (threadIdx.x == 0) total[blockIdx.x] = carry;
}

// Places.  One tile alone (hist null) needs no other launch.
template <int ITEMS>
__global__ __launch_bounds__(kSortThreads) void k_sort_place(const void* __restrict__ index, bool wide, int64_t n,
                                                             int experts, int bits, const uint32_t* __restrict__ hist,
                                                             const uint32_t* __restrict__ totals,
                                                             int32_t* __restrict__ offsets, int32_t* __restrict__ slot,
                                                             int32_t* __restrict__ source) {
  extern __shared__ uint32_t counts[];  // kSortWaves + 1 rows of experts + 1
  uint32_t* const base = counts + kSortWaves * (experts + 1);
  uint32_t key[ITEMS], rank[ITEMS];
  const int64_t first = (int64_t)blockIdx.x * kSortThreads * ITEMS;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  rank_tile<ITEMS>(index, wide, first, n, experts, bits, counts, key, rank);
  // a key's waves one after another
  for (int e = threadIdx.x; e <= experts; e += kSortThreads) {
    uint32_t t = 0;
#pragma unroll
    for (int w = 0; w < kSortWaves; ++w) {
      const uint32_t c = counts[w * (experts + 1) + e];
      counts[w * (experts + 1) + e] = t;
      t += c;
    }
    base[e] = hist != nullptr ? totals[e] : t;
  }
  __syncthreads();
  scan_experts(base, experts);
  if (blockIdx.x == 0) {
    for (int e = threadIdx.x; e <= experts; e += kSortThreads) offsets[e] = (int32_t)base[e];
  }
  if (hist != nullptr) {
    __syncthreads();
    for (int e = threadIdx.x; e <= experts; e += kSortThreads) base[e] += hist[(int64_t)e * gridDim.x + blockIdx.x];
    __syncthreads();
  }
#pragma unroll
  for (int i = 0; i < ITEMS; ++i) {
    const int64_t at = first + (int64_t)(wave * ITEMS + i) * 64 + lane;
    if (at >= n) continue;
    const int32_t p = (int32_t)(base[key[i]] + counts[wave * (experts + 1) + key[i]] + rank[i]);
    slot[at] = key[i] < (uint32_t)experts ? p : ~p;
    source[p] = (int32_t)at;
  }
}

constexpr int kMoveThreads = 256;

// Values of a row's piece times w, each rounded once.
template <class T>
__device__ __forceinline__ Piece<T> scaled(const Piece<T>& p, float w) {
  float v[Piece<T>::V];
#pragma unroll
  for (int j = 0; j < Piece<T>::V; ++j) v[j] = p.get(j) * w;
  return piece_of<T>(v);
}

// out[slot[r, j]] = x[r], zeros for an entry without an expert.  L lanes a row's
// block of L x N pieces.  Bound: HBM; 8192 x 4096 bfloat16, two entries each, in 35 us
// (201 MB, part of them in cache).
template <class T, int L, int N>
__global__ __launch_bounds__(kMoveThreads) void k_rows_out(const T* __restrict__ x, int64_t stride,
                                                           const int32_t* __restrict__ slot, T* __restrict__ out,
                                                           int64_t rows, int choices, int cols) {
  constexpr int V = Piece<T>::V;
  const int l = threadIdx.x % L, k0 = (int)blockIdx.y * L * N * V;
  const int64_t slots = rows * choices;
  for (int64_t r = (int64_t)blockIdx.x * (kMoveThreads / L) + threadIdx.x / L; r < rows;
       r += (int64_t)gridDim.x * (kMoveThreads / L)) {
    Piece<T> p[N];
#pragma unroll
    for (int n = 0; n < N; ++n) p[n].load(x + r * stride, k0 + (n * L + l) * V, cols);
    for (int j = 0; j < choices; ++j) {
      const int32_t s = slot[r * choices + j], at = s < 0 ? ~s : s;
      if (at >= slots) continue;
#pragma unroll
      for (int n = 0; n < N; ++n) {
        Piece<T> o = p[n];
        if (s < 0) o.raw = typename Piece<T>::Raw{};
        o.store(out + (int64_t)at * cols, k0 + (n * L + l) * V, cols);
      }
    }
  }
}

// The backward of k_rows_in: out[slot[r, j]] = w[r, j] dy[r] (zeros without an
// expert) and dw[r, j] = result[slot[r, j]] . dy[r] (0 without one).  HELD: the
// row's pieces stay in registers over its entries.  Bound: HBM; 8192 x 4096
// bfloat16, two entries each, in 62 us (5.4 TB/s).
template <class T, int L, int N, bool HELD>
__global__ __launch_bounds__(kMoveThreads) void k_rows_in_backward(
    const T* __restrict__ dy, int64_t stride, const T* __restrict__ results, const float* __restrict__ w,
    const int32_t* __restrict__ slot, T* __restrict__ out, float* __restrict__ dw, int64_t rows, int choices,
    int cols) {
  constexpr int V = Piece<T>::V, kRows = kMoveThreads / L;
  __shared__ float meet[2][kMoveThreads / 64];
  const int l = threadIdx.x % L;
  const int64_t slots = rows * choices;
  int turn = 0;
  for (int64_t r0 = (int64_t)blockIdx.x * kRows; r0 < rows; r0 += (int64_t)gridDim.x * kRows) {
    const bool live = r0 + threadIdx.x / L < rows;
    const int64_t r = live ? r0 + threadIdx.x / L : rows - 1;
    const T* __restrict__ row = dy + r * stride;
    Piece<T> p[N];
    if constexpr (HELD) {
#pragma unroll
      for (int n = 0; n < N; ++n) p[n].load(row, (n * L + l) * V, cols);
    }
    for (int j = 0; j < choices; ++j, turn ^= 1) {
      const int32_t s = slot[r * choices + j], at = s < 0 ? ~s : s;
      const float weight = s < 0 ? 0.0f : w != nullptr ? w[r * choices + j] : 1.0f;
      const bool there = live && at < slots;
      float dot = 0.0f;
      for (int k0 = 0; k0 < cols; k0 += L * N * V) {
        if constexpr (!HELD) {
#pragma unroll
          for (int n = 0; n < N; ++n) p[n].load(row, k0 + (n * L + l) * V, cols);
        }
        if (dw != nullptr && s >= 0 && there) {
#pragma unroll
          for (int n = 0; n < N; ++n) {
            Piece<T> q;
            q.load(results + (int64_t)at * cols, k0 + (n * L + l) * V, cols);
#pragma unroll
            for (int v = 0; v < V; ++v) dot += p[n].get(v) * q.get(v);
          }
        }
        if (out != nullptr && there) {
#pragma unroll
          for (int n = 0; n < N; ++n) {
            Piece<T> o = scaled(p[n], weight);
            if (s < 0) o.raw = typename Piece<T>::Raw{};  // whatever dy holds
            o.store(out + (int64_t)at * cols, k0 + (n * L + l) * V, cols);
          }
        }
        if constexpr (HELD) break;
      }
      if (dw == nullptr) continue;
#pragma unroll
      for (int d = 1; d < (L < 64 ? L : 64); d *= 2) dot += __shfl_xor(dot, d);
      if constexpr (L > 64) {
        if (threadIdx.x % 64 == 0) meet[turn][threadIdx.x / 64] = dot;
        __syncthreads();
        dot = 0.0f;
#pragma unroll
        for (int i = 0; i < L / 64; ++i) dot += meet[turn][i];
      }
      if (live && l == 0) dw[r * choices + j] = dot;
    }
  }
}

// y[r] = the sum over its entries, in their order, of w[r, j] result[slot[r,
// j]] (w null: 1), in float32; entries without an expert are left out.  Bound: HBM;
// 2^20 x 83 float32, one entry each, in 154 us (4.5 TB/s), 8192 x 4096 bfloat16, two, in
// 46.
template <class T, int L, int N>
__global__ __launch_bounds__(kMoveThreads) void k_rows_in(const T* __restrict__ results, int64_t stride,
                                                          const float* __restrict__ w,
                                                          const int32_t* __restrict__ slot, T* __restrict__ y,
                                                          int64_t rows, int choices, int cols) {
  constexpr int V = Piece<T>::V, kRows = kMoveThreads / L;
  __shared__ __attribute__((aligned(16))) RowsOut<T, L, N> outs[kMoveThreads / 64];
  const int l = threadIdx.x % L, k0 = (int)blockIdx.y * L * N * V, wave = (int)threadIdx.x / 64;
  const int64_t slots = rows * choices;
  for (int64_t r0 = (int64_t)blockIdx.x * kRows; r0 < rows; r0 += (int64_t)gridDim.x * kRows) {
    const int64_t r = min<int64_t>(r0 + threadIdx.x / L, rows - 1);
    float sum[N][V];
#pragma unroll
    for (int n = 0; n < N; ++n) {
#pragma unroll
      for (int v = 0; v < V; ++v) sum[n][v] = 0.0f;
    }
#pragma unroll 2
    for (int j = 0; j < choices; ++j) {
      const int32_t s = slot[r * choices + j];
      if (s < 0 || s >= slots) continue;
      const float weight = w != nullptr ? w[r * choices + j] : 1.0f;
#pragma unroll
      for (int n = 0; n < N; ++n) {
        Piece<T> p;
        load_piece(p, false, results + (int64_t)s * stride, k0 + (n * L + l) * V, cols);
#pragma unroll
        for (int v = 0; v < V; ++v) sum[n][v] += weight * p.get(v);
      }
    }
    Piece<T> o[N];
#pragma unroll
    for (int n = 0; n < N; ++n) o[n] = piece_of<T>(sum[n]);
    if (RowsOut<T, L, N>::kStaged) {  // one block of columns
      outs[wave](o, y, r0 + wave * 64 / L, rows, cols);
    } else if (r0 + threadIdx.x / L < rows) {
#pragma unroll
      for (int n = 0; n < N; ++n) {
        const int k = k0 + (n * L + l) * V;
        if (k < cols) o[n].store(y + r * cols, k, cols);
      }
    }
  }
}

// k_rows_out and k_rows_in_backward over the places, for rows that have one entry
// each and few values: out[p] = w[r] x[r] for the row r = source[p] (w null: 1; zeros
// without an expert) and dw[r] = results[p] . x[r] (dw null: not wanted).  What is
// written lies in order and leaves in whole runs: 2^20 x 83 float32 out 175 us row by
// row, 167 so; combine's gradients 249.
template <class T, int L, int N>
__global__ __launch_bounds__(kMoveThreads) void k_places_out(const T* __restrict__ x, int64_t stride,
                                                             const T* __restrict__ results,
                                                             const float* __restrict__ w,
                                                             const int32_t* __restrict__ slot,
                                                             const int32_t* __restrict__ source, T* __restrict__ out,
                                                             float* __restrict__ dw, int64_t places, int cols) {
  constexpr int V = Piece<T>::V, kRows = kMoveThreads / L;
  __shared__ __attribute__((aligned(16))) RowsOut<T, L, N> outs[kMoveThreads / 64];
  const int l = threadIdx.x % L, wave = (int)threadIdx.x / 64;
  for (int64_t p0 = (int64_t)blockIdx.x * kRows; p0 < places; p0 += (int64_t)gridDim.x * kRows) {
    const int64_t p = min<int64_t>(p0 + threadIdx.x / L, places - 1);
    const int32_t from = source[p];
    const bool known = from >= 0 && from < places, has = known && slot[known ? from : 0] == (int32_t)p;
    const int64_t r = known ? from : 0;
    const float weight = has && w != nullptr ? w[r] : 1.0f;
    Piece<T> v[N], q[N];
#pragma unroll
    for (int n = 0; n < N; ++n) {
      load_piece(v[n], n < N - 1, x + r * stride, (n * L + l) * V, cols);
      if (dw != nullptr) load_piece(q[n], n < N - 1, results + p * cols, (n * L + l) * V, cols);
    }
    if (dw != nullptr) {
      float dot = 0.0f;
#pragma unroll
      for (int n = 0; n < N; ++n) {
#pragma unroll
        for (int j = 0; j < V; ++j) dot += v[n].get(j) * q[n].get(j);
      }
#pragma unroll
      for (int d = 1; d < L; d *= 2) dot += __shfl_xor(dot, d);
      if (l == 0 && known) dw[r] = has ? dot : 0.0f;
    }
    if (out != nullptr) {
#pragma unroll
      for (int n = 0; n < N; ++n) {
        if (w != nullptr) v[n] = scaled(v[n], weight);
        if (!has) v[n].raw = typename Piece<T>::Raw{};
      }
      outs[wave](v, out, p0 + wave * 64 / L, places, cols);
    }
  }
}

// f(integral_constants L, N): lanes for rows of `pieces` 16-byte pieces, which
// take more than one block of columns from 257 pieces on.
template <class F>
void with_lanes(int64_t pieces, F&& f) {
#define SPHOPS_LANES(L, N) f(std::integral_constant<int, L>{}, std::integral_constant<int, N>{})
  if (pieces <= 4) SPHOPS_LANES(4, 1);
  else if (pieces <= 8) SPHOPS_LANES(8, 1);
  else if (pieces <= 16) SPHOPS_LANES(8, 2);
  else if (pieces <= 24) SPHOPS_LANES(8, 3);
  else if (pieces <= 32) SPHOPS_LANES(16, 2);
  else if (pieces <= 48) SPHOPS_LANES(16, 3);
  else if (pieces <= 64) SPHOPS_LANES(32, 2);
  else if (pieces <= 128) SPHOPS_LANES(64, 2);
  else SPHOPS_LANES(64, 4);
#undef SPHOPS_LANES
}

dim3 move_grid(int64_t rows, int rows_a_turn, int64_t blocks) {
  return dim3((uint32_t)std::min<int64_t>((rows + rows_a_turn - 1) / rows_a_turn, 16384), (uint32_t)blocks);
}

template <class T>
int64_t pieces_of(int64_t cols) { return (cols + Piece<T>::V - 1) / Piece<T>::V; }

int key_bits(int experts) {
  int bits = 1;
  while ((experts >> bits) != 0) ++bits;
  return bits;
}

// One workgroup's work takes no other launch.
int sort_items(int64_t n) {
  if (n <= kSortThreads) return 1;
  return n <= kSortThreads * kManyItems || n > kManyEntries ? kManyItems : kFewItems;
}
int64_t sort_tiles(int64_t n) {
  const int64_t tile = (int64_t)kSortThreads * sort_items(n);
  return (n + tile - 1) / tile;
}

// Rows of one entry each that k_places_out takes.
template <class T>
bool by_places(int choices, const int32_t* source, int64_t cols) {
  return choices == 1 && source != nullptr && pieces_of<T>(cols) <= 48;
}
// f(integral_constants L, N) for them.
template <class F>
void with_place_lanes(int64_t pieces, F&& f) {
#define SPHOPS_LANES(L, N) f(std::integral_constant<int, L>{}, std::integral_constant<int, N>{})
  if (pieces <= 4) SPHOPS_LANES(4, 1);
  else if (pieces <= 8) SPHOPS_LANES(8, 1);
  else if (pieces <= 16) SPHOPS_LANES(8, 2);
  else if (pieces <= 24) SPHOPS_LANES(8, 3);
  else if (pieces <= 32) SPHOPS_LANES(16, 2);
  else SPHOPS_LANES(16, 3);
#undef SPHOPS_LANES
}

template <class T>
void launch_places(const void* x, int64_t stride, const void* results, const float* w, const int32_t* slot,
                   const int32_t* source, void* out, float* dw, int64_t places, int64_t cols, hipStream_t st) {
  with_place_lanes(pieces_of<T>(cols), [&](auto l, auto n) {
    constexpr int L = decltype(l)::value;
    hipLaunchKernelGGL((k_places_out<T, L, decltype(n)::value>), move_grid(places, kMoveThreads / L, 1),
                       dim3(kMoveThreads), 0, st, static_cast<const T*>(x), stride, static_cast<const T*>(results), w,
                       slot, source, static_cast<T*>(out), dw, places, (int)cols);
  });
}

}  // namespace

int64_t sort_rows_workspace_words(int64_t n, int experts) {
  const int64_t tiles = sort_tiles(n);
  return tiles <= 1 ? 0 : (tiles + 1) * (experts + 1);
}

void run_sort_rows(const void* index, bool wide, int64_t n, int experts, int32_t* offsets, int32_t* slot,
                   int32_t* source, uint32_t* work, hipStream_t st) {
  const int bits = key_bits(experts);
  const uint32_t lds = (uint32_t)((kSortWaves + 1) * (experts + 1) * sizeof(uint32_t));
  const int64_t tiles = sort_tiles(n);
  auto place = [&](auto items, const uint32_t* hist, const uint32_t* totals) {
    hipLaunchKernelGGL((k_sort_place<decltype(items)::value>), dim3((uint32_t)std::max<int64_t>(tiles, 1)), dim3(kSortThreads), lds, st,
                       index, wide, n, experts, bits, hist, totals, offsets, slot, source);
  };
  const auto with_items = [&](auto&& f) {
    const int items = sort_items(n);
    if (items == 1) f(std::integral_constant<int, 1>{});
    else if (items == kFewItems) f(std::integral_constant<int, kFewItems>{});
    else f(std::integral_constant<int, kManyItems>{});
  };
  if (tiles <= 1) {
    with_items([&](auto items) { place(items, nullptr, nullptr); });
    SPHOPS_LAUNCHED();
    return;
  }
  uint32_t* const totals = work + tiles * (experts + 1);
  with_items([&](auto items) {
    hipLaunchKernelGGL((k_sort_count<decltype(items)::value>), dim3((uint32_t)tiles), dim3(kSortThreads), lds, st, index,
                       wide, n, experts, bits, work);
  });
  SPHOPS_LAUNCHED();
  hipLaunchKernelGGL(k_sort_scan, dim3((uint32_t)(experts + 1)), dim3(256), 0, st, work, (int)tiles, totals);
  SPHOPS_LAUNCHED();
  with_items([&](auto items) { place(items, work, totals); });
  SPHOPS_LAUNCHED();
}

void run_dispatch_rows(const void* x, int type, int64_t stride, const int32_t* slot, const int32_t* source, void* out,
                       int64_t rows, int choices, int64_t cols, hipStream_t st) {
  if (rows == 0) return;
  with_type(type, [&](auto t) {
    using T = decltype(t);
    if (by_places<T>(choices, source, cols)) {
      launch_places<T>(x, stride, nullptr, nullptr, slot, source, out, nullptr, rows, cols, st);
      return;
    }
    with_lanes(pieces_of<T>(cols), [&](auto l, auto n) {
      constexpr int L = decltype(l)::value, N = decltype(n)::value, V = Piece<T>::V;
      hipLaunchKernelGGL((k_rows_out<T, L, N>), move_grid(rows, kMoveThreads / L, (cols + L * N * V - 1) / (L * N * V)),
                         dim3(kMoveThreads), 0, st, static_cast<const T*>(x), stride, slot, static_cast<T*>(out), rows,
                         choices, (int)cols);
    });
  });
  SPHOPS_LAUNCHED();
}

void run_combine_rows(const void* results, int type, int64_t stride, const float* w, const int32_t* slot, void* y,
                      int64_t rows, int choices, int64_t cols, hipStream_t st) {
  if (rows == 0) return;
  with_type(type, [&](auto t) {
    using T = decltype(t);
    with_lanes(pieces_of<T>(cols), [&](auto l, auto n) {
      constexpr int L = decltype(l)::value, N = decltype(n)::value, V = Piece<T>::V;
      hipLaunchKernelGGL((k_rows_in<T, L, N>), move_grid(rows, kMoveThreads / L, (cols + L * N * V - 1) / (L * N * V)),
                         dim3(kMoveThreads), 0, st, static_cast<const T*>(results), stride, w, slot,
                         static_cast<T*>(y), rows, choices, (int)cols);
    });
  });
  SPHOPS_LAUNCHED();
}

void run_combine_rows_backward(const void* dy, int type, int64_t stride, const void* results, const float* w,
                               const int32_t* slot, const int32_t* source, void* d_results, float* dw, int64_t rows,
                               int choices, int64_t cols, hipStream_t st) {
  if (rows == 0) return;
  with_type(type, [&](auto t) {
    using T = decltype(t);
    if (by_places<T>(choices, source, cols)) {
      launch_places<T>(dy, stride, results, w, slot, source, d_results, dw, rows, cols, st);
      return;
    }
    const int64_t pieces = pieces_of<T>(cols);
    auto launch = [&](auto l, auto n, auto held) {
      constexpr int L = decltype(l)::value;
      hipLaunchKernelGGL((k_rows_in_backward<T, L, decltype(n)::value, decltype(held)::value>),
                         move_grid(rows, kMoveThreads / L, 1), dim3(kMoveThreads), 0, st, static_cast<const T*>(dy),
                         stride, static_cast<const T*>(results), w, slot, static_cast<T*>(d_results), dw, rows, choices,
                         (int)cols);
    };
    const std::integral_constant<int, 256> wide{};
    if (pieces <= 256) with_lanes(pieces, [&](auto l, auto n) { launch(l, n, std::true_type{}); });
    else if (pieces <= 512) launch(wide, std::integral_constant<int, 2>{}, std::true_type{});
    else if (pieces <= 1024) launch(wide, std::integral_constant<int, 4>{}, std::true_type{});
    else launch(wide, std::integral_constant<int, 4>{}, std::false_type{});
  });
  SPHOPS_LAUNCHED();
}

}  // namespace sphops
