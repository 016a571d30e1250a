// Linear layers of experts over rows sorted by expert, for gfx950:
//
//   y[s] = x[s] W_e^T + b_e   dx[s] = dy[s] W_e   dW_e = sum of dy[s]^T x[s]   db_e = sum of dy[s]
//
// over the rows s of expert e, offsets[e] <= s < offsets[e + 1]; rows behind the
// last expert's are zeros.  16-bit rows go to the matrix cores as they are,
// float32 ones as three bfloat16 pieces of each factor and six products
// (split16.hpp).  Sums are float32.
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

// y (slots x outs) = x (slots x cols) W_e^T + b_e, W_e (outs x cols); BACK: y = x
// W_e with W_e (cols x outs), which is the input gradient.  relu: y = max(y, 0).
// mask (slots x outs): y = 0 where it is not above 0.
template <class T, bool BACK>
__global__ __launch_bounds__(kGroupThreads) void k_group_rows(const T* __restrict__ x, int64_t xs,
                                                              const T* __restrict__ w, const T* __restrict__ b,
                                                              const T* __restrict__ mask,
                                                              const int32_t* __restrict__ offsets, T* __restrict__ y,
                                                              int64_t slots, int experts, int cols, int outs,
                                                              bool relu, int64_t mt, int nt) {
  using IA = PanelImage<T, true>;
  using IB = PanelImage<T, !BACK>;
  constexpr int P = Pieces<T>::P, V = Piece<T>::V;
  __shared__ __attribute__((aligned(16))) uint16_t room[std::max(P * (IA::kPlane + IB::kPlane), kOutbox)];
  uint16_t *const as = room, *const bs = room + P * IA::kPlane;
  int64_t m;
  int n;
  tile_of(xcd_block_id(), mt, nt, m, n);
  const GroupTile g = group_tile(offsets, experts, slots, m, kSide, true);
  if (g.group < 0) return;
  const int64_t m0 = g.lo + g.tile * kSide;
  const int n0 = n * kSide, here = (int)min<int64_t>(kSide, g.hi - m0), outs_here = min(kSide, outs - n0);
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x / 64);
  const int row0 = wave / 4 * 64, col0 = wave % 4 * 32;
  if (g.group == experts) {  // rows behind the last expert's
    for (int i = threadIdx.x; i < here * (kSide / V); i += kGroupThreads) {
      Piece<T> o;
      o.raw = typename Piece<T>::Raw{};
      o.store(y + (m0 + i / (kSide / V)) * outs, n0 + i % (kSide / V) * V, outs);
    }
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
    if ((k & (128 - kStepK)) == 128 - kStepK) sums.flush();
    __syncthreads();
  }
  sums.flush();
  float* const own = reinterpret_cast<float*>(room) + 1024 * wave;  // every wave is done with the panels
  const T* const be = b != nullptr ? b + (int64_t)g.group * outs : nullptr;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    rows_of_tile<T>(sums.value(i), own, [&](int r, int c, float (&v)[V]) {
      const int row = row0 + 32 * i + r, at = n0 + col0 + c;
      if (row >= here || at >= outs) return;
      Piece<T> o, t;
      if (be != nullptr) {
        t.load(be, at, outs);
#pragma unroll
        for (int j = 0; j < V; ++j) v[j] += t.get(j);
      }
      if (mask != nullptr) t.load(mask + (m0 + row) * outs, at, outs);
      o.raw = typename Piece<T>::Raw{};
#pragma unroll
      for (int j = 0; j < V; ++j) {
        if (relu) v[j] = v[j] <= 0.0f ? 0.0f : v[j];  // NaN stays
        if (mask != nullptr && t.get(j) <= 0.0f) v[j] = 0.0f;
        o.set(j, from_f32<T>(v[j]));
      }
      o.store(y + (m0 + row) * outs, at, outs);
    });
  }
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
  constexpr int P = Pieces<T>::P, V = Piece<T>::V;
  __shared__ __attribute__((aligned(16))) uint16_t room[std::max(P * 2 * I::kPlane, kOutbox)];
  uint16_t *const as = room, *const bs = room + P * I::kPlane;
  const uint32_t id = xcd_block_id();
  const int tiles = mt * nt, at = (int)(id % tiles);
  const int64_t piece = id / tiles;
  const int n = at % nt, m0 = at / nt * kSide, n0 = n * kSide;
  GroupTile g;
  if (part == nullptr) {
    const int e = (int)piece;
    g.group = e;
    g.lo = e == 0 ? 0 : min<int64_t>(max(offsets[e], 0), slots);
    g.hi = max<int64_t>(g.lo, min<int64_t>(offsets[e + 1], slots));
    g.tile = 0;
  } else {
    g = group_tile(offsets, experts, slots, piece, chunk, false);
    if (g.group < 0) return;
  }
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
    if ((k & (128 - kStepK)) == 128 - kStepK) sums.flush();
    __syncthreads();
  }
  sums.flush();
  const int64_t nw = (int64_t)outs * cols;
  float* const own = reinterpret_cast<float*>(room) + 1024 * wave;  // every wave is done with the panels
  float* const mine = part != nullptr ? part + piece * (nw + outs) : nullptr;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    auto put = [&](auto type, auto* to) {
      using O = decltype(type);
      rows_of_tile<O>(sums.value(i), own, [&](int r, int c, float (&v)[Piece<O>::V]) {
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

// dW and db of expert blockIdx.y: its chunks' sums in the chunks' order.
template <class T>
__global__ __launch_bounds__(256) void k_group_chunk_sum(const float* __restrict__ part,
                                                         const int32_t* __restrict__ offsets, T* __restrict__ dw,
                                                         T* __restrict__ db, int64_t slots, int experts, int64_t nw,
                                                         int outs, int64_t chunk, int64_t chunks) {
  const int e = (int)blockIdx.y;
  // the expert's first chunk: every wave counts the chunks of those before it
  int64_t before = 0, mine = 0;
  for (int base = 0; base <= e; base += 64) {
    const int i = base + (int)(threadIdx.x & 63);
    int64_t c = 0;
    if (i <= e) {
      const int64_t lo = i == 0 ? 0 : min<int64_t>(max(offsets[i], 0), slots);
      c = (max<int64_t>(lo, min<int64_t>(offsets[i + 1], slots)) - lo + chunk - 1) / chunk;
    }
    if (e >= base && e < base + 64) mine = __shfl(c, e - base);
    if (i == e) c = 0;
#pragma unroll
    for (int s = 1; s < 64; s *= 2) c += __shfl_xor(c, s);
    before += c;
  }
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
  int mt, nt;
  int64_t chunk, chunks;  // chunks 0: a workgroup takes all of an expert's rows
};
GradPlan grad_plan(int64_t slots, int experts, int64_t cols, int64_t outs) {
  GradPlan p;
  p.mt = (int)tiles_of(outs, kSide);
  p.nt = (int)tiles_of(cols, kSide);
  const int64_t tiles = (int64_t)p.mt * p.nt;
  const int64_t want = std::max<int64_t>(1, 512 / tiles);  // chunks in all
  p.chunk = std::min(kMaxGroupChunk, std::max<int64_t>(256, tiles_of(tiles_of(slots, want), kStepK) * kStepK));
  p.chunks = most_tiles(slots, experts, p.chunk);
  if (slots <= p.chunk || (tiles * experts >= 512 && slots <= 2 * kMaxGroupChunk)) {
    p.chunk = std::max<int64_t>(slots, 1);
    p.chunks = 0;
  }
  return p;
}

}  // namespace

bool group_linear_fits(int64_t slots, int experts, int64_t cols, int64_t outs) {
  const int64_t mt = most_tiles(slots, experts + 1, kSide);
  const GradPlan p = grad_plan(slots, experts, cols, outs);
  const int64_t limit = (int64_t(1) << 32) / kGroupThreads;  // threads a launch
  return mt * tiles_of(outs, kSide) < limit && mt * tiles_of(cols, kSide) < limit &&
         (int64_t)p.mt * p.nt * std::max<int64_t>(p.chunks, experts) < limit &&
         tiles_of(cols * outs + outs, 256) * experts < limit;
}

void run_group_linear(const void* x, int type, int64_t xs, const void* w, const void* b, const void* mask,
                      const int32_t* offsets, void* y, int64_t slots, int experts, int64_t cols, int64_t outs,
                      bool relu, bool back, hipStream_t st) {
  if (slots == 0) return;
  with_type(type, [&](auto t) {
    using T = decltype(t);
    const int64_t mt = most_tiles(slots, experts + 1, kSide), nt = tiles_of(outs, kSide);
    auto launch = [&](auto bk) {
      hipLaunchKernelGGL((k_group_rows<T, decltype(bk)::value>), dim3((uint32_t)(mt * nt)), dim3(kGroupThreads), 0, st,
                         static_cast<const T*>(x), xs, static_cast<const T*>(w), static_cast<const T*>(b),
                         static_cast<const T*>(mask), offsets, static_cast<T*>(y), slots, experts, (int)cols,
                         (int)outs, relu, mt, (int)nt);
    };
    if (back) launch(std::true_type{});
    else launch(std::false_type{});
  });
  SPHOPS_LAUNCHED();
}

int64_t group_weight_grad_floats(int64_t slots, int experts, int64_t cols, int64_t outs) {
  return grad_plan(slots, experts, cols, outs).chunks * (cols * outs + outs);
}

void run_group_weight_grad(const void* dy, int64_t dys, const void* x, int type, int64_t xs, const int32_t* offsets,
                           void* dw, void* db, int64_t slots, int experts, int64_t cols, int64_t outs, float* work,
                           hipStream_t st) {
  const GradPlan p = grad_plan(slots, experts, cols, outs);
  const int64_t nw = cols * outs;
  with_type(type, [&](auto t) {
    using T = decltype(t);
    const int64_t blocks = (p.chunks > 0 ? p.chunks : experts) * p.mt * p.nt;
    hipLaunchKernelGGL((k_group_weight_grad<T>), dim3((uint32_t)blocks), dim3(kGroupThreads), 0, st,
                       static_cast<const T*>(dy), dys, static_cast<const T*>(x), xs, offsets, static_cast<T*>(dw),
                       static_cast<T*>(db), p.chunks > 0 ? work : nullptr, slots, experts, (int)cols, (int)outs,
                       p.chunk, p.mt, p.nt);
    SPHOPS_LAUNCHED();
    if (p.chunks > 0)
      hipLaunchKernelGGL((k_group_chunk_sum<T>), dim3((uint32_t)tiles_of(nw + outs, 256), (uint32_t)experts), dim3(256),
                         0, st, work, offsets, static_cast<T*>(dw), static_cast<T*>(db), slots, experts, nw, (int)outs,
                         p.chunk, p.chunks);
  });
  SPHOPS_LAUNCHED();
}

}  // namespace sphops
