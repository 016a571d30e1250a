// Layer norm over rows, forward and backward, for gfx950.
//
//   m = mean x   v = mean (x - m)^2   r = 1 / sqrt(v + eps)   h = (x - m) r   y = h w + b
//   g = dy w     dx = r (g - mean g - h mean(g h))   dw = sum over rows of dy h   db = sum of dy
//
// Everything is float32 between the load of a value and the one rounding of a
// result.  A mean c rounded to float32 is off by 2^-25 of itself, which counts
// where rows lie far from zero: d = x - c is summed again and its mean e taken
// off (v = mean d^2 - e^2, h = (d - e) r).  The backward is given c and r and
// finds e beside its other two sums.
//
// c, d and e are halves and r is doubled, and c is summed in units of 2^17, which
// changes no rounding: nothing of a finite row but the sums over d overflows, a
// mask's lowest values and the difference of the largest ones included.  Where the
// squares' sum does (the sum of d does not before), r and e are 0: y is the bias,
// and no gradient reaches x.  A row that is not finite has a c that is not.
#include "rows_out.hpp"

#include <type_traits>

namespace sphops {

namespace {

constexpr float kSumUnit = 0x1p-17f, kHalfUnit = 0x1p16f;  // of c: up to 2^16 values
static_assert(kMaxRows8Cols <= 65536, "a row's sum stays in range");

// e and twice 1 / sqrt(v + eps) from a row's sums of d and of its squares.
struct Deviations {
  float e, twice;
  __device__ __forceinline__ Deviations(const float (&q)[2], float inv, float eps) {
    e = q[0] * inv;
    const float var = q[1] < __builtin_inff() ? fmaxf(q[1] * inv - e * e, 0.0f) : q[1];  // NaN stays
    twice = 1.0f / sqrtf(var + 0.25f * eps);
    if (twice == 0.0f) e = 0.0f;
  }
};

// What the backward makes halved deviations with, and r: all 0 where the squares
// overflowed, so that nothing of the row counts.
struct RowStats {
  float half, c, twice, r;
  __device__ __forceinline__ RowStats(float2 st)
      : half(st.y == 0.0f ? 0.0f : 0.5f), c(st.y == 0.0f ? 0.0f : st.x), twice(st.y), r(0.5f * st.y) {}
};

// A value of the weights, which are float32 or of the rows' type.
template <class T>
__device__ __forceinline__ float weight_at(const void* __restrict__ w, bool wide, int k) {
  return wide ? static_cast<const float*>(w)[k] : to_f32(static_cast<const T*>(w)[k]);
}

// V of them from k on, `fill` past the row's end and everywhere without weights.
template <class T>
__device__ __forceinline__ void weights_at(const void* __restrict__ w, bool wide, int k, int cols, float fill,
                                           float (&out)[Piece<T>::V]) {
  constexpr int V = Piece<T>::V;
#pragma unroll
  for (int j = 0; j < V; ++j) out[j] = fill;
  if (w == nullptr || k >= cols) return;
  if (k + V > cols) {
#pragma unroll
    for (int j = 0; j < V; ++j)
      if (k + j < cols) out[j] = weight_at<T>(w, wide, k + j);
  } else if (wide) {
#pragma unroll
    for (int i = 0; i < V / 4; ++i) {
      Piece<float> p;
      p.load(static_cast<const float*>(w), k + 4 * i, cols);
#pragma unroll
      for (int j = 0; j < 4; ++j) out[4 * i + j] = p.get(j);
    }
  } else {
    Piece<T> p;
    p.load(static_cast<const T*>(w), k, cols);
#pragma unroll
    for (int j = 0; j < V; ++j) out[j] = p.get(j);
  }
}

// Sums of a row's L lanes, K of them at a time, in every lane.  L > 64: a row's
// waves meet in LDS, two sets in turn (a wave writes a set again only after the
// other turn's barrier).
template <int L, int K, int TH>
struct RowSums {
  float part[2][K][TH / 64 + 1];
  __device__ __forceinline__ void operator()(float (&v)[K], int& turn) {
#pragma unroll
    for (int s = 1; s < (L < 64 ? L : 64); s *= 2) {
#pragma unroll
      for (int i = 0; i < K; ++i) v[i] += __shfl_xor(v[i], s);
    }
    if constexpr (L > 64) {
      const int wave = (int)threadIdx.x / 64, first = (int)threadIdx.x / L * (L / 64);
      if (threadIdx.x % 64 == 0) {
#pragma unroll
        for (int i = 0; i < K; ++i) part[turn][i][wave] = v[i];
      }
      __syncthreads();
#pragma unroll
      for (int i = 0; i < K; ++i) {
        v[i] = 0.0f;
#pragma unroll
        for (int j = 0; j < L / 64; ++j) v[i] += part[turn][i][first + j];
      }
      turn ^= 1;
    }
  }
};

// L lanes a row, which they hold in N pieces of 16 bytes each: the row is read
// once, the next one under this one's sums.  A lane keeps its columns' weights over
// all of its rows.
// Bound: HBM: 2^20 x 83 float32 in 161 us (4.3 TB/s; 20 us more with a row's pieces stored
// as they are), 8191 x 4097 bfloat16, at odd places, in 32 (4.2 TB/s), one row of 4096 in 3.
template <class T, int L, int N, int TH>
__global__ __launch_bounds__(TH) void k_norm_forward(const T* __restrict__ x, int64_t stride,
                                                     const void* __restrict__ w, const void* __restrict__ b,
                                                     bool wide, T* __restrict__ y, float2* __restrict__ stats,
                                                     int64_t rows, int cols, float eps) {
  constexpr int V = Piece<T>::V, kRows = TH / L;
  __shared__ RowSums<L, 1, TH> sum1;
  __shared__ RowSums<L, 2, TH> sum2;
  __shared__ __attribute__((aligned(16))) RowsOut<T, L, N> outs[TH / 64];
  const int l = threadIdx.x % L;
  const float inv = 1.0f / (float)cols;
  int turn1 = 0, turn2 = 0;  // of the sums
  float ww[N][V], bb[N][V];
#pragma unroll
  for (int n = 0; n < N; ++n) {
    weights_at<T>(w, wide, (n * L + l) * V, cols, 1.0f, ww[n]);
    weights_at<T>(b, wide, (n * L + l) * V, cols, 0.0f, bb[n]);
  }
  const int64_t turn = (int64_t)gridDim.x * kRows;
  Piece<T> p[N], next[N];
  auto load = [&](int64_t r0, Piece<T> (&to)[N]) {
    const int64_t r = min<int64_t>(r0 + threadIdx.x / L, rows - 1);  // lanes past the last row do it again
#pragma unroll
    for (int n = 0; n < N; ++n) load_piece(to[n], n < N - 1, x + r * stride, (n * L + l) * V, cols);
  };
  load((int64_t)blockIdx.x * kRows, next);
  for (int64_t r0 = (int64_t)blockIdx.x * kRows; r0 < rows; r0 += turn) {
    const int64_t r = min<int64_t>(r0 + threadIdx.x / L, rows - 1);
#pragma unroll
    for (int n = 0; n < N; ++n) p[n] = next[n];
    load(r0 + turn, next);  // in flight under this turn's sums
    float s[1] = {0.0f};
#pragma unroll
    for (int n = 0; n < N; ++n) {
#pragma unroll
      for (int j = 0; j < V; ++j) s[0] += p[n].get(j) * kSumUnit;
    }
    sum1(s, turn1);
    const float c = s[0] * (inv * kHalfUnit);
    float q[2] = {0.0f, 0.0f};
#pragma unroll
    for (int n = 0; n < N; ++n) {
#pragma unroll
      for (int j = 0; j < V; ++j) {
        // only the last pieces reach past the row's end (with_lanes)
        const float d = n < N - 1 || (n * L + l) * V + j < cols ? p[n].get(j) * 0.5f - c : 0.0f;
        q[0] += d;
        q[1] += d * d;
      }
    }
    sum2(q, turn2);
    const Deviations dev(q, inv, eps);
    const float e = dev.e, rstd = dev.twice;
    if (stats != nullptr && l == 0) stats[r] = float2{c, rstd};
    const float er = e * rstd;
    Piece<T> o[N];
#pragma unroll
    for (int n = 0; n < N; ++n) {
      float v[V];
#pragma unroll
      for (int j = 0; j < V; ++j) v[j] = ((p[n].get(j) * 0.5f - c) * rstd - er) * ww[n][j] + bb[n][j];
      o[n] = piece_of<T>(v);
    }
    const int wave = (int)threadIdx.x / 64;
    outs[wave](o, y, r0 + wave * 64 / L, rows, cols);
  }
}

// Rows longer than a workgroup's registers hold: a workgroup a row, read three
// times (twice from cache).
constexpr int kLongThreads = 1024;
template <class T>
__global__ __launch_bounds__(kLongThreads) void k_norm_forward_long(const T* __restrict__ x, int64_t stride,
                                                                    const void* __restrict__ w,
                                                                    const void* __restrict__ b, bool wide,
                                                                    T* __restrict__ y, float2* __restrict__ stats,
                                                                    int64_t rows, int cols, float eps) {
  constexpr int V = Piece<T>::V, TH = kLongThreads;
  __shared__ RowSums<TH, 1, TH> sum1;
  __shared__ RowSums<TH, 2, TH> sum2;
  const float inv = 1.0f / (float)cols;
  int turn1 = 0, turn2 = 0;
  for (int64_t r = blockIdx.x; r < rows; r += gridDim.x) {
    const T* __restrict__ row = x + r * stride;
    float s[1] = {0.0f};
    for (int k = threadIdx.x * V; k < cols; k += TH * V) {
      Piece<T> p;
      p.load(row, k, cols);
#pragma unroll
      for (int j = 0; j < V; ++j) s[0] += p.get(j) * kSumUnit;
    }
    sum1(s, turn1);
    const float c = s[0] * (inv * kHalfUnit);
    float q[2] = {0.0f, 0.0f};
    for (int k = threadIdx.x * V; k < cols; k += TH * V) {
      Piece<T> p;
      p.load(row, k, cols);
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const float d = k + j < cols ? p.get(j) * 0.5f - c : 0.0f;
        q[0] += d;
        q[1] += d * d;
      }
    }
    sum2(q, turn2);
    const Deviations dev(q, inv, eps);
    const float e = dev.e, rstd = dev.twice;
    if (stats != nullptr && threadIdx.x == 0) stats[r] = float2{c, rstd};
    for (int k = threadIdx.x * V; k < cols; k += TH * V) {
      Piece<T> p;
      p.load(row, k, cols);
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const int kk = min(k + j, cols - 1);
        const float ww = w != nullptr ? weight_at<T>(w, wide, kk) : 1.0f;
        const float bb = b != nullptr ? weight_at<T>(b, wide, kk) : 0.0f;
        p.set(j, from_f32<T>((p.get(j) * 0.5f - c - e) * rstd * ww + bb));
      }
      p.store(y + r * cols, k, cols);
    }
  }
}

// As the forward, with dy beside x; a lane sums its columns of dw and db over
// its rows, the workgroup's rows meet in LDS and leave as one row of `part`
// (2 x cols: dw, then db), in a fixed order.
// Bound: HBM for short rows (2^20 x 83 float32 in 248 us, 4.2 TB/s), vector work and
// the sums' latency for long ones, whose registers leave room for two waves a SIMD
// (8191 x 4097 bfloat16 in 66 us, 3.1 TB/s).
template <class T, int L, int N, int TH>
__global__ __launch_bounds__(TH, N * Piece<T>::V <= 12 ? 4 : 2) void k_norm_backward(const T* __restrict__ x, int64_t stride,
                                                      const T* __restrict__ dy, int64_t dy_stride,
                                                      const void* __restrict__ w, bool wide,
                                                      const float2* __restrict__ stats, T* __restrict__ dx,
                                                      float* __restrict__ part, int64_t rows, int cols) {
  constexpr int V = Piece<T>::V, kRows = TH / L;
  __shared__ RowSums<L, 3, TH> sums;
  __shared__ __attribute__((aligned(16))) RowsOut<T, L, N> outs[TH / 64];
  const int l = threadIdx.x % L;
  const float inv = 1.0f / (float)cols;
  int turn = 0;
  float ww[N][V], dw[N][V], db[N][V];
#pragma unroll
  for (int n = 0; n < N; ++n) {
    weights_at<T>(w, wide, (n * L + l) * V, cols, 1.0f, ww[n]);
#pragma unroll
    for (int j = 0; j < V; ++j) dw[n][j] = db[n][j] = 0.0f;
  }
  const int64_t step = (int64_t)gridDim.x * kRows;
  Piece<T> p[N], u[N], pn[N], un[N];
  float2 sn;
  auto load = [&](int64_t r0) {
    const int64_t r = min<int64_t>(r0 + threadIdx.x / L, rows - 1);
#pragma unroll
    for (int n = 0; n < N; ++n) {
      load_piece(pn[n], n < N - 1, x + r * stride, (n * L + l) * V, cols);
      load_piece(un[n], n < N - 1, dy + r * dy_stride, (n * L + l) * V, cols);
    }
    sn = stats[r];
  };
  load((int64_t)blockIdx.x * kRows);
  for (int64_t r0 = (int64_t)blockIdx.x * kRows; r0 < rows; r0 += step) {
    const bool live = r0 + threadIdx.x / L < rows;
#pragma unroll
    for (int n = 0; n < N; ++n) {
      p[n] = pn[n];
      u[n] = un[n];
    }
    const RowStats st(sn);
    load(r0 + step);  // in flight under this turn's sums
    float s[3] = {0.0f, 0.0f, 0.0f};  // of d, g and g d
#pragma unroll
    for (int n = 0; n < N; ++n) {
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const float d = n < N - 1 || (n * L + l) * V + j < cols ? p[n].get(j) * st.half - st.c : 0.0f;
        const float g = u[n].get(j) * ww[n][j];
        s[0] += d;
        s[1] += g;
        s[2] += g * d;
      }
    }
    sums(s, turn);
    const float e = s[0] * inv, mg = s[1] * inv, mgh = (s[2] - e * s[1]) * inv * st.twice;
    const float er = e * st.twice, mgr = mg * st.r, mghr = mgh * st.r;
    Piece<T> o[N];
#pragma unroll
    for (int n = 0; n < N; ++n) {
      float v[V];
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const float h = (p[n].get(j) * st.half - st.c) * st.twice - er, up = u[n].get(j);
        v[j] = (up * ww[n][j]) * st.r - mgr - h * mghr;
        if (live) {
          dw[n][j] += up * h;
          db[n][j] += up;
        }
      }
      o[n] = piece_of<T>(v);
    }
    const int wave = (int)threadIdx.x / 64;
    if (dx != nullptr) outs[wave](o, dx, r0 + wave * 64 / L, rows, cols);
  }
  if (part == nullptr) return;
  float* __restrict__ to = part + (int64_t)blockIdx.x * 2 * cols;
  if constexpr (kRows == 1) {
#pragma unroll
    for (int n = 0; n < N; ++n) {
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const int k = (n * L + l) * V + j;
        if (k < cols) {
          to[k] = dw[n][j];
          to[cols + k] = db[n][j];
        }
      }
    }
  } else {
    // a piece of every row group at a time
    __shared__ float meet[2][TH * V + TH / 8];
#pragma unroll
    for (int n = 0; n < N; ++n) {
      __syncthreads();
#pragma unroll
      for (int j = 0; j < V; ++j) {
        meet[0][threadIdx.x * V + j] = dw[n][j];
        meet[1][threadIdx.x * V + j] = db[n][j];
      }
      __syncthreads();
      for (int i = threadIdx.x; i < 2 * L * V; i += TH) {
        const int which = i / (L * V), at = i % (L * V), k = n * L * V + at;
        if (k >= cols) continue;
        float t = 0.0f;
#pragma unroll 8
        for (int g = 0; g < kRows; ++g) t += meet[which][g * L * V + at];
        to[which * cols + k] = t;
      }
    }
  }
}

// Rows too long for registers: dx by a workgroup a row, read twice.
template <class T>
__global__ __launch_bounds__(kLongThreads) void k_norm_backward_long(const T* __restrict__ x, int64_t stride,
                                                                     const T* __restrict__ dy, int64_t dy_stride,
                                                                     const void* __restrict__ w, bool wide,
                                                                     float2* __restrict__ stats, float* __restrict__ low,
                                                                     T* __restrict__ dx, int64_t rows, int cols) {
  constexpr int V = Piece<T>::V, TH = kLongThreads;
  __shared__ RowSums<TH, 3, TH> sums;
  const float inv = 1.0f / (float)cols;
  int turn = 0;
  for (int64_t r = blockIdx.x; r < rows; r += gridDim.x) {
    const T* __restrict__ row = x + r * stride;
    const T* __restrict__ up = dy + r * dy_stride;
    const RowStats st(stats[r]);
    float s[3] = {0.0f, 0.0f, 0.0f};
    for (int k = threadIdx.x * V; k < cols; k += TH * V) {
      Piece<T> p, u;
      p.load(row, k, cols);
      u.load(up, k, cols);
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const float d = k + j < cols ? p.get(j) * st.half - st.c : 0.0f;
        const float g = u.get(j) * (w != nullptr ? weight_at<T>(w, wide, min(k + j, cols - 1)) : 1.0f);
        s[0] += d;
        s[1] += g;
        s[2] += g * d;
      }
    }
    sums(s, turn);
    const float e = s[0] * inv, mg = s[1] * inv, mgh = (s[2] - e * s[1]) * inv * st.twice;
    if (low != nullptr && threadIdx.x == 0) low[r] = e;
    if (dx == nullptr) continue;
    for (int k = threadIdx.x * V; k < cols; k += TH * V) {
      Piece<T> p, u;
      p.load(row, k, cols);
      u.load(up, k, cols);
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const float g = u.get(j) * (w != nullptr ? weight_at<T>(w, wide, min(k + j, cols - 1)) : 1.0f);
        const float h = (p.get(j) * st.half - st.c - e) * st.twice;
        p.set(j, from_f32<T>(st.r * (g - mg - h * mgh)));
      }
      p.store(dx + r * cols, k, cols);
    }
  }
}

// dw and db of long rows: a workgroup takes 256 columns of a chunk of rows.
template <class T>
__global__ __launch_bounds__(256) void k_norm_columns_long(const T* __restrict__ x, int64_t stride,
                                                           const T* __restrict__ dy, int64_t dy_stride,
                                                           const float2* __restrict__ stats,
                                                           const float* __restrict__ low, float* __restrict__ part,
                                                           int64_t rows, int64_t chunk, int cols) {
  const int k = (int)blockIdx.y * 256 + threadIdx.x;
  if (k >= cols) return;
  const int64_t r0 = (int64_t)blockIdx.x * chunk, r1 = min<int64_t>(r0 + chunk, rows);
  float dw = 0.0f, db = 0.0f;
#pragma unroll 4
  for (int64_t r = r0; r < r1; ++r) {
    const float u = to_f32(dy[r * dy_stride + k]);
    const RowStats st(stats[r]);
    dw += u * ((to_f32(x[r * stride + k]) * st.half - st.c - low[r]) * st.twice);
    db += u;
  }
  float* __restrict__ to = part + (int64_t)blockIdx.x * 2 * cols;
  to[k] = dw;
  to[cols + k] = db;
}

// The sums of 32 columns of `part` (2 x cols a row: dw, then db) over its rows,
// 32 shares of them, in a fixed order.
template <class T>
__global__ __launch_bounds__(1024) void k_norm_column_sum(const float* __restrict__ part, int chunks, int cols,
                                                          bool wide, void* __restrict__ dw, void* __restrict__ db) {
  __shared__ float meet[32][33];
  const int c = threadIdx.x & 31, g = threadIdx.x >> 5, at = (int)blockIdx.x * 32 + c;
  float t = 0.0f;
  if (at < 2 * cols) {
#pragma unroll 8
    for (int i = g; i < chunks; i += 32) t += part[(int64_t)i * 2 * cols + at];
  }
  meet[g][c] = t;
  __syncthreads();
  if (g != 0 || at >= 2 * cols) return;
  t = 0.0f;
#pragma unroll
  for (int i = 0; i < 32; ++i) t += meet[i][c];
  void* const to = at < cols ? dw : db;
  if (to == nullptr) return;
  const int k = at < cols ? at : at - cols;
  if (wide) static_cast<float*>(to)[k] = t;
  else static_cast<T*>(to)[k] = from_f32<T>(t);
}

// f(integral_constants L, N) for rows of `pieces` 16-byte pieces; false: longer
// than all of them.  A row has more than L (N - 1) pieces, so only the last of a
// lane's reach past its end.
template <class F>
bool with_lanes(int64_t pieces, F&& f) {
  auto at = [&](auto l, auto n) {
    if (pieces > decltype(l)::value * decltype(n)::value) return false;
    f(l, n);
    return true;
  };
#define SPHOPS_LANES(L, N) at(std::integral_constant<int, L>{}, std::integral_constant<int, N>{})
  return SPHOPS_LANES(4, 1) || SPHOPS_LANES(8, 1) || SPHOPS_LANES(8, 2) || SPHOPS_LANES(8, 3) ||
         SPHOPS_LANES(16, 2) || SPHOPS_LANES(16, 3) || SPHOPS_LANES(32, 2) || SPHOPS_LANES(32, 3) ||
         SPHOPS_LANES(64, 2) || SPHOPS_LANES(64, 3) || SPHOPS_LANES(256, 1) || SPHOPS_LANES(256, 2) ||
         SPHOPS_LANES(256, 3) || SPHOPS_LANES(256, 4) || SPHOPS_LANES(512, 3) || SPHOPS_LANES(512, 4);
#undef SPHOPS_LANES
}

constexpr int kForwardGroups = 2048;  // workgroups that keep their weights over many rows
constexpr int kBackwardGroups = 512;  // rows of `part`
constexpr int64_t kLongChunk = 64;
// Threads of a backward's workgroup: several rows, or one (whose barriers then hold up no other).
constexpr int backward_threads(int l) { return l > 64 ? l : 512; }

template <class T>
int64_t norm_chunks(int64_t rows, int64_t cols) {
  const int64_t pieces = (cols + Piece<T>::V - 1) / Piece<T>::V;
  int64_t chunks = 0;
  const bool held = with_lanes(pieces, [&](auto l, auto) {
    constexpr int kRows = backward_threads(decltype(l)::value) / decltype(l)::value;
    chunks = std::min<int64_t>((rows + kRows - 1) / kRows, kBackwardGroups);
  });
  if (!held) chunks = std::min<int64_t>((rows + kLongChunk - 1) / kLongChunk, kBackwardGroups);
  return chunks;
}
template <class T>
int64_t norm_floats(int64_t rows, int64_t cols) {
  const int64_t pieces = (cols + Piece<T>::V - 1) / Piece<T>::V;
  return norm_chunks<T>(rows, cols) * 2 * cols + (with_lanes(pieces, [](auto, auto) {}) ? 0 : rows);
}

}  // namespace

void run_layer_norm(const void* x, int type, int64_t stride, const void* w, const void* b, bool wide, void* y,
                    float* stats, int64_t rows, int64_t cols, float eps, hipStream_t st) {
  if (rows == 0) return;
  with_type(type, [&](auto t) {
    using T = decltype(t);
    const int64_t pieces = (cols + Piece<T>::V - 1) / Piece<T>::V;
    const bool held = with_lanes(pieces, [&](auto l, auto n) {
      constexpr int L = decltype(l)::value, TH = L > 256 ? L : 256;
      const int64_t groups = std::min<int64_t>((rows + TH / L - 1) / (TH / L), kForwardGroups);
      hipLaunchKernelGGL((k_norm_forward<T, L, decltype(n)::value, TH>), dim3((uint32_t)groups), dim3(TH), 0, st,
                         static_cast<const T*>(x), stride, w, b, wide, static_cast<T*>(y),
                         reinterpret_cast<float2*>(stats), rows, (int)cols, eps);
    });
    if (!held)
      hipLaunchKernelGGL((k_norm_forward_long<T>), dim3((uint32_t)std::min<int64_t>(rows, kForwardGroups)),
                         dim3(kLongThreads), 0, st, static_cast<const T*>(x), stride, w, b, wide, static_cast<T*>(y),
                         reinterpret_cast<float2*>(stats), rows, (int)cols, eps);
  });
  SPHOPS_LAUNCHED();
}

int64_t layer_norm_backward_floats(int type, int64_t rows, int64_t cols) {
  int64_t n = 0;
  with_type(type, [&](auto t) { n = norm_floats<decltype(t)>(rows, cols); });
  return n;
}

void run_layer_norm_backward(const void* x, int64_t stride, const void* dy, int64_t dy_stride, int type,
                             const void* w, bool wide, const float* stats, void* dx, void* dw, void* db, int64_t rows,
                             int64_t cols, float* work, hipStream_t st) {
  with_type(type, [&](auto t) {
    using T = decltype(t);
    const int64_t pieces = (cols + Piece<T>::V - 1) / Piece<T>::V, chunks = norm_chunks<T>(rows, cols);
    const bool sums = dw != nullptr || db != nullptr;
    const T *px = static_cast<const T*>(x), *pdy = static_cast<const T*>(dy);
    float2* const ps = reinterpret_cast<float2*>(const_cast<float*>(stats));
    if (rows > 0) {
      const bool held = with_lanes(pieces, [&](auto l, auto n) {
        constexpr int L = decltype(l)::value, TH = backward_threads(L);
        hipLaunchKernelGGL((k_norm_backward<T, L, decltype(n)::value, TH>), dim3((uint32_t)chunks), dim3(TH), 0, st,
                           px, stride, pdy, dy_stride, w, wide, ps, static_cast<T*>(dx), sums ? work : nullptr, rows,
                           (int)cols);
      });
      if (!held) {
        float* const low = work + chunks * 2 * cols;
        hipLaunchKernelGGL((k_norm_backward_long<T>), dim3((uint32_t)std::min<int64_t>(rows, kForwardGroups)),
                           dim3(kLongThreads), 0, st, px, stride, pdy, dy_stride, w, wide, ps, low,
                           static_cast<T*>(dx), rows, (int)cols);
        if (sums)
          hipLaunchKernelGGL((k_norm_columns_long<T>), dim3((uint32_t)chunks, (uint32_t)((cols + 255) / 256)),
                             dim3(256), 0, st, px, stride, pdy, dy_stride, ps, low, work, rows,
                             (rows + chunks - 1) / chunks, (int)cols);
      }
      SPHOPS_LAUNCHED();
    }
    if (sums)
      hipLaunchKernelGGL((k_norm_column_sum<T>), dim3((uint32_t)((2 * cols + 31) / 32)), dim3(1024), 0, st, work,
                         (int)chunks, (int)cols, wide, dw, db);
  });
  SPHOPS_LAUNCHED();
}

}  // namespace sphops
