// Which rows an expert has and how a product's tiles fall on the card, for the
// host and the device (grouped.hip, expert_mlp.hip).  Offsets come from device
// memory and may hold anything: what these functions give stays inside the rows
// and the workspace all the same.
#pragma once

#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstdint>

namespace sphops {

namespace {

// Group e's rows: offsets[e] to offsets[e + 1], of the group after the last
// expert's the rows behind them all; clamped to the rows there are.
struct GroupRows {
  int64_t lo, hi;
};
__host__ __device__ __forceinline__ GroupRows group_rows(const int32_t* __restrict__ offsets, int experts, int64_t slots,
                                                         int e) {
  const auto at = [&](int i) {
    const int64_t o = offsets[i];
    return o < 0 ? int64_t(0) : o < slots ? o : slots;
  };
  GroupRows g;
  g.lo = e == 0 ? 0 : at(e);
  g.hi = e == experts ? slots : at(e + 1);
  if (g.hi < g.lo) g.hi = g.lo;
  return g;
}

// The tiles that groups of rows which do not overlap can have between them.
__host__ __device__ __forceinline__ int64_t most_tiles(int64_t slots, int64_t groups, int64_t size) {
  return slots / size + (groups < slots ? groups : slots);
}

// How a product's tiles fall on the card, which holds `room` of their workgroups at
// once: whole turns of `room` tiles, and the tiles that are left, cut along the sum
// into `slices` each where that fills a turn better.  Without cuts 8192 x 2048 ->
// 1024 float32, 272 tiles of 256 x 128 on 256 CUs, took two turns (366 us, 239 with
// them), and 955 x 1545 -> 125, 20 tiles, one long one.
//
// places: of slices that the workspace holds (slice_places).  Offsets that decrease
// give more tiles than it was made for: those are not cut.
struct Turns {
  uint32_t whole, left, slices;
};
constexpr int kMaxSlices = 16, kSliceDepth = 256;  // at most; of the sum that a slice has at least
__host__ __device__ __forceinline__ Turns turns_of(uint32_t tiles, uint32_t room, uint32_t places, int depth) {
  Turns t;
  t.whole = tiles / room * room;
  t.left = tiles - t.whole;
  t.slices = 1;
  if (t.left > 0) {
    const uint32_t deep = (uint32_t)(depth / kSliceDepth), share = places / t.left;
    const uint32_t most = deep < (uint32_t)kMaxSlices ? deep : (uint32_t)kMaxSlices;
    if (share > 1 && most > 1) t.slices = share < most ? share : most;
  }
  return t;
}
// Slices that a workspace for `tiles` tiles at most has room for.
__host__ __forceinline__ int64_t slice_places(int64_t tiles, int room) {
  return std::min<int64_t>(room, tiles * kMaxSlices);
}

}  // namespace

}  // namespace sphops
