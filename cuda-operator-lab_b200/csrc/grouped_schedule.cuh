// Groups of rows: the operands of products grouped by expert.
//
// `offsets` (int32 [groups + 1], device memory) sorts the rows of a [rows, *]
// operand into consecutive groups: group g owns rows [offsets[g],
// offsets[g + 1]).  The host never reads it (the calls stay capturable), so
// kernels clamp what they read: whatever the array holds, every row index
// stays inside [0, rows].
#pragma once

#include "common.cuh"

namespace col {

constexpr int kMaxGroups = 1024;

struct RowRange {
  int begin;
  int end;
};

// Rows of group g; all of [0, rows) where there is no offsets array.
__device__ __forceinline__ RowRange group_rows(const int* offsets, int g, int rows) {
  if (offsets == nullptr) return {0, rows};
  const int begin = min(max(offsets[g], 0), rows);
  const int end = min(max(offsets[g + 1], begin), rows);
  return {begin, end};
}

// Row tiles of the groups before each group: prefix[g + 1] - prefix[g] =
// ceil(rows of g / tile_rows).  Written by one warp to shared memory
// (prefix[0 .. groups]); the CTA synchronises before reading it.
__device__ __forceinline__ void fill_tile_prefix(int* prefix, const int* offsets, int groups,
                                                 int rows, int tile_rows, int lane) {
  int before = 0;
  for (int g0 = 0; g0 < groups; g0 += 32) {
    const int g = g0 + lane;
    int tiles = 0;
    if (g < groups) {
      const RowRange r = group_rows(offsets, g, rows);
      tiles = (r.end - r.begin + tile_rows - 1) / tile_rows;
    }
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, tiles, o);
      if (lane >= o) tiles += v;
    }
    if (g < groups) prefix[g + 1] = before + tiles;
    before += __shfl_sync(0xffffffffu, tiles, 31);
  }
  if (lane == 0) prefix[0] = 0;
}

struct TileCoords {
  int group;
  int m;  // row tile within the group
  int n;  // column tile
};

// Tile number to (group, row tile, column tile).  Within a group, kGroupRows
// row tiles at a time walk the columns together, so that the tiles in flight
// share operand rows and columns in L2.
constexpr int kGroupRows = 16;

__device__ __forceinline__ TileCoords tile_of(int tile, const int* prefix, int groups,
                                              int num_n) {
  const int q = tile / num_n;
  int lo = 0, hi = groups;  // prefix[lo] <= q < prefix[hi]
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (prefix[mid] <= q) {
      lo = mid;
    } else {
      hi = mid;
    }
  }
  const int local = tile - prefix[lo] * num_n;
  const int rows = prefix[lo + 1] - prefix[lo];
  const int band = local / (kGroupRows * num_n);
  const int first = band * kGroupRows;
  const int high = min(rows - first, kGroupRows);
  const int in_band = local - first * num_n;
  return {lo, first + in_band % high, in_band / high};
}

}  // namespace col
