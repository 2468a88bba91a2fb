// Groups of rows: the operands of products grouped by expert.
//
// `offsets` (int32 [groups + 1], device memory) sorts the rows of a [rows, *]
// operand into consecutive groups: group g owns rows [offsets[g],
// offsets[g + 1]).  The host never reads it (the calls stay capturable), so
// kernels take each offset as the largest up to it, clamped to [0, rows]:
// whatever the array holds, every row index is in range, no row has two groups
// and the number of tiles keeps its bound.
#pragma once

#include "common.cuh"

namespace col {

constexpr int kMaxGroups = 1024;

// Shared-memory tables of a CTA: first row of each group (starts[groups] ends the
// last), and the row tiles of the groups before each.
struct GroupTables {
  int* starts;
  int* prefix;
};
constexpr unsigned kGroupTableBytes = 2 * 4352;  // kMaxGroups + 1 ints each
static_assert(kGroupTableBytes / 2 >= (kMaxGroups + 1) * 4, "table size");

__device__ __forceinline__ GroupTables group_tables(void* smem) {
  return {static_cast<int*>(smem), static_cast<int*>(smem) + kGroupTableBytes / 8};
}

// Fills the tables from one warp; the CTA synchronises before reading them.
// Without offsets all rows are one group.
__device__ __forceinline__ void fill_group_tables(const GroupTables& t, const int* offsets,
                                                  int groups, int rows, int tile_rows, int lane) {
  if (offsets == nullptr) {
    if (lane == 0) {
      t.starts[0] = 0;
      t.starts[1] = rows;
      t.prefix[0] = 0;
      t.prefix[1] = (rows + tile_rows - 1) / tile_rows;
    }
    return;
  }
  int highest = 0;  // of the offsets so far
  for (int g0 = 0; g0 <= groups; g0 += 32) {
    const int g = g0 + lane;
    int start = g <= groups ? min(max(offsets[g], 0), rows) : 0;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, start, o);
      if (lane >= o) start = max(start, v);
    }
    start = max(start, highest);
    if (g <= groups) t.starts[g] = start;
    highest = __shfl_sync(0xffffffffu, start, 31);
  }
  __syncwarp();
  int before = 0;
  for (int g0 = 0; g0 < groups; g0 += 32) {
    const int g = g0 + lane;
    int tiles = 0;
    if (g < groups) tiles = (t.starts[g + 1] - t.starts[g] + tile_rows - 1) / tile_rows;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, tiles, o);
      if (lane >= o) tiles += v;
    }
    if (g < groups) t.prefix[g + 1] = before + tiles;
    before += __shfl_sync(0xffffffffu, tiles, 31);
  }
  if (lane == 0) t.prefix[0] = 0;
}

struct TileCoords {
  int group;
  int m;  // row tile within the group
  int n;  // column tile
};

// Tile number to (group, row tile, column tile).  Within a group, kGroupRows
// row tiles at a time walk the columns together, so that the tiles in flight
// share operand rows and columns in L2.  With 32, 16, 8 and 4, fastest of 12
// runs of ten launches back to back on the same inputs, measured twice: 16384 rows over 8 experts,
// gate/up 4096 x 4096 in bf16, 738-745, 735-744, 744 and 748-753 us; 8192 x 4096 x
// 14336 SwiGLU in e4m3 972-994, 925-985, 1028-1039 and 955-957 (single launches
// up to 1400, as the clock falls): no difference between 16 and 32 shows.
constexpr int kGroupRows = 32;

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
