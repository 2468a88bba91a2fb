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

}  // namespace col
