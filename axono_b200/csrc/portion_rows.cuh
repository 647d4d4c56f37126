// The table that gives the rows of a launch to sequences: sequence b has the rows row_start[b] .. row_start[b + 1] - 1.  An entry counts up
// if it is in 0 .. rows and none before it is larger; a sequence with an entry that does not is left out.  So the sequences that are left
// share no row, and every kernel that follows a table leaves out the same ones.
#pragma once

#include "common.cuh"

namespace axb {

// Whether sequence b's two entries count up; `earlier`: the largest entry before them (INT_MIN for none).
__device__ __forceinline__ bool portion_counts_up(int r0, int r1, int rows, int earlier) {
  return r0 >= 0 && r0 >= earlier && r1 >= r0 && r1 <= rows;
}

// Whether `bytes` at `other` share memory with `rows` (at least one) pieces of row_bytes that begin ld_bytes apart.
inline bool shares_memory(const void *base, int64_t ld_bytes, int64_t row_bytes, int64_t rows, const void *other, int64_t bytes) {
  const int64_t at = (int64_t)(reinterpret_cast<uintptr_t>(other) - reinterpret_cast<uintptr_t>(base));
  if (at <= 0) return at + bytes > 0;
  const int64_t row = at / ld_bytes;
  return row < rows && (at - row * ld_bytes < row_bytes || (row + 1 < rows && at + bytes > (row + 1) * ld_bytes));
}

// The sequence of a row, found by a warp, or -1; r0, r1: its entries.  Its end is the first entry above the row, so that all before are not.
// `falls`: the table does not count up around this row (every fall does so around the rows between the two entries, if there are any).
__device__ __forceinline__ int portion_sequence(const int32_t *row_start, int batch, int rows, int64_t row, int &r0, int &r1, bool &falls) {
  const int lane = threadIdx.x & 31;
  const int mine = lane <= batch ? row_start[lane] : 0x7fffffff;  // of the first 32 entries, which are all there are in most launches
  unsigned first = mine > row ? (unsigned)lane : 0x7fffffffu;
  int below = mine <= row;
  for (int i = lane + 32; i <= batch; i += 32) {
    if (row_start[i] <= row)
      ++below;
    else
      first = min(first, (unsigned)i);
  }
  first = __reduce_min_sync(0xffffffffu, first);
  below = __reduce_add_sync(0xffffffffu, below);
  falls = first <= (unsigned)batch && below != (int)first;
  if (first == 0 || first > (unsigned)batch) return -1;
  const int b = (int)first - 1;
  int earlier = lane < b ? mine : -0x7fffffff - 1;
  for (int i = lane + 32; i < b; i += 32) earlier = max(earlier, row_start[i]);
  earlier = __reduce_max_sync(0xffffffffu, earlier);
  if (b < 31) {
    r0 = __shfl_sync(0xffffffffu, mine, b);
    r1 = __shfl_sync(0xffffffffu, mine, b + 1);
  } else {
    r0 = row_start[b], r1 = row_start[b + 1];
  }
  if (portion_counts_up(r0, r1, rows, earlier)) return b;
  falls = true;
  return -1;
}

}  // namespace axb
