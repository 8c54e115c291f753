// Comparisons of row numbers that stay within 32 bits.  A table has fewer than 2^31 - 65536 rows and a window
// or a section may have as many, so that their sum with a row does not fit: it is the difference of two rows that is
// compared.  (Rows of a tile may lie up to 128 behind the table's end, which still fits.)
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace tmp {

// How far behind query row r0 the last query row lies whose window holds key row j.
__host__ __device__ inline int window_reach(int j, int r0, int window) { return (j - r0) + (window - 1); }
// Whether query row r lies behind every window that holds key row j (r >= j - 128).
__host__ __device__ inline bool beyond_window(int r, int j, int window) { return r - j >= window; }
// The query row behind the last one whose window holds a key row of [j0, j0 + rows).
__host__ __device__ inline int window_end(int j0, int rows, int window, int n) {
  const int64_t hi = (int64_t)j0 + rows + window - 1;
  return hi < n ? (int)hi : n;
}

// The row behind the last one of the section that starts at row `first` (< n).
__host__ __device__ inline int section_end(int first, int section, int n) { return section < n - first ? first + section : n; }

}  // namespace tmp
