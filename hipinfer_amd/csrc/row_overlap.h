// Whether two sets of rows in memory meet: what a call that writes rows in place of others must know. Plain host arithmetic, compiled
// alone by its test.
#pragma once
#include <cstdint>

// M rows of wx bytes from x on, lx bytes apart (lx >= wx), and M rows of wy bytes from y on, ly apart.
inline bool rows_meet(uintptr_t x, int64_t lx, int64_t wx, uintptr_t y, int64_t ly, int64_t wy, int M) {
  if (x > y) return rows_meet(y, ly, wy, x, lx, wx, M);
  const uintptr_t span = (uintptr_t)((M - 1) * lx + wx);
  for (int j = 0; j < M; j++, y += ly) {
    if (y - x >= span) return false;  // behind x's last row, as all that follow
    const int64_t d = (int64_t)(y - x), row = d / lx, at = d % lx;
    if (at < wx || (row + 1 < M && at + wy > lx)) return true;
    if (lx == ly) return false;  // every further row stands in a gap as this one does
  }
  return false;
}

// Rows that one call reads at x and writes at y: the very same ones, or apart.
inline bool in_place_or_apart(const void* x, int64_t lx, int64_t wx, const void* y, int64_t ly, int64_t wy, int M) {
  if (x == y && (lx == ly || M == 1)) return true;
  return !rows_meet((uintptr_t)x, lx, wx, (uintptr_t)y, ly, wy, M);
}
