// Whether two sets of rows in memory meet: what a call that writes rows in place of others must know. Plain host arithmetic, compiled
// alone by its test.
#pragma once
#include <cstdint>

// mx rows of wx bytes from x on, lx bytes apart (lx >= wx), and my rows of wy bytes from y on, ly apart; at least one of each.
inline bool rows_meet(uintptr_t x, int64_t lx, int64_t wx, int mx, uintptr_t y, int64_t ly, int64_t wy, int my) {
  if (x > y) return rows_meet(y, ly, wy, my, x, lx, wx, mx);
  const uintptr_t span = (uintptr_t)((mx - 1) * lx + wx);
  for (int j = 0; j < my; j++, y += ly) {
    if (y - x >= span) return false;  // behind x's last row, as all that follow
    const int64_t d = (int64_t)(y - x), row = d / lx, at = d % lx;
    if (at < wx || (row + 1 < mx && at + wy > lx)) return true;
    if (lx == ly) return false;  // every further row stands in a gap as this one does
  }
  return false;
}
inline bool rows_meet(uintptr_t x, int64_t lx, int64_t wx, uintptr_t y, int64_t ly, int64_t wy, int M) {
  return rows_meet(x, lx, wx, M, y, ly, wy, M);
}

// Rows that one call reads at x and writes at y: the very same ones, or apart.
inline bool in_place_or_apart(const void* x, int64_t lx, int64_t wx, const void* y, int64_t ly, int64_t wy, int M) {
  if (x == y && (lx == ly || M == 1)) return true;
  return !rows_meet((uintptr_t)x, lx, wx, (uintptr_t)y, ly, wy, M);
}

// A tensor of a call: m rows of w bytes, ld apart (none where p is null or m or w 0); whether the call writes it, and if it may take
// the place of one that the call reads, the number of that (whether those two may meet is in_place_or_apart's).
struct CallRows {
  const char* name;
  const void* p;
  int64_t ld, w;
  int m;
  bool out;
  int in_place = -1;
};
// One without rows.
inline CallRows call_flat(const char* name, const void* p, int64_t bytes, bool out, int in_place = -1) {
  return CallRows{name, p, bytes, bytes, 1, out, in_place};
}
// Whether two of n tensors meet though the call writes one of them; a and b: which.
template <int n>
inline bool call_rows_meet(const CallRows (&t)[n], const char*& a, const char*& b) {
  auto there = [](const CallRows& r) { return r.p && r.m > 0 && r.w > 0; };
  for (int j = 0; j < n; j++)
    for (int i = 0; i < j; i++) {
      if (!(t[i].out || t[j].out) || t[j].in_place == i || t[i].in_place == j || !there(t[i]) || !there(t[j])) continue;
      if (!rows_meet((uintptr_t)t[i].p, t[i].ld, t[i].w, t[i].m, (uintptr_t)t[j].p, t[j].ld, t[j].w, t[j].m)) continue;
      a = t[i].name;
      b = t[j].name;
      return true;
    }
  return false;
}
