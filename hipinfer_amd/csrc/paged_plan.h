// How attention over ragged row runs is cut into blocks: row tiles, and splits of a tile's keys. Plain integer arithmetic of
// one sequence at a time, used by the kernels (summed over a wave's lanes) and compiled for the host by its test.
#pragma once
#include <cstdint>

#if defined(__HIPCC__)
#define PLAN_HD __host__ __device__ __forceinline__
#else
#define PLAN_HD inline
#endif

constexpr int kPlanTile = 128;      // keys of a tile: splits are whole tiles
constexpr int kPlanMinSplit = 512;  // keys a split has at least
constexpr int kPlanNoSplit = 0x7fffff80;

// Rows of a sequence: start values are cut to the M rows there are.
PLAN_HD int plan_first(int s, int M) { return s < 0 ? 0 : s > M ? M : s; }
PLAN_HD int plan_rows(int s0, int s1, int M) {
  const int n = plan_first(s1, M) - plan_first(s0, M);
  return n > 0 ? n : 0;
}
// Keys that the row at position pos + n - 1 sees, of a table that holds cap.
PLAN_HD int plan_end(int pos, int n, int cap) {
  const int64_t e = (int64_t)pos + n;
  return e < 0 ? 0 : e > cap ? cap : (int)e;
}
// Tiles of BQ packed rows: packed row r is query head r % G of the kv head's G in token r / G.
PLAN_HD int plan_tiles(int n, int G, int BQ) { return (n * G + BQ - 1) / BQ; }
PLAN_HD int plan_tile_end(int pos, int n, int tile, int G, int BQ, int cap) {
  const int rows = (tile + 1) * BQ < n * G ? (tile + 1) * BQ : n * G;
  return plan_end(pos, (rows + G - 1) / G, cap);
}
PLAN_HD int plan_splits(int end, int L) { return end <= L ? 1 : (end + L - 1) / L; }
PLAN_HD int plan_round(int64_t keys) {
  return keys > kPlanNoSplit - kPlanTile ? kPlanNoSplit : (int)((keys + kPlanTile - 1) / kPlanTile * kPlanTile);
}
// Keys [kb, ke) of split `split` of s of a tile with `end` keys; the last ones can be empty.
PLAN_HD void plan_range(int end, int s, int split, int& kb, int& ke) {
  const int chunk = plan_round((end + s - 1) / s);
  const int64_t b = (int64_t)split * chunk;
  kb = b < end ? (int)b : end;
  ke = b + chunk < end ? (int)(b + chunk) : end;
}
// Blocks (of one kv head) that T row tiles may become: a CU each, or two each where the tiles alone are more than CUs; 0: no
// splits. So many blocks, and so many partial results, are there at most when some sequence is split.
PLAN_HD int plan_budget(int T, int Hkv, int cus) {
  const int64_t n = (int64_t)T * Hkv;
  return n >= 2 * (int64_t)cus ? 0 : (n <= cus ? cus : 2 * cus) / Hkv;
}
PLAN_HD uint32_t plan_key_tiles(int end) { return (uint32_t)(end + kPlanTile - 1) / kPlanTile; }
// The first split length to try for `work` key tiles over all row tiles (a row tile counts its sequence's), and the next
// longer one while the splits are more than the budget.
PLAN_HD int plan_length(uint32_t work, int budget) {
  const int64_t l = (int64_t)(work / (uint32_t)budget + (work % (uint32_t)budget != 0)) * kPlanTile;
  return plan_round(l < kPlanMinSplit ? kPlanMinSplit : l);
}
PLAN_HD int plan_longer(int L) { return plan_round((int64_t)L + L / 8 + 1); }
