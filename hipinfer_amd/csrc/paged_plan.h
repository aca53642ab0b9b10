// How attention over ragged row runs is cut into blocks: row tiles, and splits of a tile's keys. Plain arithmetic of one
// sequence at a time, used by the kernels (summed over a wave's lanes) and compiled for the host by its tests.
#pragma once
#include <cstdint>

#if defined(__HIPCC__)
#define PLAN_HD __host__ __device__ __forceinline__
#else
#define PLAN_HD inline
#endif
// 1 / b in fp32, off by 2^-23 of it at most: the hardware's estimate, on the host the division (a test puts in its neighbours)
#if defined(__HIP_DEVICE_COMPILE__)
#define PLAN_RCP(b) __builtin_amdgcn_rcpf(b)
#elif !defined(PLAN_RCP)
#define PLAN_RCP(b) (1.0f / (b))
#endif

constexpr int kPlanTile = 128;          // keys of a tile: splits are whole tiles, and their lengths count them
constexpr int kPlanMinSplit = 4;        // tiles a split has at least
constexpr int kPlanNoSplit = 1 << 24;   // more tiles than the 2^30 keys that a table may hold

// a / b for 0 <= a < 2^24 with a quotient below 2^22.4, so that two roundings of 2^-23 leave it off by one at most. Integer
// division is some 30 instructions, and a plan's are on the way of every block.
constexpr int kPlanDiv = 1 << 22;  // an `a` that every b >= 1 is fine with
PLAN_HD int plan_div(int a, int b) {
  const int q = (int)((float)a * PLAN_RCP((float)b)), r = a - q * b;
  return q + (r >= b ? 1 : 0) - (r < 0 ? 1 : 0);
}

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
// Packed row r is query head r % G of the kv head's G in token r / G; with magic = 2^32 / G + 1 exact below 2^28.
PLAN_HD uint32_t plan_magic(int G) { return G == 1 ? 0u : 0xffffffffu / (uint32_t)G + 1u; }
PLAN_HD int plan_token(int r, uint32_t magic) { return magic ? (int)(((uint64_t)(uint32_t)r * magic) >> 32) : r; }
// Tiles of BQ packed rows, and the keys that tile `tile` sees.
PLAN_HD int plan_tiles(int n, int G, int BQ) { return (n * G + BQ - 1) / BQ; }
PLAN_HD int plan_tile_end(int pos, int n, int tile, int G, uint32_t magic, int BQ, int cap) {
  const int rows = (tile + 1) * BQ < n * G ? (tile + 1) * BQ : n * G;
  return plan_end(pos, plan_token(rows - 1, magic) + 1, cap);
}
PLAN_HD int plan_key_tiles(int end) { return (end + kPlanTile - 1) / kPlanTile; }
// Splits of len keys, K of them each, at most S.
PLAN_HD int plan_step_splits(int len, int K, int S) {
  return len > (S - 1) * K ? S : len <= K ? 1 : plan_div(len + K - 1, K);
}
// Splits of a sequence with te key tiles.
PLAN_HD int plan_splits(int te, int L) { return te <= L ? 1 : plan_div(te + L - 1, L); }
// Keys [kb, ke) of split `split` of s of a row tile with `end` keys; the last ones can be empty.
PLAN_HD void plan_range(int end, int s, int split, int& kb, int& ke) {
  const int te = plan_key_tiles(end), chunk = s == 1 ? te : plan_div(te + s - 1, s), t0 = split * chunk, t1 = t0 + chunk;
  kb = t0 < te ? t0 * kPlanTile : end;
  ke = t1 < te ? t1 * kPlanTile : end;
}
// Blocks (of one kv head) that T row tiles may become: a CU each, or two each where the tiles alone are more than CUs; 0: no
// splits. So many blocks, and so many partial results, are there at most when some sequence is split. b1 = cus / Hkv, b2 =
// 2 cus / Hkv.
PLAN_HD int plan_budget(int T, int Hkv, int cus, int b1, int b2) {
  return T > 65535 || T * Hkv >= 2 * cus ? 0 : T * Hkv <= cus ? b1 : b2;
}
// The first split length to try for `work` key tiles over all row tiles (a row tile counts its sequence's), and the next
// longer one while the splits are more than the budget.
PLAN_HD int plan_length(uint32_t work, int budget, int least = kPlanMinSplit) {
  const int l = (int)((float)work * PLAN_RCP((float)budget)) + 1;
  return l < least ? least : l;
}
PLAN_HD int plan_longer(int L) { return L + L / 8 + 1; }
