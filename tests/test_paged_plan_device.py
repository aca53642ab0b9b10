"""The paged plans (hipinfer_amd/csrc/paged_plan.h) as the device computes them: the same text compiled for the host, with the
reciprocal one step of fp32 below, at and above the rounded 1 / b (the hardware's is within that). Division over its stated range,
and the plans of the kernel for few rows: splits by all lengths (blocks of 8 waves) and by each sequence's own (4 waves)."""
import ctypes
import os
import random
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "hipinfer_amd", "csrc")

SOURCE = r"""
#include <algorithm>
#include <cmath>
static int off = 0;
static float rcp(float b) {
  const float r = 1.0f / b;
  return off == 0 ? r : std::nextafterf(r, off < 0 ? 0.0f : INFINITY);
}
#define PLAN_RCP(b) rcp(b)
#include "paged_plan.h"
extern "C" void nudge(int by) { off = by; }
extern "C" int div_of(int a, int b) { return plan_div(a, b); }
extern "C" int step_of(int len, int K, int S) { return plan_step_splits(len, K, S); }
extern "C" int length_of(unsigned work, int budget, int least) { return plan_length(work, budget, least); }

struct Seq { int n, tiles, keys; };
static Seq seq(const int* start, const int* pos, int b, int M, int G, int COLS, int cap) {
  const int n = plan_rows(start[b], start[b + 1], M);
  return {n, plan_tiles(n, G, COLS), plan_end(pos[b], n, cap)};
}
// The kernel's walk with blocks of 8 waves: (b, tile, split, splits, place) per block; the plan knows all lengths.
extern "C" int cut_all(const int* start, const int* pos, int B, int M, int G, int COLS, int Hkv, int cap, int cus, int slots,
                       int least, int fan, int* out, int room) {
  int T = 0, longest = 0, L = kPlanNoSplit, n_out = 0, slot = 0;
  uint32_t work = 0;
  for (int b = 0; b < B; b++) {
    const Seq s = seq(start, pos, b, M, G, COLS, cap);
    T += s.tiles;
    work += (uint32_t)s.tiles * (uint32_t)plan_key_tiles(s.keys);
    if (s.tiles) longest = std::max(longest, plan_key_tiles(s.keys));
  }
  const int budget = plan_budget(T, Hkv, cus, cus / Hkv, 2 * cus / Hkv);
  if (budget > 0) {
    L = std::max(plan_length(work, budget, least), plan_div(longest + fan - 1, fan));
    for (; L < longest; L = plan_longer(L)) {
      int units = 0;
      for (int b = 0; b < B; b++) {
        const Seq s = seq(start, pos, b, M, G, COLS, cap);
        units += s.tiles * plan_splits(plan_key_tiles(s.keys), L);
      }
      if (units <= std::min(budget, slots)) break;
    }
  }
  for (int b = 0; b < B; b++) {
    const Seq s = seq(start, pos, b, M, G, COLS, cap);
    const int splits = plan_splits(plan_key_tiles(s.keys), L);
    for (int i = 0; i < s.tiles * splits; i++) {
      if (n_out == room) return -1;
      const int down = splits == 1 ? i : plan_div(i, splits), tile = s.tiles - 1 - down, split = i - down * splits;
      int* o = out + 5 * n_out++;
      o[0] = b, o[1] = tile, o[2] = split, o[3] = splits, o[4] = splits > 1 ? slot + tile * splits + split : -1;
    }
    if (splits > 1) slot += s.tiles * splits;
  }
  return n_out;
}
// With blocks of 4 waves: a sequence's splits are its own, o[4] is the tile's number.
extern "C" int cut_each(const int* start, const int* pos, int B, int M, int G, int COLS, int cap, int K, int S, int* out, int room) {
  int n_out = 0, number = 0;
  for (int b = 0; b < B; b++) {
    const Seq s = seq(start, pos, b, M, G, COLS, cap);
    const int splits = plan_step_splits(s.keys, K, S);
    for (int i = 0; i < s.tiles * splits; i++) {
      if (n_out == room) return -1;
      const int tile = splits == 1 ? i : plan_div(i, splits);
      int* o = out + 5 * n_out++;
      o[0] = b, o[1] = tile, o[2] = i - tile * splits, o[3] = splits, o[4] = number + tile;
    }
    number += s.tiles;
  }
  return n_out;
}
// Keys [first, last) of a split of a tile, as the kernel computes them.
extern "C" void keys_of(int pos, int n, int tile, int G, int COLS, int cap, int splits, int split, int* se) {
  const int len = plan_tile_end(pos, n, tile, G, plan_magic(G), COLS, cap);
  const int chunk = ((len < kPlanDiv ? plan_div(len + splits - 1, splits) : (len + splits - 1) / splits) + 7) & ~7;
  se[0] = split * chunk;
  se[1] = std::min(len, split * chunk + chunk);
}
"""


@pytest.fixture(scope="module")
def built(tmp_path_factory):
    d = tmp_path_factory.mktemp("plan")
    (d / "plan.cpp").write_text(SOURCE)
    subprocess.run(["g++", "-O1", "-std=c++17", "-ffp-contract=off", "-shared", "-fPIC", "-fsanitize=undefined",
                    "-fno-sanitize-recover=undefined", f"-I{CSRC}", "-o", str(d / "plan.so"), str(d / "plan.cpp")], check=True)
    return ctypes.CDLL(str(d / "plan.so"))


@pytest.fixture(params=[-1, 0, 1])
def plan(built, request):
    built.nudge(request.param)
    yield built
    built.nudge(0)


def test_division(plan):
    """0 <= a < 2^24, a / b < 2^22.4."""
    r = random.Random(1)
    top = int(2**22.4)
    for _ in range(100000):
        b = r.choice([r.randint(1, 40), r.randint(1, 5000), r.randint(1, 2**23)])
        most = min(2**24, top * b) - 1
        a = r.choice([r.randint(0, most), most // b * b, most // b * b - 1, r.randint(0, most // b) * b, r.randint(0, most // b) * b - 1])
        a = max(0, min(a, most))
        assert plan.div_of(a, b) == a // b, (a, b)


def test_step_splits(plan):
    """The least splits of K keys, at most S, whatever the length."""
    r = random.Random(2)
    for _ in range(50000):
        K, S = r.choice([256, 320, 512, 768, 4096]), r.choice([1, 2, 3, 8, r.randint(1, 64)])
        n = r.choice([r.randint(0, 3 * K), r.randint(0, S * K + 5), r.randint(0, S) * K, r.randint(0, 2**30), 2**30])
        assert plan.step_of(n, K, S) == max(1, min(S, -(-n // K))), (n, K, S)


def test_length_is_in_range(plan):
    """Near work / budget, never negative. A budget's tiles (at most as many, below 512) hold at most 2^23 key tiles each."""
    r = random.Random(3)
    for _ in range(20000):
        budget = r.randint(1, 511)
        work = r.choice([0, r.randint(0, 5000), r.randint(0, budget << 23), budget << 23])
        got = plan.length_of(ctypes.c_uint(work), budget, 1)
        assert 1 <= got and abs(got - (work // budget + 1)) <= 1 + work // budget // 2**21


def batch(r):
    B = r.choice([1, 1, 2, 7, 40, 100])
    G = r.choice([1, 2, 4, 6, 8, 16])
    rows = [r.choice([0, 1, 1, 2, 5, r.randint(1, 60)]) for _ in range(B)]
    pos = [r.choice([-5, -1, 0, r.randint(0, 400), r.randint(0, 50000), 2**31 - 1]) for _ in range(B)]
    cap = r.choice([128, 512, 4096, 65536, 1 << 30])
    start = [r.randint(0, 3)]
    for n in rows:
        start.append(start[-1] + n)
    return B, G, rows, pos, cap, start, start[-1] + r.randint(0, 3)


def cover(plan, units, rows, pos, G, COLS, cap):
    """Every tile has each of its splits once, and they are each of its keys once."""
    seen = {}
    for b, tile, split, splits, _ in units:
        seen.setdefault((b, tile), []).append((split, splits))
    se = (ctypes.c_int * 2)()
    for b, n in enumerate(rows):
        for tile in range(-(-n * G // COLS)):
            parts = sorted(seen.pop((b, tile)))
            assert [p[0] for p in parts] == list(range(parts[0][1]))
            at, end = 0, max(0, min(pos[b] + (min((tile + 1) * COLS, n * G) - 1) // G + 1, cap))
            for split, splits in parts:
                plan.keys_of(pos[b], n, tile, G, COLS, cap, splits, split, se)
                if se[0] < se[1]:
                    assert se[0] == at and at % 8 == 0
                    at = se[1]
            assert at == end
    assert not seen


@pytest.mark.parametrize("seed", range(80))
def test_splits_by_all_lengths(plan, seed):
    """Blocks of 8 waves: at most 32 splits of a tile, parts and blocks within the launch's."""
    r = random.Random(1000 + seed)
    Hkv, COLS, cus = r.choice([1, 2, 4, 8, 40]), r.choice([16, 32]), 256
    most = cus
    while not 0 < 2 * most * Hkv <= cus:  # the batches that take blocks of 8 waves
        B, G, rows, pos, cap, start, M = batch(r)
        most = max(min(B, M), -(-M * G // COLS))
    tiles = most if B == 1 else M * G // COLS + min(B, M)
    slots = 2 * cus // Hkv
    room = max(tiles, slots) + 1
    out = (ctypes.c_int * (5 * room))()
    ints = ctypes.c_int * (B + 1)
    n = plan.cut_all(ints(*start), ints(*pos), B, M, G, COLS, Hkv, cap, cus, slots, 1, 32, out, room)
    assert 0 <= n <= max(tiles, slots)
    units = [tuple(out[5 * i:5 * i + 5]) for i in range(n)]
    places = [u[4] for u in units if u[4] >= 0]
    assert len(set(places)) == len(places) and all(0 <= p < slots for p in places)
    assert all(u[3] <= 32 for u in units)
    cover(plan, units, rows, pos, G, COLS, cap)


@pytest.mark.parametrize("seed", range(80))
def test_splits_by_each_length(plan, seed):
    """Blocks of 4 waves: tiles numbered from 0 to at most the launch's, at most S splits each."""
    r = random.Random(2000 + seed)
    B, G, rows, pos, cap, start, M = batch(r)
    COLS, K, S = r.choice([16, 32]), r.choice([256, 320, 768, 4096]), r.randint(1, 8)
    tiles = -(-M * G // COLS) if B == 1 else M * G // COLS + min(B, M)
    room = tiles * S + 1
    out = (ctypes.c_int * (5 * room))()
    ints = ctypes.c_int * (B + 1)
    n = plan.cut_each(ints(*start), ints(*pos), B, M, G, COLS, cap, K, S, out, room)
    assert 0 <= n <= tiles * S
    units = [tuple(out[5 * i:5 * i + 5]) for i in range(n)]
    numbers = {(u[0], u[1]): u[4] for u in units}
    assert sorted(numbers.values()) == list(range(len(numbers))) and len(numbers) <= tiles
    cover(plan, units, rows, pos, G, COLS, cap)
