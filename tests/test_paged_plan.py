"""How attention over ragged row runs is cut into blocks (hipinfer_amd/csrc/paged_plan.h), compiled for the host: every visible
(row tile, key) pair belongs to exactly one block, blocks and partial results stay within what the launch provides, whatever
the lengths, and also where start leaves the rows or decreases. On the CPU; the same integer functions run on the GPU."""
import ctypes
import os
import random
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "hipinfer_amd", "csrc")

SOURCE = r"""
#include "paged_plan.h"
#include <vector>
#include <algorithm>
// The kernels' walk over the sequences, one after another: fills (b, tile, split, kb, ke, slot) per block in block order.
extern "C" int cut(const int* start, const int* pos, int B, int M, int G, int BQ, int Hkv, int cap, int cus, int slots,
                   int* out, int room) {
  int T = 0, longest = 0;
  uint32_t work = 0;
  for (int b = 0; b < B; b++) {
    const int n = plan_rows(start[b], start[b + 1], M), t = plan_tiles(n, G, BQ), e = plan_end(pos[b], n, cap);
    T += t;
    work += (uint32_t)t * plan_key_tiles(e);
    if (t) longest = std::max(longest, plan_key_tiles(e));
  }
  int L = kPlanNoSplit;
  const int budget = slots ? plan_budget(T, Hkv, cus, cus / Hkv, 2 * cus / Hkv) : 0;
  if (budget > 0)
    for (L = plan_length(work, budget); L < longest; L = plan_longer(L)) {
      int units = 0;
      for (int b = 0; b < B; b++) {
        const int n = plan_rows(start[b], start[b + 1], M);
        units += plan_tiles(n, G, BQ) * plan_splits(plan_key_tiles(plan_end(pos[b], n, cap)), L);
      }
      if (units <= std::min(budget, slots)) break;
    }
  int n_out = 0, slot = 0;
  for (int b = 0; b < B; b++) {
    const int n = plan_rows(start[b], start[b + 1], M), t = plan_tiles(n, G, BQ), s = plan_splits(plan_key_tiles(plan_end(pos[b], n, cap)), L);
    for (int i = 0; i < t * s; i++) {
      const int tile = t - 1 - i / s, split = i % s;
      int kb, ke;
      plan_range(plan_tile_end(pos[b], n, tile, G, plan_magic(G), BQ, cap), s, split, kb, ke);
      if (n_out == room) return -1;
      int* o = out + 7 * n_out++;
      o[0] = b, o[1] = tile, o[2] = split, o[3] = kb, o[4] = ke, o[5] = s > 1 ? slot + tile * s + split : -1, o[6] = s;
    }
    if (s > 1) slot += t * s;
  }
  return n_out;
}
extern "C" int budget_of(int T, int Hkv, int cus) { return plan_budget(T, Hkv, cus, cus / Hkv, 2 * cus / Hkv); }
extern "C" int token_of(int r, int G) { return plan_token(r, plan_magic(G)); }
extern "C" int tiles_of(int n, int G, int BQ) { return plan_tiles(n, G, BQ); }
"""


@pytest.fixture(scope="module")
def plan(tmp_path_factory):
    d = tmp_path_factory.mktemp("plan")
    (d / "plan.cpp").write_text(SOURCE)
    so = d / "plan.so"
    subprocess.run(["g++", "-O1", "-std=c++17", "-shared", "-fPIC", "-fsanitize=undefined", "-fno-sanitize-recover=undefined",
                    f"-I{CSRC}", "-o", str(so), str(d / "plan.cpp")], check=True)
    return ctypes.CDLL(str(so))


def cut(plan, start, pos, M, G, BQ, Hkv, cap, cus=256):
    B = len(pos)
    least = plan.tiles_of(M, G, BQ)
    slots = max(2 * cus // Hkv, 1) if plan.budget_of(least, Hkv, cus) else 0
    tiles = least if B == 1 else M * G // BQ + min(B, M)  # the launch's row tiles
    room = max(tiles, slots) + 200000
    ints = ctypes.c_int * max(1, len(start) + B)
    out = (ctypes.c_int * (7 * room))()
    n = plan.cut(ints(*start), ints(*pos), B, M, G, BQ, Hkv, cap, cus, slots, out, room)
    assert n >= 0
    return [tuple(out[7 * i:7 * i + 7]) for i in range(n)], tiles, slots


@pytest.mark.parametrize("seed", range(150))
def test_every_key_once_and_in_bounds(plan, seed):
    r = random.Random(seed)
    B = r.choice([1, 1, 2, 7, 70, 200])
    G, BQ, Hkv = r.choice([1, 2, 4, 6, 8, 16]), r.choice([64, 128]), r.choice([1, 2, 4, 8, 40, 300])
    rows = [r.choice([0, 1, 1, 5, r.randint(1, 300), r.randint(1, 3000 // B + 1)]) for _ in range(B)]
    pos = [r.choice([-5, -1, 0, r.randint(0, 400), r.randint(0, 50000), 2**31 - 1]) for _ in range(B)]
    cap = r.choice([128, 512, 4096, 65536, 1 << 30])
    front, back = r.randint(0, 3), r.randint(0, 3)
    start = [front]
    for n in rows:
        start.append(start[-1] + n)
    M = start[-1] + back
    units, tiles, slots = cut(plan, start, pos, M, G, BQ, Hkv, cap)
    assert len(units) <= max(tiles, slots)
    used = [u[5] for u in units if u[5] >= 0]
    assert len(set(used)) == len(used) and all(0 <= s < slots for s in used)
    seen = {}
    for b, tile, split, kb, ke, slot, s in units:
        assert kb % 128 == 0 or kb == ke
        seen.setdefault((b, tile), []).append((split, kb, ke, s))
    for b, n in enumerate(rows):
        for tile in range(-(-n * G // BQ)):
            last = (min((tile + 1) * BQ, n * G) - 1) // G  # token
            end = max(0, min(pos[b] + last + 1, cap))
            parts = sorted(seen.pop((b, tile)))
            assert [p[0] for p in parts] == list(range(parts[0][3]))
            at = 0
            for _, kb, ke, _ in parts:
                assert (kb, ke) == (at, ke) and ke >= kb or kb == ke == end
                at = max(at, ke)
            assert at == end
    assert not seen


@pytest.mark.parametrize("start", [[0, 3, 1, 6], [6, 4, 2, 0], [-2**31, 2**31 - 1, 0, 6], [2**31 - 1] * 4, [0, 6, 0, 6]], ids=str)
def test_bad_start_stays_in_bounds(plan, start):
    units, tiles, slots = cut(plan, start, [100, 5000, 2**31 - 1], 6, 4, 64, 8, 8192)
    for b, tile, split, kb, ke, slot, s in units:
        assert 0 <= kb <= ke <= 8192 and slot < slots


def test_token_is_exact(plan):
    r = random.Random(0)
    for G in range(1, 17):
        for _ in range(3000):
            n = r.choice([r.randint(0, 300), r.randint(0, 1 << 27), (1 << 27) - r.randint(1, 40)])
            assert plan.token_of(n, G) == n // G


def test_one_sequence_fills_the_gpu(plan):
    """Few rows after a long context: a split per CU and not more; few keys: no splits."""
    units, _, _ = cut(plan, [0, 5], [32000], 5, 4, 64, 8, 1 << 20)
    assert len(units) * 8 <= 256 and len(units) * 8 > 200
    assert len(cut(plan, [0, 5], [500], 5, 4, 64, 8, 1 << 20)[0]) == 1
