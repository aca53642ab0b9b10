"""Which of their tensors the calls of beam search and of the page pool may find in one memory, on the CPU: the rule for rows of different numbers
(hipinfer_amd/csrc/row_overlap.h), compiled for the host, against every byte of small cases, and what the C entry points refuse and
accept. Pointers here are numbers that are never followed; accepted calls end where they find no GPU (-2)."""
import ctypes
import os
import random
import re
import subprocess

import pytest
import torch

from hipinfer_amd.hipinfer import ABI, LIBRARY_PATH, _CTYPE, parse_abi
from tests.test_beam_pages_abi import NAMES, arrays

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "hipinfer_amd", "csrc")
SOURCE = """
#include "row_overlap.h"
extern "C" int meet(long long x, long long lx, long long wx, int mx, long long y, long long ly, long long wy, int my) {
  return rows_meet(x, lx, wx, mx, y, ly, wy, my);
}
"""
MB = 1 << 20  # far enough apart for any tensor here


def test_against_every_byte(tmp_path):
    (tmp_path / "meet.cpp").write_text(SOURCE)
    subprocess.run(["g++", "-O1", "-std=c++17", "-shared", "-fPIC", "-fsanitize=undefined", "-fno-sanitize-recover=undefined",
                    f"-I{CSRC}", "-o", str(tmp_path / "meet.so"), str(tmp_path / "meet.cpp")], check=True)
    meet = ctypes.CDLL(str(tmp_path / "meet.so")).meet
    ll = ctypes.c_longlong
    meet.argtypes = [ll, ll, ll, ctypes.c_int, ll, ll, ll, ctypes.c_int]
    r = random.Random(1)
    seen = [0, 0]
    for _ in range(20000):
        mx, my, wx, wy = r.randint(1, 5), r.randint(1, 5), r.randint(1, 9), r.randint(1, 9)
        lx, ly = wx + r.choice([0, 0, 3, 12]), wy + r.choice([0, 2, 9, 25])
        x, y = 100, 100 + r.choice([r.randint(-60, 60), r.randint(-12, 12)])
        cover = [{a + i * s + j for i in range(m) for j in range(w)} for a, s, w, m in ((x, lx, wx, mx), (y, ly, wy, my))]
        want = bool(cover[0] & cover[1])
        assert meet(x, lx, wx, mx, y, ly, wy, my) == want, (x, lx, wx, mx, y, ly, wy, my)
        seen[want] += 1
    assert min(seen) > 3000


def call(name, args):
    fn = getattr(ctypes.CDLL(LIBRARY_PATH), name)
    fn.argtypes = [_CTYPE[a] for a in parse_abi(ABI)[name][1]]
    return fn(*(args[a] for a in NAMES[name]))


def refused(name, args, pair, capfd):
    assert call(name, args) == -1
    err = capfd.readouterr().err
    assert re.search(rf"{name}: ({pair[0]} and {pair[1]}|{pair[1]} and {pair[0]}) must be apart", err), err


accepted = pytest.mark.skipif(torch.cuda.is_available(), reason="a GPU would run the calls")

FORK = dict(arrays(), n=2, page=16, table=MB, ldt=6, W=4, S=3, lens=2 * MB, parent=3 * MB, N=5, refs=4 * MB, pages=30, grow=1,
            table_out=5 * MB, ldo=6, lens_out=6 * MB, refs_out=7 * MB, missing=8 * MB, work=9 * MB, work_bytes=1 << 16, stream=None)
FORK_READ = ("table", "lens", "parent", "refs")
FORK_WRITTEN = ("table_out", "lens_out", "refs_out", "missing", "work")


@pytest.mark.parametrize("out", FORK_WRITTEN)
@pytest.mark.parametrize("other", FORK_READ + FORK_WRITTEN)
def test_fork(out, other, capfd):
    """A tensor that is written on the memory of any other, from its first and from a later entry on."""
    if out == other:
        return
    if (other, out) != ("refs", "refs_out"):  # (the counts in place)
        refused("hi_cache_fork", FORK | {out: FORK[other]}, (other, out), capfd)
    if other not in ("missing",) and out != "work" and (other, out) != ("refs", "refs_out"):
        refused("hi_cache_fork", FORK | {out: FORK[other] + 8}, (other, out), capfd)


@accepted
@pytest.mark.parametrize("change", [
    {}, dict(refs_out=4 * MB), dict(missing=None), dict(lens_out=3 * MB + 20), dict(lens_out=3 * MB - 20),  # behind and before parent
    dict(table_out=MB + 16, ldt=8, ldo=8),  # two tables side by side in rows of 8
    dict(lens=3 * MB),                      # what is only read
    dict(S=0, table=None, lens=None), dict(N=0, parent=None, table_out=None, lens_out=None),
    dict(N=0, parent=2 * MB, table_out=MB, lens_out=2 * MB),  # nothing is written there
], ids=str)
def test_fork_accepts(change):
    assert call("hi_cache_fork", FORK | change) == -2


COMPACT = dict(arrays(), n=2, page=16, table=MB, ldt=6, W=4, S=3, refs=4 * MB, pages=30, table_out=5 * MB, ldo=6, refs_out=7 * MB,
               moved=2 * MB, used=8 * MB, work=9 * MB, work_bytes=1 << 16, stream=None)
COMPACT_READ = ("table", "refs")
COMPACT_WRITTEN = ("table_out", "refs_out", "moved", "used", "work")
IN_PLACE = {("table", "table_out"), ("refs", "refs_out")}


@pytest.mark.parametrize("out", COMPACT_WRITTEN)
@pytest.mark.parametrize("other", COMPACT_READ + COMPACT_WRITTEN)
def test_compact(out, other, capfd):
    if out == other or (other, out) in IN_PLACE:
        return
    refused("hi_cache_compact", COMPACT | {out: COMPACT[other]}, (other, out), capfd)
    if other != "used" and out != "work":
        refused("hi_cache_compact", COMPACT | {out: COMPACT[other] + 8}, (other, out), capfd)


def test_compact_in_place(capfd):
    """moved on the table and the counts that are renamed in place."""
    base = COMPACT | dict(table_out=MB, refs_out=4 * MB)
    for at, name in ((MB, "table"), (MB + 24 + 8, "table"), (4 * MB, "refs"), (4 * MB + 116, "refs")):
        refused("hi_cache_compact", base | dict(moved=at), (name, "moved"), capfd)
        refused("hi_cache_compact", base | dict(used=at), (name, "used"), capfd)


@accepted
@pytest.mark.parametrize("change", [
    {}, dict(table_out=MB, refs_out=4 * MB), dict(used=None), dict(moved=MB + 12 * 6), dict(used=MB + 16),  # used in a gap of the table
    dict(table_out=MB + 16, ldt=8, ldo=8), dict(S=0, table=None, table_out=None),
], ids=str)
def test_compact_accepts(change):
    assert call("hi_cache_compact", COMPACT | change) == -2


BEAM = dict(logits=MB, ldl=110, scores=2 * MB, B=2, beams=4, V=100, n=8, best=3 * MB, parent=4 * MB, token=5 * MB, work=6 * MB,
            work_bytes=1 << 16, stream=None)
BEAM_READ = ("logits", "scores")
BEAM_WRITTEN = ("best", "parent", "token", "work")


@pytest.mark.parametrize("out", BEAM_WRITTEN)
@pytest.mark.parametrize("other", BEAM_READ + BEAM_WRITTEN)
def test_beam_select(out, other, capfd):
    """One sequence's block writes its places while others still read their logits and scores."""
    if out == other or (other, out) == ("scores", "best"):
        return
    refused("hi_beam_select", BEAM | {out: BEAM[other]}, (other, out), capfd)
    if out != "work":
        refused("hi_beam_select", BEAM | {out: BEAM[other] + 28}, (other, out), capfd)


@pytest.mark.parametrize("out", ["parent", "token"])
def test_beam_select_in_place(out, capfd):
    """With best in the scores' place, the other outputs are as little allowed there."""
    refused("hi_beam_select", BEAM | {"n": 4, "best": 2 * MB, out: 2 * MB}, ("scores", out), capfd)


@accepted
@pytest.mark.parametrize("change", [
    {}, dict(n=4, best=2 * MB), dict(best=2 * MB + 32), dict(parent=2 * MB + 32), dict(token=MB + 8 * 220),  # behind scores and logits
    dict(B=1, beams=1, n=5, token=MB + 200),  # one row ends with its logits, whatever its stride
], ids=str)
def test_beam_select_accepts(change):
    assert call("hi_beam_select", BEAM | change) == -2
