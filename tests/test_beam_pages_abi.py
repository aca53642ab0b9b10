"""What the C entry points of beam search and of the page pool refuse, on the CPU: bad sizes, strides, alignments, overlaps and null
pointers are found before the device is looked at (-1; nothing is launched). Pointers here are numbers that are never followed, but
for the host arrays that describe the cache tensors."""
import ctypes
import re

import pytest

from hipinfer_amd.hipinfer import ABI, LIBRARY_PATH, _CTYPE, parse_abi

NAMES = {m[1]: [a.split()[-1] for a in m[2].split(",") if a.strip()]
         for m in re.finditer(r"(\w+)\s*\(([^)]*)\)\s*;", ABI)}
P, Q, R = 1 << 20, 1 << 24, 1 << 26  # aligned addresses, far apart


def arrays(ptr=P, stride=4096, size=4096, runs=2):
    return dict(caches=(ctypes.c_void_p * 2)(P, ptr), strides=(ctypes.c_longlong * 2)(4096, stride),
                bytes=(ctypes.c_longlong * 2)(4096, size), runs=(ctypes.c_int * 2)(2, runs))


FORK = dict(arrays(), n=2, page=16, table=P, ldt=4, W=4, S=3, lens=Q, parent=Q, N=5, refs=R, pages=30, grow=1, table_out=Q + 4096, ldo=4,
            lens_out=P + 4096, refs_out=R, missing=None, work=P, work_bytes=1 << 20, stream=None)
COMPACT = {k: v for k, v in FORK.items() if k not in ("lens", "parent", "N", "grow", "lens_out", "missing")} | dict(moved=P, used=None)
BEAM = dict(logits=P, ldl=100, scores=Q, B=2, beams=4, V=100, n=8, best=P, parent=P, token=P, work=P, work_bytes=1 << 20, stream=None)
POOL = [dict(page=0), dict(page=12), dict(page=-8), dict(page=1 << 21), dict(S=-1), dict(S=8193), dict(W=0), dict(ldt=3), dict(ldo=3),
        dict(pages=0), dict(pages=(1 << 30) + 1), dict(n=-1), dict(W=1 << 27, ldt=1 << 27, ldo=1 << 27), dict(refs=None), dict(refs_out=None), dict(work=None),
        dict(work=P + 8), dict(work_bytes=100), dict(table=None), dict(table=P + 2), dict(refs=R + 2), dict(refs_out=R + 4),
        dict(refs_out=R - 100), dict(caches=None), dict(bytes=None), arrays(ptr=None), arrays(stride=4095), arrays(size=0),
        arrays(size=1 << 32, stride=1 << 33), arrays(runs=-1), arrays(runs=3), arrays(size=4000, runs=251)]
BAD = {
    "hi_cache_fork": (FORK, POOL + [
        dict(N=-1), dict(N=8193), dict(grow=-1), dict(grow=(1 << 30) + 1), dict(lens=None), dict(parent=None), dict(table_out=None),
        dict(lens_out=None), dict(lens=Q + 1), dict(parent=Q + 2), dict(lens_out=Q + 3), dict(missing=P + 1), dict(table_out=P),
        dict(table_out=P + 44), dict(table_out=P - 76), dict(lens_out=Q), dict(lens_out=Q - 16), dict(lens_out=Q + 8)]),
    "hi_cache_compact": (COMPACT, POOL + [dict(moved=None), dict(moved=P + 2), dict(used=P + 1), dict(table_out=None),
                                          dict(table_out=P + 4), dict(table_out=P, ldo=5), dict(table_out=P + 32), dict(moved=R), dict(moved=R + 116),
                                          dict(refs_out=Q, moved=Q + 8)]),
    "hi_beam_select": (BEAM, [
        dict(B=-1), dict(beams=0), dict(beams=65), dict(V=0), dict(n=0), dict(n=65), dict(beams=64, V=1 << 19, ldl=1 << 19),
        dict(B=20000), dict(logits=None), dict(scores=None), dict(best=None), dict(parent=None), dict(token=None), dict(work=None),
        dict(logits=P + 1), dict(scores=Q + 2), dict(best=P + 2), dict(parent=P + 1), dict(token=P + 3), dict(work=P + 8),
        dict(work_bytes=20), dict(ldl=99), dict(best=Q, scores=Q), dict(best=Q, scores=Q + 16), dict(best=Q + 28, scores=Q),
        dict(best=Q + 4, scores=Q, n=4)]),
}


@pytest.fixture(scope="module")
def lib():
    return ctypes.CDLL(LIBRARY_PATH)


@pytest.mark.parametrize("name", sorted(BAD))
def test_refused(lib, name, capfd):
    base, bad = BAD[name]
    assert sorted(base) == sorted(NAMES[name])
    fn = getattr(lib, name)
    fn.argtypes = [_CTYPE[a] for a in parse_abi(ABI)[name][1]]
    for change in bad:
        args = base | change
        assert fn(*(args[a] for a in NAMES[name])) == -1, change
        assert name in capfd.readouterr().err, change


def test_no_sequences_is_no_call(lib):
    fn = lib.hi_beam_select
    fn.argtypes = [_CTYPE[a] for a in parse_abi(ABI)["hi_beam_select"][1]]
    assert fn(*((BEAM | dict(B=0))[a] for a in NAMES["hi_beam_select"])) == 0


def test_work_bytes(lib):
    """0 for sizes that the calls refuse; never less for more."""
    lib.hi_cache_work_bytes.restype = lib.hi_beam_select_work_bytes.restype = ctypes.c_size_t
    for bad in [(-1, 1, 1), (1, -1, 1), (1, 1, 0), (8193, 1, 1), (1, 8193, 1)]:
        assert lib.hi_cache_work_bytes(*bad) == 0
    for bad in [(-1, 1, 9, 1), (1, 0, 9, 1), (1, 65, 9, 1), (1, 1, 0, 1), (1, 1, 9, 0), (1, 1, 9, 65), (1, 64, 1 << 19, 1), (70000, 1, 9, 1)]:
        assert lib.hi_beam_select_work_bytes(*bad) == 0
    sizes = [lib.hi_cache_work_bytes(s, n, p) for s, n, p in [(1, 0, 1), (1, 1, 1), (7, 1, 9), (7, 30, 9), (100, 30, 400), (100, 500, 400)]]
    assert sizes == sorted(sizes) and sizes[0] > 0
