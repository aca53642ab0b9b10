"""What the C entry points of the 8-bit paged cache refuse, on the CPU (as test_paged_abi.py's)."""
import ctypes

import pytest

from hipinfer_amd.hipinfer import ABI, LIBRARY_PATH, _CTYPE, parse_abi
from tests.test_paged_abi import ATTN, CACHE, NAMES, P, ROPE

NEW = dict(kexp=P, vexp=P, page_stride=2048)
ROPE8 = {k: v for k, v in ROPE.items() if k != "seq"} | NEW | dict(start=None)
ATTN8 = ATTN | NEW
CACHE8 = [c for c in CACHE if c not in (dict(page_stride=2040), dict(page_stride=2052))] + [
    dict(page_stride=2040), dict(page_stride=2056), dict(kexp=None), dict(vexp=None)]
BAD = {
    "hi_rope_cache_paged8": (ROPE8, CACHE8 + [
        dict(M=-1), dict(M=4), dict(M=2), dict(Hq=0), dict(rot=-2), dict(rot=3), dict(rot=130), dict(cs_rows=0), dict(qkv=None),
        dict(q_out=None), dict(cs=None), dict(pos=None), dict(ldq=767), dict(ldqo=511), dict(qkv=P + 1), dict(cs=P + 2),
        dict(cs=P + 4, cs_f32=1), dict(pos=P + 1), dict(start=P + 2), dict(q_out=P + 2), dict(ldqo=770)]),
    "hi_attn_paged8": (ATTN8, CACHE8 + [
        dict(M=-1), dict(M=4), dict(M=2), dict(Hq=0), dict(Hq=3, Hkv=2), dict(Hq=17, ldq=2176, ldo=2176), dict(q=None), dict(q=P + 8),
        dict(ldq=511), dict(ldq=516), dict(pos=None), dict(pos=P + 2), dict(out=None), dict(out=P + 4), dict(ldo=510), dict(ldo=508),
        dict(lse=P + 2), dict(start=P + 2), dict(M=1 << 26, B=1 << 26), dict(start=P, M=1 << 26), dict(out=P + 512)]),
}


@pytest.mark.parametrize("name", sorted(BAD))
def test_refused(name, capfd):
    base, bad = BAD[name]
    assert sorted(base) == sorted(NAMES[name])
    fn = getattr(ctypes.CDLL(LIBRARY_PATH), name)
    fn.argtypes = [_CTYPE[a] for a in parse_abi(ABI)[name][1]]
    for change in bad:
        args = base | change
        assert fn(*(args[a] for a in NAMES[name])) == -1, change
        assert name in capfd.readouterr().err, change


@pytest.mark.parametrize("name", sorted(BAD))
def test_no_rows_is_no_call(name):
    base = BAD[name][0] | dict(M=0, B=0)
    fn = getattr(ctypes.CDLL(LIBRARY_PATH), name)
    fn.argtypes = [_CTYPE[a] for a in parse_abi(ABI)[name][1]]
    assert fn(*(base[a] for a in NAMES[name])) == 0
