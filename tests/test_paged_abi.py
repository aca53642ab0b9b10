"""What the paged attention's C entry points refuse, on the CPU: bad sizes, strides, alignments and null pointers are found before
the device is looked at (-1; nothing is launched). Pointers here are numbers that are never followed."""
import ctypes
import re

import pytest

from hipinfer_amd.hipinfer import parse_abi, ABI, _CTYPE, LIBRARY_PATH

NAMES = {m[1]: [a.split()[-1] for a in m[2].split(",") if a.strip()]
         for m in re.finditer(r"(\w+)\s*\(([^)]*)\)\s*;", ABI)}
P = 1 << 20  # an aligned address

ROPE = dict(qkv=P, ldq=768, q_out=P, ldqo=768, M=3, Hq=4, Hkv=1, D=128, cs=P, cs_rows=50, cs_f32=0, rot=128, interleaved=0,
            seq=P, pos=P, kp=P, vp=P, page_stride=2048, pages=9, page=16, table=P, ldt=4, W=4, B=3, stream=None)
ATTN = dict(q=P, ldq=512, kp=P, vp=P, page_stride=2048, pages=9, page=16, table=P, ldt=4, W=4, start=None, pos=P, out=P,
            ldo=512, lse=None, M=3, B=3, Hq=4, Hkv=1, D=128, work=P, work_bytes=1 << 30, stream=None)
SHARED = {k: v for k, v in ATTN.items() if k not in ("start", "M")} | dict(shared=16)

CACHE = [dict(D=96), dict(D=0), dict(page=4), dict(page=12), dict(page=0), dict(page=-16), dict(Hkv=0), dict(Hkv=-1), dict(pages=0),
         dict(W=0), dict(ldt=3), dict(W=1 << 28, ldt=1 << 28), dict(page_stride=2040), dict(page_stride=2052), dict(page_stride=-2048),
         dict(kp=None), dict(vp=None), dict(table=None), dict(kp=P + 8), dict(vp=P + 2), dict(table=P + 2), dict(B=-1),
         dict(page=1 << 28, W=2)]
BAD = {
    "hi_rope_cache_paged": (ROPE, CACHE + [
        dict(M=-1), dict(Hq=0), dict(rot=-2), dict(rot=3), dict(rot=130), dict(cs_rows=0), dict(seq=None, M=4), dict(qkv=None),
        dict(q_out=None), dict(cs=None), dict(pos=None), dict(ldq=767), dict(ldqo=511), dict(qkv=P + 1), dict(cs=P + 2),
        dict(cs=P + 4, cs_f32=1), dict(pos=P + 1), dict(seq=P + 2)]),
    "hi_attn_paged": (ATTN, CACHE + [
        dict(M=-1), dict(M=4), dict(M=2), dict(Hq=0), dict(Hq=3, Hkv=2), dict(Hq=17, ldq=2176, ldo=2176), dict(q=None), dict(q=P + 8),
        dict(ldq=511), dict(ldq=516), dict(pos=None), dict(pos=P + 2), dict(out=None), dict(out=P + 4), dict(ldo=510), dict(ldo=508),
        dict(lse=P + 2), dict(start=P + 2), dict(M=1 << 26, B=1 << 26), dict(start=P, M=1 << 26)]),
    "hi_attn_shared": (SHARED, CACHE + [
        dict(shared=-16), dict(shared=8), dict(shared=80), dict(Hq=0), dict(Hq=17, ldq=2176, ldo=2176), dict(q=None), dict(q=P + 8),
        dict(ldq=516), dict(pos=None), dict(out=None), dict(out=P + 4), dict(ldo=510), dict(lse=P + 1), dict(B=1 << 26)]),
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


@pytest.mark.parametrize("name", ["hi_attn_paged", "hi_rope_cache_paged"])
def test_no_rows_is_no_call(lib, name):
    """No rows: 0 without a launch, also where there is no GPU."""
    base = BAD[name][0] | (dict(M=0, B=0) if name == "hi_attn_paged" else dict(M=0))
    fn = getattr(lib, name)
    fn.argtypes = [_CTYPE[a] for a in parse_abi(ABI)[name][1]]
    assert fn(*(base[a] for a in NAMES[name])) == 0


def test_work_bytes_of_bad_sizes(lib):
    lib.hi_attn_paged_work_bytes.restype = lib.hi_attn_shared_work_bytes.restype = ctypes.c_size_t
    for M, B, Hq, Hkv, D in [(-1, 1, 4, 1, 128), (1, -1, 4, 1, 128), (1, 1, 0, 1, 128), (1, 1, 4, 0, 128), (1, 1, 5, 2, 128),
                             (1, 1, 17, 1, 128), (1, 1, 4, 1, 96), (1 << 26, 1, 4, 1, 128)]:
        assert lib.hi_attn_paged_work_bytes(M, B, Hq, Hkv, D, 1) == 0
        assert lib.hi_attn_paged_work_bytes(M, B, Hq, Hkv, D, 0) == 0
        if M == B:
            assert lib.hi_attn_shared_work_bytes(B, Hq, Hkv, D) == 0
