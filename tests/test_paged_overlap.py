"""Which memory the paged cache's calls may write in place (hipinfer_amd/csrc/row_overlap.h), on the CPU: the rule, compiled for
the host, against every byte of small cases, and the C entry points' refusals. Pointers here are numbers that are never followed."""
import ctypes
import os
import random
import subprocess

import pytest

from hipinfer_amd.hipinfer import ABI, LIBRARY_PATH, _CTYPE, parse_abi
from tests.test_paged_abi import ATTN, NAMES, P, ROPE, SHARED

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "hipinfer_amd", "csrc")
SOURCE = """
#include "row_overlap.h"
extern "C" int allowed(long long x, long long lx, long long wx, long long y, long long ly, long long wy, int M) {
  return in_place_or_apart((const void*)x, lx, wx, (const void*)y, ly, wy, M);
}
"""


@pytest.fixture(scope="module")
def allowed(tmp_path_factory):
    d = tmp_path_factory.mktemp("overlap")
    (d / "overlap.cpp").write_text(SOURCE)
    subprocess.run(["g++", "-O1", "-std=c++17", "-shared", "-fPIC", "-fsanitize=undefined", "-fno-sanitize-recover=undefined",
                    f"-I{CSRC}", "-o", str(d / "overlap.so"), str(d / "overlap.cpp")], check=True)
    fn = ctypes.CDLL(str(d / "overlap.so")).allowed
    fn.argtypes = [ctypes.c_longlong] * 6 + [ctypes.c_int]
    return fn


def test_against_every_byte(allowed):
    r = random.Random(0)
    seen = [0, 0]
    for _ in range(20000):
        M = r.randint(1, 5)
        wx, wy = r.randint(1, 9), r.randint(1, 9)
        lx = wx + r.choice([0, 0, 3, 12])
        ly = r.choice([lx, wy + r.choice([0, 2, 9, 25])])
        if ly < wy:
            continue
        x, y = 100, 100 + r.choice([0, r.randint(-60, 60), r.randint(-12, 12)])
        cover = [{a + i * s + j for i in range(M) for j in range(w)} for a, s, w in ((x, lx, wx), (y, ly, wy))]
        want = not cover[0] & cover[1] or (x == y and (lx == ly or M == 1))
        assert allowed(x, lx, wx, y, ly, wy, M) == want, (x, lx, wx, y, ly, wy, M)
        seen[want] += 1
    assert min(seen) > 3000


@pytest.mark.parametrize("name,base,change", [
    ("hi_rope_cache_paged", ROPE, dict(ldqo=512)),                  # the same first row, other rows over rows still to be read
    ("hi_rope_cache_paged", ROPE, dict(q_out=P + 256)),             # a head further on
    ("hi_rope_cache_paged", ROPE, dict(qkv=P + 2 * 768, q_out=P)),  # a row before
    ("hi_attn_paged", ATTN, dict(ldo=640)),
    ("hi_attn_paged", ATTN, dict(ldo=640, start=P, M=7)),
    ("hi_attn_paged", ATTN, dict(out=P + 1024)),
    ("hi_attn_shared", SHARED, dict(ldq=640)),
    ("hi_attn_shared", SHARED, dict(out=P + 256)),
], ids=["rope-stride", "rope-head", "rope-row", "attn-stride", "runs-stride", "attn-row", "shared-stride", "shared-head"])
def test_refused(name, base, change, capfd):
    fn = getattr(ctypes.CDLL(LIBRARY_PATH), name)
    fn.argtypes = [_CTYPE[a] for a in parse_abi(ABI)[name][1]]
    args = base | change
    assert fn(*(args[a] for a in NAMES[name])) == -1
    assert "apart from it" in capfd.readouterr().err
