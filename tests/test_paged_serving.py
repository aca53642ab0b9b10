"""GPU tests of the paged cache's attention where a server takes it beyond one call's own sizes: joins of many splits,
contexts of a million keys, tables and work buffers made for the largest batch, memory that overlaps. Cache, plain
attention in float64 and tolerances are those of test_paged.py."""
import numpy as np
import pytest
import torch

from tests._util import gpu, host, rng
from tests.test_paged import Cache, attend, compare, compare_lse, dev, hi  # noqa: F401  (hi is a fixture)

pytestmark = gpu


@pytest.mark.parametrize("Hkv,G,n,p0", [(8, 4, 36, 60000), (8, 4, 16, 40000), (2, 6, 25, 70001), (1, 16, 10, 150000)])
@pytest.mark.parametrize("D", [64, 128])
def test_joins_of_joined_parts(hi, D, Hkv, G, n, p0):  # noqa: F811
    """More than 8 splits of tiles with one or two row groups: several waves of a group read the parts that one of them then
    replaces by the joined one. Every call gives the same bits, and they are right."""
    Hq = Hkv * G
    c = Cache(300 + G, [p0 + n], Hkv, D, 64)
    q = rng(301).standard_normal((n, Hq * D)).astype(np.float16)
    k, v, table = c.cuda()
    qd, start, pos = dev(q), dev(np.array([0, n], np.int32)), dev(np.array([p0], np.int32))
    work = hi.attn_paged_work(n, 1, Hq, Hkv, D, ragged=True)
    lse = torch.empty(Hq, n, device="cuda")
    first = hi.attn_paged(qd, k, v, table, pos, Hq, Hkv, start=start, work=work, lse=lse)
    some = [0, n // 2, n - 1]
    want = attend(c, [(0, p0 + t) for t in some], q[some], Hq)
    compare("joins", host(first)[some], want)
    compare_lse("joins", host(lse)[:, some], want)
    for _ in range(25):
        again = hi.attn_paged(qd, k, v, table, pos, Hq, Hkv, start=start, work=work)
        assert torch.equal(again.view(torch.int16), first.view(torch.int16))
    assert (work[:hi.ATTN_COUNTER_BYTES] == 0).all()


@pytest.mark.parametrize("B,Hq,Hkv,D", [(65535, 64, 8, 128), (65535, 32, 8, 128), (4096, 300, 300, 64), (30000, 48, 8, 128)])
def test_work_beyond_2_gib(hi, B, Hq, Hkv, D):  # noqa: F811
    """Own parts of every row and the prefix's parts, of at least a split each, have their place however many rows there are."""
    part = 4 * (D + 2)
    assert hi.lib.hi_attn_shared_work_bytes(B, Hq, Hkv, D) >= hi.ATTN_COUNTER_BYTES + 2 * B * Hq * part
    assert hi.lib.hi_attn_paged_work_bytes(B, B, Hq, Hkv, D, 0) >= hi.ATTN_COUNTER_BYTES + B * Hq * part
