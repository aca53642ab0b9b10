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


SIZES = [(32, 8, 128), (12, 2, 128), (32, 4, 64), (16, 1, 128), (7, 7, 64), (80, 80, 64), (300, 300, 64)]  # Hq, Hkv, D


@pytest.mark.parametrize("Hq,Hkv,D", SIZES)
def test_work_of_the_largest_batch(hi, Hq, Hkv, D):  # noqa: F811
    """A buffer for the largest batch is large enough for every smaller one, of either form."""
    r, need, shared = rng(310 + Hq), hi.lib.hi_attn_paged_work_bytes, hi.lib.hi_attn_shared_work_bytes
    for top_rows, top_seqs in [(70, 40), (2048, 8), (2048, 256), (600, 600), (4096, 4096), (3, 900), (1, 1), (9000, 1)]:
        most = hi.lib.hi_attn_paged_work_bytes_max(top_rows, top_seqs, Hq, Hkv, D, 1)
        step = hi.lib.hi_attn_paged_work_bytes_max(top_seqs, top_seqs, Hq, Hkv, D, 0)
        joint = hi.lib.hi_attn_shared_work_bytes_max(top_seqs, Hq, Hkv, D)
        sizes = [(top_rows, top_seqs)] + [(int(r.integers(1, top_rows + 1)), int(r.integers(1, top_seqs + 1))) for _ in range(2000)]
        sizes += [(m, b) for b in (1, 2, 3, top_seqs) for m in range(1, top_rows + 1)]
        sizes += [(m, b) for b in range(1, top_seqs + 1) for m in (b, 2 * b, 16 * b * Hkv // Hq, 32 * b * Hkv // Hq) if 1 <= m <= top_rows]
        for m, b in sizes:
            if b <= top_seqs:
                assert need(m, b, Hq, Hkv, D, 1) <= most, (m, b)
        for b in range(1, top_seqs + 1):
            assert need(b, b, Hq, Hkv, D, 0) <= step and shared(b, Hq, Hkv, D) <= joint, b
            assert b > top_rows or need(b, b, Hq, Hkv, D, 0) <= most, b


def test_one_work_buffer_for_smaller_batches(hi):  # noqa: F811
    """A server's buffers, made once for its largest batch, in calls of fewer rows and sequences: taken, with the same bits as a
    buffer of the call's own."""
    def same(a, b):  # (rows behind the cached positions are NaN)
        return torch.equal(a.view(torch.int16), b.view(torch.int16))

    Hq, Hkv, D, page = 32, 8, 128, 16
    lens = [int(n) for n in rng(320).integers(1, 900, 600)]
    c = Cache(321, [900] * 24, Hkv, D, page)
    k, v, rows = c.cuda()
    table = rows[torch.arange(600, device="cuda") % 24].contiguous()
    pos = dev(np.array(lens, np.int32) - 1)
    q = dev(rng(322).standard_normal((2048, Hq * D)).astype(np.float16))
    works = {"ragged": hi.attn_paged_work(2048, 600, Hq, Hkv, D, ragged=True), "step": hi.attn_paged_work(600, 600, Hq, Hkv, D),
             "shared": hi.attn_shared_work(600, Hq, Hkv, D)}
    for B in (600, 513, 512, 511, 64, 8, 1):
        at = q[:B], k, v, table[:B], pos[:B]
        want = hi.attn_paged(*at, Hq, Hkv)
        assert same(hi.attn_paged(*at, Hq, Hkv, work=works["step"]), want)
        assert same(hi.attn_paged(*at, Hq, Hkv, work=works["ragged"]), want)
        common = table[:1].expand(B, -1).contiguous()
        want = hi.attn_shared(q[:B], k, v, common, pos[:B], 640, Hq, Hkv)
        assert same(hi.attn_shared(q[:B], k, v, common, pos[:B], 640, Hq, Hkv, work=works["shared"]), want)
        for M in (2048, 2016, 1000, 7 * B, B):
            if M < B or M > 2048:
                continue
            start = torch.linspace(0, M, B + 1).int().cuda()
            ends = pos[:B].clamp(max=600)
            want = hi.attn_paged(q[:M], k, v, table[:B], ends, Hq, Hkv, start=start)
            assert same(hi.attn_paged(q[:M], k, v, table[:B], ends, Hq, Hkv, start=start, work=works["ragged"]), want)
    for w in works.values():
        assert (w[:hi.ATTN_COUNTER_BYTES] == 0).all()


@pytest.mark.parametrize("D,G,Hkv", [(128, 4, 8), (64, 8, 4), (128, 6, 2)], ids=["D128", "D64", "G6"])
@pytest.mark.parametrize("rows,before", [([32], [1000]), ([100], [900]), ([5] * 8, [700, 64, 0, 1500, 31, 2, 900, 333]),
                                         ([1, 300, 0, 40], [900, 0, 5, 1200])], ids=["32", "100", "8x5", "mixed"])
@pytest.mark.parametrize("times", [1, 8, 32])
def test_runs_in_wide_tables(hi, D, G, Hkv, rows, before, times):  # noqa: F811
    """A table allocated for the longest context there may be: entries behind a sequence's pages are never followed, whichever
    kernel the width selects."""
    Hq, page, M = Hkv * G, 16, sum(rows)
    lens = [p + n for p, n in zip(before, rows)]
    need = max(-(-n // page) for n in lens)
    c = Cache(330 + M, lens, Hkv, D, page, width=need * times, unused=2**31 - 1)
    q = rng(331).standard_normal((M, Hq * D)).astype(np.float16)
    k, v, table = c.cuda()
    lse = torch.empty(Hq, M, device="cuda")
    got = hi.attn_paged(dev(q), k, v, table, dev(np.array(before, np.int32)), Hq, Hkv,
                        start=dev(np.cumsum([0] + rows).astype(np.int32)), lse=lse)
    want = attend(c, [(b, p + t) for b, (p, n) in enumerate(zip(before, rows)) for t in range(n)], q, Hq)
    compare("runs", host(got), want)
    compare_lse("runs", host(lse), want)


@pytest.mark.parametrize("D,G,Hkv", [(128, 4, 8), (64, 8, 4)], ids=["D128", "D64"])
@pytest.mark.parametrize("shared", [0, 256, 4096])
@pytest.mark.parametrize("times", [1, 8, 32])
def test_steps_in_wide_tables(hi, D, G, Hkv, shared, times):  # noqa: F811
    """A decode step without a prefix, with one that is read again, and with one whose own keys share its launch."""
    B, Hq, page = 24, Hkv * G, 16
    lens = [shared + 1 + 29 * b for b in range(B)]
    need = -(-max(lens) // page)
    c = Cache(340 + shared, lens, Hkv, D, page, shared=shared, width=need * times, unused=-7)
    q = rng(341).standard_normal((B, Hq * D)).astype(np.float16)
    k, v, table = c.cuda()
    pos = dev(np.array(lens, np.int32) - 1)
    want = attend(c, [(b, n - 1) for b, n in enumerate(lens)], q, Hq)
    compare("step", host(hi.attn_paged(dev(q), k, v, table, pos, Hq, Hkv)), want)
    compare("shared", host(hi.attn_shared(dev(q), k, v, table, pos, shared, Hq, Hkv)), want)


@pytest.mark.parametrize("form", ["shared", "step", "runs"])
def test_most_sequences(hi, form):  # noqa: F811
    """As many sequences as a call takes (65535; 30000 runs), with parts beyond 2 GiB: rows from all over the batch are right."""
    D, G, Hkv, page, B = 128, 8, 8, 16, 30000 if form == "runs" else 65535
    Hq, shared = Hkv * G, 16
    c = Cache(350, [48] * 40, Hkv, D, page, shared=shared)
    k, v, rows = c.cuda()
    of = torch.arange(B, device="cuda") % 40
    table = rows[of].contiguous()
    pos = (torch.arange(B, device="cuda") % 37 + 10).int()
    q = torch.randn(B, Hq * D, device="cuda", dtype=torch.float16, generator=torch.Generator("cuda").manual_seed(351))
    if form == "shared":
        got = hi.attn_shared(q, k, v, table, pos, shared, Hq, Hkv)
    else:
        start = torch.arange(B + 1, dtype=torch.int32, device="cuda") if form == "runs" else None
        got = hi.attn_paged(q, k, v, table, pos, Hq, Hkv, start=start)
    some = [0, 1, 39, 40, 4095, 4096, 16383, 29999] + ([] if form == "runs" else [32768, 50001, 65534])
    want = attend(c, [(b % 40, b % 37 + 10) for b in some], host(q[some]), Hq)
    compare(form, host(got[some]), want)
