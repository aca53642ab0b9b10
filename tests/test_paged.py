"""GPU parity of serving from a paged key/value cache (rope_cache_paged, attn_paged, attn_shared) against plain
implementations in float64 on the CPU, at the sizes, masks and layouts where paging goes wrong: pages that end inside a
tile, rows without keys, NaN in every cache row that no position holds, table entries that are no page, strided pages, K
and V in one allocation, ragged runs of rows, padding rows, captured graphs and other streams.

Tolerances. Logits are exact fp16 products summed in fp32, so a weight w = p / l is off by its rounding to fp16 for P.V
(2^-11 of it, or half a step of 2^-24 below 2^-14, with l >= 1) and by the fp32 sums (2^-20 at these lengths); the result is
rounded to fp16 once (2^-11 of it):
    |out - ref| <= 2^-11 (1 + 2^-3) (sum w |v| + |ref|) + 2^-25 sum |v| + 2^-25.
A rotated pair is off by one rounding of fp16 and two of fp32: 2^-11 (1 + 2^-8) of |x| + |y|, or 2^-25 among subnormals.
"""
import numpy as np
import pytest
import torch

from tests._util import bits, gpu, host, rng

pytestmark = gpu


@pytest.fixture(scope="module")
def hi():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    from hipinfer_amd import hipinfer
    return hipinfer


# ------------------------------------------------------------------ a paged cache and its plain attention
class Cache:
    """Sequences of `lens` cached positions on pages in random order. Every cache row that holds no position is NaN in K
    and inf in V, unused table entries are `unused`. layout: "packed", "strided" (a gap behind every page) or "joint" (K and V
    in one allocation)."""

    def __init__(self, seed, lens, Hkv, D, page, layout="packed", unused=-1, shared=0, spare=2, sd=1.0, width=None):
        r = rng(seed)
        self.lens, self.Hkv, self.D, self.page, self.shared = list(lens), Hkv, D, page, shared
        common = shared // page
        own = [max(0, -(-n // page) - common) for n in lens]
        self.pages = common + sum(own) + spare
        order = r.permutation(self.pages)
        W = max([1, common] + [common + n for n in own]) if width is None else width
        self.table = np.full((len(lens), W), unused, np.int32)
        at = common
        for b, n in enumerate(own):
            self.table[b, :common] = order[:common]
            self.table[b, common:common + n] = order[at:at + n]
            at += n
        self.k = np.full((self.pages, Hkv, page, D), np.nan, np.float16)
        self.v = np.full((self.pages, Hkv, page, D), np.inf, np.float16)
        for b, n in enumerate(lens):
            first, last = (0, max(n, shared)) if b == 0 else (shared, n)
            for p in range(first, last, page):
                m = min(page, last - p)
                pg = self.table[b, p // page]
                self.k[pg, :, :m] = r.standard_normal((Hkv, m, D)) * sd
                self.v[pg, :, :m] = r.standard_normal((Hkv, m, D))
        self.layout = layout

    def cuda(self):
        k, v = torch.from_numpy(self.k).cuda(), torch.from_numpy(self.v).cuda()
        n = self.Hkv * self.page * self.D
        if self.layout == "joint":
            kv = torch.stack([k, v], 1).contiguous()
            k, v = kv[:, 0], kv[:, 1]
        elif self.layout == "strided":
            def spread(t):
                wide = torch.full((self.pages, n + 64), float("nan"), dtype=torch.float16, device="cuda")
                wide[:, :n] = t.reshape(self.pages, n)
                return wide[:, :n].unflatten(1, (self.Hkv, self.page, self.D))
            k, v = spread(k), spread(v)
        return k, v, torch.from_numpy(self.table).cuda()

    def seen(self, b, n):
        """(K, V) [Hkv, m, D] float64 of the keys 0 .. n - 1 of sequence b that lie on pages."""
        n = min(n, self.table.shape[1] * self.page)
        p = np.arange(max(n, 0))
        pg = self.table[b, p // self.page]
        ok = (pg >= 0) & (pg < self.pages)
        p, pg = p[ok], pg[ok]
        return (torch.from_numpy(t[pg, :, p % self.page].astype(np.float64)).transpose(0, 1).contiguous()
                for t in (self.k, self.v))


def attend(cache, rows, q, Hq):
    """rows: (sequence, position) of each row of q [M, Hq * D]; (out, tolerance, lse) in float64."""
    Hkv, D, M = cache.Hkv, cache.D, q.shape[0]
    out, tol = np.zeros((M, Hq * D)), np.zeros((M, Hq * D))
    lse = np.full((Hq, M), -np.inf)
    for m, (b, p) in enumerate(rows):
        K, V = cache.seen(b, p + 1)
        if K.shape[1] == 0:
            continue
        qm = torch.from_numpy(q[m].astype(np.float64)).view(Hkv, Hq // Hkv, D)
        x = (qm @ K.transpose(1, 2).contiguous()) / np.sqrt(D)
        total = torch.logsumexp(x, -1)
        w = torch.exp(x - total[..., None])
        o, wv, sv = w @ V, w @ V.abs(), V.abs().sum(1)[:, None].expand(-1, Hq // Hkv, -1)
        out[m] = o.reshape(-1).numpy()
        tol[m] = (2**-11 * 1.125 * (wv + o.abs()) + 2**-25 * sv + 2**-25).reshape(-1).numpy()
        lse[:, m] = (total / np.log(2.0)).reshape(-1).numpy()
    return out, tol, lse


def compare(name, got, want):
    out, tol, _ = want
    got = got.astype(np.float64)
    assert got.shape == out.shape
    bad = ~(np.abs(got - out) <= tol)
    assert not bad.any(), f"{name}: {bad.sum()} of {bad.size} off, first {np.argwhere(bad)[0]}, " \
                          f"{got[tuple(np.argwhere(bad)[0])]} for {out[tuple(np.argwhere(bad)[0])]}"


def compare_lse(name, got, want):
    """fp32 sums of at most a few thousand exp2 (each within 2^-21) and products: 2^-16 absolute on a log2 below 2^5."""
    lse = want[2]
    assert np.array_equal(np.isneginf(got), np.isneginf(lse)), name
    fine = np.isfinite(lse)
    assert (np.abs(got[fine] - lse[fine]) <= 2**-16).all(), f"{name}: lse off by {np.abs(got[fine] - lse[fine]).max()}"


def dev(a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


HEADS = [(64, 8, 4), (128, 4, 8), (128, 6, 2), (64, 1, 3), (128, 16, 1), (64, 5, 2), (128, 1, 2)]  # D, Hq / Hkv, Hkv
IDS = [f"D{d}-G{g}-Hkv{h}" for d, g, h in HEADS]


# ------------------------------------------------------------------ one row per sequence
@pytest.mark.parametrize("D,G,Hkv", HEADS, ids=IDS)
@pytest.mark.parametrize("page", [8, 16, 64, 256])
def test_decode(hi, D, G, Hkv, page):
    """Lengths around tiles, pages and split steps in one batch, an empty row among them."""
    lens = [1, 0, 7, 8, 9, 31, 32, 33, 64, 127, 129, 255, 257, 500, 777, 1030]
    c = Cache(10 + D + G + page, lens, Hkv, D, page, layout=["packed", "joint", "strided"][page % 3])
    q = rng(11 + page).standard_normal((len(lens), Hkv * G * D)).astype(np.float16)
    k, v, table = c.cuda()
    pos = dev(np.array(lens, np.int32) - 1)
    lse = torch.empty(Hkv * G, len(lens), device="cuda")
    got = hi.attn_paged(dev(q), k, v, table, pos, Hkv * G, Hkv, lse=lse)
    want = attend(c, [(b, n - 1) for b, n in enumerate(lens)], q, Hkv * G)
    compare("decode", host(got), want)
    compare_lse("decode", host(lse), want)


@pytest.mark.parametrize("B,lens", [(1, [1]), (1, [40]), (1, [2500]), (1, [9000]), (2, [6000, 17]), (70, [200]),
                                    (40, [300, 1, 1200]), (130, [65, 513])], ids=str)
@pytest.mark.parametrize("D,G,Hkv", [(128, 4, 8), (64, 8, 4)], ids=["D128", "D64"])
def test_decode_batches(hi, D, G, Hkv, B, lens):
    """From one sequence split over the GPU to more sequences than CUs."""
    lens = [lens[b % len(lens)] for b in range(B)]
    c = Cache(20 + B, lens, Hkv, D, 16)
    q = rng(21 + B).standard_normal((B, Hkv * G * D)).astype(np.float16)
    k, v, table = c.cuda()
    work = hi.attn_paged_work(B, B, Hkv * G, Hkv, D)
    pos = dev(np.array(lens, np.int32) - 1)
    got = [host(hi.attn_paged(dev(q), k, v, table, pos, Hkv * G, Hkv, work=work)) for _ in range(2)]
    compare("decode", got[0], attend(c, [(b, n - 1) for b, n in enumerate(lens)], q, Hkv * G))
    assert np.array_equal(bits(got[0]), bits(got[1])), "a kept work buffer"


@pytest.mark.parametrize("bad", [-1, -2**31, 2**31 - 1, 10**6])
def test_decode_no_pages(hi, bad):
    """Table entries that are no page leave their keys out, wherever they stand; a sequence of such only has no key."""
    D, G, Hkv, page = 128, 4, 2, 16
    lens = [700, 64, 16, 400]
    c = Cache(30, lens, Hkv, D, page)
    c.table[0, 3] = c.table[0, 20] = c.table[0, 43] = bad
    c.table[1, 0] = c.table[2, 0] = bad
    c.table[3, 1:] = bad
    q = rng(31).standard_normal((4, Hkv * G * D)).astype(np.float16)
    k, v, table = c.cuda()
    pos = dev(np.array(lens, np.int32) - 1)
    got = host(hi.attn_paged(dev(q), k, v, table, pos, Hkv * G, Hkv))
    want = attend(c, [(b, n - 1) for b, n in enumerate(lens)], q, Hkv * G)
    compare("decode", got, want)
    assert (got[2] == 0).all()
    start = dev(np.array([0, 1, 2, 3, 4], np.int32))
    compare("ragged", host(hi.attn_paged(dev(q), k, v, table, pos, Hkv * G, Hkv, start=start)), want)


def test_positions_outside(hi):
    """A position behind the table sees the keys the table holds; a negative one none, however negative."""
    D, G, Hkv, page = 64, 4, 2, 16
    c = Cache(40, [64, 64, 64, 64], Hkv, D, page)
    q = rng(41).standard_normal((4, Hkv * G * D)).astype(np.float16)
    k, v, table = c.cuda()
    pos = np.array([2**31 - 1, -1, -2**31, 64], np.int32)
    want = attend(c, [(0, 63), (1, -1), (2, -1), (3, 63)], q, Hkv * G)
    compare("decode", host(hi.attn_paged(dev(q), k, v, table, dev(pos), Hkv * G, Hkv)), want)
    start = dev(np.arange(5, dtype=np.int32))
    compare("ragged", host(hi.attn_paged(dev(q), k, v, table, dev(pos), Hkv * G, Hkv, start=start)), want)
    compare("shared", host(hi.attn_shared(dev(q), k, v, table, dev(pos), 0, Hkv * G, Hkv)), want)


@pytest.mark.parametrize("D", [64, 128])
def test_infinite_logits(hi, D):
    """Keys whose logits are -inf have weight 0, also where they come first; large finite logits do not overflow."""
    G, Hkv, page, n = 4, 2, 16, 600
    c = Cache(50, [n, n], Hkv, D, page, sd=8.0)
    q = rng(51).standard_normal((2, Hkv * G * D)).astype(np.float16) * np.float16(8)
    q[0] = np.abs(q[0])
    for p in list(range(0, 200)) + [599]:
        c.k[c.table[0, p // page], :, p % page, 0] = -np.inf
    k, v, table = c.cuda()
    pos = dev(np.array([n - 1, n - 1], np.int32))
    ref = Cache(50, [n, n], Hkv, D, page, sd=8.0)
    ref.k = np.where(np.isneginf(c.k), np.float16(-60000.0), c.k)
    ref.table = c.table
    q0 = q.copy()
    q0[0].reshape(-1, D)[:, 0] = np.float16(60000.0)  # the same keys' weights vanish
    out = host(hi.attn_paged(dev(q), k, v, table, pos, Hkv * G, Hkv))
    keep = [p for p in range(200, 599)]
    pg, at = c.table[0, np.array(keep) // page], np.array(keep) % page
    K = torch.from_numpy(c.k[pg, :, at].astype(np.float64)).transpose(0, 1).contiguous()
    V = torch.from_numpy(c.v[pg, :, at].astype(np.float64)).transpose(0, 1).contiguous()
    x = torch.from_numpy(q[0].astype(np.float64)).view(Hkv, G, D) @ K.transpose(1, 2).contiguous() / np.sqrt(D)
    w = torch.softmax(x, -1)
    o = w @ V
    tol = 2**-11 * 1.125 * (w @ V.abs() + o.abs()) + 2**-25 * V.abs().sum(1)[:, None] + 2**-25
    # logits up to 2^12: fp32 sums of D products are off by 2^-24 D of the sum of their magnitudes, an exponent of 2^-6
    tol = tol + 2**-6 * (w @ V.abs())
    assert (np.abs(out[0].astype(np.float64) - o.reshape(-1).numpy()) <= tol.reshape(-1).numpy()).all()
    assert np.isfinite(out).all()


def same_where_finite(name, got, want):
    """Within the tolerance where the result is finite, the same infinity where it is one, NaN where it is."""
    out, tol, _ = want
    got = got.astype(np.float64)
    assert np.array_equal(np.isnan(got), np.isnan(out)), f"{name}: NaN in {np.argwhere(np.isnan(got) != np.isnan(out))[:4]}"
    big = np.isinf(out)
    assert np.array_equal(got[big], out[big]), name
    fine = np.isfinite(out)
    assert (np.abs(got[fine] - out[fine]) <= tol[fine]).all(), name


@pytest.mark.parametrize("D,G,Hkv", HEADS, ids=IDS)
@pytest.mark.parametrize("form", ["ragged", "shared"])
def test_later_infinities(hi, D, G, Hkv, form):
    """Infinities and NaN in the V rows, and in the K rows, of positions that a row does not see do not reach it; in V rows
    that it sees they give what the sum gives."""
    Hq, page, n, p0 = Hkv * G, 16, 150, 90
    total = p0 + n if form == "ragged" else 8192
    c = Cache(55 + G, [total], Hkv, D, page)
    r = rng(56)
    spots = r.choice(np.arange(p0 + 20, p0 + n - 5), 9, replace=False)
    for i, p in enumerate(sorted(spots)):
        c.v[c.table[0, p // page], :, p % page, (7 * i) % D] = [np.inf, -np.inf, np.nan][i % 3]
    c.v[c.table[0, max(spots) // page], :, max(spots) % page, 7 * 2 % D] = np.inf
    last = p0 + n - 3
    c.k[c.table[0, last // page], :, last % page, :] = np.inf
    if form == "ragged":
        q = r.standard_normal((n, Hq * D)).astype(np.float16)
        k, v, table = c.cuda()
        got = host(hi.attn_paged(dev(q), k, v, table, dev(np.array([p0], np.int32)), Hq, Hkv,
                                 start=dev(np.array([0, n], np.int32))))
        at = [(0, p0 + t) for t in range(n - 3)]
        same_where_finite("ragged", got[:n - 3], attend(c, at, q[:n - 3], Hq))
        assert np.isnan(got[n - 3:]).all(), "rows that see the infinite key"
        return
    B = 60  # sequences whose last position lies in the shared part, among them some that see each of the spots
    at = [(0, int(p)) for p in r.integers(p0, last, B)]
    c.table = np.repeat(c.table, B, 0)
    q = r.standard_normal((B, Hq * D)).astype(np.float16)
    k, v, table = c.cuda()
    got = host(hi.attn_shared(dev(q), k, v, table, dev(np.array([p for _, p in at], np.int32)), total, Hq, Hkv))
    same_where_finite("shared", got, attend(c, at, q, Hq))


# ------------------------------------------------------------------ ragged batches
RAGGED = [  # rows of each sequence, cached positions before them
    ([5, 5, 5], [100, 0, 1000]),
    ([1], [0]), ([3], [0]), ([130], [0]), ([257], [70]), ([64], [2100]), ([2], [5000]),
    ([0, 7, 0, 0, 40, 1, 0], [5, 9, 0, 3, 300, 600, 20]),
    ([33, 1, 1, 128, 1, 90], [31, 700, 0, 128, 1500, 1]),
]


@pytest.mark.parametrize("D,G,Hkv", HEADS, ids=IDS)
@pytest.mark.parametrize("rows,before", RAGGED, ids=[f"rows{'_'.join(map(str, r))}" for r, _ in RAGGED])
def test_ragged(hi, D, G, Hkv, rows, before):
    page = [8, 16, 32, 128][(D + G + len(rows)) % 4]
    lens = [p + n for p, n in zip(before, rows)]
    c = Cache(60 + G + len(rows), lens, Hkv, D, page, layout=["packed", "joint", "strided"][G % 3])
    M, Hq = sum(rows), Hkv * G
    pad = 3  # rows in front of the first run and behind the last
    start = np.cumsum([pad] + rows).astype(np.int32)
    q = rng(61).standard_normal((M + 2 * pad, Hq * D)).astype(np.float16)
    q[:pad] = q[M + pad:] = np.nan
    k, v, table = c.cuda()
    wide = torch.full((M + 2 * pad, Hq * D + 8), 7.0, dtype=torch.float16, device="cuda")
    lse = torch.full((Hq, M + 2 * pad), 3.0, device="cuda")
    hi.attn_paged(dev(q), k, v, table, dev(np.array(before, np.int32)), Hq, Hkv, start=dev(start),
                  out=wide[:, :Hq * D], lse=lse)
    got = host(wide)
    assert (got[:pad] == 7).all() and (got[M + pad:] == 7).all() and (got[:, Hq * D:] == 7).all(), "rows of no sequence"
    L = host(lse)
    assert (L[:, :pad] == 3).all() and (L[:, M + pad:] == 3).all()
    at = [(b, p + t) for b, (n, p) in enumerate(zip(rows, before)) for t in range(n)]
    want = attend(c, at, q[pad:M + pad], Hq)
    compare("ragged", got[pad:M + pad, :Hq * D], want)
    compare_lse("ragged", L[:, pad:M + pad], want)


FEW = [  # few rows a sequence: one or two blocks of 16 columns, one split and many, tiles that share a sequence
    ([1], [650]), ([2], [4001]), ([1, 1, 2, 1, 3, 1], [5, 700, 33, 3000, 0, 64]), ([1] * 40, [37 * b for b in range(40)]),
    ([4, 0, 1, 0, 3], [1030, 5, 9000, 0, 257]), ([8, 1, 1, 1, 1, 1, 1, 1], [123, 0, 1, 2, 31, 32, 33, 2000]),
    ([2] * 90, [(61 * b) % 1500 for b in range(90)]), ([1] * 600, [b % 97 for b in range(600)]),
]


@pytest.mark.parametrize("D,G,Hkv", HEADS, ids=IDS)
@pytest.mark.parametrize("rows,before", FEW, ids=[f"B{len(r)}-{sum(r)}rows" for r, _ in FEW])
def test_few_rows(hi, D, G, Hkv, rows, before):
    """Runs of few rows, with entries that are no page, unwritten rows behind the last key and a kept work buffer."""
    page = [8, 16, 64][(D + G + len(rows)) % 3]
    c = Cache(200 + G + len(rows), [p + n for p, n in zip(before, rows)], Hkv, D, page, layout=["joint", "strided", "packed"][G % 3])
    for b in range(0, len(rows), 3):
        if before[b] > 3 * page:
            c.table[b, 1] = c.table[b, before[b] // page - 1] = [-1, 2**31 - 1, -2**31][b % 3]
    M, Hq = sum(rows), Hkv * G
    q = rng(201).standard_normal((M, Hq * D)).astype(np.float16)
    k, v, table = c.cuda()
    start, pos = dev(np.cumsum([0] + rows).astype(np.int32)), dev(np.array(before, np.int32))
    lse = torch.empty(Hq, M, device="cuda")
    work = hi.attn_paged_work(M, len(rows), Hq, Hkv, D, ragged=True)
    got = [host(hi.attn_paged(dev(q), k, v, table, pos, Hq, Hkv, start=start, lse=lse, work=work)) for _ in range(2)]
    want = attend(c, [(b, p + t) for b, (p, n) in enumerate(zip(before, rows)) for t in range(n)], q, Hq)
    compare("few rows", got[0], want)
    compare_lse("few rows", host(lse), want)
    assert np.array_equal(bits(got[0]), bits(got[1])), "a kept work buffer"
    assert (host(work)[:hi.ATTN_COUNTER_BYTES] == 0).all()


@pytest.mark.parametrize("D,G,Hkv", HEADS, ids=IDS)
def test_few_rows_infinities(hi, D, G, Hkv):
    """An infinite (and a NaN) V row at each of the positions of a run: only the rows from it on see it."""
    page, B, n, p0 = 16, 40, 2, 611
    for spot in (p0, p0 + 1, 300, 575, 576):
        c = Cache(210 + spot, [p0 + n] * B, Hkv, D, page)
        for b in range(B):
            c.v[c.table[b, spot // page], :, spot % page] = [np.inf, -np.inf, np.nan][b % 3]
        q = rng(211).standard_normal((B * n, Hkv * G * D)).astype(np.float16)
        k, v, table = c.cuda()
        start = dev(np.arange(0, B * n + 1, n).astype(np.int32))
        got = host(hi.attn_paged(dev(q), k, v, table, dev(np.full(B, p0, np.int32)), Hkv * G, Hkv, start=start))
        for t in range(n):
            rows = np.arange(t, B * n, n)
            if p0 + t >= spot:
                assert (~np.isfinite(got[rows])).all(), "rows that see it"
            else:
                compare("rows before it", got[rows], attend(c, [(b, p0 + t) for b in range(B)], q[rows], Hkv * G))


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("rows,before,Hkv,G", [
    ([10] * 20, [(173 * b) % 2600 for b in range(20)], 8, 4),  # tiles of 64 packed rows, some split
    ([16], [40000], 8, 4), ([16], [200001], 1, 4), ([100], [30000], 1, 8), ([40], [60000], 2, 6),  # levels of joins
], ids=["B20", "16-Hkv8", "16-Hkv1", "100-Hkv1", "40-Hkv2"])
def test_row_tiles(hi, D, rows, before, Hkv, G):
    """Runs that are too many, or whose contexts are too long, for the kernel of few rows."""
    page, Hq, M = 16, Hkv * G, sum(rows)
    c = Cache(220 + M + D, [p + n for p, n in zip(before, rows)], Hkv, D, page)
    c.table[-1, 1] = -1
    q = rng(221).standard_normal((M, Hq * D)).astype(np.float16)
    k, v, table = c.cuda()
    start, pos = dev(np.cumsum([0] + rows).astype(np.int32)), dev(np.array(before, np.int32))
    lse = torch.empty(Hq, M, device="cuda")
    work = hi.attn_paged_work(M, len(rows), Hq, Hkv, D, ragged=True)
    got = [host(hi.attn_paged(dev(q), k, v, table, pos, Hq, Hkv, start=start, lse=lse, work=work)) for _ in range(2)]
    at = [(b, p + t) for b, (p, n) in enumerate(zip(before, rows)) for t in range(n)]
    some = list(range(0, M, 1 if M * max(before) < 10**6 else 13)) + [M - 1]
    out, tol, want = attend(c, [at[m] for m in some], q[some], Hq)
    compare("row tiles", got[0][some], (out, tol, want))
    compare_lse("row tiles", host(lse)[:, some], (out, tol, want))
    assert np.array_equal(bits(got[0]), bits(got[1])), "a kept work buffer"
    assert (host(work)[:hi.ATTN_COUNTER_BYTES] == 0).all()


@pytest.mark.parametrize("T,p0,D,G,Hkv", [(700, 0, 64, 8, 4), (1000, 333, 128, 4, 8)])
def test_ragged_one_chunk(hi, T, p0, D, G, Hkv):
    """A prompt chunk over pages is the chunk over a cache slot; the two kernels agree to both their tolerances."""
    Hq = Hkv * G
    c = Cache(70, [p0 + T], Hkv, D, 16)
    q = rng(71).standard_normal((T, Hq * D)).astype(np.float16)
    k, v, table = c.cuda()
    ks, vs = (t[torch.from_numpy(c.table[0]).long().cuda()].transpose(0, 1).reshape(Hkv, -1, D).contiguous() for t in (k, v))
    ks, vs = ks.nan_to_num(), vs.nan_to_num(posinf=0.0)
    slot, slot_lse = hi.flash_prefill_lse(dev(q), ks, vs, T, p0, Hq, Hkv)
    lse = torch.empty(Hq, T, device="cuda")
    got = hi.attn_paged(dev(q), k, v, table, dev(np.array([p0], np.int32)), Hq, Hkv, start=dev(np.array([0, T], np.int32)),
                        lse=lse)
    # each is within 2^-10 1.125 (sum w |v|) of the exact value, and |v| < 2^3
    assert (got.float() - slot.float()).abs().max().item() <= 2 * 2**-10 * 1.125 * 8
    assert (lse - slot_lse).abs().max().item() <= 2**-15
    rows = [0, 1, 63, 64, 127, 128, T // 2, T - 2, T - 1]
    compare("rows", host(got)[rows], attend(c, [(0, p0 + t) for t in rows], q[rows], Hq))


@pytest.mark.parametrize("Hkv,G,n,p0", [(1, 1, 3, 40000), (1, 2, 64, 33000), (2, 4, 1, 60000), (1, 16, 40, 20000), (8, 4, 32, 9000)])
@pytest.mark.parametrize("D", [64, 128])
def test_ragged_many_splits(hi, D, Hkv, G, n, p0):
    """Few rows after a long context: up to a split per CU, joined in more than one level; a short sequence beside."""
    Hq, rows, before = Hkv * G, [n, 2], [p0, 100]
    c = Cache(75 + G, [p + m for p, m in zip(before, rows)], Hkv, D, 64)
    q = rng(76).standard_normal((n + 2, Hq * D)).astype(np.float16)
    k, v, table = c.cuda()
    start, pos = dev(np.array([0, n, n + 2], np.int32)), dev(np.array(before, np.int32))
    work = hi.attn_paged_work(n + 2, 2, Hq, Hkv, D, ragged=True)
    lse = torch.empty(Hq, n + 2, device="cuda")
    got = [host(hi.attn_paged(dev(q), k, v, table, pos, Hq, Hkv, start=start, work=work, lse=lse)) for _ in range(3)]
    at = [(b, p + t) for b, (m, p) in enumerate(zip(rows, before)) for t in range(m)]
    some = sorted({0, n // 2, n - 1, n, n + 1})
    want = attend(c, [at[m] for m in some], q[some], Hq)
    compare("ragged", got[0][some], want)
    compare_lse("ragged", host(lse)[:, some], want)
    for g in got[1:]:
        assert np.array_equal(bits(g), bits(got[0])), "a kept work buffer"
    assert (work[:16384] == 0).all(), "the counters are left at zero"


def test_one_work_buffer_for_all_forms(hi):
    """A buffer made for one form serves the others in turn (where it is large enough), each as with its own."""
    D, G, Hkv, B = 128, 4, 8, 12
    Hq, lens = Hkv * G, [2500 + 31 * b for b in range(B)]
    c = Cache(78, lens, Hkv, D, 16)
    q = dev(rng(79).standard_normal((B, Hq * D)).astype(np.float16))
    k, v, table = c.cuda()
    pos = dev(np.array(lens, np.int32) - 1)
    start = torch.arange(B + 1, dtype=torch.int32, device="cuda")
    sizes = [hi.attn_paged_work(B, B, Hq, Hkv, D), hi.attn_paged_work(B, B, Hq, Hkv, D, ragged=True),
             hi.attn_shared_work(B, Hq, Hkv, D)]
    one = max(sizes, key=lambda w: w.numel())
    one[16384:].fill_(0xff)

    def forms(work):
        yield hi.attn_paged(q, k, v, table, pos, Hq, Hkv, work=work)
        yield hi.attn_paged(q, k, v, table, pos, Hq, Hkv, start=start, work=work)
        yield hi.attn_shared(q, k, v, table, pos, 2048, Hq, Hkv, work=work)
        yield hi.attn_paged(q[:1], k, v, table[:1], pos[:1], Hq, Hkv, work=work)
    for own, shared in zip(forms(None), list(forms(one)) and forms(one)):
        assert torch.equal(own, shared)


def test_ragged_bad_start_large(hi):
    """Runs that overlap and together are more than the rows there are: the call ends, nothing outside the rows is written."""
    D, G, Hkv, M = 64, 2, 2, 700
    c = Cache(92, [900, 900, 900], Hkv, D, 16)
    q = rng(93).standard_normal((M, Hkv * G * D)).astype(np.float16)
    k, v, table = c.cuda()
    wide = torch.full((M + 4, Hkv * G * D), 7.0, dtype=torch.float16, device="cuda")
    for start in ([0, M, 0, M], [M, 0, M, 0], [-9, M + 9, 5, 2**31 - 1]):
        hi.attn_paged(dev(q), k, v, table, dev(np.array([100, 200, 3], np.int32)), Hkv * G, Hkv,
                      start=dev(np.array(start, np.int32)), out=wide[2:M + 2])
        got = host(wide)
        assert (got[:2] == 7).all() and (got[M + 2:] == 7).all()


def test_ragged_many_sequences(hi):
    """More sequences than a wave's lanes, most of one row, some empty, one long."""
    D, G, Hkv, B = 64, 8, 4, 150
    rows = [[1, 0, 1, 9][b % 4] for b in range(B)]
    before = [(37 * b) % 300 for b in range(B)]
    rows[77], before[77] = 70, 2000
    c = Cache(80, [p + n for p, n in zip(before, rows)], Hkv, D, 16)
    M, Hq = sum(rows), Hkv * G
    q = rng(81).standard_normal((M, Hq * D)).astype(np.float16)
    k, v, table = c.cuda()
    start = np.cumsum([0] + rows).astype(np.int32)
    got = hi.attn_paged(dev(q), k, v, table, dev(np.array(before, np.int32)), Hq, Hkv, start=dev(start))
    at = [(b, p + t) for b, (n, p) in enumerate(zip(rows, before)) for t in range(n)]
    compare("ragged", host(got), attend(c, at, q, Hq))


@pytest.mark.parametrize("start", [[0, 3, 1, 6], [0, -5, 4, 6], [0, 2, 100, 200], [6, 4, 2, 0], [-2**31, 2**31 - 1, 0, 6],
                                   [2**31 - 1] * 4], ids=str)
def test_ragged_bad_start(hi, start):
    """A start that decreases or leaves the rows: nothing outside the rows is read or written, and the call ends."""
    D, G, Hkv = 128, 2, 2
    c = Cache(90, [300, 300, 300], Hkv, D, 16)
    q = rng(91).standard_normal((6, Hkv * G * D)).astype(np.float16)
    k, v, table = c.cuda()
    wide = torch.full((10, Hkv * G * D), 7.0, dtype=torch.float16, device="cuda")
    hi.attn_paged(dev(q), k, v, table, dev(np.array([290, 100, 5], np.int32)), Hkv * G, Hkv,
                  start=dev(np.array(start, np.int32)), out=wide[2:8])
    got = host(wide)
    assert (got[:2] == 7).all() and (got[8:] == 7).all()


# ------------------------------------------------------------------ a shared prefix
@pytest.mark.parametrize("D,G,Hkv", HEADS, ids=IDS)
@pytest.mark.parametrize("B,shared,page", [(1, 64, 16), (3, 256, 8), (5, 1024, 64), (33, 384, 128), (9, 0, 16)])
def test_shared(hi, D, G, Hkv, B, shared, page):
    """Own parts from none to several pages; sequences shorter than the prefix, one empty."""
    own = [0, 1, 17, 300, 64, 5, 130]
    lens = [shared + own[b % len(own)] for b in range(B)]
    if B > 4:
        lens[2], lens[3], lens[4] = 0, max(shared // 2 - 3, 0), 1
    c = Cache(100 + B + D, lens, Hkv, D, page, layout=["packed", "joint", "strided"][B % 3], shared=shared)
    for b in range(1, B):  # only row 0's entries count for the prefix
        c.table[b, :shared // page] = c.table[0, :shared // page]
    Hq = Hkv * G
    q = rng(101).standard_normal((B, Hq * D)).astype(np.float16)
    k, v, table = c.cuda()
    only0 = table.clone()
    only0[1:, :shared // page] = -1
    pos = dev(np.array(lens, np.int32) - 1)
    lse = torch.empty(Hq, B, device="cuda")
    work = hi.attn_shared_work(B, Hq, Hkv, D)
    got = [host(hi.attn_shared(dev(q), k, v, t, pos, shared, Hq, Hkv, lse=lse, work=work)) for t in (table, only0)]
    want = attend(c, [(b, n - 1) for b, n in enumerate(lens)], q, Hq)
    compare("shared", got[0], want)
    compare_lse("shared", host(lse), want)
    assert np.array_equal(bits(got[0]), bits(got[1])), "the prefix is table row 0's"
    if shared:  # the same as each sequence by itself
        alone = host(hi.attn_paged(dev(q), k, v, table, pos, Hq, Hkv))
        compare("paged", alone, want)


@pytest.mark.parametrize("D,G,Hkv,B,shared,page", [
    (64, 8, 4, 70, 4096, 64), (64, 8, 4, 8, 24576, 64), (128, 4, 8, 8, 8192, 128), (128, 4, 8, 70, 2048, 16),
    (128, 6, 2, 33, 8192, 32), (64, 1, 3, 70, 8192, 128), (128, 16, 1, 40, 8192, 64), (64, 16, 1, 9, 65536, 256),
    (64, 5, 2, 64, 8192, 8), (128, 1, 2, 100, 4096, 16)])
def test_shared_once(hi, D, G, Hkv, B, shared, page):
    """Batches and prefixes where reading the prefix once is faster than once per sequence: row tiles of both heights, one
    and several, own parts in one block and in several, sequences shorter than the prefix, empty ones."""
    own = [0, 1, 17, 300, 64, 5, 130, 1100]
    lens = [shared + own[b % len(own)] for b in range(B)]
    lens[2], lens[3], lens[4] = 0, shared // 2 - 3, 1
    c = Cache(105 + B + D, lens, Hkv, D, page, layout=["packed", "joint", "strided"][B % 3], shared=shared)
    c.table[5 % B, 0] = -1  # not looked at
    want_table = c.table.copy()
    want_table[:, :shared // page] = c.table[0, :shared // page]
    Hq = Hkv * G
    q = rng(106).standard_normal((B, Hq * D)).astype(np.float16)
    k, v, table = c.cuda()
    lse = torch.empty(Hq, B, device="cuda")
    work = hi.attn_shared_work(B, Hq, Hkv, D)
    pos = dev(np.array(lens, np.int32) - 1)
    got = [host(hi.attn_shared(dev(q), k, v, table, pos, shared, Hq, Hkv, lse=lse, work=work)) for _ in range(2)]
    c.table = want_table
    rows = sorted({0, 1, 2, 3, 4, 5, 6, 7, B // 2, B - 1})
    want = attend(c, [(b, lens[b] - 1) for b in rows], q[rows], Hq)
    compare("shared", got[0][rows], want)
    compare_lse("shared", host(lse)[:, rows], want)
    assert np.array_equal(bits(got[0]), bits(got[1])), "a kept work buffer"
    alone = hi.attn_paged(dev(q), k, v, dev(want_table), pos, Hq, Hkv)
    # each is within 2^-10 1.125 (sum w |v|) of the exact value, and |v| < 2^3
    assert (alone.float() - torch.from_numpy(got[0]).cuda().float()).abs().max().item() <= 2 * 2**-10 * 1.125 * 8


def test_shared_unwritten_tail(hi):
    """All sequences shorter than the prefix: the positions behind the longest hold NaN and inf, and take no part."""
    D, G, Hkv, B, page, shared = 128, 4, 8, 40, 16, 4096
    lens = [1000 + 7 * b for b in range(B)]
    c = Cache(108, [max(lens)], Hkv, D, page, shared=0)
    c.table = np.concatenate([c.table, np.full((1, shared // page - c.table.shape[1]), c.pages - 1, np.int32)], 1)
    c.table = np.repeat(c.table, B, 0)
    Hq = Hkv * G
    q = rng(109).standard_normal((B, Hq * D)).astype(np.float16)
    k, v, table = c.cuda()
    got = hi.attn_shared(dev(q), k, v, table, dev(np.array(lens, np.int32) - 1), shared, Hq, Hkv)
    compare("shared", host(got), attend(c, [(b, n - 1) for b, n in enumerate(lens)], q, Hq))


def test_shared_long(hi):
    """A prefix over many splits, with table entries that are no page in it."""
    D, G, Hkv, B, page, shared = 128, 4, 2, 40, 16, 9600
    lens = [shared + 3 * b for b in range(B)]
    c = Cache(110, lens, Hkv, D, page, shared=shared)
    c.table[:, [7, 300, 599]] = 10**8
    Hq = Hkv * G
    q = rng(111).standard_normal((B, Hq * D)).astype(np.float16)
    k, v, table = c.cuda()
    got = hi.attn_shared(dev(q), k, v, table, dev(np.array(lens, np.int32) - 1), shared, Hq, Hkv)
    compare("shared", host(got), attend(c, [(b, n - 1) for b, n in enumerate(lens)], q, Hq))


# ------------------------------------------------------------------ rotation and cache write
def rope_case(seed, M, B, Hq, Hkv, D, rot, page, P, wide):
    r = rng(seed)
    qkv = r.standard_normal((M, (Hq + 2 * Hkv) * D)).astype(np.float16)
    ang = np.arange(P)[:, None] * (10000.0 ** (-np.arange(0, rot, 2) / max(rot, 1)))[None, :]
    cs = np.stack([np.cos(ang), np.sin(ang)], -1).astype(np.float32 if wide else np.float16)
    W = -(-P // page) + 1
    table = r.permutation(B * W).reshape(B, W).astype(np.int32)
    return qkv, cs, table


def rope_plain(qkv, cs, seq, pos, table, kp, vp, q_out, Hq, Hkv, D, inter):
    """The operator in float64 into float64 copies; (q, kp, vp, tolerance of each)."""
    page, half = kp.shape[2], cs.shape[1]
    q, k, v = (t.astype(np.float64) for t in (q_out, kp, vp))
    tq, tk = np.zeros_like(q), np.zeros_like(k)
    for m in range(qkv.shape[0]):
        b, p = seq[m], pos[m]
        if p < 0 or b < 0 or b >= table.shape[0] or p >= min(cs.shape[0], table.shape[1] * page):
            continue
        pg = table[b, p // page]
        if pg < 0 or pg >= kp.shape[0]:
            continue
        x = qkv[m, :(Hq + 2 * Hkv) * D].astype(np.float64).reshape(-1, D)
        j = np.arange(half)
        i0, i1 = (2 * j, 2 * j + 1) if inter else (j, j + half)
        y, t = x.copy(), np.zeros_like(x)
        n = Hq + Hkv
        c, s = cs[p, :, 0].astype(np.float64), cs[p, :, 1].astype(np.float64)
        y[:n, i0] = x[:n, i0] * c - x[:n, i1] * s
        y[:n, i1] = x[:n, i1] * c + x[:n, i0] * s
        for i in (i0, i1):  # fp32: two roundings of 2^-24 of the terms; fp16: one of the result
            t[:n, i] = 2**-11 * np.abs(y[:n, i]) + 2**-22 * (np.abs(x[:n, i0]) + np.abs(x[:n, i1])) + 2**-25
        q[m, :Hq * D], tq[m, :Hq * D] = y[:Hq].reshape(-1), t[:Hq].reshape(-1)
        k[pg, :, p % page], tk[pg, :, p % page] = y[Hq:n], t[Hq:n]
        v[pg, :, p % page] = y[n:]
    return q, k, v, tq, tk


@pytest.mark.parametrize("D,Hq,Hkv", [(128, 32, 8), (64, 32, 4), (128, 12, 2), (64, 3, 3)])
@pytest.mark.parametrize("rot,inter", [(1.0, False), (1.0, True), (0.5, False), (0.25, True), (-20, False), (-6, True), (0, False)])
@pytest.mark.parametrize("M", [1, 5, 200])
def test_rope_cache_paged(hi, D, Hq, Hkv, rot, inter, M):
    """Rows of several sequences in mixed order, some without a place, q into its own buffer and in place."""
    rot = int(rot * D) if rot >= 0 else -rot
    B, P, page = 4, 150, 16
    wide, odd = M != 5, rot == 20
    qkv, cs, table = rope_case(120 + D + rot, M, B, Hq, Hkv, D, rot, page, P, wide)
    if rot == 0:
        cs = np.zeros((P, 0, 2), np.float16)
    r = rng(121 + M)
    place = r.permutation(B * P)[:M]
    seq, pos = (place // P).astype(np.int32), (place % P).astype(np.int32)
    if M > 100:
        pos[3], pos[17], seq[20], seq[21], pos[30] = -1, P, -1, B, 10**9
        table[1, 2], table[2, 0] = -1, 10**7
    N = B * table.shape[1]
    kp = r.standard_normal((N, Hkv, page, D)).astype(np.float16)
    vp = r.standard_normal((N, Hkv, page, D)).astype(np.float16)
    q0 = np.full((M, Hq * D), 7.0, np.float16)
    width = qkv.shape[1] + (3 if odd else 8)
    x = torch.zeros(M, width, dtype=torch.float16, device="cuda")[:, :qkv.shape[1]]
    x.copy_(dev(qkv))
    dk, dv, dq = dev(kp), dev(vp), dev(q0)
    args = (Hq, Hkv, dev(cs), dk, dv, dev(table), dev(pos))
    hi.rope_cache_paged(x, *args, seq=dev(seq), interleaved=inter, q_out=dq)
    assert np.array_equal(bits(host(x)), bits(qkv)), "qkv stays as it was with q_out"
    q, k, v, tq, tk = rope_plain(qkv, cs, seq, pos, table, kp, vp, q0, Hq, Hkv, D, inter)
    assert (np.abs(host(dq).astype(np.float64) - q) <= tq).all(), "q"
    assert (np.abs(host(dk).astype(np.float64) - k) <= tk).all(), "k"
    assert np.array_equal(host(dv).astype(np.float64), v), "v"
    kept = host(dk)
    hi.rope_cache_paged(x, *args, seq=dev(seq), interleaved=inter)
    q2 = rope_plain(qkv, cs, seq, pos, table, kp, vp, qkv[:, :Hq * D], Hq, Hkv, D, inter)[0]
    got = host(x)
    assert (np.abs(got[:, :Hq * D].astype(np.float64) - q2) <= tq).all(), "q in place"
    assert np.array_equal(bits(got[:, Hq * D:]), bits(qkv[:, Hq * D:])), "k and v of qkv stay"
    assert np.array_equal(bits(host(dk)), bits(kept))


@pytest.mark.parametrize("layout", ["joint", "strided"])
def test_rope_cache_paged_layouts(hi, layout):
    """Strided pages, K and V in one allocation: the gaps and the other half stay as they were; no seq: row m is sequence m."""
    Hq, Hkv, D, page, B = 4, 2, 128, 16, 6
    qkv, cs, table = rope_case(130, B, B, Hq, Hkv, D, D, page, 60, False)
    pos = np.array([0, 15, 16, 59, -1, 31], np.int32)
    n = Hkv * page * D
    N = table.size
    both = torch.full((N, 2 * n + 64), 5.0, dtype=torch.float16, device="cuda")
    k = both[:, :n].unflatten(1, (Hkv, page, D))
    v = (both[:, n:2 * n] if layout == "joint" else torch.full_like(both, 5.0)[:, :n]).unflatten(1, (Hkv, page, D))
    q0 = np.zeros((B, Hq * D), np.float16)
    dq = dev(q0)
    hi.rope_cache_paged(dev(qkv), Hq, Hkv, dev(cs), k, v, dev(table), dev(pos), q_out=dq)
    base = np.full((N, Hkv, page, D), 5.0, np.float16)
    q, wk, wv, tq, tk = rope_plain(qkv, cs, np.arange(B), pos, table, base, base, q0, Hq, Hkv, D, False)
    assert (np.abs(host(dq).astype(np.float64) - q) <= tq).all()
    assert (np.abs(host(k).astype(np.float64) - wk) <= tk).all()
    assert np.array_equal(host(v).astype(np.float64), wv)
    assert (host(both)[:, 2 * n:] == 5).all()


# ------------------------------------------------------------------ the operators together, as a server calls them
def test_serving_run(hi):
    """Two prompts over a common prefix, prefilled in chunks, then decode steps for both, through the paged operators and
    through the slot caches' (rope_cache, flash_prefill, decode_attn): the same attention rows. The prefix is stored once."""
    Hq, Hkv, D, page, S = 8, 2, 128, 16, 512
    r = rng(140)
    width = (Hq + 2 * Hkv) * D
    prefix, own, steps = 160, [37, 90], 5
    ang = np.arange(S)[:, None] * (10000.0 ** (-np.arange(0, D, 2) / D))[None, :]
    cs = dev(np.stack([np.cos(ang), np.sin(ang)], -1).astype(np.float16))
    common = r.standard_normal((prefix, width)).astype(np.float16)
    rows = [r.standard_normal((n, width)).astype(np.float16) for n in own]
    kc = torch.zeros(2, Hkv, S, D, dtype=torch.float16, device="cuda")
    vc = torch.zeros_like(kc)
    kv = torch.full((60, 2, Hkv, page, D), float("nan"), dtype=torch.float16, device="cuda")
    kp, vp = kv[:, 0], kv[:, 1]
    pages = r.permutation(60).astype(np.int32)
    table = np.full((2, 24), -1, np.int32)
    table[:, :10] = pages[:10]
    table[0, 10:22], table[1, 10:22] = pages[10:22], pages[22:34]
    table = dev(table)
    q = torch.empty(prefix, Hq * D, dtype=torch.float16, device="cuda")
    tol = 2 * 2**-10 * 1.125 * 8 + 2**-6  # both attentions' roundings (|v| < 8), and the two rotations' (logits off by 2^-9)

    def same(a, b):
        assert torch.isfinite(a).all() and (a.float() - b.float()).abs().max().item() <= tol

    # the prefix as sequence 0's first positions
    ids = torch.zeros(prefix, dtype=torch.int32, device="cuda")
    at = torch.arange(prefix, dtype=torch.int32, device="cuda")
    hi.rope_cache_paged(dev(common), Hq, Hkv, cs, kp, vp, table, at, seq=ids, q_out=q)
    first = hi.attn_paged(q, kp, vp, table[:1], dev(np.zeros(1, np.int32)), Hq, Hkv, start=dev(np.array([0, prefix], np.int32)))
    for b in range(2):
        x = dev(common)
        hi.rope_cache(x, Hq, Hkv, cs, kc, vc, pos_base=0, slot_base=b)
        same(first, hi.flash_prefill(x, kc[b], vc[b], prefix, 0, Hq, Hkv))
    # both prompts' own parts in one ragged batch
    both = dev(np.concatenate(rows))
    seq = dev(np.repeat([0, 1], own).astype(np.int32))
    pos = dev(np.concatenate([prefix + np.arange(n) for n in own]).astype(np.int32))
    q2 = torch.empty(sum(own), Hq * D, dtype=torch.float16, device="cuda")
    hi.rope_cache_paged(both, Hq, Hkv, cs, kp, vp, table, pos, seq=seq, q_out=q2)
    got = hi.attn_paged(q2, kp, vp, table, dev(np.full(2, prefix, np.int32)), Hq, Hkv,
                        start=dev(np.cumsum([0] + own).astype(np.int32)))
    for b, lo in enumerate([0, own[0]]):
        x = dev(rows[b])
        hi.rope_cache(x, Hq, Hkv, cs, kc, vc, pos_base=prefix, slot_base=b)
        same(got[lo:lo + own[b]], hi.flash_prefill(x, kc[b], vc[b], own[b], prefix, Hq, Hkv))
    # decode steps
    pos = np.array([prefix + n for n in own], np.int32)
    for _ in range(steps):
        x = r.standard_normal((2, width)).astype(np.float16)
        q3 = torch.empty(2, Hq * D, dtype=torch.float16, device="cuda")
        hi.rope_cache_paged(dev(x), Hq, Hkv, cs, kp, vp, table, dev(pos), q_out=q3)
        paged = hi.attn_paged(q3, kp, vp, table, dev(pos), Hq, Hkv)
        joint = hi.attn_shared(q3, kp, vp, table, dev(pos), prefix, Hq, Hkv)
        y = dev(x)
        hi.rope_cache(y, Hq, Hkv, cs, kc, vc, pos=dev(pos))
        slot = hi.decode_attn(y, kc, vc, dev(pos), Hq, Hkv)
        same(paged, slot)
        same(joint, slot)
        pos += 1


@pytest.mark.parametrize("form", ["decode", "ragged", "shared"])
def test_captured_and_grown(hi, form):
    """One captured step, replayed while the sequences grow on the device, with eager work in between: each replay equals the
    eager call, bit for bit."""
    Hq, Hkv, D, page, B = 16, 4, 64, 16, 6
    lens = [700, 500, 450, 1500, 900, 300]
    c = Cache(150, lens, Hkv, D, page, shared=256)
    for b in range(1, B):
        c.table[b, :16] = c.table[0, :16]
    rows = 3 if form == "ragged" else 1
    q = dev(rng(151).standard_normal((B * rows, Hq * D)).astype(np.float16))
    k, v, table = c.cuda()
    pos = torch.tensor([100, 20, 280, 3, 600, 290], dtype=torch.int32, device="cuda")
    start = torch.arange(0, B * rows + 1, rows, dtype=torch.int32, device="cuda")
    out = torch.empty_like(q)

    def work():
        return hi.attn_shared_work(B, Hq, Hkv, D) if form == "shared" else \
            hi.attn_paged_work(B * rows, B, Hq, Hkv, D, ragged=form == "ragged")

    def step(out, w):
        if form == "shared":
            return hi.attn_shared(q, k, v, table, pos, 256, Hq, Hkv, out=out, work=w)
        return hi.attn_paged(q, k, v, table, pos, Hq, Hkv, start=start if form == "ragged" else None, out=out, work=w)

    w, w2 = work(), work()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(out, w)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(out, w)
    limit = torch.tensor([n - rows for n in lens], dtype=torch.int32, device="cuda")
    for i in range(6):
        out.fill_(9.0)
        graph.replay()
        eager = step(torch.empty_like(q), w2)
        torch.cuda.synchronize()
        assert torch.equal(out, eager), f"replay {i}"
        pos.copy_(torch.minimum(pos * 2 + 1, limit))


def test_pages_behind_4_gib(hi):
    """Page ids whose byte and element offsets pass 32 bits: the same bits as the same pages in a small cache."""
    D, G, Hkv, page, B = 128, 4, 8, 16, 3
    Hq, lens = Hkv * G, [700, 33, 1500]
    c = Cache(170, lens, Hkv, D, page, shared=32)
    k, v, table = c.cuda()
    N = 140000  # 4.6 GB each
    kf, vf = (torch.empty(N, Hkv, page, D, dtype=torch.float16, device="cuda") for _ in range(2))
    far = torch.from_numpy(rng(171).permutation(N - 131100)[:c.pages].astype(np.int64) + 131100).cuda()
    kf[far], vf[far] = k, v
    tf = torch.where(table >= 0, far[table.clamp(min=0).long()].int(), table)
    q = dev(rng(172).standard_normal((B, Hq * D)).astype(np.float16))
    pos = dev(np.array(lens, np.int32) - 1)
    assert torch.equal(hi.attn_paged(q, k, v, table, pos, Hq, Hkv), hi.attn_paged(q, kf, vf, tf, pos, Hq, Hkv))
    q = dev(rng(173).standard_normal((60, Hq * D)).astype(np.float16))
    start, at = dev(np.array([0, 20, 30, 60], np.int32)), dev(np.array(lens, np.int32) - np.array([20, 10, 30], np.int32))
    assert torch.equal(hi.attn_paged(q, k, v, table, at, Hq, Hkv, start=start),
                       hi.attn_paged(q, kf, vf, tf, at, Hq, Hkv, start=start))
    big = 64  # enough rows for the prefix to be read once
    tables = [t[2:3].repeat(big, 1).contiguous() for t in (table, tf)]
    q = dev(rng(174).standard_normal((big, Hq * D)).astype(np.float16))
    pos = torch.full((big,), 1499, dtype=torch.int32, device="cuda")
    assert torch.equal(hi.attn_shared(q, k, v, tables[0], pos, 1488, Hq, Hkv), hi.attn_shared(q, kf, vf, tables[1], pos, 1488, Hq, Hkv))
    qkv, cs, _ = rope_case(175, 5, 1, Hq, Hkv, D, D, page, 1600, False)
    seq, pos = dev(np.array([2, 0, 2, 1, 2], np.int32)), dev(np.array([1499, 40, 3, 32, 700], np.int32))
    for kk, vv, tt in ((k, v, table), (kf, vf, tf)):
        hi.rope_cache_paged(dev(qkv), Hq, Hkv, dev(cs), kk, vv, tt, pos, seq=seq)
    assert torch.equal(k.view(torch.int16), kf[far].view(torch.int16)) and torch.equal(v.view(torch.int16), vf[far].view(torch.int16))


@pytest.mark.parametrize("form", ["decode", "ragged", "shared", "reread"])
def test_out_in_place(hi, form):
    """out = q, a slice of the QKV rows that rope_cache_paged rotated in place: the same bits as into new rows, and the rest
    of the rows untouched."""
    D, Hq, Hkv, page = 128, 8, 2, 16
    rows = [3, 40, 1, 0, 17] if form == "ragged" else [1] * (40 if form == "shared" else 9)
    B, M, shared = len(rows), sum(rows), {"shared": 4096, "reread": 64}.get(form, 0)
    before = [shared + 37 * b for b in range(B)]
    if form == "ragged":
        before = [2500, 900, 5000, 10, 0]
    c = Cache(190, [p + n for p, n in zip(before, rows)], Hkv, D, page, shared=shared)
    for b in range(1, B):
        c.table[b, :shared // page] = c.table[0, :shared // page]
    k, v, table = c.cuda()
    pos = dev(np.array(before, np.int32))
    qkv = dev(rng(191).standard_normal((M, (Hq + 2 * Hkv) * D)).astype(np.float16))
    q, kept = qkv[:, :Hq * D], qkv[:, Hq * D:].clone()
    start = dev(np.cumsum([0] + rows).astype(np.int32))

    def run(out):
        if shared:
            return hi.attn_shared(q, k, v, table, pos, shared, Hq, Hkv, out=out)
        return hi.attn_paged(q, k, v, table, pos, Hq, Hkv, start=start if form == "ragged" else None, out=out)

    want = run(None)
    assert run(q) is q
    assert torch.equal(q, want) and torch.equal(qkv[:, Hq * D:], kept)


def test_two_streams(hi):
    """Calls on two streams at once, a work buffer each: as one after the other."""
    D, Hq, Hkv, page = 128, 32, 8, 16
    lens = [4000, 700, 2500, 90]
    c = Cache(195, lens, Hkv, D, page)
    k, v, table = c.cuda()
    pos, at = dev(np.array(lens, np.int32) - 1), dev(np.array(lens, np.int32) - 20)
    start = dev(np.arange(0, 81, 20).astype(np.int32))
    q1, q2 = (dev(rng(196 + i).standard_normal((n, Hq * D)).astype(np.float16)) for i, n in enumerate((4, 80)))
    w1, w2 = hi.attn_paged_work(4, 4, Hq, Hkv, D), hi.attn_paged_work(80, 4, Hq, Hkv, D, ragged=True)
    one = hi.attn_paged(q1, k, v, table, pos, Hq, Hkv, work=w1)
    two = hi.attn_paged(q2, k, v, table, at, Hq, Hkv, start=start, work=w2)
    a, b = [torch.empty_like(one) for _ in range(20)], [torch.empty_like(two) for _ in range(20)]
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    for x, y in zip(a, b):
        with torch.cuda.stream(s1):
            hi.attn_paged(q1, k, v, table, pos, Hq, Hkv, out=x, work=w1)
        with torch.cuda.stream(s2):
            hi.attn_paged(q2, k, v, table, at, Hq, Hkv, start=start, out=y, work=w2)
    torch.cuda.synchronize()
    for x, y in zip(a, b):
        assert torch.equal(x, one) and torch.equal(y, two)


# ------------------------------------------------------------------ refusals
def test_refusals(hi):
    D, Hq, Hkv, page, B = 128, 4, 2, 16, 3
    c = Cache(160, [40, 40, 40], Hkv, D, page)
    k, v, table = c.cuda()
    half = dict(dtype=torch.float16, device="cuda")
    q, pos = torch.zeros(B, Hq * D, **half), torch.zeros(B, dtype=torch.int32, device="cuda")
    qkv, cs = torch.zeros(B, (Hq + 2 * Hkv) * D, **half), torch.zeros(50, D // 2, 2, **half)
    start = torch.tensor([0, 1, 2, 3], dtype=torch.int32, device="cuda")

    def refused(f, *a, **kw):
        with pytest.raises(ValueError):
            f(*a, **kw)

    A, S, R = hi.attn_paged, hi.attn_shared, hi.rope_cache_paged
    refused(A, q.float(), k, v, table, pos, Hq, Hkv)
    refused(A, q.cpu(), k, v, table, pos, Hq, Hkv)
    refused(A, q, k, v, table.long(), pos, Hq, Hkv)
    refused(A, q, k, v, table, pos.long(), Hq, Hkv)
    refused(A, q, k, v, table, pos[:2], Hq, Hkv)
    refused(A, q, k, v, table, pos, Hq, Hkv + 1)
    refused(A, q, k, v, table, pos, 5, Hkv)
    refused(A, q, k, v, table, pos, 34, Hkv)
    refused(A, q[:2], k, v, table, pos, Hq, Hkv)
    refused(A, q[:, ::2], k, v, table, pos, Hq // 2, Hkv)
    refused(A, q, k, v[:, :, :8], table, pos, Hq, Hkv)
    refused(A, q, k[:, :, :8], v[:, :, :8], table, pos, Hq, Hkv)            # not packed
    refused(A, q, k[..., :64], v[..., :64], table, pos, Hq, Hkv)
    refused(A, q, k, torch.stack([v, v], 1)[:, 0], table, pos, Hq, Hkv)     # another page stride
    refused(A, q, k, v, table.t().contiguous().t(), pos, Hq, Hkv)
    refused(A, q, k, v, table, pos, Hq, Hkv, start=start[:3])
    refused(A, q, k, v, table, pos, Hq, Hkv, out=torch.zeros(B, Hq * D - 1, **half))
    refused(A, q, k, v, table, pos, Hq, Hkv, out=torch.zeros(B + 1, Hq * D, **half))
    refused(A, q, k, v, table, pos, Hq, Hkv, lse=torch.zeros(B, Hq, device="cuda"))
    refused(A, q, k, v, table, pos, Hq, Hkv, work=torch.zeros(8, dtype=torch.uint8, device="cuda"))
    for n in (4, 12, 24):  # pages that are no power of two from 8 on
        odd = torch.zeros(9, Hkv, n, D, **half)
        refused(A, q, odd, odd, table, pos, Hq, Hkv)
        refused(R, qkv, Hq, Hkv, cs, odd, odd, table, pos)
    wide = torch.zeros(9, Hkv, page, 96, **half)
    refused(A, torch.zeros(B, Hq * 96, **half), wide, wide, table, pos, Hq, Hkv)
    refused(S, q, k, v, table, pos, 8, Hq, Hkv)
    refused(S, q, k, v, table, pos, -16, Hq, Hkv)
    refused(S, q, k, v, table, pos, 16 * 4, Hq, Hkv)                        # behind the table
    refused(S, q[:2], k, v, table, pos, 16, Hq, Hkv)
    refused(R, qkv[:, :-1], Hq, Hkv, cs, k, v, table, pos)
    refused(R, qkv, Hq, Hkv, cs.double(), k, v, table, pos)
    refused(R, qkv, Hq, Hkv, torch.zeros(50, D // 2 + 1, 2, **half), k, v, table, pos)
    refused(R, qkv, Hq, Hkv, cs[:, :, :1], k, v, table, pos)
    refused(R, qkv, Hq, Hkv, cs, k, v, table[:2], pos)
    refused(R, qkv, Hq, Hkv, cs, k, v, table, pos, q_out=q[:2])
    refused(R, qkv, Hq, Hkv, cs, k, v, table, pos, seq=pos[:2])
    refused(R, qkv.float(), Hq, Hkv, cs, k, v, table, pos)
    # no rows, or no sequences: nothing to do
    empty = dict(kp=k, vp=v, table=table[:0], pos=pos[:0], Hq=Hq, Hkv=Hkv)
    assert A(torch.zeros(0, Hq * D, **half), **empty).shape == (0, Hq * D)
    assert S(torch.zeros(0, Hq * D, **half), shared=16, **empty).shape == (0, Hq * D)
    R(qkv[:0], Hq, Hkv, cs, k, v, table[:0], pos[:0])
    kept = torch.full((3, Hq * D), 7.0, **half)
    A(q, start=start[:1], out=kept, **empty)
    assert (kept == 7).all()
    none = torch.zeros(0, Hq * D, **half)
    assert A(none, k, v, table, pos, Hq, Hkv, start=torch.zeros(4, dtype=torch.int32, device="cuda")).shape == (0, Hq * D)


def test_refused_shared_beyond_32_bits(hi):
    """A `shared` that a C int would take for another number."""
    D, Hq, Hkv, page = 128, 4, 2, 16
    c = Cache(180, [40, 40], Hkv, D, page)
    k, v, table = c.cuda()
    q, pos = torch.zeros(2, Hq * D, dtype=torch.float16, device="cuda"), torch.zeros(2, dtype=torch.int32, device="cuda")
    for shared in (2**32, 2**32 + 16, -2**32):
        with pytest.raises(ValueError):
            hi.attn_shared(q, k, v, table, pos, shared, Hq, Hkv)
