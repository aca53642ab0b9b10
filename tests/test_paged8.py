"""GPU parity of the paged cache in 8 bits (rope_cache_paged8, attn_paged8) against plain implementations in float64 on the CPU.

Tolerances. Attention's keys and values are the stored ones, exact in fp16, so its bounds are those of the fp16 cache (test_paged.py).
A stored value is off by half a step of e4m3 at its page's exponent k: 2^-4 of it, or 2^-10 * 2^k among subnormals; a rotated one
by two fp32 roundings before (2^-22 of |a| + |b|). An exponent is the least with max |x| <= 448 * 2^k, where the maximum is known to
2^-22. Earlier positions that move to a larger exponent lose at most half a subnormal step, 2^-10 * 2^k: their 4 bits move whole."""
import numpy as np
import pytest
import torch

from tests._util import bits, gpu, host, rng
from tests.test_paged import FEW, HEADS, IDS, RAGGED, Cache, attend, compare, compare_lse, dev, hi  # noqa: F401  (hi is a fixture)

pytestmark = gpu
F8 = torch.float8_e4m3fn
CODES = torch.arange(256, dtype=torch.uint8).view(F8).float().numpy().astype(np.float64)  # a code's value


class Cache8(Cache):
    """test_paged's cache in 8 bits: k and v are the values that the codes stand for, NaN where no position is held."""

    def __init__(self, seed, *args, **kw):
        super().__init__(seed, *args, **kw)
        r = rng(seed + 1)
        self.kexp, self.vexp = (r.integers(-6, -1, (self.pages, self.Hkv)).astype(np.int8) for _ in range(2))
        self.kc, self.vc = self.code(self.k, self.kexp), self.code(self.v, self.vexp)
        self.values()

    @staticmethod
    def code(x, exp):
        t = torch.from_numpy(x.astype(np.float32) * 2.0 ** -exp.astype(np.float32)[:, :, None, None])
        t = torch.where(t.isinf(), torch.nan, t.clamp(-448, 448))
        return t.to(F8).view(torch.uint8).numpy()

    def values(self):
        with np.errstate(over="ignore", invalid="ignore"):
            self.k, self.v = ((CODES[c] * 2.0 ** e.astype(np.float64)[:, :, None, None]).astype(np.float16)
                              for c, e in ((self.kc, self.kexp), (self.vc, self.vexp)))

    def cuda(self):
        k, v = (torch.from_numpy(c).cuda() for c in (self.kc, self.vc))
        n = self.Hkv * self.page * self.D
        if self.layout == "joint":
            kv = torch.stack([k, v], 1).contiguous()
            k, v = kv[:, 0], kv[:, 1]
        elif self.layout == "strided":
            def spread(t):
                wide = torch.full((self.pages, n + 48), 0x7f, dtype=torch.uint8, device="cuda")
                wide[:, :n] = t.reshape(self.pages, n)
                return wide[:, :n].unflatten(1, (self.Hkv, self.page, self.D))
            k, v = spread(k), spread(v)
        return k.view(F8), v.view(F8), dev(self.kexp), dev(self.vexp), dev(self.table)


# ------------------------------------------------------------------ attention
@pytest.mark.parametrize("D,Hkv", [(64, 3), (128, 2)])
def test_every_code_at_every_exponent(hi, D, Hkv):  # noqa: F811
    """One key has weight 1: the result is its V row, and lse its logit, for all codes and exponents, in all kernels."""
    page, per = 8, 256 // D
    exps = [e for e in range(-33, 10)] + [-128, -127, -126, -100, 60, 127]
    B = per * len(exps)
    c = Cache8(1, [1] * B, Hkv, D, page, spare=0)
    for b in range(B):
        e, part = exps[b // per], b % per
        pg = c.table[b, 0]
        c.vc[pg, :, 0] = np.arange(256, dtype=np.uint8)[part * D:(part + 1) * D]
        c.vexp[pg] = e
        c.kc[pg, :, 0] = 0
        c.kc[pg, :, 0, :Hkv] = np.diag(np.full(Hkv, 0x38 + (b * 5) % 71, np.uint8))  # 1.0 to 448
        c.kexp[pg] = np.clip(e, -20, 6)
    c.values()
    with np.errstate(over="ignore", invalid="ignore"):
        want = (CODES[c.vc] * 2.0 ** np.maximum(c.vexp.astype(np.float64), -126)[:, :, None, None]).astype(np.float16)
    want = np.stack([want[c.table[b, 0], :, 0].reshape(-1) for b in range(B)])
    q = np.zeros((B, Hkv * D), np.float16)
    q[:, [h * D + h for h in range(Hkv)]] = 1
    key = np.stack([np.diagonal(c.k[c.table[b, 0], :, 0, :Hkv].astype(np.float64)) for b in range(B)], 1)
    cache = c.cuda()
    pos = dev(np.zeros(B, np.int32))
    for start in (None, dev(np.arange(B + 1, dtype=np.int32))):
        lse = torch.empty(Hkv, B, device="cuda")
        got = host(hi.attn_paged8(dev(q), *cache, pos, Hkv, Hkv, start=start, lse=lse))
        assert np.array_equal(np.isnan(got), np.isnan(want))
        fine = ~np.isnan(want)
        assert np.array_equal(got[fine], want[fine])
        x = key / np.sqrt(D) / np.log(2.0)
        assert (np.abs(host(lse) - x) <= 2**-21 * np.abs(x)).all()
    # row tiles: all of one page's positions are the same key, runs of 80 rows
    for b in (0, per * 30 + 1, per * 35):
        pg = c.table[b, 0]
        c.vc[pg, :, 1:], c.kc[pg, :, 1:] = c.vc[pg, :, :1], c.kc[pg, :, :1]
        c.values()
        cache = c.cuda()
        kp, vp, ke, ve, table = cache
        many = torch.full((1, 12), int(pg), dtype=torch.int32, device="cuda")
        out = host(hi.attn_paged8(dev(np.repeat(q[b:b + 1], 80, 0)), kp, vp, ke, ve, many, dev(np.array([3], np.int32)), Hkv, Hkv,
                                  start=dev(np.array([0, 80], np.int32)))).astype(np.float64)
        w = want[b].astype(np.float64)
        fine = np.isfinite(w)
        # equal weights w of n keys sum to 1 within n roundings of fp16 weights and the result's own
        assert (np.abs(out[:, fine] - w[fine]) <= 2**-10 * 1.125 * np.abs(w[fine]) + 2**-24).all()


@pytest.mark.parametrize("D,G,Hkv", HEADS, ids=IDS)
@pytest.mark.parametrize("page", [8, 16, 64, 256])
def test_decode(hi, D, G, Hkv, page):  # noqa: F811
    lens = [1, 0, 7, 8, 9, 31, 32, 33, 64, 127, 129, 255, 257, 500, 777, 1030]
    c = Cache8(10 + D + G + page, lens, Hkv, D, page, layout=["packed", "joint", "strided"][page % 3])
    q = rng(11 + page).standard_normal((len(lens), Hkv * G * D)).astype(np.float16)
    lse = torch.empty(Hkv * G, len(lens), device="cuda")
    got = hi.attn_paged8(dev(q), *c.cuda(), dev(np.array(lens, np.int32) - 1), Hkv * G, Hkv, lse=lse)
    want = attend(c, [(b, n - 1) for b, n in enumerate(lens)], q, Hkv * G)
    compare("decode", host(got), want)
    compare_lse("decode", host(lse), want)


@pytest.mark.parametrize("B,lens", [(1, [1]), (1, [40]), (1, [2500]), (1, [9000]), (2, [6000, 17]), (70, [200]),
                                    (40, [300, 1, 1200]), (130, [65, 513])], ids=str)
@pytest.mark.parametrize("D,G,Hkv", [(128, 4, 8), (64, 8, 4), (128, 16, 1)], ids=["D128", "D64", "G16"])
def test_decode_batches(hi, D, G, Hkv, B, lens):  # noqa: F811
    lens = [lens[b % len(lens)] for b in range(B)]
    c = Cache8(20 + B, lens, Hkv, D, 16)
    q = rng(21 + B).standard_normal((B, Hkv * G * D)).astype(np.float16)
    cache, pos = c.cuda(), dev(np.array(lens, np.int32) - 1)
    work = hi.attn_paged_work(B, B, Hkv * G, Hkv, D)
    got = [host(hi.attn_paged8(dev(q), *cache, pos, Hkv * G, Hkv, work=work)) for _ in range(2)]
    compare("decode", got[0], attend(c, [(b, n - 1) for b, n in enumerate(lens)], q, Hkv * G))
    assert np.array_equal(bits(got[0]), bits(got[1])), "a kept work buffer"


@pytest.mark.parametrize("bad", [-1, -2**31, 2**31 - 1, 10**6])
def test_no_pages(hi, bad):  # noqa: F811
    """Table entries that are no page leave their keys out; their exponents are not read."""
    D, G, Hkv, page = 128, 4, 2, 16
    lens = [700, 64, 16, 400]
    c = Cache8(30, lens, Hkv, D, page)
    c.table[0, 3] = c.table[0, 20] = c.table[0, 43] = bad
    c.table[1, 0] = c.table[2, 0] = bad
    c.table[3, 1:] = bad
    q = rng(31).standard_normal((4, Hkv * G * D)).astype(np.float16)
    cache, pos = c.cuda(), dev(np.array(lens, np.int32) - 1)
    want = attend(c, [(b, n - 1) for b, n in enumerate(lens)], q, Hkv * G)
    compare("decode", host(hi.attn_paged8(dev(q), *cache, pos, Hkv * G, Hkv)), want)
    start = dev(np.array([0, 1, 2, 3, 4], np.int32))
    compare("runs", host(hi.attn_paged8(dev(q), *cache, pos, Hkv * G, Hkv, start=start)), want)
    # a run of 90 rows over the holes
    q = rng(32).standard_normal((90, Hkv * G * D)).astype(np.float16)
    kp, vp, ke, ve, table = cache
    got = hi.attn_paged8(dev(q), kp, vp, ke, ve, table[:1], dev(np.array([605], np.int32)), Hkv * G, Hkv,
                         start=dev(np.array([0, 90], np.int32)))
    compare("row tiles", host(got), attend(c, [(0, 605 + t) for t in range(90)], q, Hkv * G))


def test_positions_outside(hi):  # noqa: F811
    D, G, Hkv, page = 64, 4, 2, 16
    c = Cache8(40, [64, 64, 64, 64], Hkv, D, page)
    q = rng(41).standard_normal((4, Hkv * G * D)).astype(np.float16)
    cache, pos = c.cuda(), dev(np.array([2**31 - 1, -1, -2**31, 64], np.int32))
    want = attend(c, [(0, 63), (1, -1), (2, -1), (3, 63)], q, Hkv * G)
    compare("decode", host(hi.attn_paged8(dev(q), *cache, pos, Hkv * G, Hkv)), want)
    start = dev(np.arange(5, dtype=np.int32))
    compare("runs", host(hi.attn_paged8(dev(q), *cache, pos, Hkv * G, Hkv, start=start)), want)


@pytest.mark.parametrize("D,G,Hkv", HEADS, ids=IDS)
@pytest.mark.parametrize("rows,before", RAGGED + FEW, ids=[f"B{len(r)}-{sum(r)}rows-{p[0]}" for r, p in RAGGED + FEW])
def test_runs(hi, D, G, Hkv, rows, before):  # noqa: F811
    """Prompt chunks, drafted and single rows; rows of no sequence in front and behind; entries that are no page."""
    page = [8, 16, 32, 128][(D + G + len(rows)) % 4]
    lens = [p + n for p, n in zip(before, rows)]
    c = Cache8(60 + G + len(rows), lens, Hkv, D, page, layout=["packed", "joint", "strided"][G % 3])
    for b in range(0, len(rows), 3):
        if before[b] > 3 * page:
            c.table[b, 1] = c.table[b, before[b] // page - 1] = [-1, 2**31 - 1, -2**31][b % 3]
    M, Hq, pad = sum(rows), Hkv * G, 3
    start = np.cumsum([pad] + rows).astype(np.int32)
    q = rng(61).standard_normal((M + 2 * pad, Hq * D)).astype(np.float16)
    q[:pad] = q[M + pad:] = np.nan
    wide = torch.full((M + 2 * pad, Hq * D + 8), 7.0, dtype=torch.float16, device="cuda")
    lse = torch.full((Hq, M + 2 * pad), 3.0, device="cuda")
    work = hi.attn_paged_work(M + 2 * pad, len(rows), Hq, Hkv, D, ragged=True)
    cache = c.cuda()
    runs = []
    for _ in range(2):
        hi.attn_paged8(dev(q), *cache, dev(np.array(before, np.int32)), Hq, Hkv, start=dev(start), out=wide[:, :Hq * D], lse=lse,
                       work=work)
        runs.append(host(wide).copy())
    got, L = runs[0], host(lse)
    assert (got[:pad] == 7).all() and (got[M + pad:] == 7).all() and (got[:, Hq * D:] == 7).all(), "rows of no sequence"
    assert (L[:, :pad] == 3).all() and (L[:, M + pad:] == 3).all()
    at = [(b, p + t) for b, (n, p) in enumerate(zip(rows, before)) for t in range(n)]
    want = attend(c, at, q[pad:M + pad], Hq)
    compare("runs", got[pad:M + pad, :Hq * D], want)
    compare_lse("runs", L[:, pad:M + pad], want)
    assert np.array_equal(bits(runs[0]), bits(runs[1])), "a kept work buffer"
    assert (host(work)[:hi.ATTN_COUNTER_BYTES] == 0).all()


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("rows,before,Hkv,G", [
    ([10] * 20, [(173 * b) % 2600 for b in range(20)], 8, 4), ([16], [40000], 8, 4), ([100], [30000], 1, 8), ([40], [60000], 2, 6),
    ([513], [1900], 8, 4), ([700], [0], 2, 5)], ids=["B20", "16-Hkv8", "100-Hkv1", "40-Hkv2", "513", "700"])
def test_row_tiles(hi, D, rows, before, Hkv, G):  # noqa: F811
    page, Hq, M = 16, Hkv * G, sum(rows)
    c = Cache8(220 + M + D, [p + n for p, n in zip(before, rows)], Hkv, D, page)
    c.table[-1, 1] = -1
    q = rng(221).standard_normal((M, Hq * D)).astype(np.float16)
    lse = torch.empty(Hq, M, device="cuda")
    got = host(hi.attn_paged8(dev(q), *c.cuda(), dev(np.array(before, np.int32)), Hq, Hkv,
                              start=dev(np.cumsum([0] + rows).astype(np.int32)), lse=lse))
    at = [(b, p + t) for b, (p, n) in enumerate(zip(before, rows)) for t in range(n)]
    some = list(range(0, M, 1 if M * max(before) < 10**6 else 13)) + [M - 1]
    want = attend(c, [at[m] for m in some], q[some], Hq)
    compare("row tiles", got[some], want)
    compare_lse("row tiles", host(lse)[:, some], want)


@pytest.mark.parametrize("D,G,Hkv", HEADS, ids=IDS)
@pytest.mark.parametrize("n", [2, 150])
def test_later_nan(hi, D, G, Hkv, n):  # noqa: F811
    """NaN in K and V rows of later positions stays out of the rows before them, and reaches those that see it."""
    Hq, page, p0 = Hkv * G, 16, 611
    for spot in (p0 + n // 2, p0 + n - 1, 300):
        c = Cache8(55 + G, [p0 + n], Hkv, D, page)
        c.vc[c.table[0, spot // page], :, spot % page, 5] = [0x7f, 0xff][spot % 2]
        if spot == p0 + n - 1:
            c.kc[c.table[0, spot // page], :, spot % page, 0] = 0x7f
        c.values()
        q = rng(56).standard_normal((n, Hq * D)).astype(np.float16)
        got = host(hi.attn_paged8(dev(q), *c.cuda(), dev(np.array([p0], np.int32)), Hq, Hkv, start=dev(np.array([0, n], np.int32))))
        before = max(0, min(n, spot - p0))
        compare("before", got[:before], attend(c, [(0, p0 + t) for t in range(before)], q[:before], Hq))
        assert np.isnan(got[before:].reshape(n - before, Hq, D)[:, :, 5]).all()


@pytest.mark.parametrize("start", [[0, 3, 1, 6], [0, -5, 4, 6], [0, 2, 100, 200], [6, 4, 2, 0], [-2**31, 2**31 - 1, 0, 6],
                                   [2**31 - 1] * 4], ids=str)
@pytest.mark.parametrize("M", [6, 700])
def test_bad_start(hi, start, M):  # noqa: F811
    """A start that decreases or leaves the rows: nothing outside the rows is read or written, and the calls end."""
    D, G, Hkv = 128, 2, 2
    Hq = Hkv * G
    c = Cache8(90, [900, 900, 900], Hkv, D, 16)
    kp, vp, ke, ve, table = c.cuda()
    q = dev(rng(91).standard_normal((M, (Hq + 2 * Hkv) * D)).astype(np.float16))
    wide = torch.full((M + 4, Hq * D), 7.0, dtype=torch.float16, device="cuda")
    s, pos = dev(np.array([v * (M // 6) if abs(v) < 1000 else v for v in start], np.int32)), dev(np.array([290, 100, 5], np.int32))
    hi.attn_paged8(q, kp, vp, ke, ve, table, pos, Hq, Hkv, start=s, out=wide[2:M + 2])
    got = host(wide)
    assert (got[:2] == 7).all() and (got[M + 2:] == 7).all()
    cs = torch.ones(1000, D // 2, 2, device="cuda")
    hi.rope_cache_paged8(q, Hq, Hkv, cs, kp, vp, ke, ve, table, pos, start=s, q_out=wide[2:M + 2])
    got = host(wide)
    assert (got[:2] == 7).all() and (got[M + 2:] == 7).all()


# ------------------------------------------------------------------ the cache write
def rotated(x, heads, cs, pos, inter):
    """float64 rotation of the first `heads` heads of x [M, H, D], and |a| + |b| of each element's pair (0 unrotated)."""
    x = x.astype(np.float64).copy()
    size = np.zeros_like(x)
    rot = 2 * cs.shape[1]
    j = np.arange(rot // 2)
    lo, up = (2 * j, 2 * j + 1) if inter else (j, j + rot // 2)
    cs = cs.astype(np.float64)[pos]
    c, s = cs[:, None, :, 0], cs[:, None, :, 1]
    a, b = x[:, :heads][..., lo].copy(), x[:, :heads][..., up].copy()
    x[:, :heads, lo], x[:, :heads, up] = a * c - b * s, b * c + a * s
    size[:, :heads, lo] = size[:, :heads, up] = np.abs(a) + np.abs(b)
    return x, size


def append_and_check(hi, c, x, Hq, cs, rows, before, inter=False, q_out=None, start=True, pad=0):
    """Appends to cache c (whose codes are updated) and checks codes, exponents, what is left alone, and q."""
    Hkv, D, page = c.Hkv, c.D, c.page
    M, B = sum(rows), len(rows)
    kp, vp, ke, ve, table = cache = c.cuda()
    old = c.kc.copy(), c.vc.copy(), c.kexp.copy(), c.vexp.copy()
    qkv = dev(x)
    first = np.cumsum([pad] + list(rows)).astype(np.int32)
    hi.rope_cache_paged8(qkv, Hq, Hkv, dev(cs), *cache, dev(np.array(before, np.int32)), start=dev(first) if start else None,
                         interleaved=inter, q_out=q_out)
    new = [host(t.contiguous().view(torch.uint8)) for t in (kp, vp)] + [host(ke), host(ve)]
    H = Hq + 2 * Hkv
    pos = np.array([p + t for n, p in zip(rows, before) for t in range(n)], np.int64)
    seq = np.array([b for b, n in enumerate(rows) for _ in range(n)], np.int64)
    cap = min(c.table.shape[1] * page, len(cs))
    ok = (pos >= 0) & (pos < cap)
    ids = np.where(ok, c.table[seq, np.clip(pos, 0, cap - 1) // page], -1)
    ok &= (ids >= 0) & (ids < c.pages)
    xr = x[pad:pad + M, :H * D].reshape(M, H, D)
    y, size = rotated(xr, Hq + Hkv, cs, np.clip(pos, 0, len(cs) - 1), inter)
    # q
    got = host(q_out if q_out is not None else qkv)[pad:pad + M, :Hq * D].reshape(M, Hq, D).astype(np.float64)
    tol = 2**-11 * 1.01 * np.abs(y[:, :Hq]) + 2**-22 * size[:, :Hq] + 2**-25
    assert (np.abs(got - y[:, :Hq])[ok] <= tol[ok]).all(), "q"
    if q_out is None:
        assert np.array_equal(bits(got[~ok].astype(np.float16)), bits(xr[~ok][:, :Hq])), "q of rows without a place"
    for which, (h0, codes, exps, oc, oe) in enumerate(((Hq, new[0], new[2], old[0], old[2]), (Hq + Hkv, new[1], new[3], old[1], old[3]))):
        t, err = y[:, h0:h0 + Hkv], 2**-22 * size[:, h0:h0 + Hkv]
        t = np.clip(t, -61440, 61440)
        touched = set()
        for pg in np.unique(ids[ok]):
            at = np.flatnonzero(ok & (ids == pg))
            off = pos[at] % page
            o0 = off.min()
            touched.add(int(pg))
            for h in range(Hkv):
                v = np.abs(t[at, h])
                most, slack = np.nanmax(np.where(np.isnan(v), 0, v)), err[at, h].max()
                k = int(exps[pg, h])
                floor = max(-32, int(oe[pg, h])) if o0 else -32
                assert floor <= k <= 8, (pg, h, k)
                assert 448 * 2.0**k >= most - slack, (pg, h, k, most)
                assert k == floor or 448 * 2.0 ** (k - 1) < most + slack, (pg, h, k, most)
                got = CODES[codes[pg, h, off]] * 2.0**k
                bad = np.isnan(t[at, h])
                assert np.array_equal(np.isnan(got), bad)
                d = np.abs(got - t[at, h])
                assert (d[~bad] <= (np.maximum(2**-4 * v, 2**-10 * 2.0**k) + err[at, h] * 1.0625)[~bad]).all(), (pg, h)
                was = CODES[oc[pg, h, :o0]] * 2.0 ** float(oe[pg, h])
                now = CODES[codes[pg, h, :o0]] * 2.0**k
                assert np.array_equal(np.isnan(was), np.isnan(now))
                live = ~np.isnan(was)
                assert (np.abs(now - was)[live] <= (2**-10 * 2.0**k if k != oe[pg, h] else 0)).all(), (pg, h)
                assert np.array_equal(codes[pg, h, off.max() + 1:], oc[pg, h, off.max() + 1:]), "behind the rows"
        rest = [p for p in range(c.pages) if p not in touched]
        assert np.array_equal(codes[rest], oc[rest]) and np.array_equal(exps[rest], oe[rest]), "other pages"
    c.kc, c.vc, c.kexp, c.vexp = new
    c.values()


def table_of(r, positions, rot, dtype):
    a = r.uniform(-np.pi, np.pi, (positions, rot // 2))
    return np.stack([np.cos(a), np.sin(a)], -1).astype(dtype)


@pytest.mark.parametrize("D,Hkv,Hq", [(128, 8, 32), (64, 4, 32), (128, 1, 1), (64, 3, 15), (128, 2, 12)])
@pytest.mark.parametrize("page", [8, 16, 32, 64, 256])
@pytest.mark.parametrize("rot,inter,dtype", [(1.0, False, np.float16), (0.5, True, np.float32), (0.5, False, np.float32), (0, False, np.float16)],
                         ids=["full", "inter", "half", "none"])
def test_append(hi, D, Hkv, Hq, page, rot, inter, dtype):  # noqa: F811
    """Chunks, single rows and empty runs; pages begun, continued (small and large values: exponents that stay and grow), filled."""
    r = rng(page + D + Hq)
    rows, before = [1, 0, 70, 5, 1, 3, 130], [0, 40, 13, 0, page + 3, 2 * page - 1, page]
    c = Cache8(300 + page, [p + n for p, n in zip(before, rows)], Hkv, D, page, layout=["packed", "joint", "strided"][Hq % 3])
    M, rot = sum(rows), int(rot * D)
    for step, sd in enumerate((1.0, 30.0, 0.01)):
        x = (r.standard_normal((M, (Hq + 2 * Hkv) * D)) * sd).astype(np.float16)
        append_and_check(hi, c, x, Hq, table_of(r, 400 + 2 * page, rot, dtype), rows, before, inter,
                         q_out=torch.empty(M, Hq * D, dtype=torch.float16, device="cuda") if step else None)


@pytest.mark.parametrize("page", [8, 16, 64, 128])
def test_append_single_rows(hi, page):  # noqa: F811
    """A decode step after the other fills pages; sequences of several lengths, some padding rows, some without a page."""
    D, Hkv, Hq, B = 128, 2, 4, 9
    r = rng(page)
    lens = [0, 1, 5, page - 1, page, page + 1, 3 * page - 2, 7, 2 * page]
    c = Cache8(310, [n + 24 for n in lens], Hkv, D, page)
    c.table[7] = -1
    c.table[4, -1] = 10**6
    cs = table_of(r, 4 * page + 24, D, np.float32)
    for t in range(20):
        x = (r.standard_normal((B, (Hq + 2 * Hkv) * D)) * 2.0 ** r.integers(-6, 7, (B, 1))).astype(np.float16)
        before = [n + t for n in lens]
        before[2] = -1 if t % 2 else -2**31
        before[8] = 2**31 - 1 if t == 5 else before[8]
        append_and_check(hi, c, x, Hq, cs, [1] * B, before, start=False)


def test_append_bits(hi):  # noqa: F811
    """Without rotation the codes are the rounding itself: every fp16 value, in pages of all magnitudes, bit for bit."""
    D, Hkv, page = 64, 1, 16
    x = np.arange(65536, dtype=np.uint16).view(np.float16)
    x = x[np.isfinite(x)]
    x = x[np.argsort(np.abs(x), kind="stable")]
    M = -(-len(x) // D)
    x = np.concatenate([x, np.zeros(M * D - len(x), np.float16)]).reshape(M, D)
    pages = -(-M // page)
    kp = torch.zeros(pages, Hkv, page, D, dtype=torch.uint8, device="cuda").view(F8)
    vp, ke, ve = torch.zeros_like(kp.view(torch.uint8)).view(F8), *(torch.zeros(pages, Hkv, dtype=torch.int8, device="cuda") for _ in "kv")
    qkv = np.concatenate([x, x, x[::-1]], 1)
    hi.rope_cache_paged8(dev(qkv), 1, Hkv, torch.empty(M + page, 0, 2, device="cuda"), kp, vp, ke, ve,
                         torch.arange(pages, dtype=torch.int32, device="cuda")[None], torch.zeros(1, dtype=torch.int32, device="cuda"),
                         start=dev(np.array([0, M], np.int32)))
    for rows, codes, exps in ((x, kp, ke), (x[::-1], vp, ve)):
        t = np.zeros((pages * page, D), np.float64)
        t[:M] = np.clip(rows.astype(np.float64), -61440, 61440)
        t = t.reshape(pages, page * D)
        m, e = np.frexp(np.abs(t).max(1))
        k = np.clip(np.where(m > 0, e - 9 + (m > 0.875), -32), -32, 8)
        assert np.array_equal(host(exps)[:, 0], k)
        want = torch.from_numpy((t * 2.0 ** -k[:, None].astype(np.float64)).astype(np.float32)).to(F8).view(torch.uint8).numpy()
        got = host(codes.view(torch.uint8)).reshape(pages * page, D)[:M]
        want = want.reshape(pages * page, D)[:M]
        assert np.array_equal(got, want)


def test_append_nonfinite(hi):  # noqa: F811
    """Infinities become the largest value, NaN stays, and neither moves the other elements' exponent beyond it."""
    D, Hkv, Hq, page = 128, 2, 2, 16
    r = rng(5)
    x = r.standard_normal((12, (Hq + 2 * Hkv) * D)).astype(np.float16)
    cols = np.arange(Hq * D, (Hq + 2 * Hkv) * D)
    x[2, cols[5]], x[3, cols[300]], x[4, cols[7]] = np.nan, np.nan, np.inf
    x[5, cols[400]], x[6, cols[9]] = -np.inf, 65504
    x[7, cols[:128]] = np.nan
    c = Cache8(320, [12], Hkv, D, page)
    with np.errstate(invalid="ignore"):
        append_and_check(hi, c, x, Hq, np.zeros((30, 0, 2), np.float32), [12], [0])
    c = Cache8(321, [1], Hkv, D, page)  # a page of NaN alone
    x[0, cols] = np.nan
    with np.errstate(invalid="ignore"):
        append_and_check(hi, c, x[:1], Hq, np.zeros((30, 0, 2), np.float32), [1], [0])
    assert (c.kexp[c.table[0, 0]] == -32).all()


@pytest.mark.parametrize("skip,pad", [(0, 1), (4, 0), (1, 7)])
def test_append_unaligned(hi, skip, pad):  # noqa: F811
    """Rows off 16-byte boundaries, other row strides, rot that is no multiple of 16."""
    D, Hkv, Hq, page = 128, 2, 3, 32
    r = rng(skip)
    wide = (r.standard_normal((90, (Hq + 2 * Hkv) * D + skip + pad)) * 3).astype(np.float16)
    for inter in (False, True):
        c = Cache8(330, [130], Hkv, D, page)
        before = host(c.cuda()[0].view(torch.uint8))
        cs = table_of(r, 200, 54, np.float16)
        full = dev(wide)
        kp, vp, ke, ve, table = c.cuda()
        out = torch.zeros(90, Hq * D + 3, dtype=torch.float16, device="cuda")
        args = (dev(np.array([37], np.int32)),)
        hi.rope_cache_paged8(full[:, skip:skip + (Hq + 2 * Hkv) * D], Hq, Hkv, dev(cs), kp, vp, ke, ve, table, *args,
                             start=dev(np.array([0, 90], np.int32)), interleaved=inter, q_out=out[:, :Hq * D])
        # the same through aligned memory
        k2, v2, ke2, ve2, _ = c.cuda()
        o2 = torch.zeros(90, Hq * D, dtype=torch.float16, device="cuda")
        x = np.ascontiguousarray(wide[:, skip:skip + (Hq + 2 * Hkv) * D])
        hi.rope_cache_paged8(dev(x), Hq, Hkv, dev(cs), k2, v2, ke2, ve2, table, *args, start=dev(np.array([0, 90], np.int32)),
                             interleaved=inter, q_out=o2)
        assert torch.equal(out[:, :Hq * D], o2) and torch.equal(ke, ke2) and torch.equal(ve, ve2)
        assert torch.equal(kp.view(torch.uint8), k2.view(torch.uint8)) and torch.equal(vp.view(torch.uint8), v2.view(torch.uint8))
        append_and_check(hi, c, x, Hq, cs, [90], [37], inter)
        assert before.shape == c.kc.shape


def test_chunks_give_the_same_codes(hi):  # noqa: F811
    """A prompt in one call, in chunks that end inside pages, and row by row: values that agree to the subnormal step."""
    D, Hkv, Hq, page, T = 128, 2, 2, 16, 75
    r = rng(9)
    x = (r.standard_normal((T, (Hq + 2 * Hkv) * D)) * 2.0 ** r.integers(-3, 4, (T, 1))).astype(np.float16)
    cs = dev(table_of(r, T, D, np.float32))
    got = []
    for cuts in ([T], [10, 7, 30, 1, 27], [1] * T):
        c = Cache8(340, [T], Hkv, D, page)
        cache = c.cuda()
        p = 0
        for n in cuts:
            hi.rope_cache_paged8(dev(x[p:p + n]), Hq, Hkv, cs, *cache, dev(np.array([p], np.int32)), start=dev(np.array([0, n], np.int32)))
            p += n
        ids = c.table[0]
        got.append([(CODES[host(a.view(torch.uint8))[ids]] * 2.0 ** host(e)[ids][:, :, None, None].astype(np.float64))
                    .transpose(0, 2, 1, 3).reshape(-1, Hkv, D)[:T] for a, e in zip(cache[:2], cache[2:4])] + [host(e)[ids] for e in cache[2:4]])
    for other in got[1:]:
        for a, b, e in ((0, 0, 2), (1, 1, 3)):
            assert np.array_equal(got[0][e], other[e])
            step = np.repeat(2.0 ** got[0][e].astype(np.float64), page, 0)[:T, :, None]
            assert (np.abs(got[0][a] - other[b]) <= 2 * 2**-10 * step).all()


# ------------------------------------------------------------------ graphs, streams, refusals
def test_captured_steps(hi):  # noqa: F811
    """A captured decode step (cache write, then attention) replayed while sequences grow, against eager calls."""
    D, G, Hkv, page, B = 128, 4, 2, 16, 5
    Hq, lens = Hkv * G, [3, 15, 16, 100, 431]
    c = Cache8(350, [n + 10 for n in lens], Hkv, D, page)
    r = rng(351)
    cs = dev(table_of(r, 500, D, np.float32))
    mine, eager = c.cuda(), c.cuda()
    qkv = torch.empty(B, (Hq + 2 * Hkv) * D, dtype=torch.float16, device="cuda").normal_()
    pos = dev(np.array(lens, np.int32))
    q, out = (torch.empty(B, Hq * D, dtype=torch.float16, device="cuda") for _ in range(2))
    work = hi.attn_paged_work(B, B, Hq, Hkv, D)
    def step(cache, out, work):
        hi.rope_cache_paged8(qkv, Hq, Hkv, cs, *cache, pos, q_out=q)
        hi.attn_paged8(q, *cache, pos, Hq, Hkv, out=out, work=work)
    scratch = c.cuda()
    step(scratch, out, work)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        step(mine, out, work)
    for t in range(8):
        qkv.copy_(dev(r.standard_normal(tuple(qkv.shape)).astype(np.float16)))
        g.replay()
        got = out.clone()
        again = torch.empty_like(out)
        step(eager, again, None)
        torch.cuda.synchronize()
        assert torch.equal(got, again) and not got.isnan().any()
        for a, b in zip(mine, eager):
            assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
        pos += 1


def test_other_stream(hi):  # noqa: F811
    """On another stream, behind work that it has to wait for."""
    D, G, Hkv, page = 64, 8, 4, 16
    c = Cache8(360, [900, 31], Hkv, D, page)
    q = rng(361).standard_normal((2, Hkv * G * D)).astype(np.float16)
    cache, pos = c.cuda(), dev(np.array([899, 30], np.int32))
    late = torch.zeros_like(cache[0].view(torch.uint8))
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        big = torch.randn(4096, 4096, device="cuda")
        for _ in range(4):
            big = big @ big
        late.copy_(cache[0].view(torch.uint8))
        got = hi.attn_paged8(dev(q), late.view(F8), *cache[1:], pos, Hkv * G, Hkv)
    s.synchronize()
    compare("stream", host(got), attend(c, [(0, 899), (1, 30)], q, Hkv * G))


def test_python_refusals(hi):  # noqa: F811
    D, Hkv, Hq, page, B = 128, 2, 8, 16, 3
    c = Cache8(370, [20, 30, 40], Hkv, D, page)
    kp, vp, ke, ve, table = c.cuda()
    pos = torch.zeros(B, dtype=torch.int32, device="cuda")
    q = torch.zeros(B, Hq * D, dtype=torch.float16, device="cuda")
    qkv = torch.zeros(B, (Hq + 2 * Hkv) * D, dtype=torch.float16, device="cuda")
    cs = torch.zeros(100, D // 2, 2, device="cuda")
    a = dict(q=q, kp=kp, vp=vp, kexp=ke, vexp=ve, table=table, pos=pos, Hq=Hq, Hkv=Hkv)
    r = dict(qkv=qkv, Hq=Hq, Hkv=Hkv, cs=cs, kp=kp, vp=vp, kexp=ke, vexp=ve, table=table, pos=pos)
    u8, f16 = kp.view(torch.uint8), torch.zeros(*kp.shape, dtype=torch.float16, device="cuda")
    cache = [dict(kp=u8), dict(vp=u8), dict(kp=f16, vp=f16), dict(kp=kp[:2]), dict(kexp=ke[:2]), dict(vexp=ve.int()),
             dict(kexp=ke.t().contiguous().t()), dict(kexp=ke.cpu()), dict(vexp=ve[:, :1]), dict(table=table.long()), dict(pos=pos[:2]),
             dict(pos=pos.float()), dict(kp=kp.cpu()), dict(Hkv=4), dict(start=pos)]
    for change in cache + [dict(q=q[:2]), dict(q=q.float()), dict(Hq=5), dict(out=q[:, :8]), dict(lse=torch.zeros(1, device="cuda")),
                           dict(work=torch.zeros(64, dtype=torch.uint8, device="cuda"))]:
        with pytest.raises(ValueError):
            hi.attn_paged8(**(a | change))
            print("not refused", change.keys())
    for change in cache + [dict(qkv=qkv[:2]), dict(qkv=qkv[:, :100]), dict(cs=cs.half().double()), dict(cs=cs[:, :, :1]),
                           dict(q_out=qkv[:, 8:]), dict(q_out=q[:2])]:
        with pytest.raises(ValueError):
            hi.rope_cache_paged8(**(r | change))
            print("not refused", change.keys())


def test_no_rows(hi):  # noqa: F811
    c = Cache8(380, [20, 30], 2, 64, 16)
    kp, vp, ke, ve, table = c.cuda()
    none = torch.zeros(0, 8 * 64, dtype=torch.float16, device="cuda")
    pos, start = torch.zeros(2, dtype=torch.int32, device="cuda"), torch.zeros(3, dtype=torch.int32, device="cuda")
    assert hi.attn_paged8(none, kp, vp, ke, ve, table, pos, 8, 2, start=start).shape == (0, 512)
    assert hi.attn_paged8(none, kp, vp, ke, ve, table[:0], pos[:0], 8, 2).shape == (0, 512)
    cs = torch.zeros(9, 32, 2, device="cuda")
    hi.rope_cache_paged8(torch.zeros(0, 12 * 64, dtype=torch.float16, device="cuda"), 8, 2, cs, kp, vp, ke, ve, table, pos, start=start)
