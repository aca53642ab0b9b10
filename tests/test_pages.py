"""GPU parity of cache_fork and cache_compact with a model in plain Python that follows the definitions page by page. Everything
is whole numbers and copies: equal, not near."""
import random

import numpy as np
import pytest
import torch

from tests._util import gpu, host

pytestmark = gpu


@pytest.fixture(scope="module")
def hi():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    from hipinfer_amd import hipinfer
    return hipinfer


def dev(a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def fork(table, lens, parent, refs, page, grow):
    """(table, lens, refs, missing, copies [(src, dst, positions)]) after a fork."""
    S, W = table.shape
    pages, N = len(refs), len(parent)
    free = [p for p in range(pages) if refs[p] == 0]
    out, olens, count = np.full((N, W), -1, np.int32), np.zeros(N, np.int32), refs.copy()
    copies, missing, seen = [], 0, set()
    for row in table:
        for e in row:
            if 0 <= e < pages:
                count[e] -= 1
    for i, p in enumerate(parent):
        if not 0 <= p < S:
            continue
        n = min(max(int(lens[p]), 0), W * page)
        heir = p not in seen
        seen.add(p)
        olens[i] = n
        for j in range(min(W, -(-(n + grow) // page))):
            e = int(table[p, j])
            there = 0 <= e < pages
            if j < n // page:
                out[i, j] = e if there else -1
            elif heir and there and refs[e] == 1:
                out[i, j] = e
            elif free:
                out[i, j] = free.pop(0)
                if there and j == n // page and n % page:
                    copies.append((e, out[i, j], n % page))
            else:
                missing += 1
    for row in out:
        for e in row:
            if e >= 0:
                count[e] += 1
    return out, olens, count, missing, copies


def compact(table, refs):
    used = np.flatnonzero(refs > 0)
    U = len(used)
    moved = np.full(len(refs), -1, np.int32)
    moved[used] = used
    src, dst = used[used >= U], [p for p in range(U) if refs[p] <= 0]
    moved[src] = dst
    count = np.zeros_like(refs)
    count[moved[used]] = refs[used]
    there = (table >= 0) & (table < len(refs))
    return np.where(there, moved[np.clip(table, 0, len(refs) - 1)], -1).astype(np.int32), count, moved, U, list(zip(src, dst))


class Pool:
    """Caches of some layers: fp16 and 8-bit ones with what belongs to a page, packed or strided, and their copies on the host."""

    def __init__(self, hi, seed, pages, page, kinds=("f16", "f8"), Hkv=2, D=64, gap=0):
        g = torch.Generator(device="cuda")
        g.manual_seed(seed)
        self.t = []
        def raw(dtype, *shape):
            n = int(np.prod(shape[1:])) * (2 if dtype == torch.float16 else 1)
            wide = torch.randint(0, 256, (pages, n + gap), dtype=torch.uint8, device="cuda", generator=g)
            return wide[:, :n].view(dtype).unflatten(1, shape[1:])
        for k in kinds:
            if k == "f16":
                self.t += [raw(torch.float16, pages, Hkv, page, D) for _ in range(2)]
            else:
                self.t += [raw(torch.uint8, pages, Hkv, page, D).view(torch.float8_e4m3fn) for _ in range(2)]
                self.t += [raw(torch.int8, pages, Hkv) for _ in range(2)]
        self.page, self.set = page, hi.cache_set(self.t, page)
        self.before = self.host()

    def host(self):
        return [t.contiguous().view(torch.uint8 if t.element_size() == 1 else torch.int16).cpu().numpy().copy() for t in self.t]

    def check(self, copies):
        for h, got in zip(self.before, self.host()):
            want = h.copy()
            for src, dst, rows in copies:
                if h.ndim == 4:
                    want[dst, :, :rows] = h[src, :, :rows]
                else:
                    want[dst] = h[src]
            assert np.array_equal(got, want)


def state(seed, S, W, pages, page, share=0.3):
    """A table of rows that share some whole pages, with lens, and counts that agree with it (some held by others too)."""
    r = random.Random(seed)
    order = list(range(pages))
    r.shuffle(order)
    table, lens = np.full((S, W), -1, np.int32), np.zeros(S, np.int32)
    refs = np.zeros(pages, np.int32)
    for s in range(S):
        n = r.randint(0, W * page)
        for j in range(-(-n // page)):
            if s and r.random() < share and table[s - 1, j] >= 0:
                table[s, j] = table[s - 1, j]
            elif order:
                table[s, j] = order.pop()
            else:
                n = min(n, j * page)
                break
            refs[table[s, j]] += 1
        lens[s] = n
    for _ in range(min(3, len(order))):  # pages of somebody else
        refs[order.pop()] += r.randint(1, 2)
    return table, lens, refs


def run_fork(hi, pool, table, lens, parent, refs, grow, in_place=False, work=None):
    dt, dl, dp, dr = dev(table), dev(lens), dev(np.array(parent, np.int32)), dev(refs)
    out = dr if in_place else torch.empty_like(dr)
    missing = torch.full((1,), -7, dtype=torch.int32, device="cuda")
    t, l = hi.cache_fork(pool.set, dt, dl, dp, dr, grow=grow, refs_out=None if in_place else out, missing=missing, work=work)
    want = fork(table, lens, parent, refs, pool.page, grow)
    assert np.array_equal(host(t), want[0])
    assert np.array_equal(host(l), want[1])
    assert np.array_equal(host(out), want[2])
    assert host(missing)[0] == want[3]
    pool.check(want[4])
    if not in_place:
        assert np.array_equal(host(dr), refs)
    assert np.array_equal(host(dt), table) and np.array_equal(host(dl), lens)
    return want


@pytest.mark.parametrize("page", [1, 8, 16, 128])
@pytest.mark.parametrize("S,N,W,grow", [(1, 1, 4, 0), (1, 4, 5, 1), (4, 4, 6, 1), (4, 1, 3, 0), (7, 13, 9, 5), (30, 70, 11, 1),
                                        (64, 64, 70, 300), (3, 1100, 4, 1)])
def test_fork(hi, page, S, N, W, grow):
    for seed in range(3):
        pages = S * W + N * 3 + 7
        table, lens, refs = state(seed, S, W, pages, page)
        r = random.Random(seed + 50)
        parent = [r.randint(-1, S) for _ in range(N)]
        pool = Pool(hi, seed, pages, page, gap=(0, 16, 4)[seed])
        run_fork(hi, pool, table, lens, parent, refs, grow, in_place=seed == 1)


def test_fork_runs_out_of_pages(hi):
    """More pages wanted than there are: the lowest rows get them, the others' entries are -1 and are counted."""
    table, lens, refs = state(5, 6, 8, 40, 8, share=0.0)
    free = int((refs == 0).sum())
    pool = Pool(hi, 1, 40, 8)
    want = run_fork(hi, pool, table, lens, [0, 0, 1, 1, 1, 2, 5, 5, 5, 4, 3, 3, 3, 3] * 3, refs, 17)
    assert want[3] > 0 and free > 0


@pytest.mark.parametrize("first", [0, 16383, 16384, 40000])
def test_fork_large_pool(hi, first):
    """Free pages behind tens of thousands of used ones, across the plan's steps; counts of a pool that ends inside one."""
    pages = 50001
    refs = np.ones(pages, np.int32)
    refs[first:first + 3] = 0
    refs[49990::3] = 0
    table, lens = np.array([[9, 8, -1, -1], [7, -1, -1, -1]], np.int32), np.array([23, 16], np.int32)
    pool = Pool(hi, 2, pages, 16, kinds=("f8",), Hkv=1)
    run_fork(hi, pool, table, lens, [0, 1, 0, 1, 0], refs, 1)


def test_fork_counts_off_alignment(hi):
    """Counts and tables that are slices of others, off 16-byte boundaries and with row strides of their own."""
    table, lens, refs = state(8, 5, 6, 60, 16)
    pool = Pool(hi, 3, 60, 16)
    wide = torch.full((5, 11), 99, dtype=torch.int32, device="cuda")
    wide[:, 3:9] = dev(table)
    some = torch.full((61,), 5, dtype=torch.int32, device="cuda")
    some[1:] = dev(refs)
    out = torch.full((7, 9), 77, dtype=torch.int32, device="cuda")
    parent = [4, 3, 3, 2, 0, 0, 1]
    t, l = hi.cache_fork(pool.set, wide[:, 3:9], dev(lens), dev(np.array(parent, np.int32)), some[1:], grow=2, table_out=out[:, 1:7])
    want = fork(table, lens, parent, refs, 16, 2)
    assert np.array_equal(host(out[:, 1:7]), want[0]) and np.array_equal(host(some[1:]), want[2])
    assert int(some[0]) == 5 and (host(out[:, 0]) == 77).all() and (host(out[:, 7:]) == 77).all()
    pool.check(want[4])


def test_fork_bad_entries(hi):
    """Entries that are no page, and lens behind the table or negative."""
    table = np.array([[3, -1, 5, 1000], [-5, 4, 60, -1], [7, 8, 9, 10]], np.int32)
    refs = np.zeros(60, np.int32)
    refs[[3, 5, 4, 7, 8, 9, 10]] = 1
    for lens in ([40, 25, 64], [1000, -3, 17]):
        pool = Pool(hi, 4, 60, 16)
        run_fork(hi, pool, table, np.array(lens, np.int32), [0, 0, 1, 1, 2, 2, -1, 3], refs, 3)


def test_fork_begins_and_ends(hi):
    """Empty rows become sequences, rows without a child are freed, all of them at once too."""
    table, lens, refs = state(9, 6, 5, 50, 8)
    table[2], lens[2] = -1, 0
    refs = np.bincount(table[table >= 0], minlength=50).astype(np.int32)
    pool = Pool(hi, 5, 50, 8)
    run_fork(hi, pool, table, lens, [2, 2, 2], refs, 20)
    pool = Pool(hi, 5, 50, 8)
    want = run_fork(hi, pool, table, lens, [-1] * 6, refs, 20, in_place=True)
    assert (want[2] == 0).all()
    pool = Pool(hi, 5, 50, 8)
    run_fork(hi, pool, table, lens, [], refs, 1)
    run_fork(hi, pool, np.zeros((0, 5), np.int32), np.zeros(0, np.int32), [0, -1], refs, 9)


def test_fork_many_layers(hi):
    """More tensors than one launch takes, pages larger than a block copies at a time, and none at all."""
    table, lens, refs = state(10, 4, 3, 30, 64)
    pool = Pool(hi, 6, 30, 64, kinds=("f16", "f8") * 23, Hkv=3, D=128)
    assert len(pool.t) > 128
    run_fork(hi, pool, table, lens, [0, 0, 1, 1, 2, 3, 3], refs, 1)
    empty = Pool.__new__(Pool)
    empty.t, empty.page, empty.set, empty.before = [], 64, hi.cache_set([], 64), []
    run_fork(hi, empty, table, lens, [0, 0, 1, 1, 2, 3, 3], refs, 1)


def test_fork_most_rows(hi):
    r = random.Random(3)
    S = 8192
    table = np.arange(S, dtype=np.int32)[:, None]
    pool = Pool(hi, 7, 3 * S, 8, kinds=("f8",), Hkv=1)
    refs = np.concatenate([np.ones(S, np.int32), np.zeros(2 * S, np.int32)])
    lens = np.array([r.randint(0, 8) for _ in range(S)], np.int32)
    run_fork(hi, pool, table, lens, [r.randrange(S) for _ in range(S)], refs, 0)


@pytest.mark.parametrize("pages,S,W", [(1, 1, 1), (2, 1, 2), (15, 2, 4), (500, 10, 20), (16384, 40, 100), (16385, 3, 7), (70001, 100, 333)])
@pytest.mark.parametrize("in_place", [False, True])
def test_compact(hi, pages, S, W, in_place):
    for seed in range(2):
        table, lens, refs = state(seed, S, W, pages, 8)
        if seed and pages > 3:
            table[0, 0], table[-1, -1], refs[pages // 2] = pages, -3, -2  # no pages, and a count gone wrong
        pool = Pool(hi, seed, pages, 8, kinds=("f8",) if pages > 1000 else ("f16", "f8"), Hkv=1, gap=(0, 16)[seed])
        dt, dr = dev(table), dev(refs)
        to, ro = (dt, dr) if in_place else (torch.empty_like(dt), torch.empty_like(dr))
        moved, used = hi.cache_compact(pool.set, dt, dr, table_out=to, refs_out=ro)
        want = compact(table, refs)
        assert np.array_equal(host(to), want[0])
        assert np.array_equal(host(ro), want[1])
        assert np.array_equal(host(moved), want[2])
        assert host(used)[0] == want[3]
        pool.check([(s, d, 8) for s, d in want[4]])


def test_compact_all_or_none(hi):
    for refs in (np.zeros(40, np.int32), np.ones(40, np.int32)):
        pool = Pool(hi, 1, 40, 16)
        t = dev(np.arange(-1, 41, dtype=np.int32).reshape(6, 7))
        moved, used = hi.cache_compact(pool.set, t, dev(refs))
        assert host(used)[0] == refs.sum()
        pool.check([])


def test_captured_fork_and_compact(hi):
    """A captured step, replayed over new parents with the program's own work in between."""
    page, S, W, pages = 8, 6, 5, 90
    table, lens, refs = state(12, S, W, pages, page)
    pool = Pool(hi, 8, pages, page)
    dt, dl, dr, dp = dev(table), dev(lens), dev(refs), dev(np.arange(S, dtype=np.int32))
    to, lo, ro = torch.empty_like(dt), torch.empty_like(dl), torch.empty_like(dr)
    t2, r2 = torch.empty_like(dt), torch.empty_like(dr)
    moved, used = torch.empty_like(dr), torch.empty(1, dtype=torch.int32, device="cuda")
    work = hi.cache_work(S, S, pages)
    def step():
        hi.cache_fork(pool.set, dt, dl, dp, dr, grow=1, table_out=to, lens_out=lo, refs_out=ro, work=work)
        hi.cache_compact(pool.set, to, ro, table_out=t2, refs_out=r2, moved=moved, used=used, work=work)
    step()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        step()
    r = random.Random(1)
    for _ in range(4):
        parent = [r.randint(-1, S - 1) for _ in range(S)]
        dp.copy_(dev(np.array(parent, np.int32)))
        fresh = [t.clone() for t in pool.t]
        pool.before = pool.host()
        g.replay()
        torch.cuda.synchronize()
        w = fork(table, lens, parent, refs, page, 1)
        c = compact(w[0], w[2])
        assert np.array_equal(host(to), w[0]) and np.array_equal(host(ro), w[2])
        assert np.array_equal(host(t2), c[0]) and np.array_equal(host(r2), c[1]) and host(used)[0] == c[3]
        for h in range(len(pool.t)):  # the fork's copies, then the compaction's
            x = pool.before[h]
            for s, d, n in w[4]:
                if x.ndim == 4:
                    x[d, :, :n] = x[s, :, :n]
                else:
                    x[d] = x[s]
        pool.check([(s, d, page) for s, d in c[4]])
        for t, f in zip(pool.t, fresh):
            t.view(torch.uint8 if t.element_size() == 1 else torch.int16).copy_(f.view(torch.uint8 if t.element_size() == 1 else torch.int16))


def test_python_refusals(hi):
    pages, page = 20, 8
    pool = Pool(hi, 1, pages, page)
    t, l, p, r = (torch.zeros(*s, dtype=torch.int32, device="cuda") for s in ((3, 4), (3,), (5,), (pages,)))
    set_ = hi.cache_set
    k = torch.zeros(pages, 2, page, 64, dtype=torch.float16, device="cuda")
    bad = [lambda: set_([k], 16), lambda: set_([k], 12), lambda: set_([k, k[:5]], page), lambda: set_([k.cpu()], page),
           lambda: set_([k.transpose(1, 2)], 2), lambda: set_([k[:, :, 0]], page), lambda: set_([k.transpose(2, 3)], 64),
           lambda: hi.cache_fork(pool.t, t, l, p, r), lambda: hi.cache_fork(pool.set, t, l, p, r[:5]),
           lambda: hi.cache_fork(pool.set, t.long(), l, p, r), lambda: hi.cache_fork(pool.set, t, l[:2], p, r),
           lambda: hi.cache_fork(pool.set, t, l, p, r, grow=-1), lambda: hi.cache_fork(pool.set, t, l, p[:3], r, table_out=t),
           lambda: hi.cache_fork(pool.set, t, l, p[:3], r, lens_out=l), lambda: hi.cache_fork(pool.set, t.cpu(), l, p, r),
           lambda: hi.cache_fork(pool.set, t, l, p, r, refs_out=r[1:]), lambda: hi.cache_fork(pool.set, t, l, p.float(), r),
           lambda: hi.cache_fork(pool.set, t, l, p, r, work=torch.zeros(64, dtype=torch.uint8, device="cuda")),
           lambda: hi.cache_fork(pool.set, t, l, p, r, missing=torch.zeros(2, dtype=torch.int32, device="cuda")),
           lambda: hi.cache_fork(pool.set, t[:, ::2], l, p, r), lambda: hi.cache_fork(pool.set, t[:1].expand(3, 4), l, p, r),
           lambda: hi.cache_compact(pool.set, t, r, table_out=t[:2]), lambda: hi.cache_compact(pool.set, t, r, moved=r[:3]),
           lambda: hi.cache_compact(pool.t, t, r), lambda: hi.cache_work(9000, 1, 5), lambda: hi.cache_work(1, 1, 0)]
    for i, f in enumerate(bad):
        with pytest.raises(ValueError):
            f()
            print("not refused", i)
