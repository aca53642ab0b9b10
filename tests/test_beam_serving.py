"""The operators together, as beam search on an 8-bit (or fp16) paged cache uses them: prompts get pages (cache_fork), go through the
cache write and attention in one ragged call, then every step selects (beam_select), forks the table (cache_fork), appends and
attends; the pool is compacted on the way, and everything is freed at the end. Each part is checked where it stands: the selection
against a stable sort in float64, attention against float64 over what the cache holds, and the cache itself against one that was
filled with the same tokens without any fork, bit for bit."""
import numpy as np
import pytest
import torch

from tests._util import gpu, host, rng
from tests.test_beam import check, select
from tests.test_paged import attend, compare, dev, hi  # noqa: F401  (hi is a fixture)

pytestmark = gpu
F8 = torch.float8_e4m3fn
V, Hq, Hkv, D, K = 912, 8, 2, 64, 4


class Pool:
    def __init__(self, hi, pages, page, bits, rows, W):
        self.hi, self.page, self.bits = hi, page, bits
        g = torch.Generator(device="cuda").manual_seed(1)
        shape = (pages, Hkv, page, D)
        if bits == 8:  # what free pages hold must not matter
            self.k, self.v = (torch.randint(0, 256, shape, dtype=torch.uint8, device="cuda", generator=g).view(F8) for _ in "kv")
            self.ke, self.ve = (torch.randint(-128, 128, (pages, Hkv), dtype=torch.int8, device="cuda", generator=g) for _ in "kv")
            self.all = [self.k, self.v, self.ke, self.ve]
        else:
            self.k, self.v = (torch.full(shape, float("nan"), dtype=torch.float16, device="cuda") for _ in "kv")
            self.all = [self.k, self.v]
        self.set = hi.cache_set(self.all, page)
        self.refs = torch.zeros(pages, dtype=torch.int32, device="cuda")
        self.table = torch.full((rows, W), -1, dtype=torch.int32, device="cuda")
        self.lens = torch.zeros(rows, dtype=torch.int32, device="cuda")
        self.missing = torch.zeros(1, dtype=torch.int32, device="cuda")

    def fork(self, parent, grow):
        self.table, self.lens = self.hi.cache_fork(self.set, self.table, self.lens, parent, self.refs, grow=grow, missing=self.missing)
        assert self.missing.item() == 0
        # counts and table agree
        t = host(self.table)
        assert np.array_equal(host(self.refs), np.bincount(t[t >= 0], minlength=len(self.refs)))

    def step(self, qkv, cs, start=None):
        """Rows at the sequences' ends: written, then attended to."""
        hi, q = self.hi, torch.empty(qkv.shape[0], Hq * D, dtype=torch.float16, device="cuda")
        if self.bits == 8:
            cache = self.k, self.v, self.ke, self.ve, self.table
            hi.rope_cache_paged8(qkv, Hq, Hkv, cs, *cache, self.lens, start=start, q_out=q)
            return q, hi.attn_paged8(q, *cache, self.lens, Hq, Hkv, start=start)
        pos, seq = self.lens, None
        if start is not None:
            n = start[1:] - start[:-1]
            seq = torch.repeat_interleave(torch.arange(len(n), device="cuda", dtype=torch.int32), n.long()).int()
            pos = (self.lens[seq.long()] + torch.arange(len(seq), device="cuda") - start[seq.long()]).int()
        hi.rope_cache_paged(qkv, Hq, Hkv, cs, self.k, self.v, self.table, pos, seq=seq, q_out=q)
        return q, hi.attn_paged(q, self.k, self.v, self.table, self.lens, Hq, Hkv, start=start)

    def raw(self, row, n):
        """What positions 0 .. n - 1 of a row hold, as bytes, and the exponents of their pages."""
        ids = self.table[row, :-(-n // self.page)].long()
        kv = [t.view(torch.uint8)[ids].transpose(1, 2).flatten(0, 1)[:n] if self.bits == 8 else
              t[ids].transpose(1, 2).flatten(0, 1)[:n].contiguous().view(torch.int16) for t in (self.k, self.v)]
        return kv + ([self.ke[ids], self.ve[ids]] if self.bits == 8 else [])

    def seen(self, row, n):
        """(K, V) [Hkv, n, D] float64: test_paged.attend's view of this cache."""
        out = []
        ids = self.table[row, :-(-n // self.page)].long()
        for t, e in ((self.k, "ke"), (self.v, "ve")):
            x = t.view(torch.uint8)[ids].view(F8).double() * 2.0 ** getattr(self, e)[ids].double()[..., None, None] if self.bits == 8 \
                else t[ids].double()
            out.append(x.transpose(0, 1).flatten(1, 2)[:, :n].cpu())
        return out


class Seen:
    """A pool in the shape that attend asks of a cache."""

    def __init__(self, pool):
        self.pool, self.Hkv, self.D = pool, Hkv, D

    def seen(self, b, n):
        return self.pool.seen(b, n)


@pytest.mark.parametrize("bits,page", [(8, 8), (8, 16), (16, 8)])
def test_beam_search(hi, bits, page):  # noqa: F811
    r = rng(bits + page)
    prompts = [[int(t) for t in r.integers(0, V, n)] for n in (5, 16, 33)]
    B, T = len(prompts), 30
    W = -(-(33 + T + 1) // page) + 1
    embed = dev((r.standard_normal((V, (Hq + 2 * Hkv) * D)) * 2.0 ** r.integers(-2, 3, (V, 1))).astype(np.float16))
    head = dev((r.standard_normal((V, Hq * D)) * 0.3).astype(np.float16))
    a = r.uniform(-np.pi, np.pi, (W * page, D // 2))
    cs = dev(np.stack([np.cos(a), np.sin(a)], -1).astype(np.float32))
    pool = Pool(hi, B * K * 2 + B * K * W, page, bits, B, W)

    pool.fork(torch.arange(B, dtype=torch.int32, device="cuda"), max(map(len, prompts)))
    start = dev(np.cumsum([0] + [len(p) for p in prompts]).astype(np.int32))
    q, out = pool.step(embed[dev(np.array(sum(prompts, [])))], cs, start)
    at = [(b, t) for b, p in enumerate(prompts) for t in range(len(p))]
    compare("prompts", host(out), attend(Seen(pool), at, host(q), Hq))
    pool.lens = pool.lens + dev(np.array([len(p) for p in prompts], np.int32))
    logits = (out[(start[1:] - 1).long()].float() @ head.float().T).half()
    scores = torch.zeros(B, device="cuda")
    history = [list(p) for p in prompts]
    beams = 1
    for t in range(T):
        best, parent, token = hi.beam_select(logits, scores, beams, K)
        check(f"step {t}", (best, parent, token), select(host(logits), host(scores), beams, K), beams)
        scores, token = best.flatten(), token.flatten()
        history = [history[p] + [k] for p, k in zip(parent.flatten().tolist(), token.tolist())]
        beams = K
        pool.fork(parent.flatten(), 1)
        if t % 7 == 6:
            before = [pool.raw(b, int(pool.lens[b])) for b in range(B * K)]
            moved, used = hi.cache_compact(pool.set, pool.table, pool.refs)
            n = int(used)
            assert (pool.refs[n:] == 0).all() and (pool.refs[:n] > 0).all() and int(pool.table.max()) < n
            for b in range(B * K):
                assert all(torch.equal(x, y) for x, y in zip(before[b], pool.raw(b, int(pool.lens[b]))))
        q, out = pool.step(embed[token.long()], cs)
        if t % 5 == 4:
            compare(f"step {t}", host(out), attend(Seen(pool), [(b, int(pool.lens[b])) for b in range(B * K)], host(q), Hq))
        pool.lens = pool.lens + 1
        logits = (out.float() @ head.float().T).half()
    # every beam's cache is that of its tokens
    for b, tokens in enumerate(history):
        n = len(prompts[b // K])
        assert int(pool.lens[b]) == len(tokens) == n + T and tokens[:n] == prompts[b // K]
        alone = Pool(hi, W, page, bits, 1, W)
        alone.fork(torch.zeros(1, dtype=torch.int32, device="cuda"), len(tokens))
        ids = dev(np.array(tokens))
        alone.step(embed[ids[:n]], cs, dev(np.array([0, n], np.int32)))
        for t in range(n, len(tokens)):
            alone.lens.fill_(t)
            alone.step(embed[ids[t:t + 1]], cs)
        for x, y in zip(pool.raw(b, len(tokens)), alone.raw(0, len(tokens))):
            assert torch.equal(x, y), b
    pool.fork(torch.full((B * K,), -1, dtype=torch.int32, device="cuda"), 1)
    assert (pool.refs == 0).all() and (pool.table == -1).all() and (pool.lens == 0).all()


def test_captured_beam_step(hi):  # noqa: F811
    """One whole step (select, fork, append, attend, logits) in a graph, replayed over two tables in turn, against eager calls."""
    page, bits, B, T = 16, 8, 2, 12
    r = rng(3)
    W = 6
    embed = dev(r.standard_normal((V, (Hq + 2 * Hkv) * D)).astype(np.float16))
    head = dev((r.standard_normal((Hq * D, V)) * 0.3).astype(np.float16))
    a = r.uniform(-np.pi, np.pi, (W * page, D // 2))
    cs = dev(np.stack([np.cos(a), np.sin(a)], -1).astype(np.float32))

    class Run:
        def __init__(self):
            self.pool = Pool(hi, 200, page, bits, B * K, W)
            p = self.pool
            p.fork(torch.arange(B * K, dtype=torch.int32, device="cuda"), 20)
            start = torch.arange(0, 20 * B * K + 1, 20, dtype=torch.int32, device="cuda")
            prompt = dev(np.repeat(rng(4).integers(0, V, (B, 20)), K, 0).reshape(-1))
            _, out = p.step(embed[prompt], cs, start)
            p.lens += 20
            self.logits = (out[19::20] @ head).contiguous()
            self.scores = dev(np.tile(np.array([0] + [-np.inf] * (K - 1), np.float32), B))
            self.out = (torch.empty(B, K, device="cuda"), *(torch.empty(B, K, dtype=torch.int32, device="cuda") for _ in range(2)))
            self.works = [hi.beam_select_work(B, K, V, K), hi.cache_work(B * K, B * K, 200), hi.attn_paged_work(B * K, B * K, Hq, Hkv, D)]
            self.q, self.o = (torch.empty(B * K, Hq * D, dtype=torch.float16, device="cuda") for _ in range(2))
            self.other = torch.empty_like(p.table), torch.empty_like(p.lens)
            self.missing = torch.zeros(1, dtype=torch.int32, device="cuda")

        def half(self, old, new):
            p = self.pool
            hi.beam_select(self.logits, self.scores, K, K, out=self.out, work=self.works[0])
            hi.cache_fork(p.set, *old, self.out[1].flatten(), p.refs, grow=1, table_out=new[0], lens_out=new[1], missing=self.missing,
                          work=self.works[1])
            qkv = embed.index_select(0, self.out[2].flatten().long())
            cache = p.k, p.v, p.ke, p.ve, new[0]
            hi.rope_cache_paged8(qkv, Hq, Hkv, cs, *cache, new[1], q_out=self.q)
            hi.attn_paged8(self.q, *cache, new[1], Hq, Hkv, out=self.o, work=self.works[2])
            new[1].add_(1)
            self.scores.copy_(self.out[0].flatten())
            hi.gemm_noalloc(self.o, headT, self.logits)

        def step(self):
            p = self.pool
            self.half((p.table, p.lens), self.other)
            self.half(self.other, (p.table, p.lens))

    headT = head.t().contiguous()
    one, two, warm = Run(), Run(), Run()
    warm.step()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        one.step()
    for t in range(T):
        g.replay()
        two.step()
        torch.cuda.synchronize()
        for x, y in ((one.logits, two.logits), (one.scores, two.scores), (one.out[1], two.out[1]), (one.out[2], two.out[2]),
                     (one.pool.table, two.pool.table), (one.pool.lens, two.pool.lens), (one.pool.refs, two.pool.refs)):
            assert torch.equal(x, y), t
        assert int(one.missing) == 0 and torch.isfinite(one.scores).all()
    assert (one.pool.lens == 20 + 2 * T).all()
