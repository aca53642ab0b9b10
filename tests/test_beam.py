"""GPU parity of beam search's selection (beam_select) against a stable sort of float64 scores on the CPU.

Tolerance. A term of a sum of exponentials is off by 2^-22 of it (the hardware's exp2) and |x - max| log2(e) 2^-23 (the argument's
rounding, whose terms are small: t 2^-t stays below 0.54), its fp32 sums of 32 and over 64 lanes by 2^-18: log sum within 2^-17, and a
score is rounded to fp32 once: |best - ref| <= 2^-17 + 2^-24 |ref|. Places must be the reference's unless two of its scores lie
within 2^-16 and are not equal; equal ones go to the lowest (beam, token)."""
import numpy as np
import pytest
import torch

from tests._util import gpu, host, rng

pytestmark = gpu


@pytest.fixture(scope="module")
def hi():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    from hipinfer_amd import hipinfer
    return hipinfer


def select(logits, scores, K, n):
    """(best, parent, token) of the float64 scores, stably sorted; what has no finite score is no candidate."""
    R, V = logits.shape
    x = logits.astype(np.float64)
    with np.errstate(all="ignore"):
        m = x.max(1, keepdims=True)
        lse = m + np.log(np.exp(x - m).sum(1, keepdims=True))
        s = scores.astype(np.float64)[:, None] + (x - lse)
    dead = ~np.isfinite(scores) | ~np.isfinite(lse[:, 0])
    s[dead] = -np.inf
    best = np.full((R // K, n), -np.inf)
    parent, token = np.full((R // K, n), -1), np.full((R // K, n), -1)
    for b in range(R // K):
        c = s[b * K:(b + 1) * K].reshape(-1)
        at = np.argsort(-c, kind="stable")[:n]
        at = at[np.isfinite(c[at])]
        best[b, :len(at)] = c[at]
        parent[b, :len(at)], token[b, :len(at)] = b * K + at // V, at % V
    return best, parent, token, s


def check(name, got, want, K):
    best, parent, token = (host(t) for t in got)
    rb, rp, rt, s = want
    assert np.array_equal(np.isneginf(best), np.isneginf(rb)), name
    fine = np.isfinite(rb)
    assert (np.abs(best[fine] - rb[fine]) <= 2**-17 + 2**-24 * np.abs(rb[fine])).all(), f"{name}: {np.abs(best[fine] - rb[fine]).max()}"
    off = (parent != rp) | (token != rt)
    for b, j in np.argwhere(off):  # another place only where the reference's scores are as good as equal, and not equal
        assert fine[b, j] and parent[b, j] // K == b, (name, b, j)
        d = abs(s[parent[b, j], token[b, j]] - rb[b, j])
        assert 0 < d <= 2**-16, (name, b, j, d)
    for b in range(len(rb)):
        places = [(p, t) for p, t in zip(parent[b], token[b]) if p >= 0]
        assert len(set(places)) == len(places), name


def dev(a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


@pytest.mark.parametrize("V", [1, 7, 8, 511, 512, 513, 2047, 2049, 8191, 32000, 32001, 128256, 151936])
@pytest.mark.parametrize("B,K,n", [(1, 1, 1), (1, 4, 8), (3, 5, 5), (2, 3, 64), (5, 2, 1), (1, 64, 64)])
def test_select(hi, V, B, K, n):
    r = rng(V + 100 * B + n)
    logits = (r.standard_normal((B * K, V)) * 2.5).astype(np.float16)
    scores = (-10 * r.random(B * K) - 5).astype(np.float32)
    check((V, B, K, n), hi.beam_select(dev(logits), dev(scores), K, n), select(logits, scores, K, n), K)


@pytest.mark.parametrize("pad,skip", [(8, 0), (3, 0), (0, 1), (5, 3)])
def test_strides(hi, pad, skip):
    """Rows that are views: other row strides, and rows that begin off 16-byte boundaries."""
    r = rng(pad + skip)
    B, K, n, V = 2, 3, 6, 5000
    wide = dev((r.standard_normal((B * K, V + pad + skip)) * 2).astype(np.float16))
    logits = wide[:, skip:skip + V]
    scores = -r.random(B * K).astype(np.float32)
    check("strides", hi.beam_select(logits, dev(scores), K, n), select(host(logits), scores, K, n), K)


def test_equal_beams(hi):
    """All beams alike, as a search begins: every candidate ties with the other beams', the lowest beam wins."""
    r = rng(1)
    K, V, n = 4, 3000, 10
    logits = np.repeat((r.standard_normal((1, V)) * 2).astype(np.float16), K, 0)
    scores = np.full(K, -1.5, np.float32)
    best, parent, token, _ = select(logits, scores, K, n)
    got = hi.beam_select(dev(logits), dev(scores), K, n)
    assert np.array_equal(host(got[1]), parent) and np.array_equal(host(got[2]), token)


@pytest.mark.parametrize("V,K,n", [(20000, 3, 64), (600, 64, 64), (100, 2, 7)])
def test_all_logits_equal(hi, V, K, n):
    """More ties than a list in LDS holds: places in order, and beams with better scores first."""
    logits = np.full((2 * K, V), 1.25, np.float16)
    scores = np.tile(np.array([-2.0] + [-1.0] * (K - 1), np.float32), 2)
    best, parent, token, _ = select(logits, scores, K, n)
    got = [host(t) for t in hi.beam_select(dev(logits), dev(scores), K, n)]
    assert np.array_equal(got[1], parent) and np.array_equal(got[2], token)
    assert np.abs(got[0] - best).max() <= 2**-17 + 2**-24 * 20


def test_sorted_vocabulary(hi):
    """Ascending and descending logits: the best candidates lie side by side in few segments."""
    V, K, n = 30000, 2, 40
    up = np.linspace(-8, 8, V).astype(np.float16)
    logits = np.stack([up, up[::-1], up[::-1], up])
    scores = np.array([-1, -1.25, -3, -2], np.float32)
    check("sorted", hi.beam_select(dev(logits), dev(scores), K, n), select(logits, scores, K, n), K)


def test_masked_and_dead(hi):
    """-inf logits are no candidates; a beam with a score that is not finite, or a NaN or +inf logit, has none; places that
    stay empty are -inf, -1, -1."""
    r = rng(3)
    K, V, n = 6, 1500, 9
    logits = (r.standard_normal((4 * K, V)) * 2).astype(np.float16)
    scores = -r.random(4 * K).astype(np.float32)
    logits[0, :1490] = -np.inf            # 10 tokens allowed
    scores[1:6] = [-np.inf, np.nan, np.inf, -1e9, -3e38]
    logits[4, 5:] = -np.inf
    logits[6:9, 100] = [np.nan, np.inf, -np.inf]
    logits[9] = -np.inf
    logits[12:18] = -np.inf               # a sequence without any candidate
    logits[15, 77] = 3.0                  # but one
    logits[18:] = -65504
    logits[18:, ::7] = 65504
    want = select(logits, scores, K, n)
    # a beam so far below the best that it does not count
    assert want[1][0].max() <= 4
    check("masked", hi.beam_select(dev(logits), dev(scores), K, n), want, K)


def test_far_beam_does_not_count(hi):
    logits = np.zeros((2, 3), np.float16)
    got = hi.beam_select(dev(logits), dev(np.array([-1.0, -3e9], np.float32)), 2, 6)
    assert host(got[1]).tolist() == [[0, 0, 0, -1, -1, -1]] and host(got[2]).tolist() == [[0, 1, 2, -1, -1, -1]]
    assert np.isneginf(host(got[0])[0, 3:]).all()


def test_out_work_and_repeat(hi):
    """Given outputs and a work buffer with anything in it; the same call gives the same bits; a smaller call in the same buffer."""
    r = rng(4)
    B, K, n, V = 3, 4, 8, 9000
    work = hi.beam_select_work(B, K, V, n)
    work.fill_(0xff)
    out = (torch.empty(B, n, device="cuda"), *(torch.empty(B, n, dtype=torch.int32, device="cuda") for _ in range(2)))
    logits, scores = dev((r.standard_normal((B * K, V)) * 3).astype(np.float16)), dev(-r.random(B * K).astype(np.float32))
    got = hi.beam_select(logits, scores, K, n, out=out, work=work)
    assert got[0] is out[0]
    first = [t.clone() for t in out]
    check("first", first, select(host(logits), host(scores), K, n), K)
    hi.beam_select(logits[:K, :100].contiguous(), scores[:K], K, 3, work=work)
    hi.beam_select(logits, scores, K, n, out=out, work=work)
    assert all(torch.equal(a, b) for a, b in zip(first, out))


def test_scores_in_place(hi):
    """With n == beams the new scores may take the old ones' place."""
    r = rng(6)
    B, K, V = 5, 4, 3000
    x, s = (r.standard_normal((B * K, V)) * 2).astype(np.float16), -r.random(B * K).astype(np.float32)
    scores = dev(s)
    out = scores.view(B, K), *(torch.empty(B, K, dtype=torch.int32, device="cuda") for _ in range(2))
    check("in place", hi.beam_select(dev(x), scores, K, out=out), select(x, s, K, K), K)
    with pytest.raises(ValueError):
        hi.beam_select(dev(x), scores[:B * K], K, 3, out=(scores[:B * 3].view(B, 3), *(t[:, :3].contiguous() for t in out[1:])))


def test_no_sequences(hi):
    got = hi.beam_select(torch.empty(0, 50, dtype=torch.float16, device="cuda"), torch.empty(0, device="cuda"), 4, 3)
    assert got[1].shape == (0, 3)


def test_captured(hi):
    """A captured selection reads new logits at every replay."""
    r = rng(5)
    B, K, n, V = 2, 4, 8, 32000
    logits, scores = torch.empty(B * K, V, dtype=torch.float16, device="cuda").normal_(), torch.zeros(B * K, device="cuda")
    out = (torch.empty(B, n, device="cuda"), *(torch.empty(B, n, dtype=torch.int32, device="cuda") for _ in range(2)))
    work = hi.beam_select_work(B, K, V, n)
    hi.beam_select(logits, scores, K, n, out=out, work=work)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        hi.beam_select(logits, scores, K, n, out=out, work=work)
    for i in range(3):
        x, s = (r.standard_normal((B * K, V)) * 2).astype(np.float16), -r.random(B * K).astype(np.float32)
        logits.copy_(dev(x))
        scores.copy_(dev(s))
        g.replay()
        torch.cuda.synchronize()
        check(f"replay {i}", out, select(x, s, K, n), K)


def test_python_refusals(hi):
    logits, scores = torch.zeros(8, 50, dtype=torch.float16, device="cuda"), torch.zeros(8, device="cuda")
    bad = [lambda: hi.beam_select(logits.float(), scores, 4), lambda: hi.beam_select(logits, scores, 3),
           lambda: hi.beam_select(logits, scores, 0), lambda: hi.beam_select(logits, scores[:7], 4),
           lambda: hi.beam_select(logits, scores.half(), 4), lambda: hi.beam_select(logits, scores.cpu(), 4),
           lambda: hi.beam_select(logits.cpu(), scores, 4), lambda: hi.beam_select(logits.t(), torch.zeros(50, device="cuda"), 5),
           lambda: hi.beam_select(logits, scores, 4, 0), lambda: hi.beam_select(logits, scores, 4, 65),
           lambda: hi.beam_select(logits, scores, 4, work=torch.zeros(16, dtype=torch.uint8, device="cuda")),
           lambda: hi.beam_select(logits[:, ::2], scores, 4), lambda: hi.beam_select(logits[0], scores, 4)]
    for f in bad:
        with pytest.raises(ValueError):
            f()
