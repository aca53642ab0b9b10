"""GPU tests of beam_select's order at scores of any size: a score that all beams of a sequence share changes nothing but the scores that
come out.

What is compared are differences of scores, so the reference is test_beam's float64 selection of the scores less the sequence's
largest one (float32 numbers less each other: exact in 64 bits, or to 2^-53 of a difference that no logit matters beside). Places
must be its places. The scores that come out are test_beam's within 2^-17 + 2^-24 of them."""
import numpy as np
import pytest
import torch

from tests._util import gpu, host, rng
from tests.test_beam import dev, hi, select  # noqa: F401  (hi is a fixture)

pytestmark = gpu
LEAST = float(np.finfo(np.float32).min)


def shifted(logits, scores, K, n):
    """select() of the scores relative to each sequence's largest finite one; best as the whole score again. The n + 1 best are equal or
    further apart than computed scores are off by, so that their order is theirs alone."""
    s = scores.astype(np.float64).reshape(-1, K)
    most = np.where(np.isfinite(s), s, -np.inf).max(1, keepdims=True)
    best, parent, token, c = select(logits, (s - most).reshape(-1), K, n)
    for x in np.sort(c.reshape(-1, K * c.shape[1]), 1)[:, ::-1][:, :n + 1]:
        gaps = -np.diff(x[np.isfinite(x)])
        assert ((gaps == 0) | (gaps > 2**-15)).all()
    live = best > -2.0**31
    return np.where(live, best + most, -np.inf), np.where(live, parent, -1), np.where(live, token, -1)


def agree(name, hi, logits, scores, K, n):
    want = shifted(logits, scores, K, n)
    got = hi.beam_select(dev(logits), dev(scores), K, n)
    best, parent, token = (host(t) for t in got)
    assert np.array_equal(parent, want[1]) and np.array_equal(token, want[2]), name
    fine = want[1] >= 0
    assert np.isneginf(best[~fine]).all(), name
    assert (np.abs(best[fine] - want[0][fine]) <= 2**-17 + 2**-24 * np.abs(want[0][fine])).all(), name


@pytest.mark.parametrize("score", [0.0, -1e5, -1e9, -1e12, -1e15, -1e16, -1e17, -1e20, -1e30, LEAST, 1e12, 1e20, -LEAST])
@pytest.mark.parametrize("K,n,V", [(4, 8, 32000), (1, 4, 999), (8, 8, 4097), (3, 64, 600)])
def test_one_large_score(hi, score, K, n, V):  # noqa: F811
    """All beams of a sequence at one score (a request that is masked with the lowest float): n candidates, by their logits, 2^-4
    apart and in any beam."""
    r = rng(V + K)
    B = 2
    logits = np.full((B, K * V), -20, np.float16)
    for b in range(B):
        top = r.permutation(K * V)[:100 * K]
        logits[b, top] = np.maximum(8 - np.arange(100 * K) * 2.0**-4, -20)
    logits = logits.reshape(B * K, V)
    agree((score, K, n, V), hi, logits, np.full(B * K, score, np.float32), K, n)


@pytest.mark.parametrize("score", [-1e5, -1e9, -1e12, -1e17, LEAST])
def test_scores_a_step_apart(hi, score):  # noqa: F811
    """Beams at neighbouring float32 scores: the lower one's candidates follow while they are within 2^31 of the best, and count no
    longer beyond."""
    r = rng(11)
    K, V, n = 3, 5, 15
    logits = (np.arange(2 * K * V).reshape(2 * K, V) * 0.25 - r.integers(0, 2, (2 * K, V))).astype(np.float16)
    up = np.nextafter(np.float32(score), np.float32(0))
    scores = np.array([score, up, score, up, score, np.nextafter(up, np.float32(0))], np.float32)
    agree(score, hi, logits, scores, K, n)


@pytest.mark.parametrize("score", [-1e17, LEAST])
def test_ties_and_dead_beams_at_a_large_score(hi, score):  # noqa: F811
    """Equal rows at one large score: the lowest (beam, token) wins; beams that have ended and logits of -inf have no candidates there
    either."""
    r = rng(12)
    K, V, n = 4, 3000, 20
    row = r.permutation(V).astype(np.float64) * 2.0**-6 - 30
    logits = np.repeat(row[None].astype(np.float16), 2 * K, 0)
    logits[1, 7:] = -np.inf
    scores = np.full(2 * K, score, np.float32)
    scores[2], scores[5] = -np.inf, np.nan
    agree(score, hi, logits, scores, K, n)


def test_large_scores_among_others(hi):  # noqa: F811
    """Sequences with ordinary scores and with large ones in one call, and the call in place."""
    r = rng(13)
    B, K, V = 6, 4, 2500
    logits = (r.standard_normal((B * K, V)) * 2.5).astype(np.float16)
    scores = -r.random(B * K).astype(np.float32)
    scores[K:2 * K], scores[3 * K:4 * K] = -1e20, LEAST
    want = shifted(logits, scores, K, K)
    d = dev(scores)
    out = d.view(B, K), *(torch.empty(B, K, dtype=torch.int32, device="cuda") for _ in range(2))
    best, parent, token = (host(t) for t in hi.beam_select(dev(logits), d, K, out=out))
    assert np.array_equal(parent, want[1]) and np.array_equal(token, want[2])
    assert (np.abs(best - want[0]) <= 2**-17 + 2**-24 * np.abs(want[0])).all()
