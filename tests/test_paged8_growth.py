"""GPU tests of what stored values of the 8-bit cache are off by, over pages whose exponents grow again and again.

Bound. When it is written at its page's exponent k0 a value x is off by 2^-4 |x| at most, or by half a subnormal step, 2^-10 * 2^k0. At
each growth to k1 < k2 < ... <= k its code moves exactly or is rounded to a subnormal code, by 2^-10 * 2^ki at most. These half
steps are of different powers of two up to 2^k: less than 2^-9 * 2^k together. x is exact here: fp16 V, and K that is not turned
(cosine 1, sine 0)."""
import numpy as np
import pytest
import torch

from tests._util import gpu, host, rng
from tests.test_paged8 import CODES, F8, dev, hi  # noqa: F401  (hi is a fixture)

pytestmark = gpu


def append(hi, x, Hq, Hkv, D, page, cuts):
    """The stored values [2][T, Hkv, D] (K, V) and their exponents [2][T, Hkv] after calls of so many rows each."""
    T = len(x)
    W = -(-T // page)
    g = torch.Generator(device="cuda")
    g.manual_seed(1)
    kp, vp = (torch.randint(0, 256, (W, Hkv, page, D), dtype=torch.uint8, device="cuda", generator=g).view(F8) for _ in range(2))
    ke, ve = (torch.randint(-128, 128, (W, Hkv), dtype=torch.int8, device="cuda", generator=g) for _ in range(2))
    table = torch.arange(W, dtype=torch.int32, device="cuda").flip(0).view(1, W).contiguous()
    cs = torch.zeros(T, D // 2, 2, device="cuda")
    cs[:, :, 0] = 1
    p = 0
    for n in cuts:
        hi.rope_cache_paged8(dev(x[p:p + n]), Hq, Hkv, cs, kp, vp, ke, ve, table, dev(np.array([p], np.int32)),
                             start=dev(np.array([0, n], np.int32)))
        p += n
    assert p == T
    exps = [np.repeat(host(e)[::-1].astype(np.float64), page, 0)[:T] for e in (ke, ve)]
    codes = [CODES[host(c.view(torch.uint8))[::-1]].transpose(0, 2, 1, 3).reshape(-1, Hkv, D)[:T] for c in (kp, vp)]
    return [c * 2.0 ** e[:, :, None] for c, e in zip(codes, exps)], exps


@pytest.mark.parametrize("page", [8, 16, 64])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("falling", [False, True])
def test_values_after_growth(hi, D, page, falling):  # noqa: F811
    Hq, Hkv, T = 1, 2, 75
    r = rng(page + D)
    size = 2.0 ** (np.arange(T) % page % 20 - 12)  # rows of a page grow (or fall) by a binary order each
    if falling:
        size = size[::-1]
    x = (r.standard_normal((T, (Hq + 2 * Hkv) * D)) * size[:, None]).astype(np.float16)
    want = [x[:, (Hq + i * Hkv) * D:(Hq + (i + 1) * Hkv) * D].reshape(T, Hkv, D).astype(np.float64) for i in range(2)]
    for cuts in ([T], [1] * T, [3, 20, 1, 1, 30, 9, 11]):
        got, exps = append(hi, x, Hq, Hkv, D, page, cuts)
        for g, w, e in zip(got, want, exps):
            assert (np.abs(g - w) < 2.0**-4 * np.abs(w) + 2.0**-9 * 2.0 ** e[:, :, None]).all(), cuts
            for p in range(0, T, page):  # the least exponent that holds the page, however it came
                most = np.abs(w[p:p + page]).max((0, 2))
                k = np.clip(np.ceil(np.log2(most / 448)), -32, 8)
                assert np.array_equal(e[p], k)
            normal = np.abs(w) >= 2.0**-6 * 2.0 ** e[:, :, None]  # rounded once
            assert (np.abs(g - w)[normal] <= 2.0**-4 * np.abs(w[normal])).all()
