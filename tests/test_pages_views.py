"""GPU tests of cache_fork over tables that are views of one buffer, against test_pages' model."""
import numpy as np
import pytest
import torch

from tests._util import gpu, host
from tests.test_pages import Pool, dev, fork, hi, state  # noqa: F401  (hi is a fixture)

pytestmark = gpu


@pytest.mark.parametrize("S,parent,first", [(6, [5, 0, 0, -1, 2, 2], 0), (7, [1, 1, 3], 1), (3, [0, 0, 0, 2, 2, 1, 1, 1], 0)])
def test_two_tables_in_one_buffer(hi, S, parent, first):  # noqa: F811
    """The old and the new table as the two halves of wider rows: nothing else in the buffer changes."""
    W, pages, page, grow = 9, 200, 16, 20
    table, lens, refs = state(S + 40, S, W, pages, page)
    pool = Pool(hi, S, pages, page)
    N = len(parent)
    both = torch.full((max(S, N), 2 * W + 3), 77, dtype=torch.int32, device="cuda")
    old, new = (both[:n, h * (W + 1):h * (W + 1) + W] for n, h in ((S, first), (N, 1 - first)))
    old.copy_(dev(table))
    before = host(both)
    dr = dev(refs)
    missing = torch.zeros(1, dtype=torch.int32, device="cuda")
    t, l = hi.cache_fork(pool.set, old, dev(lens), dev(np.array(parent, np.int32)), dr, grow=grow, table_out=new, missing=missing)
    want = fork(table, lens, parent, refs, page, grow)
    assert t is new and np.array_equal(host(new), want[0]) and np.array_equal(host(l), want[1])
    assert np.array_equal(host(dr), want[2]) and host(missing)[0] == want[3]
    pool.check(want[4])
    got = host(both)
    at = (1 - first) * (W + 1)
    before[:N, at:at + W] = want[0]
    assert np.array_equal(got, before)


def test_new_lens_on_parent_are_refused(hi):  # noqa: F811
    """Waves of a row's block read parent while another writes the row's length: not one memory."""
    table, lens, refs = state(3, 4, 5, 60, 8)
    pool = Pool(hi, 3, 60, 8)
    parent, dr = dev(np.array([0, 0, 1, 3], np.int32)), dev(refs)
    for bad in (dict(lens_out=parent), dict(missing=parent[1:2]), dict(table_out=dr[:20].view(4, 5))):
        with pytest.raises(ValueError):
            hi.cache_fork(pool.set, dev(table), dev(lens), parent, dr, **bad)
    assert np.array_equal(host(dr), refs) and host(parent).tolist() == [0, 0, 1, 3]
    pool.check([])
