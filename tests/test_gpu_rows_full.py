"""Accepted drafts of sequences whose pages end before their rows do."""
import numpy as np
import pytest

import rows_oracle as ro
import sheep_amd as sa
from sheep_amd import serving
from test_gpu_rows import ints

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def device():
    sa.init(0)


@pytest.mark.parametrize("over", [0, 1, 3, 5, 6, 40, 2 ** 31 - 1 - 48])
def test_accept_past_the_last_page(over):
    """A sequence's len says where its new rows lie, also where that is past its last
    slot: its kept rows' lengths are len - m + n_kept, and only rows that have a
    slot, at places that are slots, are moved."""
    rng = np.random.default_rng(3)
    page, pages, hd, m = 16, 3, 64, 6
    cap = page * pages
    pool = rng.integers(0, 1 << 16, (pages, page, 1, hd)).astype(np.uint16)
    bufs = [sa.DevBuf.of(pool), sa.DevBuf.of(pool ^ 1)]
    pg = serving.Pages(*bufs, ints([[2, 0, 1]]), pages, page, 1, pages, 1, hd)
    tok, parent = [9, 5, 6, 7, 8, 3], [-1, 0, 0, 2, 2, 4]
    pick = [6, 0, 8, 0, 3, 1]
    path = ro.walk(tok, parent, pick, 8)
    assert path == [0, 2, 4, 5]
    n = cap + over
    n_kept, kept, nxt, ln = ints([-9]), ints([-9] * 8), ints([-9] * 8), ints([-9])
    serving.accept(pg, m, ints([0, m]), ints([n]), ints(tok), ints(parent), ints(pick), 8, n_kept, kept, nxt, ln)
    assert n_kept.read(np.int32)[0] == 4 and kept.read(np.int32).tolist() == path + [-1] * 4
    assert nxt.read(np.int32).tolist() == [6, 8, 3, 1] + [-1] * 4
    assert ln.read(np.int32)[0] == n - m + 4
    for buf, p in zip(bufs, (pool, pool ^ 1)):
        at = p[[2, 0, 1]].reshape(cap, hd)
        want = at.copy()
        for j, i in enumerate(path):
            f, t = n - m + i, n - m + j
            if f < cap:
                want[t] = at[f]
        np.testing.assert_array_equal(buf.read(np.uint16).reshape(pages, page, 1, hd)[[2, 0, 1]].reshape(cap, hd), want)
