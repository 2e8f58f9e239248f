"""The cache in pages and the verification of drafts at values, scores and sizes far from the ordinary ones.

Tolerances as in test_gpu_paged.py; what a value must not change is equal bit for bit.
"""
import numpy as np
import pytest

from tests.test_gpu_paged import BF16, F16, F32, Attend, Cache, to_type

pytestmark = pytest.mark.gpu
WILD = (np.nan, np.inf, -np.inf)


def with_value(c, name, b, row, col, value):
    """The pool of K or V (kv head 0) with one more value, for an upload."""
    pool = c.pools[name].copy()
    pool[c.where(b, np.array([row]))[0, 0, col]] = to_type(np.array([value], np.float32), c.dtype)[0]
    return pool


# -- values that are not finite ------------------------------------------------------
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("p", [50, 3000])
@pytest.mark.parametrize("hd,G", [(64, 32), (128, 40), (128, 71), (40, 64), (256, 16), (256, 20)])
def test_a_draft_does_not_reach_the_tokens_before_it(hip, hd, G, p, dtype):
    """Groups of query heads as large as the kernels' tiles, so that a tile's rows are all one token's."""
    n = 3
    c = Cache([(p, n), (33, 1)], 1, hd, 16, dtype, 0, 7)
    r = Attend(c, G)
    r.call()
    r.check()
    clean = r.result()
    for at in range(1, n):
        for what in WILD:
            c.v.upload(with_value(c, "V", 0, p + at, 5, what))
            r.call()
            got = r.result()
            assert np.array_equal(got[:at], clean[:at]), (at, what)
            assert np.array_equal(got[n:], clean[n:]), (at, what)
            assert not np.isfinite(got[at:n, :, 5]).any()
            assert np.array_equal(np.delete(got[at:n], 5, 2), np.delete(clean[at:n], 5, 2))
    c.v.upload(c.pools["V"])
