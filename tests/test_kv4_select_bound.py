"""What a page's score bounds (paged 4-bit selection), on the oracle's arithmetic."""

import math

import numpy as np
import pytest

from oracle import kv4


def units(q):
    """The queries' power of two and their whole numbers (oracle/kv4.py, select)."""
    G, D = q.shape
    s = kv4.exponent(np.abs(q).max(), -100) + max(0, math.ceil(math.log2(G * D / 1024)))
    return s, np.rint(q.astype(np.float64) * 2.0 ** -s)


def page(rng, n, D):
    """Keys of a page that are alike: its bounds are tight."""
    x = rng.standard_normal((1, D)) + 0.02 * rng.standard_normal((n, D))
    held = kv4.values(*kv4.quantise(x.astype(np.float32)))
    bound, e = kv4.bounds(held)
    return held, bound, e


@pytest.mark.parametrize("G,D", [(1, 64), (4, 128), (8, 128), (32, 128), (64, 256)])
@pytest.mark.parametrize("outlier", [1.0, 100.0])
def test_a_page_score_bounds_its_keys_up_to_the_queries_rounding(G, D, outlier):
    rng = np.random.default_rng(G + D)
    passed = 0
    for _ in range(200):
        held, bound, e = page(rng, 16, D)
        q = rng.standard_normal((G, D)).astype(np.float32)
        q[:, 5] *= outlier
        s, z = units(q)
        assert np.abs(z).max() <= 127 and np.abs(z * 2.0 ** s - q).max() <= 2.0 ** (s - 1)
        score = np.maximum(z[:, None] * bound[0], z[:, None] * bound[1]).sum() * 2.0 ** (e + s)
        assert (z * 2.0 ** s @ held.astype(np.float64).T).sum(0).max() <= score  # of the rounded queries
        margin = 2.0 ** (s - 1) * G * np.abs(bound.astype(np.float64)).max(0).sum() * 2.0 ** e
        best = (q.astype(np.float64) @ held.astype(np.float64).T).sum(0).max()
        assert best <= score + margin
        passed += best > score
    assert outlier == 1.0 or passed > 0  # the margin is needed
