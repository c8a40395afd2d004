"""The bound of oracle.kv4.attention sees a single lost or added key (CPU only)."""

from __future__ import annotations

import numpy as np
import pytest

from kv4_keys import telling_pool, telling_queries
from oracle import kv4 as O


@pytest.mark.parametrize("keys", [1, 31, 129, 1000, 9001, 40000])
def test_one_key_more_or_less_leaves_the_bound(keys):
    """A key is at least (5/6) e^-1 of its dim's mean share, and the bounds around the
    right and the wrong result together 2^-10 of the sum and 2^-7 of what the signs
    leave of it, its root: 0.3 / n against 2^-10 + 2^-7 / sqrt(n) allows n of a few
    hundred keys of a dim, 128 times as many in all."""
    rng = np.random.default_rng(keys)
    per = -(-keys // 128) + 1
    m = rng.permutation(per)[None]
    pages = telling_pool(rng, m, per, 1)
    k, v = (O.get(pages, m[0], w)[: keys + 1] for w in "kv")
    q = telling_queries(rng, 1, 1, 128).astype(np.float64)
    ok = np.arange(keys + 1)[None] < keys
    out, tol = O.attention(q, k, v, ok)
    some = {0, keys - 1, keys, keys // 2, *(int(x) for x in rng.integers(0, keys, 20))}
    for j in some - ({0} if keys == 1 else set()):
        other = ok.copy()
        other[0, j] ^= True
        wrong = O.attention(q, k, v, other)[0]
        assert np.any(np.abs(wrong - out) > 2 * tol), j


def test_scores_are_small_and_every_key_has_its_dim():
    rng = np.random.default_rng(0)
    m = rng.permutation(20).reshape(2, 10)
    pages = telling_pool(rng, m, 21, 3)
    v = O.get(pages, m[1], "v")
    assert np.all((v != 0).sum(-1) == 1) and np.all(np.abs(v).max(-1) >= 5)
    q = telling_queries(rng, 64, 3, 128)
    s = np.einsum("rhd,khd->rhk", q, O.get(pages, m[1], "k")) / np.sqrt(128)
    assert np.abs(s).max() < 1.5
