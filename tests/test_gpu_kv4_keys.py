"""Attention over the 4-bit cache sees just the keys that it should: caches in
which a single lost or added key leaves the bound (kv4_keys.py), at the edges of
steps, splits, pages, cut units, windows, sinks and frames."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from kv4_keys import telling_pool, telling_queries
from test_gpu_kv4 import BF, _attend, _check, _map, _status

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _clean(cuda):
    _status()
    yield


def _case(batch, kvh, grp, start, rows, kw, *, seed=0, counts=None, starts=None, bad=()):
    rng = np.random.default_rng(seed + 31 * start + rows)
    per = -(-(start + rows) // 128)
    m = _map(rng, batch, per, batch * per + 1)
    pages = telling_pool(rng, m, batch * per + 1, kvh)
    for b, p in bad:
        m[b, p] = -1
    q = torch.from_numpy(telling_queries(rng, batch, rows, kvh * grp * 128)).to(BF)
    use = [n for n, x in (("starts", starts), ("counts", counts)) if x is not None]
    _check(*_attend(rng, pages, m, starts or [start] * batch, counts or [rows] * batch, rows, kvh * grp, q=q,
                    use=use, **kw))
    assert _status() == (1 if bad else 0)


# one query row: a step of 32 keys, a CTA's eight warps, clusters of 2, 4 and 8
# splits, the workspace, several heads
@pytest.mark.parametrize("start", [0, 30, 31, 32, 127, 128, 254, 255, 256, 511, 700, 1023, 1100, 2047, 4098, 8191, 9000, 30000])
@pytest.mark.parametrize("kvh,grp", [(1, 1), (3, 4)])
def test_every_key_of_a_decoding_step(start, kvh, grp):
    _case(1, kvh, grp, start, 1, {})


@pytest.mark.parametrize("batch,kvh,grp,start,rows", [
    (1, 1, 12, 9000, 1), (1, 2, 5, 4500, 3), (1, 1, 1, 9000, 20), (1, 2, 1, 4000, 33), (48, 2, 1, 4200, 1),
    (20, 8, 1, 700, 1), (5, 6, 2, 2600, 1),
    (1, 1, 1, 9000, 150), (1, 2, 1, 3000, 500), (2, 3, 1, 2000, 400), (1, 2, 2, 1100, 257), (3, 1, 3, 130, 129)])
def test_every_key_of_several_rows(batch, kvh, grp, start, rows):
    _case(batch, kvh, grp, start, rows, {})


@pytest.mark.parametrize("rows,start", [(1, 9000), (1, 700), (3, 4097), (12, 3000), (140, 2000), (300, 5000)])
@pytest.mark.parametrize("kw", [dict(window=1), dict(window=33, sinks=33), dict(window=128, sinks=127), dict(window=129, sinks=128),
                                dict(window=500, sinks=129), dict(window=1000, sinks=1), dict(tokens=60, window=3, sinks=2),
                                dict(tokens=128, window=2, sinks=1), dict(tokens=77)])
def test_every_key_of_windows_sinks_and_frames(rows, start, kw):
    _case(1, 2, 2, start, rows, kw)


@pytest.mark.parametrize("rows,start", [(1, 3000), (40, 900), (300, 1500)])
@pytest.mark.parametrize("kw", [{}, dict(window=200, sinks=40), dict(tokens=50, window=9, sinks=1)])
def test_every_key_of_ragged_batches_with_bad_pages(rows, start, kw):
    starts = [start, 0, start - 1, start // 2, 127]
    counts = [rows, rows, (rows + 1) // 2, 0, rows]
    _case(5, 2, 1, start, rows, kw, starts=starts, counts=counts)
    _case(2, 2, 1, start, rows, {}, bad=[(0, 0), (1, start // 128 - 1)])
