"""Attention over the 4-bit cache at the ends of the rules that choose its way:
many query heads to a K/V head, many sequences."""

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


def _case(batch, kvh, grp, start, rows, **kw):
    rng = np.random.default_rng(grp + rows)
    per = -(-(start + rows) // 128)
    m = _map(rng, batch, per, batch * per + 1)
    q = torch.from_numpy(telling_queries(rng, batch, rows, kvh * grp * 128)).to(BF)
    _check(*_attend(rng, telling_pool(rng, m, batch * per + 1, kvh), m, [start] * batch, [rows] * batch, rows, kvh * grp,
                    q=q, **kw))
    assert _status() == 0


@pytest.mark.parametrize("grp,rows,start,kw", [
    (255, 1, 200, {}), (255, 5, 600, {}), (256, 1, 200, {}), (256, 4, 600, dict(window=90, sinks=3)),
    (257, 3, 500, {}), (300, 1, 900, {}), (300, 7, 400, dict(tokens=5, window=30, sinks=1)), (700, 2, 300, {})])
def test_groups_of_hundreds_of_heads(grp, rows, start, kw):
    """A row tile is less than a query row's heads, or little more."""
    _case(1, 1, grp, start, rows, **kw)


@pytest.mark.parametrize("batch", [1150, 1160, 1190])
def test_more_sequences_than_the_cut_list_holds(batch):
    """Up to 1152 pairs of a row tile and a sequence can be cut; more are whole units."""
    _case(batch, 1, 1, 31, 100)
