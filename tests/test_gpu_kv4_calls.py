"""The 4-bit K/V cache on a device: calls that test_gpu_kv4.py leaves out."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import kv4 as O

pytestmark = pytest.mark.gpu

BF, F32 = torch.bfloat16, torch.float32


def _status():
    from kvp.attention import read_status
    return read_status()


@pytest.fixture(autouse=True)
def _clean(cuda):
    _status()
    yield


@pytest.mark.parametrize("rows", [1, 12, 300])
def test_reads_and_attention_agree_on_any_bytes(rows):
    """A row that sees only its own key returns that key's V (a weight of 1,
    whose roundings are 2^-11 and the result's 2^-8: below 1/128 of the value),
    which is what a read returns: scale bytes that are never written too."""
    from kvp import kv4
    rng = np.random.default_rng(rows)
    host = rng.integers(0, 256, (4, 2, O.PAGE_HEAD), dtype=np.uint8)
    assert (host.reshape(4, 2, 16, O.BLOCK)[..., 1088:] > O.TOP_BYTE).any()
    pages = torch.from_numpy(host).cuda()
    q = torch.zeros(rows, 256, dtype=BF, device="cuda")
    out = torch.full_like(q, 7.0)
    kv4.attn(q, pages, out, heads=2, start=100, window=1)
    got = out.double().cpu().numpy()
    for dtype in (BF, F32):
        v = torch.empty(rows, 256, dtype=dtype, device="cuda")
        kv4.read(pages, None, v, start=100)
        v = v.double().cpu().numpy()
        assert np.array_equal(v, O.get(host, range(4), "v")[100: 100 + rows].reshape(rows, 256))
        assert np.all(np.abs(got - v) <= np.abs(v) / 128)
    assert _status() == 0
