"""The 4-bit cache without a GPU: what the entry points refuse before any
device work, the format's arithmetic, and the CPU restatement against plain
formulas."""

from __future__ import annotations

import ctypes as C

import numpy as np
import pytest
import torch

from kvp._lib import Kv4Attn, Kv4Rows, Kv4Span, KvpError, lib
from oracle import kv4 as O

ERR_ARG = -1

SPAN = dict(pages=0x10000, page_map=0x20000, starts=0, counts=0, n_pages=8, kv_heads=2, batch=2,
            map_stride=4, start=5, rows=100)
ROWS = dict(k=0x30000, v=0x40000, row_stride=256, batch_stride=25600, elem_bytes=2)
ATTN = dict(q=0x50000, out=0x60000, q_row_stride=512, q_batch_stride=51200, out_row_stride=512,
            out_batch_stride=51200, heads=4, tokens=1, window=0, sinks=0)


def _call(fn, struct, base, span_kw, kw):
    s = Kv4Span(**{**SPAN, **span_kw})
    x = struct(**{**base, **kw})
    return getattr(lib(), fn)(C.byref(s), C.byref(x), None)


BAD_SPAN = [
    dict(pages=0), dict(pages=0x10008), dict(n_pages=0), dict(n_pages=1 << 31), dict(kv_heads=0),
    dict(kv_heads=5000), dict(batch=-1), dict(rows=-1), dict(map_stride=0),
    dict(map_stride=1 << 24),                       # 2^31 rows
    dict(page_map=0x20002), dict(starts=0x20001), dict(counts=0x20003),
    dict(page_map=0, n_pages=7),                    # two sequences of four pages
    dict(start=-1), dict(start=413),                # rows up to 513 of 512
]


@pytest.mark.parametrize("bad", BAD_SPAN)
@pytest.mark.parametrize("fn,struct,base", [("kvp_kv4_write", Kv4Rows, ROWS),
                                            ("kvp_kv4_read", Kv4Rows, ROWS),
                                            ("kvp_attn_kv4", Kv4Attn, ATTN)])
def test_refuses_bad_spans(fn, struct, base, bad):
    assert _call(fn, struct, base, bad, {}) == ERR_ARG
    assert b"kv4" in lib().kvp_last_error()


@pytest.mark.parametrize("fn", ["kvp_kv4_write", "kvp_kv4_read"])
@pytest.mark.parametrize("bad", [
    dict(elem_bytes=1), dict(elem_bytes=8), dict(k=0, v=0), dict(k=0x30008), dict(v=0x40004),
    dict(row_stride=252), dict(row_stride=128),     # not 16 bytes; rows overlap
    dict(batch_stride=25601), dict(batch_stride=-25600),
    dict(elem_bytes=4, row_stride=258),
])
def test_refuses_bad_rows(fn, bad):
    assert _call(fn, Kv4Rows, ROWS, {}, bad) == ERR_ARG


def test_refuses_overlapping_outputs_and_missing_operands():
    assert _call("kvp_kv4_read", Kv4Rows, ROWS, {}, dict(batch_stride=0)) == ERR_ARG
    assert b"overlap" in lib().kvp_last_error()
    assert _call("kvp_kv4_write", Kv4Rows, ROWS, {}, dict(v=0)) == ERR_ARG
    L = lib()
    assert L.kvp_kv4_write(None, None, None) == ERR_ARG
    assert L.kvp_kv4_read(None, None, None) == ERR_ARG
    assert L.kvp_attn_kv4(None, None, None) == ERR_ARG


def test_refuses_outputs_that_overlap_in_either_order():
    """Sequence by sequence, or row by row with the sequences inside, and nothing between."""
    rows = dict(row_stride=3 * 256 - 8, batch_stride=256)       # 3 sequences of 100 rows
    span = dict(batch=3, rows=100, page_map=0x20000)
    assert _call("kvp_kv4_read", Kv4Rows, ROWS, span, dict(rows, batch_stride=248)) == ERR_ARG
    assert _call("kvp_kv4_read", Kv4Rows, ROWS, span, rows) == ERR_ARG
    assert b"overlap" in lib().kvp_last_error()
    assert _call("kvp_kv4_read", Kv4Rows, ROWS, span, dict(v=ROWS["k"])) == ERR_ARG
    assert b"overlap" in lib().kvp_last_error()
    assert _call("kvp_attn_kv4", Kv4Attn, ATTN, span, dict(out_row_stride=3 * 512 - 8, out_batch_stride=512)) == ERR_ARG
    assert b"overlap" in lib().kvp_last_error()


@pytest.mark.parametrize("bad", [
    dict(heads=3), dict(heads=0), dict(tokens=0), dict(window=-1), dict(sinks=-1), dict(q=0),
    dict(out=0), dict(q=0x50002), dict(out=0x60008), dict(q_row_stride=516), dict(out_row_stride=508),
    dict(q_row_stride=256), dict(out_row_stride=0), dict(out_batch_stride=512), dict(q_batch_stride=-8),
])
def test_refuses_bad_attention(bad):
    assert _call("kvp_attn_kv4", Kv4Attn, ATTN, {}, bad) == ERR_ARG
    assert b"attn_kv4" in lib().kvp_last_error()


def test_page_bytes():
    assert lib().kvp_kv4_page_bytes(12) == 12 * 18432
    assert lib().kvp_kv4_page_bytes(0) == ERR_ARG


def test_python_refuses_without_a_device():
    from kvp import kv4
    pages = torch.zeros(2, 2, kv4.PAGE_HEAD_BYTES, dtype=torch.uint8)
    k = torch.zeros(4, 256, dtype=torch.bfloat16)
    with pytest.raises(KvpError, match="CUDA"):
        kv4.write(pages, k, k)
    with pytest.raises(KvpError, match="agree"):
        kv4.write(pages, k, k.float())
    with pytest.raises(KvpError, match="heads"):
        kv4.write(pages, k[:, :128], k[:, :128])
    with pytest.raises(KvpError, match="expected"):
        kv4.write(pages, k.half(), k.half())
    with pytest.raises(KvpError, match="needs k and v"):
        kv4.write(pages, k, None)
    with pytest.raises(KvpError, match="no rows"):
        kv4.read(pages, None, None)
    with pytest.raises(KvpError, match="uint8"):
        kv4.read(pages[..., ::2], k, k)
    with pytest.raises(KvpError, match="shape"):
        kv4.attn(k, pages, k[:3], heads=2)


# ------------------------------------------------------------- the format

def test_every_value_is_exact_in_bf16():
    x = np.arange(-8, 8)[:, None] * O.SCALES[None, :]
    assert np.array_equal(O.bf16(x), x)


def test_no_value_is_clipped_and_errors_stay_below_half_a_scale():
    """s >= amax / 7 / (1 + 1/16), so amax / s <= 7.4375 rounds to 7."""
    rng = np.random.default_rng(0)
    x = O.bf16(rng.standard_normal((512, 128)) * np.exp2(rng.uniform(-9, 9, (512, 1))))
    n, byte = O.quantise(x)
    err = np.abs(O.values(n, byte) - x).reshape(512, 8, 16)
    assert np.all(err <= O.SCALES[byte][..., None] / 2)
    assert np.abs(n).max() == 7


def test_put_and_get_are_inverse_and_touch_only_their_row():
    rng = np.random.default_rng(1)
    pages = rng.integers(0, 256, (3, 2, O.PAGE_HEAD), dtype=np.uint8)
    before = {w: O.get(pages, [0, 1, 2], w) for w in "kv"}
    x = rng.standard_normal(256)
    for w in "kv":
        O.put(pages, 1, 77, w, x)
        after = O.get(pages, [0, 1, 2], w)
        want = O.values(*O.quantise(x.reshape(2, 128)))
        assert np.array_equal(after[128 + 77], want)
        keep = np.arange(384) != 128 + 77
        assert np.array_equal(after[keep], before[w][keep])
    # every byte of a block belongs to exactly one field
    seen = np.zeros(O.BLOCK, int)
    for w in "kv":
        t = O._TAB[w].reshape(-1, 3)
        for at in set(map(tuple, t[:, :2])):
            seen[at[0]] += 1
        for sc in set(t[:, 2]):
            seen[sc] += 2
    assert np.all(seen == 2)


def test_visible_follows_the_frames():
    ok = O.visible([0, 3, 9], 10, tokens=2, window=2, sinks=1)
    assert np.array_equal(np.nonzero(ok[0])[0], [0, 1])
    assert np.array_equal(np.nonzero(ok[1])[0], [0, 1, 2, 3])
    assert np.array_equal(np.nonzero(ok[2])[0], [0, 1, 6, 7, 8, 9])
    assert O.visible([5], 6, tokens=1).all()


def test_oracle_attention_is_softmax():
    rng = np.random.default_rng(2)
    q, k, v = (rng.standard_normal((5, h, 128)) for h in (4, 2, 2))
    ok = np.tril(np.ones((5, 5), bool))
    ok[2] = False
    out, tol = O.attention(q, k, v, ok)
    for r in range(5):
        for h in range(4):
            if r == 2:
                assert np.all(out[r, h] == 0)
                continue
            s = k[: r + 1, h // 2] @ q[r, h] / np.sqrt(128)
            w = np.exp(s - s.max())
            assert np.allclose(out[r, h], w @ v[: r + 1, h // 2] / w.sum(), atol=1e-12)
    assert np.all(tol >= 0)


def test_packed_arguments_are_the_c_structures():
    """kvp.kv4 packs its arguments; the layouts are those of include/kvp.h."""
    from kvp import kv4
    s = Kv4Span(1, 2, 3, 4, 5, 6, 7, 8, 9, 10)
    assert kv4._SPAN(1, 2, 3, 4, 5, 6, 7, 8, 9, 10) == bytes(s)
    r = Kv4Rows(1, 2, 3, 4, 5)
    assert kv4._ROWS(1, 2, 3, 4, 5) == bytes(r)
    a = Kv4Attn(1, 2, 3, 4, 5, 6, 7, 8, 9, 10)
    assert kv4._ATTN(1, 2, 3, 4, 5, 6, 7, 8, 9, 10) == bytes(a)
