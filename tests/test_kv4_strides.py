"""K and V rows of different strides: what kvp_kv4_write_kv and kvp.kv4 refuse and pass on (CPU only)."""

from __future__ import annotations

import ctypes as C

import pytest
import torch

from kvp._lib import Kv4Rows, Kv4Span, KvpError, lib

ERR_ARG = -1
SPAN = Kv4Span(0x10000, 0x20000, 0, 0, 8, 2, 2, 4, 5, 100)
K = dict(k=0x30000, v=0, row_stride=256, batch_stride=25600, elem_bytes=2)
V = dict(k=0, v=0x40000, row_stride=768, batch_stride=76800, elem_bytes=2)


@pytest.mark.parametrize("k,v", [
    (dict(k=0), {}), ({}, dict(v=0)), (dict(k=0x30008), {}), ({}, dict(v=0x40008)),
    ({}, dict(elem_bytes=4)), (dict(elem_bytes=3), dict(elem_bytes=3)),
    (dict(row_stride=128), {}), ({}, dict(row_stride=128)), ({}, dict(row_stride=770)),
    (dict(batch_stride=-25600), {}), ({}, dict(batch_stride=-8)), ({}, dict(batch_stride=4)),
])
def test_refusals(k, v):
    L = lib()
    assert L.kvp_kv4_write_kv(C.byref(SPAN), C.byref(Kv4Rows(**{**K, **k})), C.byref(Kv4Rows(**{**V, **v})), None) == ERR_ARG
    assert b"kv4_write" in L.kvp_last_error()


def test_missing_structures():
    L, k, v = lib(), Kv4Rows(**K), Kv4Rows(**V)
    for args in ((None, C.byref(k), C.byref(v)), (C.byref(SPAN), None, C.byref(v)), (C.byref(SPAN), C.byref(k), None)):
        assert L.kvp_kv4_write_kv(*args, None) == ERR_ARG


@pytest.fixture
def calls(monkeypatch):
    """kvp.kv4 with tensors that claim to be on device 0; the library's calls."""
    from kvp import kv4
    seen = []
    monkeypatch.setattr(kv4, "_call", lambda fn, what, dev, stream, span, *rows: seen.append((what, rows)))
    monkeypatch.setattr(torch.Tensor, "get_device", lambda self: 0)
    return kv4, seen


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_what_is_passed_on(calls, dtype):
    kv4, seen = calls
    pages = torch.zeros(4, 2, kv4.PAGE_HEAD_BYTES, dtype=torch.uint8)
    k = torch.zeros(2, 5, 256, dtype=dtype)
    v = torch.zeros(2, 5, 768, dtype=dtype)[..., 512:]
    size = k.element_size()
    kv4.write(pages, k, v)
    kv4.write(pages, k, torch.zeros_like(k))
    kv4.read(pages, k, v)
    kv4.read(pages, k, None)
    apart = (kv4._ROWS(k.data_ptr(), 0, 256, 1280, size), kv4._ROWS(0, v.data_ptr(), 768, 3840, size))
    assert [w for w, _ in seen] == ["kvp_kv4_write_kv", "kvp_kv4_write", "kvp_kv4_read", "kvp_kv4_read", "kvp_kv4_read"]
    assert seen[0][1] == apart and (seen[2][1] + seen[3][1]) == apart
    assert seen[4][1] == (apart[0],)
    with pytest.raises(KvpError, match="overlap"):
        kv4.read(pages, k, torch.as_strided(k, (2, 5, 256), (256, 512, 1)))
    # strides of single rows and sequences mean nothing
    del seen[:]
    kv4.write(pages, k[:1, :1], v[:1, :1])
    assert [w for w, _ in seen] == ["kvp_kv4_write"]


@pytest.mark.parametrize("stream", [None, 77])
def test_a_call_on_another_device_than_the_current_one(monkeypatch, stream):
    """The device is made current for the call, and its current stream is the call's."""
    from kvp import kv4
    log = []

    class Device:
        def __init__(self, d): self.d = d
        def __enter__(self): log.append(("enter", self.d))
        def __exit__(self, *a): log.append(("exit", self.d))

    monkeypatch.setattr(kv4, "_current_device", lambda: 0)
    monkeypatch.setattr(kv4, "_raw_stream", lambda dev: 1000 + dev)
    monkeypatch.setattr(torch.cuda, "device", Device)
    fn = lambda *a: log.append(a) or 0
    kv4._call(fn, "kvp_kv4_write", 1, stream, b"span", b"rows")
    assert log == [("enter", 1), (b"span", b"rows", 1001 if stream is None else stream), ("exit", 1)]
    del log[:]
    kv4._call(fn, "kvp_kv4_write", 0, stream, b"span", b"rows")
    assert log == [(b"span", b"rows", 1000 if stream is None else stream)]
    with pytest.raises(RuntimeError):                # (KvpError; other tests reload the module that defines it)
        kv4._call(lambda *a: -1, "kvp_kv4_write", 1, stream, b"span", b"rows")
    assert log[-1] == ("exit", 1)
