"""The 4-bit K/V cache and attention over it (kvp_kv4_write, kvp_kv4_read,
kvp_attn_kv4; include/kvp.h).

A cache is a pool of pages of 128 rows, a uint8 CUDA tensor [n_pages,
kv_heads, 18432] (``alloc_pages``), and an int32 page map [batch, pages] that
gives each sequence's pages in order (None: sequence b owns pages b *
(n_pages // batch) and up).  Rows are [batch, rows, heads * 128] or, for one
sequence, [rows, heads * 128]; only their last dimension has to be
contiguous, so slices of a fused QKV buffer work, V beside a K of its own
too.  A call touches the rows [start, start + rows) of every sequence;
``starts`` (int32 device tensor [batch]) gives each sequence its own start,
``counts`` fewer rows.

    pages = kv4.alloc_pages(n, kv_heads)
    kv4.write(pages, k, v, page_map=m, start=s)          # the new rows
    kv4.attn(q, pages, out, page_map=m, heads=h, start=s, tokens=1560, window=6, sinks=1)

Everything is queued on the current stream of the tensors' device, or on
``stream`` (a raw cudaStream_t).  Fails loudly without libkvp.so.
"""

from __future__ import annotations

import struct

import torch

from . import KvpError
from ._lib import check, lib

PAGE_ROWS = 128
PAGE_HEAD_BYTES = 18432

_ROW_TYPES = (torch.bfloat16, torch.float32)
_Q_TYPES = (torch.bfloat16,)
_MAX_INT = 2 ** 31
# kvp_kv4_span, kvp_kv4_rows and kvp_kv4_attn in native layout (a packed
# bytes object costs a fifth of a filled ctypes structure)
_SPAN = struct.Struct("@PPPPqiiiii4x").pack
_ROWS = struct.Struct("@PPqqi4x").pack
_ATTN = struct.Struct("@PPqqqqiiii").pack
# the current stream's handle without building a Stream object, the current
# device without asking whether CUDA is up (a tensor is on it)
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or \
    (lambda dev: torch.cuda.current_stream(dev).cuda_stream)
_current_device = getattr(torch._C, "_cuda_getDevice", None) or torch.cuda.current_device


def alloc_pages(n_pages: int, kv_heads: int, device="cuda"):
    """An unwritten pool (any bytes stand for finite values)."""
    return torch.empty(n_pages, kv_heads, PAGE_HEAD_BYTES, dtype=torch.uint8, device=device)


def _bad(what: str):
    raise KvpError(f"kv4: {what}")


def _ints(t, name: str, batch: int, dev: int, dims: int) -> int:
    shape = t.shape
    if t.dtype is not torch.int32 or len(shape) != dims or shape[0] != batch or not t.is_contiguous():
        _bad(f"{name} must be a contiguous int32 [{batch}{', pages' if dims == 2 else ''}] tensor")
    if t.get_device() != dev:
        _bad(f"tensors on {t.device} and cuda:{dev}")
    return t.data_ptr()


def _args(pages, a, b, names: str, types, heads, page_map, start: int, starts, counts):
    """Checks the pool, the row tensors a and b (b may be None; heads None: the
    pool's) and the rest; (device, packed span, a's row and batch stride, b's).
    One function, because calls of several cost a microsecond of the seven that
    a call of the package takes."""
    shape = pages.shape
    if len(shape) != 3 or shape[2] != PAGE_HEAD_BYTES or pages.dtype is not torch.uint8 or \
            not pages.is_contiguous():
        _bad(f"pages must be a contiguous uint8 [n_pages, kv_heads, {PAGE_HEAD_BYTES}] tensor")
    n_pages, kv_heads, _ = shape
    width = (kv_heads if heads is None else heads) * 128
    shape, strides, dtype = a.shape, a.stride(), a.dtype
    if dtype not in types:
        _bad(f"{names} of {dtype}, expected one of {[str(d) for d in types]}")
    if len(shape) == 3:
        batch, rows, d = shape
        bs, rs, es = strides
    elif len(shape) == 2:
        batch, bs = 1, 0
        rows, d = shape
        rs, es = strides
    else:
        _bad(f"{names} must be [rows, heads * 128] or [batch, rows, heads * 128]")
    if d != width or es != 1:
        _bad(f"{names} need {width // 128} heads of 128 contiguous elements, got {tuple(shape)}")
    b_rs, b_bs = rs, bs
    if b is not None:
        if b.dtype is not dtype or b.shape != shape:
            _bad(f"{names} must agree in shape and type")
        if (other := b.stride()) != strides:
            if other[-1] != 1:
                _bad(f"{names} need {width // 128} heads of 128 contiguous elements")
            b_rs, b_bs = other[-2], other[0] if len(other) == 3 else 0
    # the strides of single rows and sequences mean nothing
    if rows < 2:
        rs = b_rs = width
    if batch < 2:
        bs = b_bs = 0
    dev = pages.get_device()
    if dev < 0:
        _bad("pages must be a CUDA tensor")
    if a.get_device() != dev or (b is not None and b.get_device() != dev):
        _bad(f"tensors on {a.device if b is None else f'{a.device}, {b.device}'} and cuda:{dev}")
    if page_map is None:
        stride, map_ptr = n_pages // max(batch, 1), 0
    else:
        map_ptr = _ints(page_map, "page_map", batch, dev, 2)
        stride = page_map.shape[1]
    if not (0 <= start < _MAX_INT and rows < _MAX_INT and stride < _MAX_INT and batch < _MAX_INT):
        _bad(f"start {start}, rows {rows}, batch {batch} or {stride} pages out of range")
    return dev, _SPAN(pages.data_ptr(), map_ptr,
                      0 if starts is None else _ints(starts, "starts", batch, dev, 1),
                      0 if counts is None else _ints(counts, "counts", batch, dev, 1),
                      n_pages, kv_heads, batch, stride, start, rows), rs, bs, b_rs, b_bs


def _call(fn, what, dev, stream, *args):
    if dev == _current_device():
        rc = fn(*args, _raw_stream(dev) if stream is None else stream)
    else:
        with torch.cuda.device(dev):
            rc = fn(*args, _raw_stream(dev) if stream is None else stream)
    if rc < 0:
        check(rc, what)


def _kv(pages, k, v, page_map, start, starts, counts):
    """Checks; (device, packed span, packed rows, v's rows if their strides are others)."""
    some, other = (k, v) if k is not None else (v, None)
    if some is None:
        _bad("no rows")
    dev, span, rs, bs, v_rs, v_bs = _args(pages, some, other, "k and v", _ROW_TYPES, None, page_map, start, starts,
                                          counts)
    k_at, v_at, size = 0 if k is None else k.data_ptr(), 0 if v is None else v.data_ptr(), some.element_size()
    if other is not None and (rs != v_rs or bs != v_bs):
        return dev, span, _ROWS(k_at, 0, rs, bs, size), _ROWS(0, v_at, v_rs, v_bs, size)
    return dev, span, _ROWS(k_at, v_at, rs, bs, size), None


def write(pages, k, v, *, page_map=None, start: int = 0, starts=None, counts=None,
          stream=None) -> None:
    """Quantises rows k, v (bf16 or fp32) into the cache."""
    if k is None or v is None:
        _bad("write needs k and v")
    dev, span, rows, v_rows = _kv(pages, k, v, page_map, start, starts, counts)
    if v_rows is None:
        _call(lib().kvp_kv4_write, "kvp_kv4_write", dev, stream, span, rows)
    else:
        _call(lib().kvp_kv4_write_kv, "kvp_kv4_write_kv", dev, stream, span, rows, v_rows)


def read(pages, k, v, *, page_map=None, start: int = 0, starts=None, counts=None,
         stream=None) -> None:
    """Fills k and v (bf16 or fp32; either may be None) with the rows' values."""
    dev, span, rows, v_rows = _kv(pages, k, v, page_map, start, starts, counts)
    if v_rows is not None and k.data_ptr() == v.data_ptr():
        _bad("the output rows overlap")
    _call(lib().kvp_kv4_read, "kvp_kv4_read", dev, stream, span, rows)
    if v_rows is not None:
        _call(lib().kvp_kv4_read, "kvp_kv4_read", dev, stream, span, v_rows)


def attn(q, pages, out, *, heads: int, page_map=None, start: int = 0, starts=None, counts=None,
         tokens: int = 1, window: int = 0, sinks: int = 0, stream=None) -> None:
    """out = attention of query rows q (bf16) over the cache: the row at
    position p, in frame f = p // tokens, sees the cached rows up to the end of
    its frame (and of this call's rows) that lie in the last `window` frames
    (0: all) or the first `sinks` frames.  The call's own rows are keys: write
    them first.  out may be q."""
    dev, span, qr, qb, orow, obatch = _args(pages, q, out, "q and out", _Q_TYPES, heads, page_map, start, starts,
                                            counts)
    if not (0 < tokens < _MAX_INT and 0 <= window < _MAX_INT and 0 <= sinks < _MAX_INT):
        _bad(f"tokens {tokens}, window {window} or sinks {sinks} out of range")
    _call(lib().kvp_attn_kv4, "kvp_attn_kv4", dev, stream, span,
          _ATTN(q.data_ptr(), out.data_ptr(), qr, qb, orow, obatch, heads, tokens, window, sinks))
