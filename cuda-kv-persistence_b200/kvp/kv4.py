"""The 4-bit K/V cache and attention over it (kvp_kv4_write, kvp_kv4_read,
kvp_attn_kv4; include/kvp.h).

A cache is a pool of pages of 128 rows, a uint8 CUDA tensor [n_pages,
kv_heads, 18432] (``alloc_pages``), and an int32 page map [batch, pages] that
gives each sequence's pages in order (None: sequence b owns pages b *
(n_pages // batch) and up).  Rows are [batch, rows, heads * 128] or, for one
sequence, [rows, heads * 128]; only their last dimension has to be
contiguous, so slices of a fused QKV buffer work.  A call touches the rows
[start, start + rows) of every sequence; ``starts`` (int32 device tensor
[batch]) gives each sequence its own start, ``counts`` fewer rows.

    pages = kv4.alloc_pages(n, kv_heads)
    kv4.write(pages, k, v, page_map=m, start=s)          # the new rows
    kv4.attn(q, pages, out, page_map=m, heads=h, start=s, tokens=1560, window=6, sinks=1)

Everything is queued on the current stream of the tensors' device, or on
``stream`` (a raw cudaStream_t).  Fails loudly without libkvp.so.
"""

from __future__ import annotations

import ctypes as C

from ._lib import Kv4Attn, Kv4Rows, Kv4Span, KvpError, check, lib

PAGE_ROWS = 128
PAGE_HEAD_BYTES = 18432


def alloc_pages(n_pages: int, kv_heads: int, device="cuda"):
    """An unwritten pool (any bytes stand for finite values)."""
    import torch
    return torch.empty(n_pages, kv_heads, PAGE_HEAD_BYTES, dtype=torch.uint8, device=device)


def _bad(what: str):
    raise KvpError(f"kv4: {what}")


def _rows3(t, name: str, dtypes, heads: int):
    """(batch, rows, row stride, batch stride) of a row tensor."""
    if t.dtype not in dtypes:
        _bad(f"{name} is {t.dtype}, expected one of {[str(d) for d in dtypes]}")
    if t.dim() == 2:
        b, (n, d), rs, bs = 1, t.shape, t.stride(0), 0
    elif t.dim() == 3:
        (b, n, d), rs, bs = t.shape, t.stride(1), t.stride(0)
    else:
        _bad(f"{name} must be [rows, heads * 128] or [batch, rows, heads * 128]")
    if d != heads * 128 or t.stride(-1) != 1:
        _bad(f"{name} needs {heads} heads of 128 contiguous elements, got {tuple(t.shape)}")
    # the strides of single rows and sequences mean nothing
    return b, n, rs if n > 1 else d, bs if b > 1 else 0


def _span(pages, batch: int, rows: int, page_map, start: int, starts, counts, tensors):
    import torch
    if pages.dtype != torch.uint8 or pages.dim() != 3 or pages.shape[2] != PAGE_HEAD_BYTES or \
            not pages.is_contiguous():
        _bad(f"pages must be a contiguous uint8 [n_pages, kv_heads, {PAGE_HEAD_BYTES}] tensor")
    dev = pages.device
    if dev.type != "cuda":
        _bad("pages must be a CUDA tensor")
    n_pages = pages.shape[0]
    if page_map is None:
        stride = n_pages // batch if batch else n_pages
    else:
        if page_map.dtype != torch.int32 or page_map.dim() != 2 or page_map.shape[0] != batch or \
                not page_map.is_contiguous():
            _bad(f"page_map must be a contiguous int32 [{batch}, pages] tensor")
        stride = page_map.shape[1]
    for t, name in ((starts, "starts"), (counts, "counts")):
        if t is not None and (t.dtype != torch.int32 or tuple(t.shape) != (batch,) or
                              not t.is_contiguous()):
            _bad(f"{name} must be a contiguous int32 [{batch}] tensor")
    for t in (page_map, starts, counts, *tensors):
        if t is not None and t.device != dev:
            _bad(f"tensors on {t.device} and {dev}")
    if not (0 <= start < 2 ** 31 and rows < 2 ** 31):
        _bad(f"start {start}, rows {rows} out of range")
    return Kv4Span(pages.data_ptr(), 0 if page_map is None else page_map.data_ptr(),
                   0 if starts is None else starts.data_ptr(),
                   0 if counts is None else counts.data_ptr(), n_pages, pages.shape[1], batch,
                   stride, start, rows)


def _call(fn, what, dev, stream, *args):
    import torch
    if stream is None:
        stream = torch.cuda.current_stream(dev).cuda_stream
    if dev.index == torch.cuda.current_device():
        check(fn(*args, int(stream)), what)
    else:
        with torch.cuda.device(dev):
            check(fn(*args, int(stream)), what)


def _kv(pages, k, v, page_map, start, starts, counts):
    import torch
    some = k if k is not None else v
    if some is None:
        _bad("no rows")
    if pages.dim() != 3:
        _bad("pages must be [n_pages, kv_heads, bytes]")
    heads = pages.shape[1]
    types = (torch.bfloat16, torch.float32)
    shape = _rows3(some, "k" if k is not None else "v", types, heads)
    if k is not None and v is not None and (_rows3(v, "v", types, heads) != shape or
                                            k.dtype != v.dtype):
        _bad("k and v must agree in shape, strides and type")
    b, n, rs, bs = shape
    span = _span(pages, b, n, page_map, start, starts, counts, (k, v))
    rows = Kv4Rows(0 if k is None else k.data_ptr(), 0 if v is None else v.data_ptr(), rs, bs,
                   some.element_size())
    return span, rows


def write(pages, k, v, *, page_map=None, start: int = 0, starts=None, counts=None,
          stream=None) -> None:
    """Quantises rows k, v (bf16 or fp32) into the cache."""
    if k is None or v is None:
        _bad("write needs k and v")
    span, rows = _kv(pages, k, v, page_map, start, starts, counts)
    _call(lib().kvp_kv4_write, "kvp_kv4_write", pages.device, stream, C.byref(span), C.byref(rows))


def read(pages, k, v, *, page_map=None, start: int = 0, starts=None, counts=None,
         stream=None) -> None:
    """Fills k and v (bf16 or fp32; either may be None) with the rows' values."""
    span, rows = _kv(pages, k, v, page_map, start, starts, counts)
    _call(lib().kvp_kv4_read, "kvp_kv4_read", pages.device, stream, C.byref(span), C.byref(rows))


def attn(q, pages, out, *, heads: int, page_map=None, start: int = 0, starts=None, counts=None,
         tokens: int = 1, window: int = 0, sinks: int = 0, stream=None) -> None:
    """out = attention of query rows q (bf16) over the cache: the row at
    position p, in frame f = p // tokens, sees the cached rows up to the end of
    its frame (and of this call's rows) that lie in the last `window` frames (0: all) or the
    first `sinks` frames.  The call's own rows are keys: write them first."""
    import torch
    bf = (torch.bfloat16,)
    b, n, qr, qb = _rows3(q, "q", bf, heads)
    ob, on, orow, obatch = _rows3(out, "out", bf, heads)
    if (ob, on) != (b, n):
        _bad("q and out must agree in shape")
    span = _span(pages, b, n, page_map, start, starts, counts, (q, out))
    a = Kv4Attn(q.data_ptr(), out.data_ptr(), qr, qb, orow, obatch, heads, tokens, window, sinks)
    _call(lib().kvp_attn_kv4, "kvp_attn_kv4", pages.device, stream, C.byref(span), C.byref(a))
