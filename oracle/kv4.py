"""CPU restatement of the 4-bit K/V cache and of attention over it, in 64
bits (the format's definition: include/kvp.h and csrc/kv4.h).

* ``quantise`` / ``values`` -- rows to codes and scale bytes and back
* ``put`` / ``get``         -- rows into and out of a pool's bytes
* ``attention``             -- block-causal attention with window and sinks,
  and the bound on a bf16 kernel's error that its roundings imply
"""

from __future__ import annotations

import math

import numpy as np
import torch

PAGE, HEAD, PAGE_HEAD, BLOCK = 128, 128, 18432, 1152
SCALES = np.array([(1 + m / 8) * 2.0 ** (e - 15) for e in range(32) for m in range(8)])
TOP_BYTE = 215                                   # the largest scale that is written
TOP = 7 * SCALES[TOP_BYTE]


def bf16(x: np.ndarray) -> np.ndarray:
    return torch.from_numpy(np.ascontiguousarray(x, np.float32)).to(torch.bfloat16).double().numpy()


def quantise(x: np.ndarray):
    """x [..., 128] -> integers n [..., 128] in [-7, 7], scale bytes [..., 8]."""
    x = bf16(x)
    x = np.clip(np.where(np.isnan(x), 0.0, x), -TOP, TOP)
    g = x.reshape(*x.shape[:-1], 8, 16)
    want = np.abs(g).max(-1) / 7
    # nearest scale, the upper one half-way (want * 7 and the bounds are exact)
    s = SCALES[: TOP_BYTE + 1]
    middle = (s[1:] + s[:-1]) / 2 * 7
    byte = np.searchsorted(middle, np.abs(g).max(-1), side="right")
    assert byte.shape == want.shape
    r = np.abs(g) / SCALES[byte][..., None]            # exact enough: halves are exact quotients
    n = np.sign(g) * np.floor(r + 0.5)
    assert np.abs(n).max(initial=0) <= 7
    return n.reshape(x.shape).astype(np.int64), byte.astype(np.uint8)


def values(n: np.ndarray, byte: np.ndarray) -> np.ndarray:
    return (n.reshape(*n.shape[:-1], 8, 16) * SCALES[byte][..., None]).reshape(n.shape)


def _at(which: str, row: int, dim: int):
    """Byte and nibble of a code, byte of its scale, inside an 8-row block."""
    word, d = divmod(dim, 8)
    bit = 4 * (d // 2) + 16 * (d % 2)
    grp = dim // 16
    if which == "k":
        return row * 64 + word * 4 + bit // 8, bit % 8, 512 + row * 8 + grp
    return 576 + grp * 64 + row * 8 + (word % 2) * 4 + bit // 8, bit % 8, 1088 + grp * 8 + row


_TAB = {w: np.array([[_at(w, r, d) for d in range(HEAD)] for r in range(8)]) for w in "kv"}


def put(pages: np.ndarray, page: int, row: int, which: str, x: np.ndarray) -> None:
    """One row x [kv_heads * 128] into row `row` of a page (uint8 [n, heads, 18432])."""
    heads = pages.shape[1]
    n, byte = quantise(x.reshape(heads, HEAD))
    blk, r = divmod(row, 8)
    for d in range(HEAD):
        at, bit, sc = _TAB[which][r, d]
        b = pages[page, :, blk * BLOCK + at]
        pages[page, :, blk * BLOCK + at] = (b & ~np.uint8(15 << bit)) | ((n[:, d] + 8) << bit).astype(np.uint8)
        pages[page, :, blk * BLOCK + sc] = byte[:, d // 16]


def get(pages: np.ndarray, page_ids, which: str) -> np.ndarray:
    """All rows of the pages: float64 [len(page_ids) * 128, heads, 128]."""
    t = pages[np.asarray(page_ids)].reshape(len(page_ids), pages.shape[1], 16, BLOCK)
    at, bit, sc = (_TAB[which][..., i] for i in range(3))
    n = ((t[..., at] >> bit.astype(np.uint8)) & 15).astype(np.int64) - 8
    # [page, head, block, row, dim]; V's scale bytes count up to the largest that is written
    x = n * SCALES[t[..., sc] if which == "k" else np.minimum(t[..., sc], TOP_BYTE)]
    return x.transpose(0, 2, 3, 1, 4).reshape(-1, pages.shape[1], HEAD)


def visible(pos, end: int, *, tokens: int, window: int = 0, sinks: int = 0) -> np.ndarray:
    """bool [len(pos), end]: which keys the queries at positions pos see."""
    pos = np.asarray(pos)[:, None]
    key = np.arange(end)[None, :]
    f, kf = pos // tokens, key // tokens
    ok = kf <= f
    if window:
        ok &= (kf > f - window) | (kf < sinks)
    return ok


def attention(q, k, v, ok):
    """q [rows, heads, 128], k / v [keys, kv_heads, 128], ok bool [rows, keys]
    -> out [rows, heads, 128] and a bound on |kernel - out|.

    The bound counts the kernels' roundings, each at most half a step.
    Weights P to fp16, the largest of a row at 2^7 or above: 2^-11 of each, or
    half of fp16's smallest step of 2^-24, which is 2^-25 / 2^7 = 2^-32 of the
    largest and so of the sum of the weights, for every key: 2^-32 sum |v|.
    These enter the numerator alone.  The scores' fp32 sums of 128 products
    (each partial sum off by 2^-23 of the sum of magnitudes, so a weight by d =
    130 * 2^-23 * max sum |q k| / sqrt(128)), the exponent's argument and the
    exponential itself (2^-21 (1 + max |score|)): numerator and denominator.  The
    sums over keys: 2^-23 each, at most 2^9 deep.  V is exact.  The result to
    bf16: 2^-8 of it, the errors before included."""
    q, k, v = (torch.as_tensor(np.asarray(x, np.float64)) for x in (q, k, v))
    ok = torch.as_tensor(ok)
    rows, heads = q.shape[:2]
    kvh = k.shape[1]
    grp = heads // kvh
    out = torch.zeros(rows, heads, HEAD, dtype=torch.float64)
    tol = torch.zeros_like(out)
    for h in range(heads):
        kk, vv = k[:, h // grp], v[:, h // grp]
        s = (q[:, h] @ kk.T / math.sqrt(HEAD)).masked_fill(~ok, -math.inf)
        m = s.amax(-1, keepdim=True) if s.shape[1] else torch.full((rows, 1), -math.inf, dtype=torch.float64)
        w = torch.exp(s - torch.where(m == -math.inf, 0.0, m))
        tot = w.sum(-1, keepdim=True)
        w = w / torch.where(tot == 0, 1.0, tot)
        o = w @ vv
        a = w @ vv.abs()
        mag = (q[:, h].abs() @ kk.abs().T / math.sqrt(HEAD)).masked_fill(~ok, 0.0)
        mag = mag.amax(-1, keepdim=True) if mag.shape[1] else torch.zeros(rows, 1, dtype=torch.float64)
        d = 130 * 2.0 ** -23 * mag + 2.0 ** -21 * (1 + mag)
        out[:, h] = o
        before = (2.0 ** -11 + 2 * d + 2.0 ** -14) * a + 2.0 ** -32 * (ok.double() @ vv.abs())
        tol[:, h] = (1 + 2.0 ** -8) * before + 2.0 ** -8 * o.abs()
    return out.numpy(), tol.numpy()
