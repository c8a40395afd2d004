"""Caches in which every key shows: key j of a head has one value other than
0 in V, at dim (5 j + 3 j // 128 + 11 h) % 128 and of either sign, and K is
small enough that no weight is far from its neighbours'.  A dim then sums every
128th key, so that a key that is lost, or seen where it is hidden, changes it by
more than the roundings that oracle.kv4.attention counts, up to tens of thousands
of keys (test_kv4_keys.py)."""

from __future__ import annotations

import numpy as np

from oracle import kv4 as O

ONE = 8 * 15                     # the scale byte of 1.0


def dim_of(key, head):
    return (5 * key + 3 * (key // 128) + 11 * head) % 128


def telling_pool(rng, page_map, n_pages, heads):
    """Pages of batch * per * 128 keys as above, uint8 [n_pages, heads, 18432]."""
    pages = np.zeros((n_pages, heads, 16, O.BLOCK), np.uint8)
    pages[..., :512] = rng.integers(1, 256, pages[..., :512].shape)
    pages[..., 512:576] = rng.integers(8 * 11, 8 * 12, pages[..., 512:576].shape)     # 2^-4 .. 2^-3
    pages[..., 576:1088] = 0x88
    pages[..., 1088:] = ONE
    at = O._TAB["v"]                                                # [row, dim]: byte, bit, scale byte
    for seq in page_map:
        key = np.arange(len(seq) * 128)
        for h in range(heads):
            byte, bit, _ = at[key % 8, dim_of(key, h)].T
            code = np.where(rng.random(len(key)) < 0.5, rng.integers(1, 4, len(key)), rng.integers(13, 16, len(key)))
            where = (seq[key // 128], h, key % 128 // 8, byte)
            pages[where] = (0x88 & ~(15 << bit)) | (code << bit)
    return pages.reshape(n_pages, heads, O.PAGE_HEAD)


def telling_queries(rng, *shape):
    """Query rows that give K of telling_pool scores of at most a few tenths."""
    return (0.25 * rng.standard_normal(shape)).astype(np.float32)
