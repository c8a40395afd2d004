"""The 4-bit K/V cache and attention over it on a device (kvp.kv4) against
the 64-bit restatement in oracle/kv4.py.

Writes are compared byte for byte over the whole pool, reads value for value;
attention within the bound that oracle.kv4.attention derives from its
roundings."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import kv4 as O

pytestmark = pytest.mark.gpu

BF, F32 = torch.bfloat16, torch.float32


def _pool(rng, n, heads):
    """Pages of arbitrary bytes."""
    return rng.integers(0, 256, (n, heads, O.PAGE_HEAD), dtype=np.uint8)


def _calm_pool(rng, n, heads):
    """Pages whose rows are all quantised normal values (fast: scales and codes drawn)."""
    p = _pool(rng, n, heads).reshape(n, heads, 16, O.BLOCK)
    for a, b in ((512, 576), (1088, 1152)):
        p[..., a:b] = rng.integers(8 * 12, 8 * 14, p[..., a:b].shape)   # scales 2^-3 .. 2^-1
    return p.reshape(n, heads, O.PAGE_HEAD)


def _map(rng, batch, per, n):
    return rng.permutation(n)[: batch * per].reshape(batch, per).astype(np.int32)


def _status():
    from kvp.attention import read_status
    return read_status()


@pytest.fixture(autouse=True)
def _clean(cuda):
    _status()
    yield


def _expect_write(pages, m, starts, counts, k, v):
    want = pages.copy()
    for b in range(m.shape[0]):
        for i in range(counts[b]):
            page, row = m[b, (starts[b] + i) // 128], (starts[b] + i) % 128
            if 0 <= page < pages.shape[0]:
                O.put(want, page, row, "k", k[b, i])
                O.put(want, page, row, "v", v[b, i])
    return want


WRITES = [  # batch, heads, start, rows
    (1, 1, 0, 1), (1, 12, 4095, 1), (3, 2, 127, 2), (2, 3, 5, 8), (1, 2, 8, 16), (2, 2, 121, 150),
    (1, 5, 0, 129), (1, 1, 250, 300),
]


@pytest.mark.parametrize("batch,heads,start,rows", WRITES)
@pytest.mark.parametrize("dtype", [BF, F32])
def test_write_then_read(batch, heads, start, rows, dtype):
    from kvp import kv4
    rng = np.random.default_rng(start + rows)
    per = -(-(start + rows) // 128)
    pages = _pool(rng, batch * per + 2, heads)
    m = _map(rng, batch, per, batch * per + 2)
    x = [torch.from_numpy(rng.standard_normal((batch, rows, heads * 128)).astype(np.float32) *
                          np.exp2(rng.uniform(-6, 6, (batch, rows, 1))).astype(np.float32)).to(dtype)
         for _ in range(2)]
    dev = torch.from_numpy(pages).cuda()
    mm = torch.from_numpy(m).cuda()
    kv4.write(dev, x[0].cuda(), x[1].cuda(), page_map=mm, start=start)
    want = _expect_write(pages, m, [start] * batch, [rows] * batch, *(t.float().numpy() for t in x))
    assert np.array_equal(dev.cpu().numpy(), want)
    out = [torch.full((batch, rows, heads * 128), 7.0, dtype=dtype, device="cuda") for _ in range(2)]
    kv4.read(dev, *out, page_map=mm, start=start)
    for t, w in zip(out, "kv"):
        for b in range(batch):
            ref = O.get(want, m[b], w)[start: start + rows].reshape(rows, -1)
            assert np.array_equal(t[b].double().cpu().numpy(), ref)
    assert _status() == 0


def test_write_ties_zeros_and_tiny_values():
    """Exact halves of a step (both signs), halves between two scales, zero
    groups, denormals, values at the format's two ends."""
    from kvp import kv4
    rows = []
    for s in (1.0, 1.125, 1.875, 2.0 ** -15, 1.5 * 2.0 ** -9, 3840.0):
        g = np.zeros(128)
        g[:16] = np.array([7, -7, 6.5, -6.5, 0.5, -0.5, 1.5, -1.5, 2.5, 3.5, -4.5, 5.5, 0, 0.25, 0.75, -0.75]) * s
        rows.append(g)
    for q in range(8, 16):                                # amax / 7 half-way between two scales
        g = np.zeros(128)
        g[0], g[17], g[33] = 7 * (q + 0.5) / 8, 7 * (q + 0.5) / 8 * (1 + 2.0 ** -7), 7 * (q + 0.5) / 8 * (1 - 2.0 ** -7)
        rows.append(g)
    rows.append(np.zeros(128))
    rows.append(np.full(128, 1e-40))
    rows.append(np.full(128, -2.0 ** -17))
    rows.append(np.linspace(-26880, 26880, 128))
    x = torch.from_numpy(np.array(rows, np.float32)).to(BF)
    pages = np.zeros((1, 1, O.PAGE_HEAD), np.uint8)
    dev = torch.from_numpy(pages).cuda()
    kv4.write(dev, x.cuda(), (-x).cuda())
    want = _expect_write(pages, np.zeros((1, 1), int), [0], [len(rows)], x[None].float().numpy(),
                         -x[None].float().numpy())
    assert np.array_equal(dev.cpu().numpy(), want)
    assert _status() == 0


def test_write_every_bf16_mantissa():
    """All 256 positive mantissas of two binades as group maxima, and as members under a fixed maximum."""
    from kvp import kv4
    vals = torch.arange(0x3F00, 0x4100, dtype=torch.int32).to(torch.int16).view(BF).float().numpy()  # [0.5, 8)
    x = np.zeros((len(vals), 128), np.float32)
    x[:, 0::16] = vals[:, None]
    x[:, 1::16] = vals[:, None] * 0.5
    x[:, 2::16] = -np.abs(vals[::-1, None])
    for g in range(8):
        x[:, 16 * g + 3] = [3.5, 7, 7.875, 6.5625, 13, 26.25, 49, 56][g]
    t = torch.from_numpy(x).to(BF)
    pages = np.zeros((4, 1, O.PAGE_HEAD), np.uint8)
    dev = torch.from_numpy(pages).cuda()
    kv4.write(dev, t.cuda(), t.cuda())
    want = _expect_write(pages, np.arange(4)[None], [0], [len(vals)], t[None].float().numpy(), t[None].float().numpy())
    assert np.array_equal(dev.cpu().numpy(), want)


@pytest.mark.parametrize("value", [float("nan"), float("inf"), -float("inf"), 27136.0, -3e38])
@pytest.mark.parametrize("dtype", [BF, F32])
def test_write_of_values_beyond_the_format(value, dtype):
    from kvp import kv4
    x = torch.randn(3, 128, generator=torch.Generator().manual_seed(0)).to(dtype)
    x[1, 37] = value
    pages = np.zeros((1, 1, O.PAGE_HEAD), np.uint8)
    dev = torch.from_numpy(pages).cuda()
    kv4.write(dev, x.cuda(), x.cuda())
    want = _expect_write(pages, np.zeros((1, 1), int), [0], [3], x[None].float().numpy(), x[None].float().numpy())
    assert np.array_equal(dev.cpu().numpy(), want)
    assert _status() == 8


def test_write_strided_rows_device_starts_counts_and_bad_pages():
    from kvp import kv4
    rng = np.random.default_rng(9)
    batch, heads, rows, per = 5, 2, 140, 4
    n = batch * per
    pages = _pool(rng, n, heads)
    m = _map(rng, batch, per, n)
    m[0, 1] = -1
    m[1, 1] = n
    starts = np.array([120, 120, 0, 372, -1], np.int32)
    counts = np.array([140, 20, 0, 140, 3], np.int32)
    fused = torch.from_numpy(rng.standard_normal((batch, rows, 3 * heads * 128)).astype(np.float32)).to(BF)
    k, v = fused[..., 256:512], fused[..., 512:]
    dev = torch.from_numpy(pages).cuda()
    fd = fused.cuda()
    args = dict(page_map=torch.from_numpy(m).cuda(), starts=torch.from_numpy(starts).cuda(),
                counts=torch.from_numpy(counts).cuda())
    kv4.write(dev, fd[..., 256:512], fd[..., 512:], **args)
    want = _expect_write(pages, m, starts, np.where((starts < 0) | (starts + counts > 512), 0, counts),
                         k.float().numpy(), v.float().numpy())
    assert np.array_equal(dev.cpu().numpy(), want)
    assert _status() == 1
    # read: bad pages are zeros; rows behind a count and refused sequences stay
    out = torch.full((batch, rows, 3 * heads * 128), 7.0, dtype=BF, device="cuda")
    kv4.read(dev, out[..., :256], None, **args)
    kv4.read(dev, None, out[..., 512:], **args)
    assert _status() == 1
    got = out.double().cpu().numpy()
    assert np.all(got[..., 256:512] == 7)
    for b in range(batch):
        c = counts[b] if starts[b] >= 0 else 0
        if starts[b] + counts[b] > 512:
            c = 0
        for w, sl in (("k", slice(0, 256)), ("v", slice(512, 768))):
            ids = np.clip(m[b], 0, n - 1)
            ref = O.get(want, ids, w).reshape(512, -1)
            for p in range(per):
                if not 0 <= m[b, p] < n:
                    ref[128 * p: 128 * p + 128] = 0
            assert np.array_equal(got[b, :c, sl], ref[max(starts[b], 0): max(starts[b], 0) + c])
            assert np.all(got[b, c:, sl] == 7)


def test_no_page_map_and_empty_calls():
    from kvp import kv4
    rng = np.random.default_rng(4)
    pages = _pool(rng, 6, 1)
    dev = torch.from_numpy(pages).cuda()
    x = torch.from_numpy(rng.standard_normal((3, 130, 128)).astype(np.float32)).to(BF)
    kv4.write(dev, x.cuda(), x.cuda(), start=100)
    m = np.arange(6).reshape(3, 2)
    want = _expect_write(pages, m, [100] * 3, [130] * 3, x.float().numpy(), x.float().numpy())
    assert np.array_equal(dev.cpu().numpy(), want)
    e = torch.empty(3, 0, 128, dtype=BF, device="cuda")
    kv4.write(dev, e, e)
    kv4.read(dev, e, None)
    kv4.attn(e, dev, torch.empty_like(e), heads=1)
    assert np.array_equal(dev.cpu().numpy(), want)
    assert _status() == 0


# ---------------------------------------------------------------- attention

def _attend(rng, pages, m, starts, counts, rows, heads, *, use=("start",), q=None, **kw):
    """(kernel output, 64-bit output, bound) of one call; rows behind a count stay 7."""
    from kvp import kv4
    batch = m.shape[0]
    if q is None:
        q = torch.from_numpy(rng.standard_normal((batch, rows, heads * 128)).astype(np.float32)).to(BF)
    out = torch.full((batch, rows, heads * 128), 7.0, dtype=BF, device="cuda")
    args = {}
    if "starts" in use:
        args["starts"] = torch.tensor(np.asarray(starts), dtype=torch.int32, device="cuda")
    else:
        args["start"] = int(starts[0])
    if "counts" in use:
        args["counts"] = torch.tensor(np.asarray(counts), dtype=torch.int32, device="cuda")
    kv4.attn(q.cuda(), torch.from_numpy(pages).cuda(), out, page_map=torch.from_numpy(m).cuda(),
             heads=heads, **args, **kw)
    want = np.full((batch, rows, heads, 128), 7.0)
    tol = np.zeros_like(want)
    opt = {"tokens": 1, **kw}
    for b in range(batch):
        c = counts[b]
        if c == 0:
            continue
        end = starts[b] + c
        pg = m[b, : -(-end // 128)]
        ids = np.clip(pg, 0, pages.shape[0] - 1)
        k, v = (O.get(pages, ids, w)[:end] for w in "kv")
        ok = O.visible(np.arange(starts[b], end), end, **opt)
        ok &= np.repeat((pg >= 0) & (pg < pages.shape[0]), 128)[None, :end]
        want[b, :c], tol[b, :c] = O.attention(q[b, :c].double().numpy().reshape(c, heads, 128), k, v, ok)
    shape = (batch, rows, heads * 128)
    return out.double().cpu().numpy(), want.reshape(shape), tol.reshape(shape)


def _check(got, want, tol):
    d = np.abs(got - want)
    assert np.all(d <= tol), (float(np.nanmax(d)), float(np.nanmax(d / np.maximum(tol, 1e-30))))


ATTN = [  # batch, kv_heads, group, start, rows, options
    (1, 1, 1, 0, 1, {}),                                        # the first token
    (1, 12, 1, 4098, 1, {}),
    (2, 3, 1, 127, 1, {}), (2, 3, 1, 128, 1, {}), (1, 2, 1, 15, 1, {}), (1, 2, 1, 16, 1, {}),
    (3, 2, 4, 300, 1, {}), (1, 1, 8, 777, 1, {}), (1, 1, 9, 500, 1, {}), (1, 2, 16, 129, 1, {}),
    (1, 1, 17, 200, 1, {}), (1, 1, 5, 130, 3, {}), (2, 2, 7, 61, 4, {}),
    (2, 2, 2, 1000, 1, dict(window=100, sinks=4)), (2, 2, 2, 1000, 1, dict(window=1)),
    (1, 2, 1, 1000, 1, dict(window=128, sinks=200)), (1, 2, 1, 1000, 1, dict(window=990, sinks=20)),
    (1, 2, 1, 700, 2, dict(window=17, sinks=1)), (1, 1, 1, 50, 1, dict(window=1000, sinks=1000)),
    (1, 2, 3, 0, 130, {}), (1, 1, 1, 0, 257, dict(window=64, sinks=3)), (2, 2, 1, 37, 100, {}),
    (1, 2, 1, 120, 60, dict(tokens=60)), (1, 2, 1, 180, 180, dict(tokens=60, window=2, sinks=1)),
    (1, 1, 2, 300, 100, dict(tokens=100, window=1)), (1, 3, 1, 390, 260, dict(tokens=130, window=3, sinks=1)),
    (1, 1, 1, 33, 50, dict(tokens=40, window=2)),               # frames cut by start and end
    (1, 1, 1, 0, 300, dict(tokens=1000)),                       # one frame, not complete
    (1, 2, 1, 1560, 1560, dict(tokens=1560)),
    (1, 1, 3, 0, 700, dict(tokens=7, window=20, sinks=2)),
    # splits: in a cluster, over the workspace (few, many, 9 to 16 rows)
    (1, 4, 1, 2500, 1, {}), (1, 1, 1, 9000, 1, {}), (1, 1, 12, 9000, 1, {}), (1, 2, 3, 9000, 2, dict(window=6000, sinks=100)),
    (48, 2, 1, 4200, 1, {}),
    # units cut between CTAs: one unit for all of them, several, masked pages at the cuts
    (1, 1, 1, 9000, 20, {}), (1, 1, 1, 6000, 300, dict(tokens=100, window=20, sinks=3)), (2, 3, 1, 2000, 400, {}),
    (1, 2, 2, 3000, 500, dict(window=900, sinks=130)), (1, 1, 4, 1500, 750, dict(tokens=250, window=5, sinks=1)),
]


@pytest.mark.parametrize("batch,kvh,grp,start,rows,kw", ATTN)
def test_attention(batch, kvh, grp, start, rows, kw):
    rng = np.random.default_rng(start * 7 + rows)
    per = -(-(start + rows) // 128)
    pages = _calm_pool(rng, batch * per + 1, kvh)
    m = _map(rng, batch, per, batch * per + 1)
    _check(*_attend(rng, pages, m, [start] * batch, [rows] * batch, rows, kvh * grp, **kw))
    assert _status() == 0


@pytest.mark.parametrize("seed", range(24))
def test_attention_of_drawn_shapes(seed):
    """Any batch, heads, rows, frames, window, sinks, starts and counts."""
    rng = np.random.default_rng(1000 + seed)
    kvh, grp, batch = int(rng.integers(1, 4)), int(rng.choice([1, 1, 2, 3, 5, 8])), int(rng.integers(1, 5))
    rows = int(rng.choice([1, 1, 2, 3, 17, 40, 129, 260, 400]))
    per = int(rng.integers(-(-rows // 128), 12))
    T = int(rng.choice([1, 1, 7, 60, 128, 300]))
    kw = dict(tokens=T, window=int(rng.choice([0, 1, 2, 5, 40])) * int(rng.choice([1, 1, 9])), sinks=int(rng.integers(0, 3)))
    starts = [int(rng.integers(0, per * 128 - rows + 1)) for _ in range(batch)]
    counts = [int(rng.integers(0, rows + 1)) if rng.random() < 0.4 else rows for _ in range(batch)]
    pages = _calm_pool(rng, batch * per + 1, kvh)
    m = _map(rng, batch, per, batch * per + 1)
    _check(*_attend(rng, pages, m, starts, counts, rows, kvh * grp, use=("starts", "counts"), **kw))
    assert _status() == 0


@pytest.mark.parametrize("rows,grp,kw", [(1, 1, {}), (1, 4, dict(window=50, sinks=2)), (6, 1, {}),
                                         (70, 2, {}), (70, 2, dict(tokens=10, window=3, sinks=1)),
                                         (300, 1, dict(tokens=64, window=2))])
def test_ragged_batches(rows, grp, kw):
    """Starts and counts on the device: empty, short and refused sequences."""
    rng = np.random.default_rng(rows)
    starts, counts = [0, 511 - rows, 200, 3, 40], [rows, rows, 0, (rows + 1) // 2, rows]
    pages = _calm_pool(rng, 25, 2)
    m = _map(rng, 5, 4, 25)
    _check(*_attend(rng, pages, m, starts, counts, rows, 2 * grp, use=("starts", "counts"), **kw))
    assert _status() == 0


@pytest.mark.parametrize("rows", [1, 200])
def test_refused_sequences_are_left_alone(rows):
    from kvp import kv4
    rng = np.random.default_rng(3)
    pages = torch.from_numpy(_calm_pool(rng, 8, 1)).cuda()
    q = torch.randn(4, rows, 128, device="cuda").to(BF)
    for starts, counts in (([-1, 0, 0, 256 - rows + 1], [rows] * 4), ([0] * 4, [rows, -1, rows + 1, rows])):
        out = torch.full_like(q, 7.0)
        kv4.attn(q, pages, out, heads=1, starts=torch.tensor(starts, dtype=torch.int32, device="cuda"),
                 counts=torch.tensor(counts, dtype=torch.int32, device="cuda"))
        assert _status() == 1
        for b in range(4):
            fits = 0 <= starts[b] and 0 <= counts[b] <= rows and starts[b] + counts[b] <= 256
            assert bool((out[b] == 7).all()) != fits


@pytest.mark.parametrize("rows,start", [(1, 600), (150, 450), (1, 9000), (150, 3450)])
def test_bad_pages_are_no_keys(rows, start):
    rng = np.random.default_rng(5)
    per = -(-(start + rows) // 128)
    pages = _calm_pool(rng, per + 1, 2)
    m = _map(rng, 1, per, per + 1)
    m[0, 1], m[0, 3] = -5, per + 1
    _check(*_attend(rng, pages, m, [start], [rows], rows, 4))
    assert _status() == 1
    m[:] = -1                                       # no key at all: rows of zeros
    got, want, _ = _attend(rng, pages, m, [start], [rows], rows, 4)
    assert np.all(want == 0) and np.all(got == 0)
    assert _status() == 1


@pytest.mark.parametrize("rows", [1, 140])
def test_pages_outside_the_window_are_not_looked_up(rows):
    rng = np.random.default_rng(6)
    start = 1000
    pages = _calm_pool(rng, 12, 2)
    m = _map(rng, 1, 9, 12)
    m[0, 1:6] = 1 << 30                             # freed
    _check(*_attend(rng, pages, m, [start], [rows], rows, 2, window=150, sinks=5))
    assert _status() == 0


@pytest.mark.parametrize("rows,kw", [(1, {}), (3, dict(window=9, sinks=1)), (200, dict(tokens=50, window=2, sinks=1))])
def test_arbitrary_bytes_where_no_key_is(rows, kw):
    """Rows behind the last one and hidden rows hold arbitrary bytes, scales that are never written among them."""
    rng = np.random.default_rng(8)
    start = 500
    per = -(-(start + rows) // 128) + 1
    calm, wild = _calm_pool(rng, per, 1), _pool(rng, per, 1)
    m = np.arange(per, dtype=np.int32)[None]
    end = start + rows
    ok = O.visible(np.arange(start, end), end, **{"tokens": 1, **kw}).any(0)
    seen = np.zeros(per * 128, bool)
    seen[:end] = ok
    seen = seen.reshape(per, 1, 16, 8)
    c, w = (x.reshape(per, 1, 16, O.BLOCK) for x in (calm, wild))
    for a, sh, ax in ((0, (8, 64), 3), (512, (8, 8), 3), (576, (8, 8, 8), 4), (1088, (8, 8), 4)):
        size = int(np.prod(sh))
        cv, wv = (x[..., a: a + size].reshape(per, 1, 16, *sh) for x in (c, w))
        mask = np.expand_dims(seen, tuple(range(4, 3 + len(sh)))) if ax == 3 else \
            np.expand_dims(seen, (3, *range(5, 3 + len(sh))))
        c[..., a: a + size] = np.where(mask, cv, wv).reshape(per, 1, 16, size)
    _check(*_attend(rng, c.reshape(per, 1, -1), m, [start], [rows], rows, 2, **kw))


@pytest.mark.parametrize("rows", [1, 5, 150])
def test_queries_that_are_not_finite_spoil_their_own_rows_only(rows):
    rng = np.random.default_rng(11)
    pages = _calm_pool(rng, 4, 1)
    m = np.arange(4, dtype=np.int32)[None]
    q = torch.from_numpy(rng.standard_normal((1, rows, 512)).astype(np.float32)).to(BF)
    q[0, 0, 5], q[0, 0, 130] = float("nan"), float("inf")
    got, want, tol = _attend(rng, pages, m, [200], [rows], rows, 4, q=q)
    assert np.all(np.isnan(got[0, 0, :256]))
    sel = np.ones_like(want, bool)
    sel[0, 0, :256] = False
    assert np.all(np.abs(got - want)[sel] <= tol[sel])


@pytest.mark.parametrize("rows", [1, 160])
def test_steep_scores(rows):
    """Scores that rise and fall by hundreds along the keys: the running maximum moves often."""
    rng = np.random.default_rng(12)
    start, heads = 700, 2
    per = -(-(start + rows) // 128)
    pages = _calm_pool(rng, per, heads)
    p = pages.reshape(per, heads, 16, O.BLOCK)
    p[..., 512:576] = rng.integers(8 * 10, 8 * 19, p[..., 512:576].shape)   # K scales 2^-5 .. 2^4
    m = _map(rng, 1, per, per)
    _check(*_attend(rng, p.reshape(per, heads, -1), m, [start], [rows], rows, heads))


def test_offsets_beyond_32_bits():
    """A pool of over 4 GB: the sequence's pages are its last ones."""
    from kvp import kv4
    rng = np.random.default_rng(13)
    heads = 16
    n = (1 << 32) // (heads * O.PAGE_HEAD) + 40
    small = _calm_pool(rng, 3, heads)
    pages = torch.zeros(n, heads, O.PAGE_HEAD, dtype=torch.uint8, device="cuda")
    pages[n - 3:] = torch.from_numpy(small).cuda()
    m = torch.tensor([[n - 2, n - 1, n - 3]], dtype=torch.int32, device="cuda")
    x = torch.from_numpy(rng.standard_normal((2, heads * 128)).astype(np.float32)).to(BF)
    kv4.write(pages, x.cuda(), x.cuda(), page_map=m, start=255)
    want = _expect_write(small, np.array([[1, 2, 0]]), [255], [2], x[None].float().numpy(), x[None].float().numpy())
    assert np.array_equal(pages[n - 3:].cpu().numpy(), want)
    assert not bool(pages[: n - 3].any())
    k = torch.empty(2, heads * 128, dtype=BF, device="cuda")
    kv4.read(pages, k, None, page_map=m, start=255)
    assert np.array_equal(k.double().cpu().numpy().reshape(2, heads, 128), O.get(want, [1, 2, 0], "k")[255:257])
    for rows in (1, 130):
        q = torch.from_numpy(rng.standard_normal((rows, heads * 128)).astype(np.float32)).to(BF)
        out = torch.empty(rows, heads * 128, dtype=BF, device="cuda")
        s = 300 - rows
        kv4.attn(q.cuda(), pages, out, heads=heads, page_map=m, start=s)
        kk, vv = (O.get(want, [1, 2, 0], w)[:300] for w in "kv")
        o, tol = O.attention(q.double().numpy().reshape(rows, heads, 128), kk, vv,
                             O.visible(np.arange(s, 300), 300, tokens=1))
        _check(out.double().cpu().numpy().reshape(o.shape), o, tol)


@pytest.mark.parametrize("rows,heads", [(1, 2), (1, 12), (90, 2), (400, 4)])
def test_strided_queries_and_the_same_call_twice(rows, heads):
    """q and out as slices of wider buffers; results do not change from call to call."""
    from kvp import kv4
    rng = np.random.default_rng(14)
    pages = torch.from_numpy(_calm_pool(rng, 24, 2)).cuda()
    wide = torch.from_numpy(rng.standard_normal((2, rows, 3 * heads * 128)).astype(np.float32)).to(BF).cuda()
    q = wide[..., heads * 128: 2 * heads * 128]
    a = torch.full_like(wide, 7.0)
    b, c = (torch.empty(2, rows, heads * 128, dtype=BF, device="cuda") for _ in range(2))
    for o, x in ((a[..., : heads * 128], q), (b, q.contiguous()), (c, q)):
        kv4.attn(x, pages, o, heads=heads, start=1000)
    assert torch.equal(a[..., : heads * 128], b) and torch.equal(b, c)
    assert bool((a[..., heads * 128:] == 7).all())


@pytest.mark.parametrize("kw", [{}, dict(window=700, sinks=150), dict(tokens=90, window=4, sinks=1)])
def test_many_units_cut_where_they_do_not_divide(kw):
    """150 units of 12 pages: each CTA goes from one sequence's or head's to
    the next; one and two query tiles, sequences of no rows between them."""
    rng = np.random.default_rng(len(kw))
    batch, kvh, rows, per = 15, 10, 130, 12
    starts = [per * 128 - rows - int(x) for x in rng.integers(0, 400, batch)]
    counts = [int(x) for x in rng.choice([rows, rows, 100, 129, 7, 0], batch)]
    starts[3], counts[3] = 0, rows
    pages = _calm_pool(rng, batch * per, kvh)
    got, want, tol = _attend(rng, pages, _map(rng, batch, per, batch * per), starts, counts, rows, kvh,
                             use=("starts", "counts"), **kw)
    _check(got, want, tol)
    assert _status() == 0


@pytest.mark.parametrize("rows", [1, 3, 130])
def test_sequences_inside_rows_in_place_and_shared_queries(rows):
    """Row-major batches ([rows, batch, ...] seen as [batch, rows, ...]) in
    writes, reads and attention; out = q; one q for all sequences."""
    from kvp import kv4
    rng = np.random.default_rng(rows)
    host = _calm_pool(rng, 3 * 34, 2)

    def draw(n, d):
        return torch.from_numpy(rng.standard_normal((n, 3, d)).astype(np.float32)).to(BF).cuda().transpose(0, 1)

    k, v, q = draw(rows, 256), draw(rows, 256), draw(rows, 512)
    a, b = (torch.from_numpy(host).cuda() for _ in range(2))
    kv4.write(a, k, v, start=4100)
    kv4.write(b, k.contiguous(), v.contiguous(), start=4100)
    assert torch.equal(a, b)
    for dtype in (BF, F32):
        x, y = (torch.empty(rows, 3, 256, dtype=dtype, device="cuda").transpose(0, 1) for _ in range(2))
        w = [torch.empty(3, rows, 256, dtype=dtype, device="cuda") for _ in range(2)]
        kv4.read(a, x, y, start=4100)
        kv4.read(a, *w, start=4100)
        assert torch.equal(x, w[0]) and torch.equal(y, w[1])
    want = torch.empty(3, rows, 512, dtype=BF, device="cuda")
    kv4.attn(q.contiguous(), a, want, heads=4, start=4100)
    out = torch.empty(rows, 3, 512, dtype=BF, device="cuda").transpose(0, 1)
    kv4.attn(q, a, out, heads=4, start=4100)
    assert torch.equal(out, want)
    one = q[:1].expand(3, rows, 512)
    kv4.attn(one, a, out, heads=4, start=4100)
    kv4.attn(one.contiguous(), a, want, heads=4, start=4100)
    assert torch.equal(out, want)
    mine = one.contiguous()
    kv4.attn(mine, a, mine, heads=4, start=4100)
    assert torch.equal(mine, want)
    assert _status() == 0


@pytest.mark.parametrize("rows", [1, 40, 300])
@pytest.mark.parametrize("kw", [dict(tokens=2 ** 31 - 1), dict(window=2 ** 31 - 1), dict(sinks=2 ** 31 - 1, window=1),
                                dict(tokens=2 ** 31 - 1, window=2 ** 31 - 1, sinks=2 ** 31 - 1),
                                dict(tokens=3, window=2 ** 31 - 1)])
def test_options_at_their_ends(rows, kw):
    """Frames, windows and sinks beyond anything cached hide nothing."""
    rng = np.random.default_rng(rows)
    got, want, tol = _attend(rng, _calm_pool(rng, 12, 1), _map(rng, 1, 12, 12), [1000], [rows], rows, 2, **kw)
    _check(got, want, tol)
    assert _status() == 0


@pytest.mark.parametrize("rows,far", [(1, 0), (1, 6000), (130, 0), (130, 3000)])
def test_graphs_replay_and_do_not_share_workspaces(rows, far):
    """Two captured calls replayed at once on two streams, starts moved between replays."""
    from kvp import kv4
    rng = np.random.default_rng(15)
    pages = torch.from_numpy(_calm_pool(rng, 32 + far // 128, 2)).cuda()
    qs = [torch.from_numpy(rng.standard_normal((1, rows, 512)).astype(np.float32)).to(BF).cuda() for _ in range(2)]
    starts = [torch.tensor([1500 + far + 300 * i], dtype=torch.int32, device="cuda") for i in range(2)]
    outs = [torch.zeros_like(q) for q in qs]
    graphs = []
    for q, st, o in zip(qs, starts, outs):
        kv4.attn(q, pages, o, heads=4, starts=st)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            kv4.attn(q, pages, o, heads=4, starts=st)
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in range(2)]
    for move in (0, 700):
        for st in starts:
            st += move
        torch.cuda.synchronize()
        for _ in range(5):
            for g, s in zip(graphs, streams):
                with torch.cuda.stream(s):
                    g.replay()
        torch.cuda.synchronize()
        for q, st, o in zip(qs, starts, outs):
            ref = torch.zeros_like(q)
            kv4.attn(q, pages, ref, heads=4, starts=st)
            assert torch.equal(o, ref)
    assert _status() == 0


@pytest.mark.parametrize("rows,start", [(1, 300), (1, 4000), (1, 9000), (40, 900), (300, 700), (300, 9000)])
@pytest.mark.parametrize("wait", [False, True])
def test_calls_follow_one_another(rows, start, wait):
    """Kernels are launched before what precedes them ends: rows, queries, starts,
    pages and outputs that the call before, or another kernel, has just written
    or read.  With and without a wait in between the results are the same."""
    from kvp import kv4
    gen = torch.Generator(device="cuda").manual_seed(rows + start)
    pages = kv4.alloc_pages(80, 2).random_(0, 256, generator=gen)
    x = torch.randn(20, rows, 256, device="cuda", generator=gen).to(BF)
    results = []
    for pause in (True, wait):
        p, q = pages.clone(), torch.zeros(rows, 512, dtype=BF, device="cuda")
        k, v = (torch.zeros_like(x[0]) for _ in range(2))
        at = torch.full((1,), start, dtype=torch.int32, device="cuda")
        out, back, outs = torch.zeros_like(q), torch.zeros_like(x[0]), []
        torch.cuda.synchronize()
        for i in range(20):
            for step in (lambda: k.copy_(x[i]), lambda: v.copy_(x[19 - i]), lambda: q.copy_(x[i].repeat(1, 2)),
                         lambda: kv4.write(p, k, v, starts=at), lambda: kv4.attn(q, p, out, heads=4, starts=at),
                         lambda: q.copy_(out), lambda: kv4.attn(q, p, q, heads=4, starts=at),
                         lambda: kv4.write(p, q[:, :256], q[:, 256:], starts=at),
                         lambda: kv4.read(p, back, None, starts=at),
                         lambda: outs.append(torch.cat((out, q, back), 1)), lambda: at.add_(i % 3 - 1)):
                step()
                if pause:
                    torch.cuda.synchronize()
        results.append(torch.stack(outs).view(torch.int16))       # (bits: arbitrary bytes make scores that overflow)
    assert torch.equal(results[0], results[1])
    assert _status() in (0, 8)          # some of them are written back, beyond the format


@pytest.mark.parametrize("rows,start", [(1, 300), (1, 9000), (200, 900)])
def test_captured_after_copies_fills_and_other_streams(rows, start):
    """A graph in which a copy, a fill and a second stream's work come before
    the calls, replayed with new rows."""
    from kvp import kv4
    gen = torch.Generator(device="cuda").manual_seed(rows + start)
    x = torch.randn(3, rows, 256, device="cuda", generator=gen).to(BF)
    pages, src = kv4.alloc_pages(80, 2).fill_(0x77), x[0].clone()
    k, back = torch.zeros_like(src), torch.zeros_like(src)
    q, out = torch.zeros(rows, 512, dtype=BF, device="cuda"), torch.zeros(rows, 512, dtype=BF, device="cuda")
    other = torch.cuda.Stream()

    def calls():
        k.copy_(src)
        kv4.write(pages, k, k, start=start)
        here = torch.cuda.current_stream()
        other.wait_stream(here)
        with torch.cuda.stream(other):
            q[:, :256].copy_(src)
            kv4.read(pages, back, None, start=start)
        here.wait_stream(other)
        out.zero_()
        kv4.attn(q, pages, out, heads=4, start=start)

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        calls()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        calls()
    for i in (1, 2):
        src.copy_(x[i])
        graph.replay()
        torch.cuda.synchronize()
        got = out.clone(), back.clone()
        calls()
        torch.cuda.synchronize()
        assert torch.equal(got[0], out) and torch.equal(got[1], back)
        assert bool((back.float() - x[i].float()).abs().max() < 0.5) and bool(out.any())
    assert _status() == 0


def test_two_streams_at_once():
    from kvp import kv4
    rng = np.random.default_rng(16)
    pages = torch.from_numpy(_calm_pool(rng, 64, 2)).cuda()
    qs = [torch.from_numpy(rng.standard_normal((1, r, 256)).astype(np.float32)).to(BF).cuda() for r in (1, 1, 200, 200)]
    refs = [torch.empty_like(q) for q in qs]
    for q, o in zip(qs, refs):
        kv4.attn(q, pages, o, heads=2, start=7000)
    outs = [torch.zeros_like(q) for q in qs]
    streams = [torch.cuda.Stream() for _ in qs]
    torch.cuda.synchronize()
    for _ in range(4):
        for q, o, s in zip(qs, outs, streams):
            kv4.attn(q, pages, o, heads=2, start=7000, stream=s.cuda_stream)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(outs, refs))


def test_python_refusals_on_a_device():
    from kvp import kv4
    from kvp._lib import KvpError
    pages = kv4.alloc_pages(4, 2)
    k = torch.zeros(2, 3, 256, dtype=BF, device="cuda")
    m = torch.zeros(2, 2, dtype=torch.int32, device="cuda")
    for kw, what in ((dict(page_map=m.long()), "int32"), (dict(page_map=m[:1]), "page_map"),
                     (dict(page_map=m.cpu()), "tensors on"), (dict(starts=m[0, :1]), "starts"),
                     (dict(counts=m[0].long()), "counts"), (dict(start=-1), "out of range"),
                     (dict(start=254), "do not fit"), (dict(page_map=m, start=254), "do not fit")):
        with pytest.raises(KvpError, match=what):
            kv4.write(pages, k, k, **kw)
    with pytest.raises(KvpError, match="multiple of kv_heads"):
        kv4.attn(k[..., :128], pages, torch.empty_like(k[..., :128]), heads=1)
    with pytest.raises(KvpError, match="overlap"):
        kv4.attn(k, pages, torch.empty(1, 3, 256, dtype=BF, device="cuda").expand(2, 3, 256), heads=2)
    assert _status() == 0


def test_a_video_loop_then_tokens():
    """Write, attend and read back as they are used: four frames in chunks
    with a window and a sink frame, then single tokens appended to them."""
    from kvp import kv4
    rng = np.random.default_rng(17)
    T, kvh, heads, frames = 150, 2, 4, 4
    total = T * frames + 3
    per = -(-total // 128)
    host = _pool(rng, per, kvh)
    pages = torch.from_numpy(host).cuda()
    m = _map(rng, 1, per, per)
    mm = torch.from_numpy(m).cuda()
    x = [torch.from_numpy(rng.standard_normal((total, kvh * 128)).astype(np.float32)).to(BF) for _ in range(2)]
    q = torch.from_numpy(rng.standard_normal((total, heads * 128)).astype(np.float32)).to(BF)
    xd, qd = [t.cuda() for t in x], q.cuda()
    out = torch.zeros(total, heads * 128, dtype=BF, device="cuda")
    steps = [(0, T, dict(tokens=T, window=2, sinks=1)), (T, 2 * T, dict(tokens=T, window=2, sinks=1)),
             (3 * T, T, dict(tokens=T, window=2, sinks=1))]
    steps += [(4 * T + i, 1, dict(window=200, sinks=5)) for i in range(3)]
    for s, n, kw in steps:
        sl = slice(s, s + n)
        kv4.write(pages, xd[0][sl], xd[1][sl], page_map=mm, start=s)
        kv4.attn(qd[sl], pages, out[sl], page_map=mm, heads=heads, start=s, **kw)
    back = [torch.empty_like(t) for t in xd]
    kv4.read(pages, *back, page_map=mm)
    vals = [O.values(*O.quantise(t.float().numpy().reshape(total, kvh, 128))) for t in x]
    for t, w in zip(back, vals):
        assert np.array_equal(t.double().cpu().numpy().reshape(w.shape), w)
    for s, n, kw in steps:
        o, tol = O.attention(q[s: s + n].double().numpy().reshape(n, heads, 128), vals[0][: s + n], vals[1][: s + n],
                             O.visible(np.arange(s, s + n), s + n, **{"tokens": 1, **kw}))
        _check(out[s: s + n].double().cpu().numpy().reshape(o.shape), o, tol)
    assert _status() == 0
