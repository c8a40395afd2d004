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


def _staged(seed):
    """A manager with five queued rows of 2 x 256 floats: (manager, k, v, slots' sources)."""
    from kvp.manager import KVTileManager
    gen = torch.Generator(device="cuda").manual_seed(seed)
    k, v = (torch.randn(50, 256, device="cuda", generator=gen) for _ in range(2))
    m = KVTileManager(20 * 2048, 20 * 2048)
    assert m.init() and m.arena_init(20 * 2048, 512)
    m.arena_begin_step()
    src = []
    for r in (3, 4, 5, 40, 41):
        ok, slot = m.arena_stage(k[r].data_ptr(), 1024, v[r].data_ptr(), 1024)
        assert ok and slot == len(src)
        src.append(r)
    assert m.pending_copies() == 10
    return m, k, v, src


def test_queued_copies_of_the_managers_go_first():
    """Staging calls queue their row copies up to the next launch: a write may
    take its rows from the arena, a read may fill rows that a copy reads."""
    import ctypes as C

    from kvp import kv4
    from kvp._lib import Kv4Attn, Kv4Rows, Kv4Span, lib
    L = lib()
    pages = kv4.alloc_pages(1, 2)
    span = Kv4Span(pages.data_ptr(), 0, 0, 0, 1, 2, 1, 1, 0, 5)

    m, k, v, src = _staged(1)
    arena = m.arena_device_ptr()
    rows = Kv4Rows(arena, arena + 1024, 512, 0, 4)
    bad = Kv4Rows(arena, arena + 1024, 510, 0, 4)
    assert L.kvp_kv4_write(C.byref(span), C.byref(bad), None) == -1 and m.pending_copies() == 10
    assert L.kvp_kv4_write(C.byref(span), C.byref(rows), None) == 0 and m.pending_copies() == 0
    back = [torch.empty(5, 256, device="cuda") for _ in range(2)]
    kv4.read(pages, *back)
    for t, x in zip(back, (k, v)):
        want = O.values(*O.quantise(x[src].double().cpu().numpy().reshape(5, 2, 128))).reshape(5, 256)
        assert np.array_equal(t.double().cpu().numpy(), want)
    m.close()

    m, k, v, src = _staged(2)
    kept = k.clone()
    kv4.read(pages, k[3:8], None)                    # over three of the rows to be copied
    assert m.pending_copies() == 0 and not torch.equal(k, kept)
    staged = Kv4Rows(m.arena_device_ptr(), m.arena_device_ptr() + 1024, 512, 0, 4)
    assert L.kvp_kv4_write(C.byref(span), C.byref(staged), None) == 0
    kv4.read(pages, back[0], None)
    want = O.values(*O.quantise(kept[src].double().cpu().numpy().reshape(5, 2, 128))).reshape(5, 256)
    assert np.array_equal(back[0].double().cpu().numpy(), want)
    m.close()

    m, k, v, src = _staged(3)
    q = torch.zeros(5, 256, dtype=BF, device="cuda")
    attn = Kv4Attn(q.data_ptr(), q.data_ptr(), 256, 0, 256, 0, 2, 1, 0, 0)
    assert L.kvp_attn_kv4(C.byref(span), C.byref(attn), None) == 0 and m.pending_copies() == 0
    m.close()
    assert _status() == 0


@pytest.mark.parametrize("batch,rows,start", [(1, 1, 5), (3, 1, 127), (1, 40, 3), (2, 150, 121)])
@pytest.mark.parametrize("dtype", [BF, F32])
def test_k_and_v_of_different_strides(batch, rows, start, dtype):
    """K a tensor of its own (or with the sequences inside the rows), V a slice of a fused projection."""
    from kvp import kv4
    gen = torch.Generator(device="cuda").manual_seed(rows)
    v = torch.randn(batch, rows, 768, device="cuda", generator=gen).to(dtype)[..., 512:]
    own = torch.randn(batch, rows, 256, device="cuda", generator=gen).to(dtype)
    inside = own.transpose(0, 1).contiguous().transpose(0, 1)
    host = np.random.default_rng(rows).integers(0, 256, (3 * batch, 2, O.PAGE_HEAD), dtype=np.uint8)
    want = torch.from_numpy(host).cuda()
    kv4.write(want, own, v.contiguous(), start=start)
    fused = torch.full((batch, rows, 768), 7.0, dtype=dtype, device="cuda")
    for k in (own, inside):
        got = torch.from_numpy(host).cuda()
        kv4.write(got, k, v, start=start)
        assert torch.equal(got, want)
        swapped = torch.from_numpy(host).cuda()
        kv4.write(want2 := torch.from_numpy(host).cuda(), v.contiguous(), own, start=start)
        kv4.write(swapped, v, k, start=start)
        assert torch.equal(swapped, want2)
        back = torch.empty_like(k)
        kv4.read(got, back, fused[..., 512:], start=start)
        for t, w in ((back, "k"), (fused[..., 512:], "v")):
            for b in range(batch):
                ids = range(3 * b, 3 * b + 3)
                ref = O.get(want.cpu().numpy(), ids, w)[start: start + rows].reshape(rows, 256)
                assert np.array_equal(t[b].double().cpu().numpy(), ref)
    assert bool((fused[..., :512] == 7).all())
    assert _status() == 0


@pytest.mark.parametrize("rows,start", [(1, 300), (1, 4000), (1, 9000), (12, 5000), (40, 900), (300, 700), (300, 9000)])
@pytest.mark.parametrize("mode", ["queued", "paused", "captured"])
def test_what_a_call_has_written_is_what_the_next_one_reads(rows, start, mode):
    """Copies, writes, attention and reads back to back.  A row's key is four times
    its query, 22 or more above any other score, so its output is its own value: off
    by half a scale, max / 14 * 17 / 16 < 0.4, and bf16's rounding, if pages, starts and
    queries are those of this iteration, and nowhere near if they are the last one's."""
    from kvp import kv4
    gen = torch.Generator(device="cuda").manual_seed(rows + start)
    pages = kv4.alloc_pages(80, 2).random_(0, 256, generator=gen)
    field = pages.view(80, 2, 16, O.BLOCK)
    for a in (512, 1088):
        field[..., a: a + 64] = torch.randint(96, 112, field[..., a: a + 64].shape, device="cuda", generator=gen)
    x = torch.randn(12, rows, 256, device="cuda", generator=gen).to(BF)
    src = x[0].clone()
    k, v, back = (torch.zeros_like(src) for _ in range(3))
    q, out = (torch.zeros(rows, 512, dtype=BF, device="cuda") for _ in range(2))
    again = torch.zeros_like(q)
    at = torch.full((1,), start, dtype=torch.int32, device="cuda")

    def wide(t):                                       # K/V head h for query heads 2h and 2h + 1
        return t.view(rows, 2, 1, 128).expand(rows, 2, 2, 128).reshape(rows, 512)

    steps = [lambda: torch.mul(src, 4, out=k), lambda: v.copy_(src), lambda: q.copy_(wide(src)),
             lambda: kv4.write(pages, k, v, starts=at), lambda: kv4.attn(q, pages, out, heads=4, starts=at),
             lambda: kv4.read(pages, None, back, starts=at), lambda: kv4.attn(q, pages, again, heads=4, starts=at),
             lambda: kv4.write(pages, v, k, starts=at),    # (another content, until the next iteration)
             lambda: at.add_(1)]

    def once():
        for step in steps:
            step()
            if mode == "paused":
                torch.cuda.synchronize()

    if mode == "captured":
        side = torch.cuda.Stream()
        with torch.cuda.stream(side):
            once()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            once()
        torch.cuda.synchronize()
    outs = []
    for i in range(12):
        src.copy_(x[i])
        graph.replay() if mode == "captured" else once()
        outs.append(torch.cat((out, again, back), 1))
    got = torch.stack(outs).float()
    want = torch.stack([torch.cat((wide(y), wide(y), y), 1) for y in x]).float()
    assert bool(((got - want).abs() < 0.5).all())
    assert float((got[1:] - got[:-1]).abs().amax((1, 2)).min()) > 2
    assert _status() == 0


@pytest.mark.parametrize("rows,start", [(1, 300), (1, 1200), (1, 9000), (12, 9000), (40, 900), (300, 900), (300, 9000)])
def test_the_first_attention_of_a_process_is_captured(rows, start):
    """One call on a device comes before the first capture there; a write will do."""
    import subprocess
    import sys
    from pathlib import Path
    code = f"""
import sys
sys.path.insert(0, {str(Path(__file__).resolve().parents[1] / 'cuda-kv-persistence_b200')!r})
import torch
from kvp import kv4
from kvp.attention import read_status
pages = kv4.alloc_pages(80, 2).fill_(0x69)
x = torch.randn({rows}, 256, device="cuda", generator=torch.Generator("cuda").manual_seed(0)).to(torch.bfloat16)
kv4.write(pages, x, x, start={start})
torch.cuda.synchronize()
out, back, ref = torch.zeros_like(x), torch.zeros_like(x), torch.zeros_like(x)
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    kv4.attn(x, pages, out, heads=2, start={start})
    kv4.read(pages, back, None, start={start})
graph.replay()
kv4.attn(x, pages, ref, heads=2, start={start})
torch.cuda.synchronize()
assert torch.equal(out, ref) and bool(out.any()) and bool((back.float() - x.float()).abs().max() < 0.5)
assert read_status() == 0
"""
    done = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=120)
    assert done.returncode == 0, done.stderr[-2000:]


@pytest.mark.parametrize("dtype", [BF, F32])
def test_calls_at_once_on_neighbouring_rows(dtype):
    """Writes that run at once may share a block of eight rows, and reads and attention
    go on beside them on rows that they do not touch."""
    from kvp import kv4
    gen = torch.Generator(device="cuda").manual_seed(1)
    cuts = [0, 13, 14, 15, 40, 41, 122, 131, 256, 259, 300]
    x = torch.randn(2, 300, 256, device="cuda", generator=gen).to(dtype)
    host = np.random.default_rng(1).integers(0, 256, (3, 2, O.PAGE_HEAD), dtype=np.uint8)
    want = torch.from_numpy(host).cuda()
    kv4.write(want, x[0], x[1])
    q = torch.randn(5, 256, device="cuda", generator=gen).to(BF)
    ref, k = torch.empty_like(q), torch.empty(84, 256, dtype=dtype, device="cuda")
    kv4.attn(q, want, ref, heads=2, start=295)
    got = torch.from_numpy(host).cuda()
    streams = [torch.cuda.Stream() for _ in cuts[1:]]
    torch.cuda.synchronize()
    for _ in range(20):
        got.copy_(torch.from_numpy(host))
        torch.cuda.synchronize()
        for s, a, b in zip(streams, cuts, cuts[1:]):
            kv4.write(got, x[0, a:b], x[1, a:b], start=a, stream=s.cuda_stream)
        torch.cuda.synchronize()
        assert torch.equal(got, want)
        outs = [torch.empty_like(q) for _ in streams]
        kv4.write(got, x[0, 10:12], x[1, 10:12], start=10, stream=streams[0].cuda_stream)    # as they are
        kv4.read(got, k, None, start=300, stream=streams[1].cuda_stream)
        for s, o in zip(streams[2:], outs[2:]):
            kv4.attn(q, got, o, heads=2, start=295, window=200, stream=s.cuda_stream)
        torch.cuda.synchronize()
        assert all(torch.equal(o, outs[2]) for o in outs[2:])
    kv4.attn(q, got, outs[0], heads=2, start=295)
    assert torch.equal(outs[0], ref)
    assert _status() == 0
