"""The 4-bit K/V cache and the attention that reads it: what is measured.

Three operators of ``kvp.kv4``:

* ``write`` -- quantises K and V rows as they enter the cache (its cases read
  the rows back, so that they return the values the cache stands for);
* ``read``  -- reads rows of the cache back;
* ``attn``  -- attention over the cache, block-causal by frames, with a
  sliding window and first frames ("sinks") that stay visible; with one token
  per frame it is a language model's causal attention, with one query row its
  decoding step.

The cache is a pool of pages, uint8 [pages][kv_heads][18432]: 128 rows of one
head, as 16 blocks of 8 rows.  A block is K codes [8 rows][64 B], K scales
[8 rows][8], V codes [8 groups][8 rows][8 B], V scales [8 groups][8 rows]
(1152 bytes).  Every 16 dims share one scale byte (eeeee mmm, the value
(1 + m/8) * 2^(e - 15)); a code is 4 bits, value (code - 8) * scale.  Eight
dims make a 32-bit word: dim 2i in bits [4i, 4i+4), dim 2i+1 16 bits higher.

``own`` false: the plain form, in elementary torch operations.
"""

import math
import sys
from pathlib import Path

import torch

own = False

HEAD = 128            # head dim
PAGE = 128            # rows of a page
PAGE_HEAD = 18432     # bytes of one head's share of a page
BLOCK = 1152          # bytes of 8 rows of one head


def _kv4():
    root = str(Path(__file__).resolve().parents[1] / "cuda-kv-persistence_b200")
    if root not in sys.path:
        sys.path.insert(0, root)
    from kvp import kv4
    return kv4


def _dev():
    return "cuda" if torch.cuda.is_available() else "cpu"


# ------------------------------------------------------------------- cases

def _case(name, op, **kw):
    c = {"name": name, "op": op, "batch": 1, "heads": 12, "kv_heads": 12, "start": 0, "rows": 1,
         "ragged": 0, "tokens": 1, "window": 0, "sinks": 0, "dtype": "bf16"}
    c.update(kw)
    return c


def listed():
    return [
        # one new token of four sequences enters the cache: the append of a decoding step
        _case("write_token", "write", batch=4, start=4095),
        # one 30 x 52 latent frame of 12 heads, the per-frame append of the autoregressive loop
        _case("write_frame", "write", rows=1560, start=3 * 1560),
        # all 21 frames of a clip at once: filling the cache from existing K/V
        _case("write_clip", "write", rows=21 * 1560),
        # a frame read back in bf16, e.g. to hand it to the bf16 kernels
        _case("read_frame", "read", rows=1560, start=7 * 1560),
        # two ragged prompts read back in fp32, as a check or a conversion does
        _case("read_prompt_fp32", "read", batch=2, kv_heads=8, heads=8, rows=6001, start=129,
              dtype="fp32"),
        # one decoding step of one short sequence: latency counts
        _case("decode_token", "attn", start=4098),
        # a serving batch of unequal lengths, four query heads to a K/V head
        _case("decode_batch", "attn", batch=16, heads=32, kv_heads=8, start=8190, ragged=1),
        # one very long sequence
        _case("decode_long", "attn", start=131070),
        # decoding with a window and four first tokens that stay visible
        _case("decode_sinks", "attn", batch=8, start=32760, ragged=1, window=4096, sinks=4),
        # one frame of queries over all 21 frames: the autoregressive video step
        _case("frame_step", "attn", rows=1560, start=20 * 1560, tokens=1560),
        # a chunk of three frames, the last six frames visible and the first one kept
        _case("frame_sinks", "attn", rows=3 * 1560, start=18 * 1560, tokens=1560, window=6, sinks=1),
        # a token-causal prompt of odd length, three query heads to a K/V head, window and sinks
        _case("prompt_window", "attn", heads=24, kv_heads=8, rows=4097, window=1024, sinks=4),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["write", "read", "decode", "decode", "frame", "prompt"])
    kv = rng.choice([1, 2, 4, 5, 8, 12, 16])
    group = rng.choice([1, 1, 2, 3, 4, 7, 8])
    if op in ("write", "read"):
        rows = _log(rng, 1, 32760)
        batch = _log(rng, 1, max(1, min(16, 32760 * 12 // (rows * kv))))
        c = _case("", op, batch=batch, heads=kv, kv_heads=kv, rows=max(1, min(rows, 32760 * 12 // (batch * kv))),
                  start=rng.randrange(0, 4096), dtype=rng.choice(["bf16", "bf16", "fp32"]))
    elif op == "decode":
        start = _log(rng, 1, 131070)
        batch = _log(rng, 1, max(1, min(32, 131070 * 12 // (start * kv))))
        start = min(start, 131070 * 12 // (batch * kv))
        win = rng.choice([0, 0, 1]) * _log(rng, 16, 8192)
        c = _case("", "attn", batch=batch, heads=kv * group, kv_heads=kv, start=start,
                  ragged=rng.choice([0, 1]), rows=rng.choice([1, 1, 1, 2, 4]), window=win,
                  sinks=rng.randrange(0, 9) if win else 0)
    elif op == "frame":
        tokens = _log(rng, 60, 1560)
        total = rng.randrange(2, 22)
        frames = rng.randrange(1, min(3, total) + 1)
        win = rng.choice([0, 1]) * rng.randrange(frames, total + 1)
        if not win:
            frames = 1
        c = _case("", "attn", rows=frames * tokens, start=(total - frames) * tokens, tokens=tokens,
                  window=win, sinks=rng.randrange(0, 3) if win else 0)
    else:
        rows = _log(rng, 17, 6000)
        batch = max(1, min(rng.choice([1, 1, 2, 3]), 6000 // rows))
        heads = max(1, min(24 // kv, group))
        win = rng.choice([0, 1]) * _log(rng, 16, 4096)
        c = _case("", "attn", batch=batch, heads=kv * heads, kv_heads=kv, rows=rows,
                  start=rng.choice([0, rng.randrange(0, 2048)]), ragged=rng.choice([0, 1]),
                  window=win, sinks=rng.randrange(0, 9) if win else 0)
    del c["name"]
    return c


def _starts(case):
    """The first new row's position in each sequence; ragged batches differ by a fixed rule."""
    s, b = case["start"], case["batch"]
    return [s - (s * i) // (2 * b) if case["ragged"] else s for i in range(b)]


def _span(case, pos, limit):
    """Key rows [0, s) and [lo, hi) that the query at position pos sees (s <= lo)."""
    T, W, S = case["tokens"], case["window"], case["sinks"]
    f = pos // T
    hi = min((f + 1) * T, limit)
    lo = max(f - W + 1, 0) * T if W else 0
    return min(S * T, lo, hi), lo, hi


def work(case):
    b, kv, h, n = case["batch"], case["kv_heads"], case["heads"], case["rows"]
    size = 4 if case["dtype"] == "fp32" else 2
    plain = 2 * b * n * kv * HEAD * size          # K and V as rows
    packed = b * n * kv * (BLOCK // 8)            # K and V in the cache
    if case["op"] == "write":                     # rows in, cache out; cache in, rows out
        return {"bytes": 2 * plain + 2 * packed, "flops": 0}
    if case["op"] == "read":
        return {"bytes": plain + packed, "flops": 0}
    pairs = keys = 0
    for s in _starts(case):
        first, last = _span(case, s, s + n), _span(case, s + n - 1, s + n)
        keys += last[2] - max(first[1], first[0]) + min(max(first[0], last[0]), first[1])
        for i in range(n):
            a, lo, hi = _span(case, s + i, s + n)
            pairs += a + hi - lo
    return {"bytes": 2 * b * n * h * HEAD * 2 + keys * kv * (BLOCK // 8),
            "flops": 4 * HEAD * pairs * h}


# ------------------------------------------------------- the format, plainly

def _quantise(x):
    """x [..., 128] -> codes uint8 [..., 128], scale bytes uint8 [..., 8] (32-bit arithmetic)."""
    x = x.to(torch.bfloat16).float().unflatten(-1, (8, 16))
    m, e = torch.frexp(x.abs().amax(-1) / 7)
    q = torch.floor(m * 16 + 0.5)                                  # 4 bits, halves up
    up = q == 16
    q, e = torch.where(up, 8.0, q), e + up.to(e.dtype)
    e = torch.where(m == 0, -99, e) + 14                           # s = q/8 * 2^(e - 15)
    q, e = torch.where(e < 0, 8.0, q), e.clamp(min=0)
    q, e = torch.where(e > 31, 15.0, q), e.clamp(max=31)
    byte = (e * 8 + (q.int() - 8)).to(torch.uint8)
    s = torch.ldexp(q, e - 18).unsqueeze(-1)
    n = torch.floor(x.abs() / s + 0.5).clamp(max=7) * torch.sign(x)
    return (n + 8).to(torch.uint8).flatten(-2), byte


def _pack(codes):
    """codes uint8 [..., 128] -> bytes uint8 [..., 64], eight dims to a little-endian word."""
    c = codes.unflatten(-1, (16, 4, 2))                            # word, i, parity
    c = c.transpose(-1, -2).unflatten(-1, (2, 2))                  # word, parity, byte, nibble
    return (c[..., 0] | (c[..., 1] << 4)).flatten(-3)


def _unpack(b):
    """The inverse of _pack."""
    b = b.unflatten(-1, (16, 2, 2))
    c = torch.stack((b & 15, b >> 4), -1).flatten(-2)              # word, parity, i
    return c.transpose(-1, -2).flatten(-3)


def _value(codes, byte):
    b = byte.int()
    s = torch.ldexp((8 + (b & 7)).float(), (b >> 3) - 18)
    return ((codes.float() - 8).unflatten(-1, (8, 16)) * s.unsqueeze(-1)).flatten(-2)


def _fields(pages):
    """Views of a pool: K codes, K scales, V codes, V scales, indexed [page, head, block, ...]."""
    t = pages.unflatten(-1, (16, BLOCK))
    return (t[..., :512].unflatten(-1, (8, 64)), t[..., 512:576].unflatten(-1, (8, 8)),
            t[..., 576:1088].unflatten(-1, (8, 8, 8)), t[..., 1088:].unflatten(-1, (8, 8)))


def _places(page_map, start, rows):
    """Page, block and row in the block of rows [start, start + rows) of every sequence."""
    pos = torch.arange(start, start + rows, device=page_map.device)
    page = page_map[:, pos // PAGE].long().flatten()
    pos = pos.repeat(page_map.shape[0])
    return page, pos % PAGE // 8, pos % 8


def _plain_write(pages, page_map, start, k, v):
    page, blk, row = _places(page_map, start, k.shape[1])
    kc, ks, vc, vs = _fields(pages)
    heads = pages.shape[1]
    c, s = _quantise(k.flatten(0, 1).unflatten(-1, (heads, HEAD)))
    kc[page, :, blk, row] = _pack(c)
    ks[page, :, blk, row] = s
    c, s = _quantise(v.flatten(0, 1).unflatten(-1, (heads, HEAD)))
    vc[page, :, blk, :, row] = _pack(c).unflatten(-1, (8, 8))
    vs[page, :, blk, :, row] = s


def _plain_read(pages, page_map, start, rows, dtype):
    page, blk, row = _places(page_map, start, rows)
    kc, ks, vc, vs = _fields(pages)
    k = _value(_unpack(kc[page, :, blk, row]), ks[page, :, blk, row])
    v = _value(_unpack(vc[page, :, blk, :, row].flatten(-2)), vs[page, :, blk, :, row])
    b = page_map.shape[0]
    return tuple(x.flatten(-2).unflatten(0, (b, rows)).to(dtype) for x in (k, v))


def _plain_attn(q, pages, page_map, starts, case):
    b, n = q.shape[:2]
    kv, group = case["kv_heads"], case["heads"] // case["kv_heads"]
    used = -(-(max(_starts(case)) + n) // PAGE)
    pm = page_map[:, :used].long()
    kc, ks, vc, vs = _fields(pages)
    # [b, page, head, block, row, ...] -> [b, head, key, dim]
    k = _value(_unpack(kc[pm]), ks[pm]).transpose(1, 2).flatten(2, 4)
    v = _value(_unpack(vc[pm].transpose(-3, -2).flatten(-2)), vs[pm].transpose(-1, -2))
    v = v.transpose(1, 2).flatten(2, 4)
    pos = starts.view(b, 1).long() + torch.arange(n, device=q.device)
    key = torch.arange(k.shape[2], device=q.device)
    T, W, S = case["tokens"], case["window"], case["sinks"]
    f = pos // T
    hi = torch.minimum((f + 1) * T, starts.view(b, 1).long() + n).unsqueeze(-1)
    lo = ((f - W + 1).clamp(min=0) * T if W else torch.zeros_like(f)).unsqueeze(-1)
    hidden = ~((key < hi) & ((key >= lo) | (key < S * T)))
    # rows of a K/V head: (query row, query head of the group)
    x = q.float().view(b, n, kv, group, HEAD).permute(0, 2, 1, 3, 4).flatten(2, 3) / math.sqrt(HEAD)
    hidden = hidden.unsqueeze(2).expand(b, n, group, key.numel()).flatten(1, 2).unsqueeze(1)
    s = (x @ k.transpose(-1, -2)).masked_fill_(hidden, -math.inf)
    m = s.amax(-1, keepdim=True)
    p = s.sub_(torch.where(m == -math.inf, 0.0, m)).exp_()
    total = p.sum(-1, keepdim=True)
    o = (p @ v) / torch.where(total == 0, 1.0, total)
    o = o.unflatten(2, (n, group)).permute(0, 2, 1, 3, 4).reshape(b, n, -1)
    return o.to(torch.bfloat16)


# ----------------------------------------------------------- prepare and run

def _rows(gen, *shape):
    """K or V rows: normal values, a few dims of each head far larger, as keys have them."""
    x = torch.randn(*shape, generator=gen, device=gen.device)
    w = torch.exp(0.5 * torch.randn(shape[-1], generator=gen, device=gen.device))
    return x.mul_(w)


def prepare(case, seed):
    dev = _dev()
    gen = torch.Generator(device=dev).manual_seed(seed)
    b, n, kv = case["batch"], case["rows"], case["kv_heads"]
    dtype = torch.float32 if case["dtype"] == "fp32" else torch.bfloat16
    starts = _starts(case)
    per = -(-(max(starts) + n) // PAGE)
    pool = b * per + 3
    page_map = torch.randperm(pool, generator=gen, device=dev)[: b * per].view(b, per).int()
    s = {"case": case, "page_map": page_map.contiguous(),
         "starts": torch.tensor(starts, dtype=torch.int32, device=dev)}
    if case["op"] == "write":
        s["pages"] = torch.zeros(pool, kv, PAGE_HEAD, dtype=torch.uint8, device=dev)
        s["k"] = _rows(gen, b, n, kv * HEAD).to(dtype)
        s["v"] = _rows(gen, b, n, kv * HEAD).to(dtype)
    else:
        # a pool written before: any 16 values quantise to codes with one at the end of the range
        pages = torch.empty(pool, kv, PAGE_HEAD, dtype=torch.uint8, device=dev)
        kc, ks, vc, vs = _fields(pages)
        for p0 in range(0, pool, 64):
            t = slice(p0, min(p0 + 64, pool))
            m = t.stop - t.start
            c, e = _quantise(_rows(gen, m, 16, 8, kv * HEAD).unflatten(-1, (kv, HEAD)).permute(0, 3, 1, 2, 4))
            kc[t], ks[t] = _pack(c), e
            c, e = _quantise(_rows(gen, m, 16, 8, kv * HEAD).unflatten(-1, (kv, HEAD)).permute(0, 3, 1, 2, 4))
            vc[t], vs[t] = _pack(c).unflatten(-1, (8, 8)).transpose(-3, -2), e.transpose(-1, -2)
        s["pages"] = pages
    if case["op"] == "attn":
        s["q"] = torch.randn(b, n, case["heads"] * HEAD, generator=gen, device=dev).to(torch.bfloat16)
        s["out"] = torch.empty_like(s["q"])
    else:
        s["k_out"] = torch.empty(b, n, kv * HEAD, dtype=dtype, device=dev)
        s["v_out"] = torch.empty_like(s["k_out"])
    return s


def run(s):
    case = s["case"]
    if own:
        kv4 = _kv4()
        if case["op"] == "attn":
            kv4.attn(s["q"], s["pages"], s["out"], page_map=s["page_map"], heads=case["heads"],
                     tokens=case["tokens"], window=case["window"], sinks=case["sinks"],
                     **({"starts": s["starts"]} if case["ragged"] else {"start": case["start"]}))
            return {"out": s["out"]}
        if case["op"] == "write":
            kv4.write(s["pages"], s["k"], s["v"], page_map=s["page_map"], start=case["start"])
        kv4.read(s["pages"], s["k_out"], s["v_out"], page_map=s["page_map"], start=case["start"])
        return {"k": s["k_out"], "v": s["v_out"]}
    if case["op"] == "attn":
        return {"out": _plain_attn(s["q"], s["pages"], s["page_map"], s["starts"], case)}
    if case["op"] == "write":
        _plain_write(s["pages"], s["page_map"], case["start"], s["k"], s["v"])
    k, v = _plain_read(s["pages"], s["page_map"], case["start"], case["rows"], s["k_out"].dtype)
    return {"k": k, "v": v}


# ----------------------------------------------------------------- 64 bits

def _exact_rows(x):
    """What the cache holds for rows x [..., D]: thresholds and a table of all scales, in 64 bits."""
    dev = x.device
    scales = torch.tensor([(8 + m) * 2.0 ** (e - 18) for e in range(32) for m in range(8)],
                          dtype=torch.float64, device=dev)
    g = x.to(torch.bfloat16).double().unflatten(-1, (-1, 16))
    # the nearest scale to amax / 7, the upper one in the middle between two
    middle = 7 * (scales[1:] + scales[:-1]) / 2
    s = scales[torch.searchsorted(middle, g.abs().amax(-1), right=True)].unsqueeze(-1)
    n = torch.zeros_like(g)
    for level in range(1, 8):
        n += g.abs() >= (level - 0.5) * s
    return (n * s * torch.sign(g)).flatten(-2)


def _exact_cache(pages, ids, head, which):
    """One head's rows of the pages `ids`, decoded byte by byte: [len(ids) * 128, 128] in 64 bits."""
    dev = pages.device
    t = pages[ids, head].long().view(len(ids), 16, BLOCK)
    dim = torch.arange(HEAD, device=dev)
    row = torch.arange(8, device=dev).unsqueeze(1)
    word, bit = dim // 8, dim % 8 // 2 * 4 + dim % 2 * 16
    if which == "k":
        code_at, scale_at = row * 64 + word * 4, 512 + row * 8 + dim // 16
    else:
        code_at, scale_at = 576 + dim // 16 * 64 + row * 8 + word % 2 * 4, 1088 + dim // 16 * 8 + row
    code = (t[:, :, code_at + bit // 8] >> (bit % 8)) & 15
    byte = t[:, :, scale_at]
    scale = (1 + (byte % 8).double() / 8) * torch.pow(2.0, (byte // 8 - 15).double())
    return ((code - 8).double() * scale).view(-1, HEAD)


def exact(case, seed):
    s = prepare(case, seed)
    starts, n = _starts(case), case["rows"]
    pm = s["page_map"].long()
    if case["op"] == "write":
        return {"k": _exact_rows(s["k"]), "v": _exact_rows(s["v"])}
    if case["op"] == "read":
        got = {}
        for which in ("k", "v"):
            out = torch.empty(case["batch"], n, case["kv_heads"], HEAD, dtype=torch.float64,
                              device=pm.device)
            for b in range(case["batch"]):
                for h in range(case["kv_heads"]):
                    out[b, :, h] = _exact_cache(s["pages"], pm[b], h, which)[starts[b]: starts[b] + n]
            got[which] = out.flatten(-2)
        return got
    group = case["heads"] // case["kv_heads"]
    out = torch.empty(case["batch"], n, case["heads"], HEAD, dtype=torch.float64, device=pm.device)
    q = s["q"].double().unflatten(-1, (case["heads"], HEAD))
    for b in range(case["batch"]):
        end = starts[b] + n
        sees = torch.tensor([_span(case, starts[b] + i, end) for i in range(n)], device=pm.device)
        ids = pm[b, : -(-end // PAGE)]
        key = torch.arange(end, device=pm.device)
        ok = (key < sees[:, :1]) | ((key >= sees[:, 1:2]) & (key < sees[:, 2:]))
        for h in range(case["kv_heads"]):
            k = _exact_cache(s["pages"], ids, h, "k")[:end]
            v = _exact_cache(s["pages"], ids, h, "v")[:end]
            for g in range(h * group, (h + 1) * group):
                x = torch.where(ok, q[b, :, g] @ k.T * HEAD ** -0.5, -torch.inf)
                w = torch.exp(x - torch.logsumexp(x, -1, keepdim=True))
                out[b, :, g] = torch.nan_to_num(w) @ v
    return {"out": out.flatten(-2)}
