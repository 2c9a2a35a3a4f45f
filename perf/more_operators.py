"""More operators of the paged KV cache: one case per way a serving program calls them.

A cache held in 4 bits: numbers of 1 + 2 + 1 bits with a power of two per 32 of
them, which a step's keys and values are rounded to ("append"), and which
attention reads, from one token to prompts and shared prefixes ("attend",
"prefix").  Positions with several axes, for images and video, on the way into
a cache of any type ("append").  And the pages themselves: samples that go on
from a common beginning ("fork", with the freeing of what they held), pages
moved to the front of a cache that is to shrink ("compact"), pages copied into
another cache of the same sizes ("copy").  A case's "kind" names the entry
point.  Heads, dims and pages are those of the 64 KiB KV pages that the
benchmark moves (8 heads of 128 in bf16, 16 tokens a page), with other common
shapes around them.

`own` false: plain torch operations in 32 bits.  `own` true: the framework's
operators.  exact() is the definition in 64 bits, sequence by sequence.
"""
import math
import random

import numpy as np
import torch

own = False

DEV = "cuda"
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "e4m3": torch.float8_e4m3fn, "e2m1": torch.uint8}
E4M3_MAX = 448.0
K_SCALE, V_SCALE = 1 / 32, 1 / 64  # of 8-bit caches
GROUP = 32  # numbers that share a scale
# Bytes of scales, 2^(byte - 127), that leave 6 times the scale within the rows' type, and half of it no less than its least.
SCALE_BYTES = {"bf16": (1, 252), "fp16": (104, 140)}
FILL = -7  # what a table holds where nothing is written


def _append(name, tokens, q_heads=32, kv_heads=8, dim=128, page=16, dtype="bf16", cache="bf16", heads_first=False,
            rotary=128, pairs=False, axes=0, turns=False, seconds=False, far=8192):
    return dict(name=name, kind="append", tokens=tokens, q_heads=q_heads, kv_heads=kv_heads, dim=dim, page=page,
                dtype=dtype, cache=cache, heads_first=heads_first, rotary=rotary, pairs=pairs, axes=axes, turns=turns,
                seconds=seconds, far=far)


def _attend(name, batch, q, kv, q_heads=32, kv_heads=8, dim=128, page=16, dtype="bf16", heads_first=False,
            ragged=True, cap=0.0, slopes=False, window=0, docs=0, prefix_mask=False, prefix=0, lens=1):
    return dict(name=name, kind="prefix" if prefix else "attend", batch=batch, q=q, kv=kv, q_heads=q_heads,
                kv_heads=kv_heads, dim=dim, page=page, dtype=dtype, cache="e2m1", heads_first=heads_first,
                ragged=ragged, cap=cap, slopes=slopes, window=window, docs=docs, prefix_mask=prefix_mask,
                prefix=prefix, lens=lens)


def _pages_of(name, kind, pages, kv_heads=8, dim=128, page=16, cache="bf16", heads_first=False, seqs=1, children=0,
              length=1, more=0, part=1.0, lens=1):
    return dict(name=name, kind=kind, pages=pages, kv_heads=kv_heads, dim=dim, page=page, dtype="bf16", cache=cache,
                heads_first=heads_first, seqs=seqs, children=children, length=length, more=more, part=part, lens=lens)


def listed():
    return [
        # One decode step of nine chats about images into a 4-bit cache: launches' latency.
        _append("append-9-axes-e2m1", 9, cache="e2m1", axes=3),
        # A video's tokens at (time, height, width), time in seconds.
        _append("append-6001-axes", 6001, axes=3, turns=True, seconds=True),
        # Several prompts' tokens of a whole batch into a 4-bit cache.
        _append("append-16384-e2m1", 16384, heads_first=True, page=64, cache="e2m1"),
        # A single user's decode step: latency.
        _attend("decode-1x700-e2m1", 1, 1, 700, ragged=False),
        # A serving batch's decode step over ragged contexts.
        _attend("decode-64x16384-e2m1", 64, 1, 16384, heads_first=True),
        # Capped scores in a sliding window, wide heads, pages that are no power of two.
        _attend("decode-33x6000-cap-e2m1", 33, 1, 6000, q_heads=16, dim=256, page=24, dtype="fp16", heads_first=True,
                cap=50.0, window=4096),
        # A chunk of a long prompt behind what is in the cache already.
        _attend("prompt-2048of8192-e2m1", 1, 2048, 8192, page=64, heads_first=True, ragged=False),
        # Many requests on one long document.
        _attend("prefix-64x32768-e2m1", 64, 1, 32768 + 1024, heads_first=True, prefix=32768),
        # A few samples from one chat, dropped again: latency.
        _pages_of("fork-4", "fork", 512, seqs=2, children=4, length=700, more=16),
        # A search's step: many sequences go on from a few, each with room for its next tokens.
        _pages_of("fork-256", "fork", 12000, seqs=16, children=256, length=5000, more=100, cache="e4m3", page=32),
        # A cache of 0.8 GB, three fifths of it free, brought together at its front.
        _pages_of("compact-12000", "compact", 12000, seqs=48, length=4000),
        # A 4-bit cache's pages into another cache, whose pages hold one head after the other.
        _pages_of("copy-3001-e2m1", "copy", 8000, cache="e2m1", part=0.375),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["append", "append", "decode", "decode", "prompt", "prefix", "fork", "compact", "copy"])
    q_heads, kv_heads = rng.choice([(32, 8), (8, 8), (16, 2), (28, 4), (12, 12), (40, 8), (16, 1), (64, 8)])
    dim = rng.choice([64, 128, 128, 128, 256])
    dtype = rng.choice(["bf16", "bf16", "fp16"])
    common = dict(kv_heads=kv_heads, dim=dim, heads_first=rng.random() < 0.5, page=rng.choice([1, 8, 16, 16, 24, 32, 64, 128]))
    if kind == "append":
        axes = rng.choice([0, 2, 3, 3])
        cache = rng.choice(["e2m1", "e2m1", dtype, "e4m3"]) if axes else "e2m1"
        c = _append("", _log(rng, 1, 16384 * 4096 // ((q_heads + kv_heads) * dim * 5) + 1), q_heads=q_heads,
                    dtype=dtype, cache=cache, rotary=rng.choice([dim, dim, dim // 2, dim // 4 + 2]),
                    pairs=rng.random() < 0.4, axes=axes, turns=rng.random() < 0.5,
                    seconds=bool(axes) and rng.random() < 0.4, far=rng.choice([4096, 65536, 1 << 20]), **common)
    elif kind in ("fork", "compact", "copy"):
        common["cache"] = rng.choice(["bf16", "e4m3", "e2m1"])
        lens = rng.randint(1, 1 << 30)
        most = max(64, min(40000, (1 << 29) // (common["page"] * kv_heads * dim * 2 * 2)))
        pages = _log(rng, 64, most)
        if kind == "copy":
            c = _pages_of("", kind, pages, part=rng.uniform(0.02, 0.45), lens=lens, **common)
        else:
            seqs = _log(rng, 1, 32)
            length = max(1, int(pages * common["page"] / seqs * rng.uniform(0.05, 0.45)))
            children = _log(rng, 1, 256) if kind == "fork" else 0
            more = _log(rng, 1, max(2, pages * common["page"] // (8 * children))) if children else 0
            c = _pages_of("", kind, pages, seqs=seqs, children=children, length=length, more=more, lens=lens, **common)
    else:
        extra = dict(q_heads=q_heads, dtype=dtype, cap=rng.choice([0.0, 0.0, 30.0, 50.0]), slopes=rng.random() < 0.3,
                     lens=rng.randint(1, 1 << 30), ragged=rng.random() < 0.7, **common)
        if kind == "decode":
            batch = _log(rng, 1, 128)
            extra["window"] = rng.choice([0, 0, _log(rng, 16, 4096)])
            c = _attend("", batch, rng.choice([1, 1, 1, 2, 5]),
                        _log(rng, 16, min(16384, 400_000_000 // (batch * kv_heads * dim))), **extra)
        elif kind == "prompt":
            most = max(64, min(2048, (2048 * 4096) // (q_heads * dim)))
            q = _log(rng, 17, most)
            batch = _log(rng, 1, max(1, most // q))
            extra["docs"] = rng.choice([0, 0, rng.randint(2, 12)])
            extra["prefix_mask"] = rng.random() < 0.4
            extra["window"] = rng.choice([0, 0, 0, _log(rng, 64, 2048)])
            past = rng.choice([0, 0, _log(rng, 1, 4096)])
            c = _attend("", batch, q, q + past, **extra)
        else:
            batch = _log(rng, 2, 64)
            q = rng.choice([1, 1, 1, 3, 8])
            prefix = _log(rng, 64, min(32768, (1 << 27) // (kv_heads * dim), (1 << 35) // (batch * q * q_heads * dim)))
            own_len = _log(rng, 8, min(1024, (1 << 26) // (batch * kv_heads * dim)))
            c = _attend("", batch, q, prefix + max(own_len, q), prefix=prefix, **extra)
    del c["name"]
    return c


# --------------------------------------------------------------- the batch

def _pages(n, page):
    return -(-n // page)


def _lengths(case):
    """Lengths (q_len, kv_len) of every sequence; they are the case's, so that work() knows them."""
    rng = random.Random(case["lens"] * 7919 + case["batch"])
    q = [case["q"]] * case["batch"]
    kv = [case["kv"]] * case["batch"]
    for b in range(case["batch"]):
        if case["ragged"] and b:  # the first sequence keeps the full lengths
            if case["q"] > 8:
                q[b] = _log(rng, max(1, case["q"] // 16), case["q"])
            own_kv = case["kv"] - case["prefix"]
            kv[b] = case["prefix"] + max(q[b], _log(rng, max(1, own_kv // 16), own_kv))
    return q, kv


def _marks(case):
    """Per token, sequence after sequence: where its document starts and where the prefix that it sees ends."""
    rng = random.Random(case["lens"] * 104729 + case["kv"])
    start, end = [], []
    for q, kv in zip(*_lengths(case)):
        pos = np.arange(kv - q, kv)
        cuts = np.array(sorted([0] + [rng.randint(1, max(1, kv - 1)) for _ in range(max(0, case["docs"] - 1))]))
        at = np.searchsorted(cuts, pos, side="right") - 1
        lens = np.diff(np.append(cuts, kv))
        seen = np.array([rng.randint(0, int(n) // 2) for n in lens])
        start.append(cuts[at])
        end.append(cuts[at] + seen[at])
    return np.concatenate(start).astype(np.int32), np.concatenate(end).astype(np.int32)


def _visible(case):
    """Per token (position, first visible key, end of the visible keys), in numpy."""
    q, kv = _lengths(case)
    pos = np.concatenate([np.arange(k - n, k) for n, k in zip(q, kv)])
    length = np.repeat(kv, q)
    start, end = _marks(case)
    lo = np.maximum(0, start if case["docs"] else 0)
    lo = np.maximum(lo, pos - case["window"] + 1) if case["window"] else np.broadcast_to(lo, pos.shape)
    hi = np.minimum(length, np.maximum(pos + 1, end)) if case["prefix_mask"] else pos + 1
    return pos, lo, hi


def _family(case):
    """Sequences in a pool of pages, and what goes on from them: lengths, children's (parent, shared length, room)."""
    rng = random.Random(case["lens"] * 6151 + case["pages"])
    lens = [case["length"]] + [_log(rng, max(1, case["length"] // 8), case["length"]) for _ in range(case["seqs"] - 1)]
    kids = []
    for _ in range(case["children"]):
        b = rng.randrange(case["seqs"])
        n = lens[b] if rng.random() < 0.6 else rng.randint(1, lens[b])
        kids.append((b, n, n + rng.randint(1, max(1, case["more"]))))
    return lens, kids


def _row_bytes(case):
    """Bytes of a token's keys and values."""
    n = 2 * case["kv_heads"] * case["dim"]
    return {"e2m1": n // 2 + n // GROUP, "e4m3": n}.get(case["cache"], 2 * n)


def work(case):
    if case["kind"] == "append":
        t, d = case["tokens"], case["dim"]
        heads = case["q_heads"] + case["kv_heads"]
        written = _row_bytes(case)
        if case["cache"] == "e2m1":  # and read back as rows
            written += _row_bytes(case) + 4 * case["kv_heads"] * d
        return dict(bytes=t * (2 * d * (2 * case["q_heads"] + 2 * case["kv_heads"]) + written + 8 + 4 * max(1, case["axes"])),
                    flops=t * heads * case["rotary"] * 3)
    if case["kind"] == "copy":
        return dict(bytes=2 * int(case["part"] * case["pages"]) * case["page"] * _row_bytes(case), flops=0)
    if case["kind"] in ("fork", "compact"):
        lens, kids = _family(case)
        ps = case["page"]
        if case["kind"] == "fork":
            tokens = sum(n % ps for _, n, _ in kids)
            entries = sum(2 * (n // ps) + _pages(room, ps) for _, n, room in kids)
        else:
            used = sum(_pages(n, ps) for n in lens)
            # The live pages lie anywhere: those past the front move.
            tokens = ps * used * max(0, case["pages"] - used) // case["pages"]
            entries = 2 * used + 2 * case["pages"]
        return dict(bytes=2 * tokens * _row_bytes(case) + 4 * entries + 4 * case["pages"], flops=0)
    q, kv = _lengths(case)
    pos, lo, hi = _visible(case)
    first = np.concatenate([[0], np.cumsum(q)])
    keys = sum(max(0, int(hi[a:b].max()) - max(case["prefix"], int(lo[a:b].min())))
               for a, b in zip(first[:-1], first[1:]) if b > a)
    if case["prefix"]:
        keys += max(0, case["prefix"] - int(lo.min()))
    pairs = int(np.maximum(0, hi - lo).sum()) * case["q_heads"]
    return dict(bytes=keys * _row_bytes(case) + len(pos) * case["q_heads"] * (4 * case["dim"] + 4),
                flops=4 * case["dim"] * pairs)


# ---------------------------------------------------------------- 4-bit numbers

MAGNITUDES = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _to_e2m1(x, dtype):
    """x [..., dim] in 32 bits -> (bytes of two numbers, the first in the low half; bytes of scales)."""
    g = x.unflatten(-1, (-1, GROUP))
    top = g.abs().amax(-1)
    # The least power of two of which the largest is at most seven: what lies between six and seven is rounded to six.
    byte = ((top.view(torch.int32) + 0x1FFFFF) >> 23) - 2
    byte = byte.clamp(*SCALE_BYTES[dtype])
    y = g * ((254 - byte) << 23).view(torch.float32)[..., None]
    a = y.abs()
    code = ((a > 0.25).to(torch.uint8) + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5) + (a >= 3.5) + (a > 5))
    code = (code + 8 * torch.signbit(y)).to(torch.uint8).flatten(-2)
    return code[..., 0::2] | (code[..., 1::2] << 4), byte.to(torch.uint8)


def _from_e2m1(codes, scales):
    """The values in 32 bits, [..., dim]."""
    table = torch.tensor(MAGNITUDES + tuple(-m for m in MAGNITUDES), device=codes.device)
    both = torch.stack((codes & 15, codes >> 4), -1).flatten(-2)
    x = table[both.int()].unflatten(-1, (-1, GROUP))
    return (x * (scales.int() << 23).view(torch.float32)[..., None]).flatten(-2)


# ------------------------------------------------------------------ inputs

def _rand(gen, *shape):
    return torch.randn(*shape, generator=gen, device=DEV, dtype=torch.float32)


def _cache(case, gen, num_pages, fill, heads_first=None):
    """Pages as one block each, keys before values (before their scales): the blocks, and views [pages, page, heads, ...]."""
    heads_first = case["heads_first"] if heads_first is None else heads_first
    h, ps, d = case["kv_heads"], case["page"], case["dim"]
    inner = (h, ps) if heads_first else (ps, h)
    order = (0, 2, 1, 3) if heads_first else (0, 1, 2, 3)
    c = {"num_pages": num_pages}
    if case["cache"] == "e2m1":
        rows = ps * h
        size = -(-rows * (d + d // GROUP * 2) // 16) * 16
        c["blocks"] = torch.zeros(num_pages, size, device=DEV, dtype=torch.uint8)
        at = 0
        for name, width in (("k", d // 2), ("v", d // 2), ("k_scales", d // GROUP), ("v_scales", d // GROUP)):
            c[name] = c["blocks"][:, at:at + rows * width].unflatten(1, (*inner, width)).permute(order)
            at += rows * width
        if fill:
            # Keys have dims of a larger spread than others, after their rotation too.
            wide = 1 + 3 * (torch.rand(d, generator=gen, device=DEV) < 0.06)
            for first in range(0, num_pages, 2048):
                part = slice(first, first + 2048)
                for name in ("k", "v"):
                    x = _rand(gen, *c[name][part].shape[:3], d)
                    codes, scales = _to_e2m1(x * wide if name == "k" else x, case["dtype"])
                    c[name][part], c[name + "_scales"][part] = codes, scales
        return c
    c["blocks"] = torch.zeros(num_pages, 2, *inner, d, device=DEV, dtype=TYPES[case["cache"]])
    if fill:
        scale = torch.tensor([K_SCALE, V_SCALE], device=DEV).view(2, 1, 1, 1)
        for first in range(0, num_pages, 4096):
            part = c["blocks"][first:first + 4096]
            x = _rand(gen, *part.shape)
            part.copy_(((x / scale).clamp(-E4M3_MAX, E4M3_MAX) if case["cache"] == "e4m3" else x).to(c["blocks"].dtype))
    c["k"], c["v"] = c["blocks"][:, 0].permute(order), c["blocks"][:, 1].permute(order)
    return c


def _grid(case, rng):
    """Positions [axes][tokens] of frames, row by row."""
    t = case["tokens"]
    side = max(2, min(64, int(round(t ** (1 / 3) * 2))))
    wide = max(2, int(side * rng.uniform(0.6, 1.8)))
    at = np.arange(t)
    first = int(rng.integers(0, max(1, case["far"] - t)))
    axes = [at // (side * wide), at // wide % side, at % wide][-case["axes"]:]
    pos = np.stack([first + a for a in axes])
    if case["seconds"]:
        pos = pos.astype(np.float32)
        pos[0] = first + axes[0] * np.float32(0.48)
    return pos


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    rng = np.random.default_rng(seed)
    dtype = TYPES[case["dtype"]]
    s = dict(case)
    s["error"] = torch.zeros(1, dtype=torch.int32, device=DEV)
    if case["kind"] == "append":
        _prepare_append(s, case, gen, rng, dtype)
    elif case["kind"] in ("fork", "compact", "copy"):
        _prepare_pages(s, case, gen, rng)
    else:
        _prepare_attention(s, case, gen, rng, dtype)
    return s


def _prepare_append(s, case, gen, rng, dtype):
    t, hq, hk, d, page = (case[n] for n in ("tokens", "q_heads", "kv_heads", "dim", "page"))
    # Half of the pages are another batch's; a projection's output holds q, k and v of a token side by side.
    pages = 2 * _pages(t, page)
    s["cache_of"] = _cache(case, gen, pages, False)
    rows = _rand(gen, t, (hq + 2 * hk) * d).to(dtype)
    s["q_rows"], s["k_rows"], s["v_rows"] = (x.unflatten(1, (-1, d)) for x in rows.split([hq * d, hk * d, hk * d], 1))
    place = rng.permutation(pages)[:_pages(t, page)].astype(np.int64)
    at = np.arange(t)
    s["slots"] = torch.from_numpy(place[at // page] * page + at % page).to(DEV)
    half = case["rotary"] // 2
    if case["axes"]:
        pos = _grid(case, rng)
        s["positions"] = torch.from_numpy(pos if case["seconds"] else pos.astype(np.int32)).to(DEV)
        i = np.arange(half)
        axis = i % case["axes"] if case["turns"] else i * case["axes"] // max(1, half)
        s["axis"] = torch.from_numpy(axis.astype(np.uint8)).to(DEV)
    else:
        first = int(rng.integers(0, max(1, case["far"] - t)))
        s["positions"] = torch.from_numpy((first + at).astype(np.int32)).to(DEV)
    s["inv_freq"] = torch.from_numpy((10000.0 ** (-np.arange(half) / half)).astype(np.float32)).to(DEV)
    s["q_out"] = torch.empty(t, hq, d, device=DEV, dtype=dtype)
    if case["cache"] == "e2m1":
        s["k_out"], s["v_out"] = (torch.empty(t, hk, d, device=DEV, dtype=dtype) for _ in range(2))


def _prepare_attention(s, case, gen, rng, dtype):
    hq, d, page = case["q_heads"], case["dim"], case["page"]
    q_len, kv_len = _lengths(case)
    own_pages = [_pages(n - case["prefix"], page) for n in kv_len]
    shared = _pages(case["prefix"], page)
    place = rng.permutation(sum(own_pages) + shared + 3).astype(np.int32)  # three free pages
    s["cache_of"] = _cache(case, gen, len(place), True)
    table = np.zeros((case["batch"], max(own_pages)), np.int32)
    used = shared
    for b, n in enumerate(own_pages):
        table[b, :n] = place[used:used + n]
        used += n
    s["prefix_table"] = torch.from_numpy(place[:shared].copy()).to(DEV)
    s["table"] = torch.from_numpy(table).to(DEV)
    s["q_start"] = torch.from_numpy(np.concatenate([[0], np.cumsum(q_len)]).astype(np.int32)).to(DEV)
    s["kv_len"] = torch.tensor(kv_len, dtype=torch.int32, device=DEV)
    s["tokens"], s["max_q"], s["max_kv"] = sum(q_len), max(q_len), max(kv_len)
    s["q_rows"] = (1.5 * _rand(gen, s["tokens"], hq, d)).to(dtype)
    start, end = _marks(case)
    s["doc_start"] = torch.from_numpy(start).to(DEV) if case["docs"] else None
    s["prefix_end"] = torch.from_numpy(end).to(DEV) if case["prefix_mask"] else None
    s["slope"] = (2.0 ** (-8.0 * torch.arange(1, hq + 1, device=DEV) / hq)).float() if case["slopes"] else None
    s["out"] = torch.empty(s["tokens"], hq, d, device=DEV, dtype=dtype)
    s["lse"] = torch.empty(s["tokens"], hq, device=DEV, dtype=torch.float32)
    s["scale"] = d ** -0.5


def _prepare_pages(s, case, gen, rng):
    n, ps = case["pages"], case["page"]
    s["cache_of"] = _cache(case, gen, n, True)
    if case["kind"] == "copy":
        count = int(case["part"] * n)
        more = n + 5
        s["to"] = _cache(case, gen, more, False, heads_first=not case["heads_first"])
        copies = np.stack([rng.permutation(n)[:count], rng.permutation(more)[:count], np.full(count, ps),
                           np.zeros(count)], 1)
        s["copies"] = torch.from_numpy(copies.astype(np.int32)).to(DEV)
        return
    lens, kids = _family(case)
    pages = [_pages(k, ps) for k in lens]
    place = rng.permutation(n).astype(np.int32)[:sum(pages)]
    table = np.full((len(lens), max(pages) + 3), FILL, np.int32)
    refs = np.zeros(n, np.int32)
    refs[place] = 1
    used = 0
    for b, k in enumerate(pages):
        table[b, :k] = place[used:used + k]
        used += k
    s["table"], s["refs"] = torch.from_numpy(table).to(DEV), torch.from_numpy(refs).to(DEV)
    s["lens"] = torch.tensor(lens, dtype=torch.int32, device=DEV)
    if case["kind"] == "fork":
        width = max(_pages(room, ps) for _, _, room in kids) + 1
        s["child_table"] = torch.full((len(kids) + 2, width), FILL, dtype=torch.int32, device=DEV)  # two rows are others'
        s["child"] = torch.from_numpy(rng.permutation(len(kids) + 2)[:len(kids)].astype(np.int32)).to(DEV)
        for i, name in enumerate(("parent", "shared", "room")):
            s[name] = torch.tensor([k[i] for k in kids], dtype=torch.int32, device=DEV)
        s["copies"] = torch.zeros(len(kids), 4, dtype=torch.int32, device=DEV)
    else:
        s["new_table"] = torch.full_like(s["table"], FILL)
        s["new_refs"], s["page_map"] = torch.full_like(s["refs"], FILL), torch.full_like(s["refs"], FILL)
        s["copies"] = torch.zeros(max(1, n // 2), 4, dtype=torch.int32, device=DEV)
        s["num_copies"] = torch.zeros(1, dtype=torch.int32, device=DEV)


# ---------------------------------------------------------------- one pass

def run(s):
    if s["kind"] == "append":
        return (_own_append if own else _plain_append)(s)
    if s["kind"] == "fork":
        return (_own_fork if own else _plain_fork)(s)
    if s["kind"] == "compact":
        return (_own_compact if own else _plain_compact)(s)
    if s["kind"] == "copy":
        return (_own_copy if own else _plain_copy)(s)
    return (_own_attention if own else _plain_attention)(s)


def _own_cache(s, name="cache_of"):
    """The cache's descriptor, which a program makes once with its pages."""
    import gfd_amd

    c = s[name]
    if "handle" not in c:
        k = c["k"]
        sizes = dict(num_pages=k.shape[0], page_size=k.shape[1], num_heads=k.shape[2], head_dim=s["dim"])
        places = dict(k=k.data_ptr(), v=c["v"].data_ptr(), page_stride=k.stride(0), slot_stride=k.stride(1),
                      head_stride=k.stride(2))
        if s["cache"] == "e2m1":
            c["handle"] = gfd_amd.KV4Cache(k_scales=c["k_scales"].data_ptr(), v_scales=c["v_scales"].data_ptr(),
                                           scale_page_stride=c["k_scales"].stride(0), **places, **sizes)
        else:
            c["handle"] = gfd_amd.KVCache(
                dtype={"bf16": gfd_amd.BF16, "fp16": gfd_amd.FP16, "e4m3": gfd_amd.E4M3}[s["cache"]], k_scale=K_SCALE,
                v_scale=V_SCALE, **places, **sizes)
        s["type"] = gfd_amd.BF16 if s["dtype"] == "bf16" else gfd_amd.FP16
    return c["handle"]


def _now(s):
    return dict(error_flag=s["error"].data_ptr(), stream=torch.cuda.current_stream().cuda_stream)


def _own_append(s):
    import gfd_amd

    cache = _own_cache(s)
    q, k, v, out, pos = s["q_rows"], s["k_rows"], s["v_rows"], s["q_out"], s["positions"]
    rows = gfd_amd.KVRows(
        q=q.data_ptr(), k=k.data_ptr(), v=v.data_ptr(), q_out=out.data_ptr(), q_stride=q.stride(0),
        k_stride=k.stride(0), v_stride=v.stride(0), q_out_stride=out.stride(0),
        positions=None if s["axes"] else pos.data_ptr(), slots=s["slots"].data_ptr(),
        inv_freq=s["inv_freq"].data_ptr(), num_tokens=q.shape[0], num_q_heads=q.shape[1], rotary_dim=s["rotary"],
        interleaved=int(s["pairs"]), dtype=s["type"])
    axes = None
    if s["axes"]:
        axes = gfd_amd.RotaryAxes(positions=pos.data_ptr(), axis=s["axis"].data_ptr(), axis_stride=pos.stride(0),
                                  token_stride=pos.stride(1), num_axes=s["axes"], float_positions=int(s["seconds"]))
    gfd_amd.kv_append(cache, rows, axes=axes, **_now(s))
    if s["cache"] != "e2m1":
        return dict(q=out, cache=s["cache_of"]["blocks"])
    k, v = s["k_out"], s["v_out"]
    back = gfd_amd.KVRead(k=k.data_ptr(), v=v.data_ptr(), k_stride=k.stride(0), v_stride=v.stride(0),
                          slots=s["slots"].data_ptr(), num_tokens=k.shape[0], dtype=s["type"])
    gfd_amd.kv_read(cache, back, **_now(s))
    return dict(q=out, k=k, v=v)


def _own_attention(s):
    import gfd_amd

    cache = _own_cache(s)
    q, out, table = s["q_rows"], s["out"], s["table"]
    call = gfd_amd.Attention(
        q=q.data_ptr(), out=out.data_ptr(), lse=s["lse"].data_ptr(), q_stride=q.stride(0), out_stride=out.stride(0),
        q_start=s["q_start"].data_ptr(), kv_len=s["kv_len"].data_ptr(), block_table=table.data_ptr(),
        table_stride=table.stride(0), doc_start=s["doc_start"].data_ptr() if s["docs"] else None,
        prefix_end=s["prefix_end"].data_ptr() if s["prefix_mask"] else None,
        slopes=s["slope"].data_ptr() if s["slopes"] else None, scale=s["scale"], softcap=s["cap"], window=s["window"],
        batch=s["batch"], num_tokens=s["tokens"], max_q_len=s["max_q"], max_kv_len=s["max_kv"],
        num_q_heads=q.shape[1], dtype=s["type"])
    if "workspace" not in s:  # kept, as a program keeps it for its largest batch
        s["workspace"] = torch.empty(gfd_amd.attention_workspace_bytes(cache, call, s["prefix"]), dtype=torch.uint8,
                                     device=DEV)
    more = dict(workspace=s["workspace"].data_ptr(), workspace_bytes=s["workspace"].numel(), **_now(s))
    if s["prefix"]:
        gfd_amd.shared_prefix_attention(cache, call, s["prefix_table"].data_ptr(), s["prefix"], **more)
    else:
        gfd_amd.paged_attention(cache, call, **more)
    return dict(out=out, lse=s["lse"])


def _own_pool(s):
    """The pool's descriptor and what its calls need, which a program makes once with its pages."""
    import gfd_amd

    if "pool" not in s:
        s["pool"] = gfd_amd.KVPool(refs=s["refs"].data_ptr(), num_pages=s["pages"], page_size=s["page"])
        s["workspace"] = torch.empty(gfd_amd.kv_pool_workspace_bytes(s["pool"], s["children"]), dtype=torch.uint8,
                                     device=DEV)
    return s["pool"], dict(workspace=s["workspace"].data_ptr(), workspace_bytes=s["workspace"].numel())


def _own_fork(s):
    import gfd_amd

    cache, (pool, space) = _own_cache(s), _own_pool(s)
    table, kids, copies = s["table"], s["child_table"], s["copies"]
    call = gfd_amd.KVFork(table=table.data_ptr(), child_table=kids.data_ptr(), table_stride=table.stride(0),
                          child_stride=kids.stride(0), rows=table.shape[0], child_rows=kids.shape[0],
                          parent=s["parent"].data_ptr(), child=s["child"].data_ptr(), len=s["shared"].data_ptr(),
                          capacity=s["room"].data_ptr(), copies=copies.data_ptr(), num=s["children"])
    gfd_amd.kv_fork(pool, call, **space, **_now(s))
    gfd_amd.kv_copy_pages(cache, cache, copies.data_ptr(), s["children"], **_now(s))
    gfd_amd.kv_free(pool, kids.data_ptr(), kids.stride(0), kids.shape[0], s["child"].data_ptr(), s["room"].data_ptr(),
                    s["children"], **_now(s))
    return dict(table=kids, copies=copies, refs=s["refs"], cache=s["cache_of"]["blocks"])


def _own_compact(s):
    import gfd_amd

    cache, (pool, space) = _own_cache(s), _own_pool(s)
    table, new, copies = s["table"], s["new_table"], s["copies"]
    call = gfd_amd.KVCompact(new_refs=s["new_refs"].data_ptr(), table=table.data_ptr(), new_table=new.data_ptr(),
                             table_stride=table.stride(0), new_stride=new.stride(0), len=s["lens"].data_ptr(),
                             rows=table.shape[0], page_map=s["page_map"].data_ptr(), copies=copies.data_ptr(),
                             num_copies=s["num_copies"].data_ptr())
    gfd_amd.kv_compact(pool, call, **space, **_now(s))
    gfd_amd.kv_copy_pages(cache, cache, copies.data_ptr(), copies.shape[0], count=s["num_copies"].data_ptr(), **_now(s))
    return dict(table=new, refs=s["new_refs"], page_map=s["page_map"], copies=copies, num_copies=s["num_copies"],
                cache=s["cache_of"]["blocks"])


def _own_copy(s):
    import gfd_amd

    gfd_amd.kv_copy_pages(_own_cache(s, "to"), _own_cache(s), s["copies"].data_ptr(), s["copies"].shape[0], **_now(s))
    return dict(cache=s["to"]["blocks"])


def _rotate(x, cos, sin, pairs):
    r = 2 * cos.shape[-1]
    if pairs:
        a, b = x[..., 0:r:2], x[..., 1:r:2]
        turned = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
    else:
        a, b = x[..., :r // 2], x[..., r // 2:r]
        turned = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
    return torch.cat((turned, x[..., r:]), -1)


def _plain_append(s):
    pos = s["positions"].double()
    pos = pos[s["axis"].long()].T[:, None] if s["axes"] else pos[:, None, None]
    angle = pos * s["inv_freq"].double()  # far positions: 64 bits
    cos, sin = angle.cos().float(), angle.sin().float()
    q = _rotate(s["q_rows"].float(), cos, sin, s["pairs"]).to(s["q_rows"].dtype)
    k, v = _rotate(s["k_rows"].float(), cos, sin, s["pairs"]), s["v_rows"].float()
    page, slot, c = s["slots"] // s["page"], s["slots"] % s["page"], s["cache_of"]
    if s["cache"] == "e2m1":
        for name, x in (("k", k), ("v", v)):
            c[name][page, slot], c[name + "_scales"][page, slot] = _to_e2m1(x, s["dtype"])
        back = {name: _from_e2m1(c[name][page, slot], c[name + "_scales"][page, slot]).to(q.dtype) for name in ("k", "v")}
        return dict(q=q, **back)
    if s["cache"] == "e4m3":
        k, v = (k / K_SCALE).clamp(-E4M3_MAX, E4M3_MAX), (v / V_SCALE).clamp(-E4M3_MAX, E4M3_MAX)
    kind = torch.uint8 if s["cache"] == "e4m3" else c["blocks"].dtype  # an 8-bit float is stored as its bits
    c["k"].view(kind)[page, slot] = k.to(c["blocks"].dtype).view(kind)
    c["v"].view(kind)[page, slot] = v.to(c["blocks"].dtype).view(kind)
    return dict(q=q, cache=c["blocks"])


def _plain_keys(s, name, table, n):
    """[..., n keys, heads, dim] in 32 bits through a table of pages."""
    j = torch.arange(n, device=DEV)
    page, slot, c = table[..., j // s["page"]].long(), j % s["page"], s["cache_of"]
    return _from_e2m1(c[name][page, slot], c[name + "_scales"][page, slot])


def _plain_attention(s):
    hq, hk, d, pre = s["q_heads"], s["kv_heads"], s["dim"], s["prefix"]
    b, n, g, t = s["batch"], s["max_q"], hq // hk, s["tokens"]
    first, count = s["q_start"][:-1, None], s["q_start"].diff()[:, None]
    i = torch.arange(n, device=DEV)
    tok = torch.where(i < count, first + i, t).long()  # [b, n]; t: no token
    at = tok.clamp(max=t - 1)
    pos = s["kv_len"][:, None] - count + i
    lo = s["doc_start"][at].clamp(min=0) if s["docs"] else torch.zeros_like(pos)
    lo = torch.maximum(lo, pos - s["window"] + 1) if s["window"] else lo
    hi = torch.maximum(pos + 1, s["prefix_end"][at]) if s["prefix_mask"] else pos + 1
    hi = torch.minimum(hi, s["kv_len"][:, None])
    q = s["q_rows"][at].float().view(b, n, hk, g, d).permute(0, 2, 3, 1, 4).reshape(b, hk, g * n, d)
    k, v = (_plain_keys(s, name, s["table"], s["max_kv"] - pre).transpose(1, 2) for name in ("k", "v"))
    x = q @ k.transpose(2, 3).contiguous()  # [b, hk, g * n, own keys]
    if pre:  # the shared keys, once for all rows
        pk, pv = (_plain_keys(s, name, s["prefix_table"], pre).transpose(0, 1) for name in ("k", "v"))
        rows = q.transpose(0, 1).reshape(hk, b * g * n, d)
        y = (rows @ pk.transpose(1, 2).contiguous()).view(hk, b, g * n, pre).transpose(0, 1)
        x = torch.cat((y, x), 3)
    x = x.view(b, hk, g, n, -1).mul_(s["scale"])
    if s["cap"]:
        x = x.div_(s["cap"]).tanh_().mul_(s["cap"])
    j = torch.arange(x.shape[-1], device=DEV)
    if s["slopes"]:
        x = x - s["slope"].view(hk, g, 1, 1) * (pos[..., None] - j).abs()[:, None, None]
    seen = (j >= lo[..., None]) & (j < hi[..., None])
    x = x.masked_fill_(~seen[:, None, None], -math.inf)
    top = x.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, 0.0, top)
    x = x.sub_(top).exp_()
    total = x.sum(-1, keepdim=True)
    x = x.view(b, hk, g * n, -1)
    o = x[..., pre:] @ v.contiguous()
    if pre:
        p = x[..., :pre].transpose(0, 1).reshape(hk, b * g * n, pre)
        o += (p @ pv.contiguous()).view(hk, b, g * n, d).transpose(0, 1)
    o = o.view(b, hk, g, n, d) / torch.where(total == 0, 1.0, total)
    lse = (top + total.log()).squeeze(-1)
    out = torch.empty(t + 1, hq, d, device=DEV, dtype=s["q_rows"].dtype)
    out[tok] = o.permute(0, 3, 1, 2, 4).reshape(b, n, hq, d).to(out.dtype)
    norm = torch.empty(t + 1, hq, device=DEV)
    norm[tok] = lse.permute(0, 3, 1, 2).reshape(b, n, hq)
    return dict(out=out[:t], lse=norm[:t])


def _planes(s, c):
    """Views [pages, slot, head, ...] of whatever a page holds, as bits."""
    kind = torch.uint8 if s["cache"] in ("e4m3", "e2m1") else c["blocks"].dtype
    return [c[n].view(kind) for n in ("k", "v", "k_scales", "v_scales") if n in c]


def _plain_copy(s):
    src, dst = s["copies"][:, 0].long(), s["copies"][:, 1].long()
    for x, y in zip(_planes(s, s["cache_of"]), _planes(s, s["to"])):
        y[dst] = x[src]  # all slots
    return dict(cache=s["to"]["blocks"])


def _plain_fork(s):
    ps, n, refs = s["page"], s["children"], s["refs"]
    kids, width = s["child_table"], s["child_table"].shape[1]
    full, part, end = s["shared"] // ps, s["shared"] % ps, (s["room"] + ps - 1) // ps
    need = (end - full).long()
    j = torch.arange(width, device=DEV)
    from_parent = j < full[:, None]
    old = s["table"][s["parent"].long()[:, None], j.clamp(max=s["table"].shape[1] - 1)]
    fresh = (j >= full[:, None]) & (j < end[:, None])
    rank = (need.cumsum(0) - need)[:, None] + (j - full[:, None])
    free = (refs != 0).int().sort(stable=True)[1].int()  # free pages first, in order
    new = torch.where(rank < (refs == 0).sum(), free[rank.clamp(0, len(free) - 1)], -1)
    row = kids[s["child"].long()]
    row = torch.where(from_parent, old, torch.where(fresh, new, row))
    kids[s["child"].long()] = row
    used = (from_parent | fresh) & (row >= 0)
    refs.index_add_(0, row.clamp(min=0).flatten(), used.flatten().int())
    last = full.long()[:, None]
    src = s["table"][s["parent"].long()[:, None], last].squeeze(1)
    dst = row.gather(1, last).squeeze(1)
    some = (part > 0) & (dst >= 0)
    nothing = torch.zeros_like(part)
    s["copies"].copy_(torch.stack((torch.where(some, src, -1), torch.where(some, dst, -1),
                                   torch.where(some, part, 0), nothing), 1))
    some = some.nonzero().squeeze(1)
    page, to, slot = src[some].long()[:, None], dst[some].long()[:, None], torch.arange(ps, device=DEV)
    take = (slot < part[some][:, None])[..., None, None]
    for x in _planes(s, s["cache_of"]):
        x[to, slot] = torch.where(take, x[page, slot], x[to, slot])
    refs.index_add_(0, row.clamp(min=0).flatten(), -used.flatten().int())  # and freed again
    return dict(table=kids, copies=s["copies"], refs=refs, cache=s["cache_of"]["blocks"])


def _plain_compact(s):
    used = s["refs"] != 0
    n, ps = s["pages"], s["page"]
    at = torch.arange(n, device=DEV)
    live = used.sum()
    src = (used & (at >= live)).nonzero().squeeze(1)
    dst = (~used & (at < live)).nonzero().squeeze(1)
    where = torch.where(used, at, -1)
    where[src] = dst
    s["page_map"].copy_(where)
    s["new_refs"].copy_(torch.where(at < live, s["refs"], 0))
    s["new_refs"][dst] = s["refs"][src]
    j = torch.arange(s["table"].shape[1], device=DEV)
    named = j < ((s["lens"] + ps - 1) // ps)[:, None]
    s["new_table"].copy_(torch.where(named, where[s["table"].clamp(min=0).long()].int(), s["new_table"]))
    moves = torch.stack((src, dst, torch.full_like(src, ps), torch.zeros_like(src)), 1).int()
    s["copies"][:len(src)] = moves
    s["num_copies"].fill_(len(src))
    for x in _planes(s, s["cache_of"]):
        x[dst] = x[src]
    return dict(table=s["new_table"], refs=s["new_refs"], page_map=s["page_map"], copies=s["copies"],
                num_copies=s["num_copies"], cache=s["cache_of"]["blocks"])


# ------------------------------------------------------- the definition, 64 bits

def _nearest4(x, dtype):
    """x [..., dim] in 64 bits as a 4-bit cache holds it: the nearest multiples of its group's power of two, ties to even."""
    g = x.unflatten(-1, (-1, GROUP))
    lo, hi = SCALE_BYTES[dtype]
    power = torch.full(g.shape[:-1], lo - 127, device=DEV, dtype=torch.float64)
    top = g.abs().amax(-1)
    for e in range(lo - 127, hi - 127):  # the least of which the largest is at most seven times
        if bool((top > 7 * 2.0 ** e).any()):
            power = torch.where(top > 7 * 2.0 ** e, float(e + 1), power)
    unit = 2.0 ** power[..., None]
    a = (g / unit).abs().clamp(max=6)
    step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0))
    return ((a / step).round() * step * unit * g.sign()).flatten(-2)


def _values4(codes, scales):
    """What 4-bit numbers stand for, in 64 bits, from their bits."""
    n = torch.stack((codes & 15, codes >> 4), -1).flatten(-2).double()
    sign = torch.where(n >= 8, -1.0, 1.0)
    n = n % 8
    exponent, odd = (n / 2).floor(), n % 2
    x = torch.where(exponent == 0, odd / 2, 2.0 ** (exponent - 1) * (1 + odd / 2)) * sign
    return x * (2.0 ** (scales.double() - 127)).repeat_interleave(GROUP, -1)


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "append":
        return _exact_append(case, s)
    if case["kind"] in ("attend", "prefix"):
        return _exact_attention(case, s)
    return _exact_pages(case, s)


def _exact_append(case, s):
    half = case["rotary"] // 2
    pos = s["positions"].double()
    if case["axes"]:
        pos = torch.stack([pos[a] for a in s["axis"].tolist()], 1)[:, None]
    else:
        pos = pos[:, None, None]
    turn = torch.polar(torch.ones((), device=DEV, dtype=torch.float64), pos * s["inv_freq"].double())

    def rotated(x):
        x = x.double().clone()
        a = slice(0, 2 * half, 2) if case["pairs"] else slice(0, half)
        b = slice(1, 2 * half, 2) if case["pairs"] else slice(half, 2 * half)
        z = torch.complex(x[..., a], x[..., b]) * turn
        x[..., a], x[..., b] = z.real, z.imag
        return x

    q, k, v = rotated(s["q_rows"]), rotated(s["k_rows"]), s["v_rows"].double()
    if case["cache"] == "e2m1":
        return dict(q=q, k=_nearest4(k, case["dtype"]), v=_nearest4(v, case["dtype"]))
    blocks = s["cache_of"]["blocks"].double()
    order = (0, 2, 1, 3) if case["heads_first"] else (0, 1, 2, 3)
    page, slot = (torch.from_numpy(x).to(DEV) for x in np.divmod(s["slots"].cpu().numpy(), case["page"]))
    for i, (x, scale) in enumerate(((k, K_SCALE), (v, V_SCALE))):
        x = (x / scale).clamp(-E4M3_MAX, E4M3_MAX) if case["cache"] == "e4m3" else x
        blocks[:, i].permute(order)[page, slot] = x
    return dict(q=q, cache=blocks)


def _exact_attention(case, s):
    group, pre, c = case["q_heads"] // case["kv_heads"], case["prefix"], s["cache_of"]
    positions, los, his = (torch.from_numpy(x.copy()).to(DEV) for x in _visible(case))
    out = torch.zeros(s["tokens"], case["q_heads"], case["dim"], device=DEV, dtype=torch.float64)
    lse = torch.full((s["tokens"], case["q_heads"]), -math.inf, device=DEV, dtype=torch.float64)
    t0 = 0
    for b, (nq, nk) in enumerate(zip(*_lengths(case))):
        t = slice(t0, t0 + nq)
        t0 += nq
        j = torch.arange(nk, device=DEV)
        own_j = (j - pre).clamp(min=0)
        pages = s["table"][b][own_j // case["page"]].long()
        slot = own_j % case["page"]
        if pre:
            shared = j.clamp(max=pre - 1)
            pages = torch.where(j < pre, s["prefix_table"][shared // case["page"]].long(), pages)
            slot = torch.where(j < pre, shared % case["page"], slot)
        seen = (j >= los[t, None]) & (j < his[t, None])
        far = (positions[t, None] - j).abs().double()
        for h in range(case["kv_heads"]):
            k, v = (_values4(c[name][pages, slot, h], c[name + "_scales"][pages, slot, h]) for name in ("k", "v"))
            for head in range(h * group, (h + 1) * group):
                x = s["q_rows"][t, head].double() @ k.T * s["scale"]
                if case["cap"]:
                    x = case["cap"] * torch.tanh(x / case["cap"])
                if case["slopes"]:
                    x = x - s["slope"][head].double() * far
                x = x.masked_fill(~seen, -math.inf)
                norm = torch.logsumexp(x, 1)
                lse[t, head] = norm
                some = norm > -math.inf
                out[t, head] = torch.exp(x - torch.where(some, norm, 0.0)[:, None]) @ v
    return dict(out=out, lse=lse)


def _exact_pages(case, s):
    """Bits are copied: nothing is rounded but what a cache of floats held before."""
    blocks = s["cache_of"]["blocks"]
    if case["cache"] == "e2m1":
        return None
    order = (0, 2, 1, 3) if case["heads_first"] else (0, 1, 2, 3)
    ps = case["page"]
    if case["kind"] == "copy":
        to = torch.zeros(s["to"]["blocks"].shape, device=DEV, dtype=torch.float64)
        for a, b, _, _ in s["copies"].cpu().numpy():
            to[b] = blocks[a].transpose(1, 2).double()
        return dict(cache=to)
    got = blocks.double()
    refs = s["refs"].cpu().numpy()
    if case["kind"] == "fork":
        free = iter(np.flatnonzero(refs == 0).tolist())
        for b, n, room in _family(case)[1]:
            new = [next(free, None) for _ in range(_pages(room, ps) - n // ps)]
            if n % ps and new[0] is not None:
                src = int(s["table"][b, n // ps])
                for i in (0, 1):
                    x, y = blocks[:, i].permute(order), got[:, i].permute(order)
                    y[new[0], :n % ps] = x[src, :n % ps].double()
        return dict(table=None, copies=None, refs=None, cache=got)
    live = int((refs != 0).sum())
    for a, b in zip(np.flatnonzero(refs[live:] != 0) + live, np.flatnonzero(refs[:live] == 0)):
        got[int(b)] = blocks[int(a)].double()
    return dict(table=None, refs=None, page_map=None, copies=None, num_copies=None, cache=got)
