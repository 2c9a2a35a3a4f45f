"""The operators of the paged KV cache: one case per way a serving program calls them.

A cache that the gather paths fill page by page also has to take a step's new
keys and values, rotated to their positions ("append"), and to be read by
attention: from one token per sequence up to whole prompts ("attend"), and for
a batch that shares a long prefix ("prefix").  A case's "kind" names the
entry point.  Heads, dims and pages are those of the 64 KiB KV pages that the
benchmark moves (8 heads of 128 in bf16, 16 tokens a page, keys before values)
and of the 4 KiB tokens of its headline workload (pages of one token), with
other common shapes around them.

`own` false: plain torch operations in 32 bits.  `own` true: the framework's
operators.  exact() is the definition in 64 bits, sequence by sequence.
"""
import math
import random

import numpy as np
import torch

own = False

DEV = "cuda"
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "e4m3": torch.float8_e4m3fn}
E4M3_MAX = 448.0
K_SCALE, V_SCALE = 1 / 32, 1 / 64  # what values of a few units leave of the e4m3 range


def _append(name, tokens, q_heads=32, kv_heads=8, dim=128, page=16, dtype="bf16", cache="bf16", heads_first=False,
            rotary=128, pairs=False, far=8192):
    return dict(name=name, kind="append", tokens=tokens, q_heads=q_heads, kv_heads=kv_heads, dim=dim, page=page,
                dtype=dtype, cache=cache, heads_first=heads_first, rotary=rotary, pairs=pairs, far=far)


def _attend(name, batch, q, kv, q_heads=32, kv_heads=8, dim=128, page=16, dtype="bf16", cache="bf16",
            heads_first=False, ragged=True, cap=0.0, slopes=False, window=0, docs=0, prefix_mask=False, prefix=0,
            lens=1):
    return dict(name=name, kind="prefix" if prefix else "attend", batch=batch, q=q, kv=kv, q_heads=q_heads,
                kv_heads=kv_heads, dim=dim, page=page, dtype=dtype, cache=cache, heads_first=heads_first,
                ragged=ragged, cap=cap, slopes=slopes, window=window, docs=docs, prefix_mask=prefix_mask,
                prefix=prefix, lens=lens)


def listed():
    return [
        # One decode step of eight sequences: a launch's latency.
        _append("append-8", 8),
        # A prompt's tokens at far positions, pairs side by side, half of the dims rotated, pages of one 4 KiB token.
        _append("append-4097-pairs", 4097, page=1, dtype="fp16", cache="fp16", rotary=64, pairs=True, far=1 << 20),
        # Several prompts' tokens of a whole batch into an 8-bit cache.
        _append("append-16384-e4m3", 16384, heads_first=True, page=64, cache="e4m3"),
        # A single user's decode step: latency.
        _attend("decode-1x700", 1, 1, 700, ragged=False),
        # A serving batch's decode step over ragged contexts.
        _attend("decode-64x8192", 64, 1, 8192),
        # Capped scores in a sliding window, wide heads, an 8-bit cache with pages that are no power of two.
        _attend("decode-33x6000-cap-e4m3", 33, 1, 6000, q_heads=16, dim=256, page=24, cache="e4m3", heads_first=True,
                cap=50.0, window=4096),
        # A chunk of a long prompt behind what is in the cache already.
        _attend("prompt-4096of16384", 1, 4096, 16384, ragged=False),
        # Packed documents, with capped scores.
        _attend("prompt-8192-docs-cap", 1, 8192, 8192, page=64, ragged=False, cap=30.0, docs=9),
        # Ragged prompts with a distance bias, each with a prefix that all of its tokens see.
        _attend("prompts-7x1500-bias-prefix", 7, 1500, 1900, q_heads=16, kv_heads=16, dim=64, page=32, dtype="fp16",
                cache="fp16", heads_first=True, slopes=True, prefix_mask=True),
        # A few chats on one short system prompt: latency.
        _attend("prefix-8x1024", 8, 1, 1024 + 64, prefix=1024),
        # Many requests on one long document.
        _attend("prefix-64x32768", 64, 1, 32768 + 1024, prefix=32768),
        # Drafted tokens verified, odd lengths, distance bias, an 8-bit cache of fewer heads.
        _attend("prefix-17x4-e4m3", 17, 4, 5001 + 700, q_heads=28, kv_heads=4, page=32, cache="e4m3", slopes=True,
                prefix=5001),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["append", "decode", "decode", "prompt", "prompt", "prefix", "prefix"])
    q_heads, kv_heads = rng.choice([(32, 8), (8, 8), (16, 2), (28, 4), (12, 12), (40, 8), (16, 1), (64, 8)])
    dim = rng.choice([64, 128, 128, 128, 256])
    dtype = rng.choice(["bf16", "bf16", "fp16"])
    common = dict(q_heads=q_heads, kv_heads=kv_heads, dim=dim, dtype=dtype, cache=rng.choice([dtype, dtype, "e4m3"]),
                  heads_first=rng.random() < 0.4, page=rng.choice([1, 8, 16, 16, 24, 32, 64, 128]))
    if kind == "append":
        c = _append("", _log(rng, 1, 16384 * 4096 // ((q_heads + kv_heads) * dim * 5) + 1),
                    rotary=rng.choice([dim, dim, dim // 2, dim // 4 + 2]), pairs=rng.random() < 0.4,
                    far=rng.choice([4096, 65536, 1 << 20]), **common)
    else:
        extra = dict(cap=rng.choice([0.0, 0.0, 30.0, 50.0]), slopes=rng.random() < 0.3, lens=rng.randint(1, 1 << 30),
                     ragged=rng.random() < 0.7, **common)
        if kind == "decode":
            batch = _log(rng, 1, 128)
            extra["window"] = rng.choice([0, 0, _log(rng, 16, 4096)])
            c = _attend("", batch, rng.choice([1, 1, 1, 2, 5]),
                        _log(rng, 16, min(16384, 200_000_000 // (batch * kv_heads * dim))), **extra)
        elif kind == "prompt":
            q = _log(rng, 17, 4096)
            batch = _log(rng, 1, max(1, 4096 // q))
            extra["docs"] = rng.choice([0, 0, rng.randint(2, 12)])
            extra["prefix_mask"] = rng.random() < 0.4
            extra["window"] = rng.choice([0, 0, 0, _log(rng, 64, 2048)])
            past = rng.choice([0, 0, _log(rng, 1, 4096)])
            c = _attend("", batch, q, q + past, **extra)
        else:
            batch = _log(rng, 2, 64)
            prefix = _log(rng, 64, min(32768, (1 << 27) // (kv_heads * dim)))
            own_len = _log(rng, 8, min(1024, (1 << 26) // (batch * kv_heads * dim)))
            q = rng.choice([1, 1, 1, 3, 8])
            c = _attend("", batch, q, prefix + max(own_len, q), prefix=prefix, **extra)
    del c["name"]
    return c


# --------------------------------------------------------------- the batch

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


def _pages(n, page):
    return -(-n // page)


def work(case):
    size = 1 if case["cache"] == "e4m3" else 2
    if case["kind"] == "append":
        t, d = case["tokens"], case["dim"]
        heads = case["q_heads"] + case["kv_heads"]
        return dict(bytes=t * (2 * d * (2 * case["q_heads"] + 2 * case["kv_heads"]) + size * 2 * case["kv_heads"] * d
                               + 12), flops=t * heads * case["rotary"] * 3)
    q, kv = _lengths(case)
    pos, lo, hi = _visible(case)
    first = np.concatenate([[0], np.cumsum(q)])
    keys = sum(max(0, int(hi[a:b].max()) - max(case["prefix"], int(lo[a:b].min())))
               for a, b in zip(first[:-1], first[1:]) if b > a)
    if case["prefix"]:
        keys += max(0, case["prefix"] - int(lo.min()))
    pairs = int(np.maximum(0, hi - lo).sum()) * case["q_heads"]
    return dict(bytes=keys * 2 * size * case["kv_heads"] * case["dim"]
                + len(pos) * case["q_heads"] * (4 * case["dim"] + 4), flops=4 * case["dim"] * pairs)


# ------------------------------------------------------------------ inputs

def _rand(gen, *shape):
    return torch.randn(*shape, generator=gen, device=DEV, dtype=torch.float32)


def _cache(case, gen, num_pages, fill):
    """Pages as one block each, keys before values; views [pages, page, heads, dim] of both."""
    inner = (case["kv_heads"], case["page"]) if case["heads_first"] else (case["page"], case["kv_heads"])
    blocks = torch.zeros(num_pages, 2, *inner, case["dim"], device=DEV, dtype=TYPES[case["cache"]])
    if fill:
        scale = torch.tensor([K_SCALE, V_SCALE], device=DEV).view(2, 1, 1, 1)
        for first in range(0, num_pages, 4096):
            part = blocks[first:first + 4096]
            x = _rand(gen, *part.shape)
            part.copy_(((x / scale).clamp(-E4M3_MAX, E4M3_MAX) if case["cache"] == "e4m3" else x).to(blocks.dtype))
    order = (0, 2, 1, 3) if case["heads_first"] else (0, 1, 2, 3)
    return blocks, blocks[:, 0].permute(order), blocks[:, 1].permute(order)


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    rng = np.random.default_rng(seed)
    dtype = TYPES[case["dtype"]]
    hq, hk, d, page = case["q_heads"], case["kv_heads"], case["dim"], case["page"]
    s = dict(case)
    if case["kind"] == "append":
        t = case["tokens"]
        # Half of the pages are another batch's; a projection's output holds q, k and v of a token side by side.
        pages = 2 * _pages(t, page)
        s["blocks"], s["k_pages"], s["v_pages"] = _cache(case, gen, pages, False)
        rows = _rand(gen, t, (hq + 2 * hk) * d).to(dtype)
        s["q_rows"], s["k_rows"], s["v_rows"] = (x.unflatten(1, (-1, d)) for x in rows.split([hq * d, hk * d, hk * d], 1))
        place = rng.permutation(pages)[:_pages(t, page)].astype(np.int64)
        at = np.arange(t)
        s["slots"] = torch.from_numpy(place[at // page] * page + at % page).to(DEV)
        first = int(rng.integers(0, max(1, case["far"] - t)))
        s["positions"] = torch.from_numpy((first + at).astype(np.int32)).to(DEV)
        half = case["rotary"] // 2
        s["inv_freq"] = torch.from_numpy((10000.0 ** (-np.arange(half) / half)).astype(np.float32)).to(DEV)
        s["q_out"] = torch.empty(t, hq, d, device=DEV, dtype=dtype)
        return s
    q_len, kv_len = _lengths(case)
    own_pages = [_pages(n - case["prefix"], page) for n in kv_len]
    shared = _pages(case["prefix"], page)
    place = rng.permutation(sum(own_pages) + shared + 3).astype(np.int32)  # three free pages
    s["blocks"], s["k_pages"], s["v_pages"] = _cache(case, gen, len(place), True)
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
    return s


# ---------------------------------------------------------------- one pass

def run(s):
    if s["kind"] == "append":
        return (_own_append if own else _plain_append)(s)
    return (_own_attention if own else _plain_attention)(s)


def _own_cache(s):
    """The cache's descriptor, which a program makes once with its pages."""
    import gfd_amd

    if "handle" not in s:
        k = s["k_pages"]
        s["handle"] = gfd_amd.KVCache(
            k=k.data_ptr(), v=s["v_pages"].data_ptr(), page_stride=k.stride(0), slot_stride=k.stride(1),
            head_stride=k.stride(2), num_pages=k.shape[0], page_size=k.shape[1], num_heads=k.shape[2],
            head_dim=k.shape[3], dtype={"bf16": gfd_amd.BF16, "fp16": gfd_amd.FP16, "e4m3": gfd_amd.E4M3}[s["cache"]],
            k_scale=K_SCALE, v_scale=V_SCALE)
        s["type"] = gfd_amd.BF16 if s["dtype"] == "bf16" else gfd_amd.FP16
        s["error"] = torch.zeros(1, dtype=torch.int32, device=DEV)
    return s["handle"]


def _own_append(s):
    import gfd_amd

    cache = _own_cache(s)
    q, k, v, out = s["q_rows"], s["k_rows"], s["v_rows"], s["q_out"]
    rows = gfd_amd.KVRows(
        q=q.data_ptr(), k=k.data_ptr(), v=v.data_ptr(), q_out=out.data_ptr(), q_stride=q.stride(0),
        k_stride=k.stride(0), v_stride=v.stride(0), q_out_stride=out.stride(0), positions=s["positions"].data_ptr(),
        slots=s["slots"].data_ptr(), inv_freq=s["inv_freq"].data_ptr(), num_tokens=q.shape[0],
        num_q_heads=q.shape[1], rotary_dim=s["rotary"], interleaved=int(s["pairs"]), dtype=s["type"])
    gfd_amd.kv_append(cache, rows, error_flag=s["error"].data_ptr(), stream=torch.cuda.current_stream().cuda_stream)
    return dict(q=out, cache=s["blocks"])


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
    more = dict(workspace=s["workspace"].data_ptr(), workspace_bytes=s["workspace"].numel(),
                error_flag=s["error"].data_ptr(), stream=torch.cuda.current_stream().cuda_stream)
    if s["prefix"]:
        gfd_amd.shared_prefix_attention(cache, call, s["prefix_table"].data_ptr(), s["prefix"], **more)
    else:
        gfd_amd.paged_attention(cache, call, **more)
    return dict(out=out, lse=s["lse"])


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
    angle = s["positions"].double()[:, None, None] * s["inv_freq"].double()  # far positions: 64 bits
    cos, sin = angle.cos().float(), angle.sin().float()
    q = _rotate(s["q_rows"].float(), cos, sin, s["pairs"])
    k, v = _rotate(s["k_rows"].float(), cos, sin, s["pairs"]), s["v_rows"].float()
    if s["cache"] == "e4m3":
        k, v = (k / K_SCALE).clamp(-E4M3_MAX, E4M3_MAX), (v / V_SCALE).clamp(-E4M3_MAX, E4M3_MAX)
    page, slot = s["slots"] // s["page"], s["slots"] % s["page"]
    kind = torch.uint8 if s["cache"] == "e4m3" else s["blocks"].dtype  # an 8-bit float is stored as its bits
    s["k_pages"].view(kind)[page, slot] = k.to(s["blocks"].dtype).view(kind)
    s["v_pages"].view(kind)[page, slot] = v.to(s["blocks"].dtype).view(kind)
    return dict(q=q.to(s["q_rows"].dtype), cache=s["blocks"])


def _plain_keys(s, pages, table, n):
    """[..., n keys, heads, dim] in 32 bits through a table of pages."""
    j = torch.arange(n, device=DEV)
    kind = torch.uint8 if s["cache"] == "e4m3" else pages.dtype
    return pages.view(kind)[table[..., j // s["page"]].long(), j % s["page"]].view(pages.dtype).float()


def _plain_attention(s):
    hq, hk, d, pre = s["q_heads"], s["kv_heads"], s["dim"], s["prefix"]
    ks, vs = (K_SCALE, V_SCALE) if s["cache"] == "e4m3" else (1.0, 1.0)
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
    k, v = (_plain_keys(s, p, s["table"], s["max_kv"] - pre).transpose(1, 2) for p in (s["k_pages"], s["v_pages"]))
    x = q @ k.transpose(2, 3).contiguous()  # [b, hk, g * n, own keys]
    if pre:  # the shared keys, once for all rows
        pk, pv = (_plain_keys(s, p, s["prefix_table"], pre).transpose(0, 1) for p in (s["k_pages"], s["v_pages"]))
        rows = q.transpose(0, 1).reshape(hk, b * g * n, d)
        y = (rows @ pk.transpose(1, 2).contiguous()).view(hk, b, g * n, pre).transpose(0, 1)
        x = torch.cat((y, x), 3)
    x = x.view(b, hk, g, n, -1).mul_(s["scale"] * ks)
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
    o = o.view(b, hk, g, n, d) / torch.where(total == 0, 1.0, total) * vs
    lse = (top + total.log()).squeeze(-1)
    out = torch.empty(t + 1, hq, d, device=DEV, dtype=s["q_rows"].dtype)
    out[tok] = o.permute(0, 3, 1, 2, 4).reshape(b, n, hq, d).to(out.dtype)
    norm = torch.empty(t + 1, hq, device=DEV)
    norm[tok] = lse.permute(0, 3, 1, 2).reshape(b, n, hq)
    return dict(out=out[:t], lse=norm[:t])


# ------------------------------------------------------- the definition, 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "append":
        turn = torch.polar(torch.ones((), device=DEV, dtype=torch.float64),
                           s["positions"].double()[:, None, None] * s["inv_freq"].double())
        half = case["rotary"] // 2

        def rotated(x):
            x = x.double().clone()
            a = slice(0, 2 * half, 2) if case["pairs"] else slice(0, half)
            b = slice(1, 2 * half, 2) if case["pairs"] else slice(half, 2 * half)
            z = torch.complex(x[..., a], x[..., b]) * turn
            x[..., a], x[..., b] = z.real, z.imag
            return x

        blocks = s["blocks"].double()
        order = (0, 2, 1, 3) if case["heads_first"] else (0, 1, 2, 3)
        slots = s["slots"].cpu().numpy()
        page, slot = (torch.from_numpy(x).to(DEV) for x in np.divmod(slots, case["page"]))
        for i, (x, scale) in enumerate(((rotated(s["k_rows"]), K_SCALE), (s["v_rows"].double(), V_SCALE))):
            x = (x / scale).clamp(-E4M3_MAX, E4M3_MAX) if case["cache"] == "e4m3" else x
            blocks[:, i].permute(order)[page, slot] = x
        return dict(q=rotated(s["q_rows"]), cache=blocks)
    ks, vs = (K_SCALE, V_SCALE) if case["cache"] == "e4m3" else (1.0, 1.0)
    group, pre = case["q_heads"] // case["kv_heads"], case["prefix"]
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
            k = s["k_pages"][:, :, h].float()[pages, slot].double() * ks if case["cache"] == "e4m3" else \
                s["k_pages"][pages, slot, h].double()
            v = s["v_pages"][:, :, h].float()[pages, slot].double() * vs if case["cache"] == "e4m3" else \
                s["v_pages"][pages, slot, h].double()
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
