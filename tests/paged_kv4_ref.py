"""A cache of 4-bit numbers for the paged cache's tests: the numbers and their
scales in 64 bits, and pages of them in any layout, with every slot that no
test token uses poisoned by scales that say NaN.  What reads the pages is
paged_kv_ref's: a Pages4 has the values that its bits stand for.
"""
import numpy as np

import paged_kv_ref as ref
from paged_kv_ref import BF16, FP16

GROUP = 32
MAGNITUDES = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])
VALUES = np.concatenate([MAGNITUDES, -MAGNITUDES])
# The scales that an append writes, by the rows' type.
SCALES = {BF16: (1, 252), FP16: (104, 140)}
NAN = 255


def powers(byte):
    return np.where(byte == NAN, np.nan, 2.0 ** (byte.astype(np.float64) - 127))


def scale_bytes(x, dtype):
    """x [..., dims] -> [..., dims / 32]: the least power of two of which the largest magnitude is at most seven."""
    top = np.abs(x.reshape(*x.shape[:-1], x.shape[-1] // GROUP, GROUP)).max(-1)
    lo, hi = SCALES[dtype]
    e = np.ceil(np.log2(np.maximum(top, 2.0 ** -160) / 7))  # near the power: settled below
    e = np.where(top > 7 * 2.0 ** e, e + 1, np.where(top <= 7 * 2.0 ** (e - 1), e - 1, e))
    byte = np.clip(np.nan_to_num(e, nan=0, posinf=0) + 127, lo, hi).astype(np.uint8)
    return np.where(np.isfinite(top), byte, NAN).astype(np.uint8)


def codes(x, byte):
    """The nearest numbers, ties to the even code, saturated: [..., dims] of 0..15."""
    with np.errstate(invalid="ignore"):
        y = x.reshape(*x.shape[:-1], x.shape[-1] // GROUP, GROUP) / powers(byte)[..., None]
    y = np.where(np.isnan(y), 0.0, y).reshape(x.shape)
    a = np.minimum(np.abs(y), 6.0)
    hi = np.clip(np.searchsorted(MAGNITUDES, a), 0, 7)
    lo = np.maximum(hi - 1, 0)
    up, down = MAGNITUDES[hi] - a, a - MAGNITUDES[lo]
    pick = np.where((up < down) | ((up == down) & (hi % 2 == 0)), hi, lo)
    return (pick | np.where(np.signbit(y), 8, 0)).astype(np.uint8)


def packed(code):
    return (code[..., 0::2] | (code[..., 1::2] << 4)).astype(np.uint8)


def unpacked(numbers):
    return np.stack([numbers & 15, numbers >> 4], -1).reshape(*numbers.shape[:-1], 2 * numbers.shape[-1])


def values(numbers, byte):
    """What bytes of numbers and of scales stand for."""
    x = VALUES[unpacked(numbers)]
    return (x.reshape(*x.shape[:-1], x.shape[-1] // GROUP, GROUP) * powers(byte)[..., None]).reshape(x.shape)


def encode(x, dtype):
    """(bytes of numbers, bytes of scales) of x."""
    byte = scale_bytes(x, dtype)
    return packed(codes(x, byte)), byte


class Pages4:
    """Keys and values of some sequences in pages of 4-bit numbers, the rest of the pages NaN.

    layout: "block" [page](keys, values, their scales), slots outside heads; "heads" the same, heads outside slots;
    "apart" four arrays; "padded" a block with gaps between slots, parts and pages."""

    dtype = 3

    def __init__(self, rng, lengths, page_size, heads, dim, rows=BF16, layout="block", prefix=0, spread=1.0, spare=3):
        self.page_size, self.heads, self.dim, self.layout = page_size, heads, dim, layout
        own = [-(-n // page_size) for n in lengths]
        shared = -(-prefix // page_size)
        self.num_pages = sum(own) + shared + spare
        place = rng.permutation(self.num_pages).astype(np.int32)
        self.table = np.full((max(len(lengths), 1), max(own + [1])), 0x7FFFFFF0, np.int32)  # never read past the lengths
        self.prefix_table = place[:shared].copy()
        used = shared
        for b, n in enumerate(own):
            self.table[b, :n] = place[used:used + n]
            used += n
        row, ps, n = dim // 2, page_size, self.num_pages
        self.slot, self.head = (row, ps * row) if layout == "heads" else (heads * row, row)
        if layout == "padded":
            self.slot, self.head = heads * (row + 16) + 32, row + 16
        part = ps * heads * row if layout != "padded" else ps * self.slot
        if layout == "apart":
            self.page, self.scale_page = part, part // 16
            offsets = [0, n * part, 2 * n * part, 2 * n * part + n * (part // 16)]
            total = 2 * n * part + 2 * n * (part // 16)
        else:
            gap = 48 if layout == "padded" else 0
            offsets = [0, part + gap, 2 * part + gap, 2 * part + gap + part // 16 + gap // 16]
            self.page = self.scale_page = -(-(offsets[3] + part // 16 + gap) // 16) * 16
            total = n * self.page
        self.offsets = dict(zip(("k", "v", "k_scales", "v_scales"), offsets))
        self.words = rng.integers(0, 256, total).astype(np.uint8)
        self.k = [np.zeros((m + prefix, heads, dim)) for m in lengths]
        self.v = [np.zeros((m + prefix, heads, dim)) for m in lengths]
        for p in range(n):
            for s in range(ps):
                for which in ("k_scales", "v_scales"):
                    self.view(p, s, which)[:] = NAN
        for which in ("k", "v"):
            pre = self.store(which, self.prefix_table, self.numbers(rng, prefix, rows, spread))
            for b, m in enumerate(lengths):
                mine = self.store(which, self.table[b], self.numbers(rng, m, rows, spread))
                getattr(self, which)[b] = np.concatenate([pre, mine])

    def numbers(self, rng, n, rows, spread):
        """Values of different sizes from group to group."""
        x = rng.standard_normal((n, self.heads, self.dim)) * spread
        size = 2.0 ** rng.integers(-3, 3, (n, self.heads, self.dim // GROUP))
        return encode(x * np.repeat(size, GROUP, -1), rows)

    def store(self, which, table, bits):
        for j, (numbers, byte) in enumerate(zip(*bits)):
            self.view(table[j // self.page_size], j % self.page_size, which)[:] = numbers
            self.view(table[j // self.page_size], j % self.page_size, which + "_scales")[:] = byte
        return values(*bits)

    def view(self, page, slot, which):
        """[heads, bytes] of one slot: of "k" and "v", or of their scales."""
        scales = which.endswith("_scales")
        inside = int(slot) * self.slot // (16 if scales else 1)
        first = self.offsets[which] + int(page) * (self.scale_page if scales else self.page) + inside
        return np.lib.stride_tricks.as_strided(self.words[first:], (self.heads, self.dim // (32 if scales else 2)),
                                               (self.head // (16 if scales else 1), 1))


class OneHead:
    """One head's keys and values of one sequence, for attention64."""

    def __init__(self, pages, b, head):
        self.heads = 1
        self.k, self.v = ([x[b][:, head:head + 1]] for x in (pages.k, pages.v))


def handle(pages, words):
    import gfd_amd

    return gfd_amd.KV4Cache(
        **{name: words.ptr + at for name, at in pages.offsets.items()}, page_stride=pages.page, slot_stride=pages.slot,
        head_stride=pages.head, scale_page_stride=pages.scale_page, num_pages=pages.num_pages,
        page_size=pages.page_size, num_heads=pages.heads, head_dim=pages.dim)


def rotated(x, positions, inv_freq, interleaved, axis=None):
    """x [T, heads, dim] turned by positions ([T], or [axes, T] with axis per pair); (y, how far 32 bits may leave it)."""
    half = len(inv_freq)
    at = positions[axis] .T if axis is not None else np.repeat(np.asarray(positions)[:, None], half, 1)
    angle = at.astype(np.float64) * inv_freq.astype(np.float64)
    c, s = np.cos(angle)[:, None], np.sin(angle)[:, None]
    ia, ib = (np.arange(0, 2 * half, 2), np.arange(1, 2 * half, 2)) if interleaved else (
        np.arange(half), np.arange(half, 2 * half))
    y, off = x.copy(), np.zeros_like(x)
    a, b = x[..., ia], x[..., ib]
    with np.errstate(invalid="ignore"):
        y[..., ia], y[..., ib] = a * c - b * s, b * c + a * s
        # cos and sin to within 4 steps of 1, two products and a sum.
        off[..., ia] = off[..., ib] = 8 * ref.F32 * (np.abs(a) + np.abs(b))
    return y, off
