"""The paged cache's operators in 64 bits, and what their tests share.

Element types in numpy (bf16 and e4m3 as bit patterns), a cache in pages of
any layout with every slot that no test token uses poisoned by NaN, and the
definitions of kv_append and paged attention, row by row, from the formulas.

Tolerances count roundings.  A rounding to a type is off by at most half a
step, U[type] relative (bf16 2^-8 / 2 ... see below); a 32-bit operation by
2^-24.  Attention's result has one rounding of the output, one of each weight
to the 16-bit type of its product with the values, and 32-bit sums.
"""
import numpy as np

BF16, FP16, E4M3 = 0, 1, 2
# Half a step relative to the value: finfo(type).eps / 2.
U = {BF16: 2.0 ** -8, FP16: 2.0 ** -11, E4M3: 2.0 ** -4}
F32 = 2.0 ** -24


def _e4m3_table():
    v = np.zeros(256)
    for b in range(256):
        e, m = (b >> 3) & 15, b & 7
        x = (m / 8) * 2.0 ** -6 if e == 0 else (1 + m / 8) * 2.0 ** (e - 7)
        v[b] = np.nan if b & 127 == 127 else (-x if b & 128 else x)
    return v


E4M3_VALUES = _e4m3_table()


def encode(x, dtype):
    """float -> the type's bits, to nearest, ties to even (e4m3: saturated)."""
    x = np.asarray(x, np.float64)
    if dtype == FP16:
        return x.astype(np.float16).view(np.uint16)
    if dtype == BF16:
        u = x.astype(np.float32).view(np.uint32).astype(np.uint64)
        r = ((u + 0x7FFF + ((u >> 16) & 1)) >> 16).astype(np.uint16)
        return np.where(np.isnan(x), np.uint16(0x7FC0), r).astype(np.uint16)
    mags = E4M3_VALUES[:127]
    a = np.minimum(np.abs(np.nan_to_num(x, nan=0.0)), 448.0)
    hi = np.clip(np.searchsorted(mags, a), 0, 126)
    lo = np.maximum(hi - 1, 0)
    up = mags[hi] - a
    down = a - mags[lo]
    pick = np.where((up < down) | ((up == down) & (hi % 2 == 0)), hi, lo)
    bits = np.where(np.isnan(x), 127, pick | np.where(np.signbit(x), 128, 0))
    return bits.astype(np.uint8)


def decode(bits, dtype):
    if dtype == FP16:
        return bits.view(np.float16).astype(np.float64)
    if dtype == BF16:
        return (bits.astype(np.uint32) << 16).view(np.float32).astype(np.float64)
    return E4M3_VALUES[bits]


def quantised(rng, shape, dtype, spread=1.0):
    """(bits, values) of normal numbers that the type holds."""
    bits = encode(rng.standard_normal(shape) * spread, dtype)
    return bits, decode(bits, dtype)


class Pages:
    """Keys and values of some sequences in pages, the rest of the pages NaN.

    layout: "block" [page][2][slot][head][dim], "heads" [page][2][head][slot][dim],
    "apart" [page][slot][head][dim] twice, "padded" block with gaps between
    slots and pages."""

    def __init__(self, rng, lengths, page_size, heads, dim, dtype, layout="block", prefix=0, k_scale=1.0,
                 v_scale=1.0, spread=1.0, spare=3):
        self.page_size, self.heads, self.dim, self.dtype, self.layout = page_size, heads, dim, dtype, layout
        self.k_scale, self.v_scale = (k_scale, v_scale) if dtype == E4M3 else (1.0, 1.0)
        own = [-(-n // page_size) for n in lengths]
        shared = -(-prefix // page_size)
        self.num_pages = sum(own) + shared + spare
        place = rng.permutation(self.num_pages).astype(np.int32)
        width = max(own + [1])
        self.table = np.full((max(len(lengths), 1), width), 0x7FFFFFF0, np.int32)  # never read past the lengths
        self.prefix_table = place[:shared].copy()
        used = shared
        for b, n in enumerate(own):
            self.table[b, :n] = place[used:used + n]
            used += n
        ps, h, d = page_size, heads, dim
        gap = 16 if layout == "padded" else 0
        if layout == "heads":
            self.strides = (2 * h * ps * d, d, ps * d)
            self.v_offset = h * ps * d
        elif layout == "apart":
            self.strides = (ps * h * d, h * d, d)
            self.v_offset = self.num_pages * ps * h * d
        else:
            slot = h * d + gap
            self.strides = (2 * ps * slot + 3 * gap, slot, d)
            self.v_offset = ps * slot
        self.words = np.full(2 * self.num_pages * self.strides[0] if layout == "apart" else
                             self.num_pages * self.strides[0], 127 if dtype == E4M3 else
                             (0x7FC0 if dtype == BF16 else 0x7E00), np.uint8 if dtype == E4M3 else np.uint16)
        self.k = [np.zeros((n + prefix, h, d)) for n in lengths]
        self.v = [np.zeros((n + prefix, h, d)) for n in lengths]
        pre = [quantised(rng, (prefix, h, d), dtype, spread) for _ in range(2)]
        for which, at in ((0, 0), (1, self.v_offset)):
            for j in range(prefix):
                self.view(self.prefix_table[j // ps], j % ps, at)[:] = pre[which][0][j]
        for b, n in enumerate(lengths):
            for which, at in ((0, 0), (1, self.v_offset)):
                bits, values = quantised(rng, (n, h, d), dtype, spread)
                for j in range(n):
                    self.view(self.table[b, j // ps], j % ps, at)[:] = bits[j]
                whole = np.concatenate([pre[which][1], values]) * (self.v_scale if which else self.k_scale)
                (self.v if which else self.k)[b] = whole

    def view(self, page, slot, at=0):
        """[heads, dim] of one slot in the flat words."""
        first = at + int(page) * self.strides[0] + int(slot) * self.strides[1]
        return np.lib.stride_tricks.as_strided(self.words[first:], (self.heads, self.dim),
                                               (self.strides[2] * self.words.itemsize, self.words.itemsize))


def intervals(q_lens, kv_lens, window=0, doc_start=None, prefix_end=None):
    """Per token (sequence, position, lo, hi)."""
    out = []
    t = 0
    for b, (n, kv) in enumerate(zip(q_lens, kv_lens)):
        for i in range(n):
            pos = kv - n + i
            lo = max(0, int(doc_start[t]) if doc_start is not None else 0)
            if window:
                lo = max(lo, pos - window + 1)
            hi = min(kv, max(pos + 1, int(prefix_end[t])) if prefix_end is not None else pos + 1)
            out.append((b, pos, lo, hi))
            t += 1
    return out


def attention64(q, pages, rows, dtype, scale, softcap=0.0, slopes=None):
    """q [T, heads, dim] values; (out, lse, tol_out, tol_lse)."""
    T, hq, d = q.shape
    group = hq // pages.heads
    out, lse = np.zeros((T, hq, d)), np.full((T, hq), -np.inf)
    tol, tol_lse = np.zeros((T, hq, d)), np.zeros((T, hq))
    for t, (b, pos, lo, hi) in enumerate(rows):
        if hi <= lo:
            continue
        j = np.arange(lo, hi)
        for h in range(hq):
            k, v = pages.k[b][lo:hi, h // group], pages.v[b][lo:hi, h // group]
            s = k @ q[t, h] * scale
            # A sum of d products in 32 bits, in any order, and the operations after it.
            err = (d + 8) * F32 * (np.abs(k) @ np.abs(q[t, h]) * scale)
            if softcap > 0:
                s = softcap * np.tanh(s / softcap)
                err = err + 8 * F32 * softcap
            if slopes is not None:
                far = slopes[h] * np.abs(pos - j)
                s = s - far
                err = err + 4 * F32 * (far + np.abs(s))
            m = s.max()
            w = np.exp(s - m)
            total = w.sum()
            out[t, h] = (w / total) @ v
            lse[t, h] = m + np.log(total)
            # Scores enter as exp(s - m): an error e of both is 2 e of the weight, and the
            # exponent's own argument is rounded (a few steps of |s - m|, which no weight
            # over 2^-40 has above 28).
            rel = 2 * err.max() + 64 * F32
            spread = (w / total) @ np.abs(v)
            tol[t, h] = U[dtype] * np.abs(out[t, h]) + (1.01 * U[dtype] + 1.01 * rel + 2 * len(j) * F32) * spread + 1e-30
            if dtype == FP16:  # steps no longer shrink below 2^-24
                tol[t, h] += 2.0 ** -25 + 2.0 ** -25 * np.abs(v).max() * len(j)
            tol_lse[t, h] = err.max() + (16 + 2 * len(j)) * F32 * (1 + abs(lse[t, h]))
    return out, lse, tol, tol_lse


def rotate64(x, positions, inv_freq, interleaved):
    """x [T, heads, dim] values; (rotated, how far 32 bits may leave it)."""
    r = 2 * len(inv_freq)
    angle = positions.astype(np.float64)[:, None] * inv_freq.astype(np.float64)
    c, s = np.cos(angle)[:, None], np.sin(angle)[:, None]
    ia, ib = (np.arange(0, r, 2), np.arange(1, r, 2)) if interleaved else (np.arange(r // 2), np.arange(r // 2, r))
    y, off = x.copy(), np.zeros_like(x)
    a, b = x[..., ia], x[..., ib]
    y[..., ia], y[..., ib] = a * c - b * s, b * c + a * s
    # cos and sin to within 4 steps of 1, two products and a sum.
    off[..., ia] = off[..., ib] = 8 * F32 * (np.abs(a) + np.abs(b))
    return y, off
