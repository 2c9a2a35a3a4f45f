"""kv_append into a 4-bit cache, with positions of one and of several axes, and kv_read, on the GPU against their
definitions in 64 bits.

What a cache holds is decided by a 32-bit result, off by `off` at most: its scale is that of a group whose numbers are
all off by as much either way, and its number lies between those of x - off and x + off at that scale."""
import numpy as np
import pytest

import gfd_amd
import paged_kv4_ref as ref4
import paged_kv_ref as ref
import test_gpu_paged_kv as gpu
from paged_kv_ref import BF16, E4M3, FP16
from test_gpu_paged_kv import close, up

pytestmark = pytest.mark.gpu

PAGE = 5


@pytest.fixture(autouse=True, scope="module")
def device():
    assert gfd_amd.device_count() > 0, "no GPU visible to libgfd_amd.so"
    assert gfd_amd.lib().gfd_set_device(0) == 0


def held(got, byte, x, off, dtype, what):
    """The values and scale bytes of rows x [..., dim] against the definition."""
    top = np.abs(x).reshape(*x.shape[:-1], -1, 32)
    wide = off.reshape(top.shape)
    least = ref4.scale_bytes(np.maximum(top - wide, 0).reshape(x.shape), dtype)
    most = ref4.scale_bytes((top + wide).reshape(x.shape), dtype)
    nan = most == ref4.NAN
    assert ((byte == ref4.NAN) == nan).all(), what
    assert ((least <= byte) & (byte <= most))[~nan].all(), what + ": scales"
    lo, hi = (ref4.values(ref4.packed(ref4.codes(np.nan_to_num(x + d, posinf=0, neginf=0), byte)), byte)
              for d in (-off, off))
    fine = ~np.repeat(nan, 32, -1)
    assert np.isnan(got[~fine]).all(), what
    bad = fine & ~((lo <= got) & (got <= hi))
    assert not bad.any(), "%s: %d of %d at %s: %r outside %r .. %r of %r" % (
        what, bad.sum(), bad.size, np.argwhere(bad)[0], got[bad][0], lo[bad][0], hi[bad][0], x[bad][0])


class Step:
    """One step's rows on the device."""

    def __init__(self, rng, tokens, hq, hk, d, dtype, rotary, num_pages, axes=0, float_positions=False, turns=False,
                 special=None, pairs=False, with_q=True, in_place=False, axes_last=False, far=1 << 20):
        self.tokens, self.hq, self.hk, self.d, self.dtype, self.pairs = tokens, hq, hk, d, dtype, pairs
        q_bits, k_bits, v_bits = (ref.quantised(rng, (tokens, h, d), dtype, 1.5)[0] for h in (hq, hk, hk))
        if special is not None:
            n = min(len(special), d)
            k_bits[0, 0, :n] = v_bits[0, 0, :n] = ref.encode(special[:n], dtype)
            v_bits[-1, -1] = ref.encode(np.zeros(d), dtype)
        self.q, self.k, self.v = (ref.decode(x, dtype) for x in (q_bits, k_bits, v_bits))
        self.fused = np.concatenate([x.reshape(tokens, -1) for x in (q_bits, k_bits, v_bits)], 1)
        self.slots = rng.permutation(num_pages * PAGE)[:tokens].astype(np.int64)
        if tokens > 3:
            self.slots[2] = -1
        half = rotary // 2
        self.inv_freq = (10000.0 ** (-np.arange(half) / max(half, 1))).astype(np.float32)
        self.axis, shape = None, (tokens,)
        if axes:
            i = np.arange(half)
            self.axis = (i % axes if turns else i * axes // max(half, 1)).astype(np.uint8)
            shape = (axes, tokens)
        self.positions = rng.integers(0, far, shape).astype(np.int32)
        if float_positions:
            self.positions = (self.positions * np.float32(0.37)).astype(np.float32)
        self.positions.reshape(-1)[0] = 0
        if tokens > 3 and not float_positions:
            self.positions.reshape(-1)[3] = 0x7FFFFFFF
        given = np.ascontiguousarray(self.positions.T) if axes_last else self.positions
        self.buffers = dict(rows=up(self.fused), slots=up(self.slots), positions=up(given), inv=up(self.inv_freq),
                            axis=up(self.axis if axes else np.zeros(1, np.uint8)), error=up(np.zeros(1, np.int32)))
        p = {k: b.ptr for k, b in self.buffers.items()}
        self.q_out = gfd_amd.DeviceBuffer(tokens * hq * d * 2 + 64)
        self.q_out.fill(0xA5)
        width = self.fused.shape[1]
        self.with_q, self.in_place = with_q, in_place
        self.rows = gfd_amd.KVRows(
            q=p["rows"] if with_q else None, k=p["rows"] + hq * d * 2, v=p["rows"] + (hq + hk) * d * 2,
            q_out=None if not with_q else p["rows"] if in_place else self.q_out.ptr, q_stride=width, k_stride=width,
            v_stride=width, q_out_stride=width if in_place else hq * d, positions=None if axes else p["positions"],
            slots=p["slots"], inv_freq=p["inv"], num_tokens=tokens, num_q_heads=hq, rotary_dim=rotary,
            interleaved=int(pairs), dtype=dtype)
        self.axes = None
        if axes:
            self.axes = gfd_amd.RotaryAxes(positions=p["positions"], axis=p["axis"],
                                           axis_stride=1 if axes_last else tokens,
                                           token_stride=axes if axes_last else 1, num_axes=axes,
                                           float_positions=int(float_positions))

    def append(self, cache, stream=None):
        gfd_amd.kv_append(cache, self.rows, error_flag=self.buffers["error"].ptr, stream=stream, axes=self.axes)
        gfd_amd.synchronize()

    def errors(self):
        return int(self.buffers["error"].download(4).view(np.int32)[0])

    def turned(self, x):
        return ref4.rotated(x, self.positions, self.inv_freq, self.pairs, self.axis)

    def check_q(self):
        n = self.tokens * self.hq * self.d
        raw, width = self.q_out.download(), self.fused.shape[1]
        assert (raw[n * 2:] == 0xA5).all()
        after = self.buffers["rows"].download().view(np.uint16)[:self.fused.size].reshape(self.fused.shape)
        own = self.hq * self.d
        assert (after[:, own:] == self.fused[:, own:]).all() and (self.in_place or (after == self.fused).all())
        got = after[:, :own].copy() if self.in_place else raw[:n * 2].view(np.uint16)
        if not self.with_q:
            assert (got == 0xA5A5).all()
            return
        want, off = self.turned(self.q)
        close(ref.decode(got.reshape(self.q.shape), self.dtype), want, ref.U[self.dtype] * np.abs(want) + 1.01 * off +
              (2.0 ** -25 if self.dtype == FP16 else 0), "q")


def append4(seed, layout, dtype, d, rotary, tokens, hq=6, hk=2, **kw):
    rng = np.random.default_rng(seed)
    num_pages = 2 * -(-tokens // PAGE) + 1
    pages = ref4.Pages4(rng, [0], PAGE, hk, d, dtype, layout, spare=num_pages)
    before = pages.words.copy()
    s = Step(rng, tokens, hq, hk, d, dtype, rotary, num_pages, **kw)
    words = up(pages.words)
    s.append(ref4.handle(pages, words))
    assert s.errors() == 0
    pages.words = words.download()[:len(before)]
    at = [t for t in range(tokens) if s.slots[t] >= 0]
    for which, (x, off) in (("k", s.turned(s.k)), ("v", (s.v, np.zeros_like(s.v)))):
        bits = [np.stack([pages.view(s.slots[t] // PAGE, s.slots[t] % PAGE, w) for t in at]) for w in
                (which, which + "_scales")]
        held(ref4.values(*bits), bits[1], x[at], off[at], dtype, which)
    s.check_q()
    # Everything else is as it was.
    for t in at:
        for which in ("k", "v", "k_scales", "v_scales"):
            now = pages.view(s.slots[t] // PAGE, s.slots[t] % PAGE, which)
            pages.words, after = before, pages.words
            now[:] = pages.view(s.slots[t] // PAGE, s.slots[t] % PAGE, which)
            pages.words = after
    assert (pages.words == before).all(), "written outside the tokens' slots"


@pytest.mark.parametrize("layout", ["block", "heads", "apart", "padded"])
@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("d,rotary,pairs", [(128, 128, False), (128, 64, True), (64, 18, False), (256, 256, True),
                                            (256, 0, False), (64, 2, True), (128, 96, False), (128, 16, False),
                                            (256, 66, False), (64, 64, False), (256, 256, False)])
def test_append(layout, dtype, d, rotary, pairs):
    append4(1, layout, dtype, d, rotary, 13, pairs=pairs)


@pytest.mark.parametrize("tokens", [1, 2, 64, 300, 1000])
@pytest.mark.parametrize("with_q", [True, False])
def test_append_of_few_and_many_tokens(tokens, with_q):
    append4(2, "block", BF16, 128, 128, tokens, with_q=with_q)


@pytest.mark.parametrize("d,rotary,pairs", [(64, 64, False), (64, 32, True), (128, 50, False)])
def test_append_of_four_tokens_a_workgroup(d, rotary, pairs):
    append4(3, "heads", BF16, d, rotary, 8195, hq=1, hk=1, pairs=pairs)


@pytest.mark.parametrize("hq,hk", [(1, 1), (7, 7), (28, 4), (64, 8)])
def test_append_of_every_head_count(hq, hk):
    append4(4, "heads", FP16, 64, 64, 21, hq=hq, hk=hk)


def test_append_turns_queries_in_place():
    append4(5, "block", FP16, 128, 128, 9, in_place=True)
    append4(5, "block", FP16, 128, 128, 9, in_place=True, pairs=True)
    append4(5, "block", BF16, 128, 50, 9, in_place=True)


@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_append_of_values_at_the_ends(dtype):
    big, small = (3.38e38, 2.0 ** -133) if dtype == BF16 else (65504.0, 2.0 ** -24)
    for special in ([big, -big, 1.0], [small, -small, 3 * small], [-0.0, 0.0], [big / 8, small, -7.0],
                    [7.0, 6.0, 5.0, 3.5, 2.5, 1.75, 1.25, 0.75, 0.25], [np.inf, 1.0], [1.0, -np.inf], [np.nan]):
        x = np.zeros(32)
        x[:len(special)] = special
        append4(6, "block", dtype, 64, 0, 5, special=x)


def test_a_slot_outside_the_cache_is_reported_and_the_others_are_written():
    rng = np.random.default_rng(7)
    pages = ref4.Pages4(rng, [0], 16, 2, 128, spare=2)
    rows = up(np.full((3, 2, 128), 0x3F80, np.uint16))
    for bad in (32, 1 << 40, 0x7FFFFFFFFFFFFFFF):
        words, error, slots = up(pages.words), up(np.zeros(1, np.int32)), up(np.array([3, bad, 31], np.int64))
        cache = ref4.handle(pages, words)
        gfd_amd.kv_append(cache, gfd_amd.KVRows(k=rows.ptr, v=rows.ptr, k_stride=256, v_stride=256, slots=slots.ptr,
                                                num_tokens=3, dtype=BF16), error_flag=error.ptr)
        gfd_amd.synchronize()
        assert int(error.download(4).view(np.int32)[0]) == gfd_amd.KV_ERR_PAGE
        out = [gfd_amd.DeviceBuffer(3 * 512) for _ in range(2)]
        for o in out:
            o.fill(0xA5)
        gfd_amd.kv_read(cache, gfd_amd.KVRead(k=out[0].ptr, v=out[1].ptr, k_stride=256, v_stride=256, slots=slots.ptr,
                                              num_tokens=3, dtype=BF16), error_flag=error.ptr)
        gfd_amd.synchronize()
        for o in out:
            got = o.download().view(np.uint16).reshape(3, 256)
            assert (got[[0, 2]] == 0x3F80).all() and (got[1] == 0xA5A5).all()


# ------------------------------------------------------------ positions of several axes

@pytest.mark.parametrize("d,rotary,pairs", [(128, 128, False), (128, 64, True), (64, 18, False), (256, 66, False)])
@pytest.mark.parametrize("axes,turns,seconds,last", [(3, False, False, False), (3, True, True, False),
                                                     (2, True, False, True), (1, False, False, False),
                                                     (200, False, False, False)])
def test_append_at_positions_of_several_axes(d, rotary, pairs, axes, turns, seconds, last):
    append4(10, "block", BF16, d, rotary, 13, pairs=pairs, axes=axes, turns=turns, float_positions=seconds, axes_last=last)


def append16(seed, layout, dtype, cache, d, rotary, tokens, hq=6, hk=2, **kw):
    """Into the other caches."""
    rng = np.random.default_rng(seed)
    num_pages = 2 * -(-tokens // PAGE) + 1
    pages = ref.Pages(rng, [0], PAGE, hk, d, cache, layout, k_scale=1 / 32, v_scale=1 / 64, spare=num_pages)
    s = Step(rng, tokens, hq, hk, d, dtype, rotary, num_pages, **kw)
    words = up(pages.words)
    s.append(gpu.handle(pages, words))
    assert s.errors() == 0
    pages.words = words.download().view(pages.words.dtype)[:len(pages.words)]
    at = [t for t in range(tokens) if s.slots[t] >= 0]
    for first, (x, off), scale in ((0, s.turned(s.k), pages.k_scale), (pages.v_offset, (s.v, 0 * s.v), pages.v_scale)):
        got = ref.decode(np.stack([pages.view(s.slots[t] // PAGE, s.slots[t] % PAGE, first) for t in at]), cache)
        y, o = x[at] / scale, off[at] / scale
        if cache == E4M3:
            y = np.clip(y, -448, 448)
            tol = np.maximum(ref.U[E4M3] * np.abs(y), 2.0 ** -10) + 1.07 * o + 2 * ref.F32 * np.abs(y)
        else:
            tol = ref.U[cache] * np.abs(y) + 1.01 * o + (2.0 ** -25 if cache == FP16 else 0)
        close(got, y, tol, "cache")
    s.check_q()


@pytest.mark.parametrize("dtype,cache", [(BF16, BF16), (FP16, FP16), (BF16, E4M3), (FP16, E4M3)])
@pytest.mark.parametrize("d,rotary,pairs", [(128, 128, False), (128, 64, True), (64, 18, False)])
@pytest.mark.parametrize("axes,turns,seconds,last", [(3, False, False, False), (2, True, True, True)])
def test_append_to_other_caches_at_positions_of_several_axes(dtype, cache, d, rotary, pairs, axes, turns, seconds, last):
    append16(11, "block", dtype, cache, d, rotary, 13, pairs=pairs, axes=axes, turns=turns, float_positions=seconds,
             axes_last=last)


def test_append_of_many_tokens_at_positions_of_several_axes():
    append16(12, "heads", BF16, BF16, 64, 64, 8195, hq=1, hk=1, axes=3)


@pytest.mark.parametrize("four", [False, True])
def test_one_axis_is_the_rows_own_position(four):
    """The same bits with the positions given either way."""
    got = []
    for axes in (0, 1):
        rng = np.random.default_rng(13)
        pages = (ref4.Pages4(rng, [0], PAGE, 2, 128, spare=9) if four else ref.Pages(rng, [0], PAGE, 2, 128, BF16, spare=9))
        s = Step(rng, 13, 6, 2, 128, BF16, 128, 9, axes=axes)
        words = up(pages.words)
        s.append((ref4 if four else gpu).handle(pages, words))
        got.append(np.concatenate([words.download(), s.q_out.download()]))
    assert (got[0] == got[1]).all()


@pytest.mark.parametrize("four", [False, True])
def test_a_pair_of_no_axis_is_reported_and_not_turned(four):
    rng = np.random.default_rng(14)
    pages = (ref4.Pages4(rng, [0], PAGE, 2, 128, spare=9) if four else ref.Pages(rng, [0], PAGE, 2, 128, BF16, spare=9))
    s = Step(rng, 9, 6, 2, 128, BF16, 128, 9, axes=3)
    s.axis[[5, 63]] = 3, 255
    s.buffers["axis"].upload(s.axis)
    words = up(pages.words)
    s.append((ref4 if four else gpu).handle(pages, words))
    assert s.errors() == gfd_amd.KV_ERR_AXIS
    s.positions = np.concatenate([s.positions, np.zeros((253, 9), np.int32)])
    s.check_q()


# ------------------------------------------------------------ read

@pytest.mark.parametrize("layout", ["block", "heads", "apart", "padded"])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("dtype,cache", [(BF16, BF16), (FP16, FP16), (BF16, E4M3), (FP16, E4M3), (BF16, 3), (FP16, 3)])
def test_read(layout, d, dtype, cache):
    rng = np.random.default_rng(20)
    hk, tokens, width = 3, 37, 3 * d + 16
    if cache == 3:
        pages = ref4.Pages4(rng, [tokens], PAGE, hk, d, dtype, layout)
    else:
        pages = ref.Pages(rng, [tokens], PAGE, hk, d, cache, layout, k_scale=1 / 32, v_scale=1 / 64, spread=20.0)
    words, error = up(pages.words), up(np.zeros(1, np.int32))
    order = rng.permutation(tokens)
    slots = pages.table[0, order // PAGE].astype(np.int64) * PAGE + order % PAGE
    slots[4] = -1
    bufs = [gfd_amd.DeviceBuffer(tokens * width * 2 + 64) for _ in range(2)]
    for with_k, with_v in ((1, 1), (1, 0), (0, 1)):
        for b in bufs:
            b.fill(0xA5)
        keep = up(slots)
        gfd_amd.kv_read((ref4 if cache == 3 else gpu).handle(pages, words), gfd_amd.KVRead(
            k=bufs[0].ptr if with_k else None, v=bufs[1].ptr if with_v else None, k_stride=width, v_stride=width,
            slots=keep.ptr, num_tokens=tokens, dtype=dtype), error_flag=error.ptr)
        gfd_amd.synchronize()
        assert int(error.download(4).view(np.int32)[0]) == 0
        for b, want, asked in ((bufs[0], pages.k[0], with_k), (bufs[1], pages.v[0], with_v)):
            raw = b.download()
            rows = raw[:tokens * width * 2].view(np.uint16).reshape(tokens, width)
            if not asked:
                assert (raw == 0xA5).all()
                continue
            assert (raw[tokens * width * 2:] == 0xA5).all() and (rows[:, 3 * d:] == 0xA5A5).all()
            assert (rows[4] == 0xA5A5).all()
            got = ref.decode(rows[:, :3 * d].copy(), dtype).reshape(tokens, hk, d)
            # Held exactly by the type, but for an 8-bit number times its scale.
            want = want[order]
            tol = (ref.U[dtype] * 1.01 * np.abs(want) + (2.0 ** -25 if dtype == FP16 else 0)) if cache == E4M3 else 0 * want
            live = np.arange(tokens) != 4
            close(got[live], want[live], tol[live], "rows")
