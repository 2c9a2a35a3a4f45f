"""Batches that fill the card many times over: a workgroup walks a range of more keys than it looks up at once.

All sequences read the same pages, so that the cache stays small; the oracle takes some of them."""
import numpy as np
import pytest

import gfd_amd
import paged_kv_ref as ref
from paged_kv_ref import BF16, E4M3, FP16
from test_gpu_paged_kv import Attend, close

pytestmark = pytest.mark.gpu

KV = 4000


@pytest.fixture(autouse=True, scope="module")
def device():
    assert gfd_amd.device_count() > 0, "no GPU visible to libgfd_amd.so"
    assert gfd_amd.lib().gfd_set_device(0) == 0


def batch_of(rng, batch, q, hq, hk, d, dtype, cache, lengths, **kw):
    """(call, its pages, lengths of the sequences); the first of them are `lengths`."""
    pages = ref.Pages(rng, [KV], 16, hk, d, cache, "heads", k_scale=1 / 32, v_scale=1 / 64,
                      spread=20.0 if cache == E4M3 else 1.0)
    kv = rng.integers(1, KV + 1, batch).tolist()
    kv[:len(lengths)] = lengths
    pages.table = np.repeat(pages.table, batch, 0)
    return pages, kv, lambda: Attend(rng, pages, [q] * batch, kv, hq, dtype, **kw)


EDGES = [KV, 1, 1023, 1024, 1025, 1151, 1152, 1153, 2047, 2048, 2049, 2176, 2177, 2432, 2433, 3328, 3329, 3456, 3999]


@pytest.mark.parametrize("batch", [1100, 2400, 5000])  # ranges of 1152 and 2432 keys, and whole contexts
@pytest.mark.parametrize("q,hq,d,dtype,cache", [(1, 8, 64, BF16, BF16), (1, 8, 128, FP16, FP16), (2, 20, 64, BF16, E4M3),
                                                (1, 64, 256, BF16, BF16)])
def test_ranges_of_several_pieces(batch, q, hq, d, dtype, cache):
    rng = np.random.default_rng(90)
    window = 3000 if q == 2 else 0
    pages, kv, make = batch_of(rng, batch, q, hq, 2, d, dtype, cache, EDGES, window=window)
    a = make()
    rows = ref.intervals([q] * batch, kv, window=window)
    pick = [t for t, r in enumerate(rows) if r[0] < (len(EDGES) if d == 64 else 10)]
    want, want_lse, tol, tol_lse = ref.attention64(a.q[pick], pages, [(0,) + rows[t][1:] for t in pick], dtype,
                                                   float(np.float32(a.scale)))
    out, lse = a.run()
    assert a.errors() == 0 and np.isfinite(out).all()
    none = np.isneginf(want_lse)
    close(out[pick], want, tol, "out")
    assert (np.isneginf(lse[pick]) == none).all()
    close(np.where(none, 0, lse[pick]), np.where(none, 0, want_lse), tol_lse, "lse")
    again, _ = a.run()
    assert (again == out).all()


@pytest.mark.parametrize("at", [900, 1100, 2999])  # in the first and the second piece, and the last key
def test_a_value_that_is_no_number_in_a_later_piece(at):
    rng = np.random.default_rng(91)
    pages, kv, make = batch_of(rng, 2400, 2, 8, 2, 64, BF16, BF16, [3000] * 8)
    pages.view(pages.table[0, at // 16], at % 16, pages.v_offset)[:, 3] = 0x7F80  # infinite
    a = make()
    rows = ref.intervals([2] * 2400, kv)
    out, lse = a.run()
    want, _, tol, _ = ref.attention64(a.q[:16], pages, [(0,) + r[1:] for r in rows[:16]], BF16, float(np.float32(a.scale)))
    sees = np.array([lo <= at < hi for _, _, lo, hi in rows[:16]])
    others = np.arange(64) != 3
    close(out[:16][:, :, others], want[:, :, others], tol[:, :, others], "other dims")
    close(out[:16][~sees], want[~sees], tol[~sees], "tokens that do not see it")
    assert sees.any() and (out[:16][sees][:, :, 3] == np.inf).all() and np.isfinite(lse[:16]).all()


def test_a_bad_page_in_a_later_piece_is_reported_and_read_as_nothing():
    rng = np.random.default_rng(92)
    pages, kv, make = batch_of(rng, 2400, 1, 8, 2, 64, BF16, BF16, [3000, 3000])
    pages.table[0, 70] = pages.num_pages  # keys 1120 to 1135 of the first sequence
    a = make()
    out, lse = a.run()
    assert a.errors() == gfd_amd.KV_ERR_PAGE
    j = np.r_[0:1120, 1136:3000]
    for t in (0, 1):
        j = np.r_[0:1120, 1136:3000] if t == 0 else np.arange(3000)
        for h in range(8):
            s = pages.k[0][j, h // 4] @ a.q[t, h] * a.scale
            w = np.exp(s - s.max())
            v = pages.v[0][j, h // 4]
            # Weights and the output are rounded once, 2^-8 relative; 32-bit sums are far below a tenth of that.
            close(out[t, h], w / w.sum() @ v, 2.1 * 2.0 ** -8 * (w / w.sum() @ np.abs(v)) + 1e-3 * 2.0 ** -8, "row %d" % t)


@pytest.mark.parametrize("batch", [1100, 5000])
def test_a_prefix_before_ranges_of_several_pieces(batch):
    rng = np.random.default_rng(93)
    prefix = 70
    pages = ref.Pages(rng, [KV], 16, 2, 64, FP16, prefix=prefix)
    pages.table = np.repeat(pages.table, batch, 0)
    kv = (prefix + rng.integers(1, KV + 1, batch)).tolist()
    kv[:6] = [prefix + n for n in (KV, 1, 1024, 1025, 1153, 2177)]
    a = Attend(rng, pages, [1] * batch, kv, 8, FP16, prefix=prefix)
    rows = [(0, n - 1, 0, n) for n in kv[:12]]
    want, want_lse, tol, tol_lse = ref.attention64(a.q[:12], pages, rows, FP16, float(np.float32(a.scale)))
    out, lse = a.run()
    assert a.errors() == 0 and np.isfinite(out).all()
    close(out[:12], want, tol, "out")
    close(lse[:12], want_lse, tol_lse, "lse")


@pytest.mark.parametrize("batch", [1, 9])
def test_a_shared_prefix_in_pieces(batch):
    """A prefix of 140800 keys whose table names the same ten pages again and again, with 64 heads: its ranges are of
    more than a piece where few rows share it."""
    rng = np.random.default_rng(94)
    heads, d, page, times = 64, 64, 64, 220
    period = 10 * page
    prefix = period * times
    pages = ref.Pages(rng, [1] * batch, page, heads, d, BF16, prefix=period)
    pages.prefix_table = np.tile(pages.prefix_table, times)
    a = Attend(rng, pages, [1] * batch, [prefix + 1] * batch, heads, BF16, prefix=prefix)
    out, lse = a.run()
    assert a.errors() == 0
    for t in range(batch):
        for h in range(0, heads, 7):
            k, v = pages.k[t][:, h], pages.v[t][:, h]  # a period and the token's own key
            s = k @ a.q[t, h] * float(np.float32(a.scale))
            w = np.exp(s - s.max()) * np.r_[np.full(period, times), 1]
            w, total = w / w.sum(), s.max() + np.log(w.sum())
            # Scores: d + 8 steps of 2^-24 of their magnitudes, twice in a weight; sums over all keys in any order, one
            # step for each of a wave's; weights and output rounded once.
            err = (d + 8) * ref.F32 * (np.abs(k) @ np.abs(a.q[t, h]) * a.scale).max()
            rel = 2 * err + (64 + 2 * 1152) * ref.F32
            tol = 2.0 ** -8 * np.abs(w @ v) + (1.01 * 2.0 ** -8 + 1.01 * rel) * (w @ np.abs(v)) + 1e-30
            close(out[t, h], w @ v, tol, "out")
            assert abs(lse[t, h] - total) <= err + (16 + 2 * 1152) * ref.F32 * (1 + abs(total))
