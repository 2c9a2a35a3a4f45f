"""4-bit caches whose batches fill the card many times over: a workgroup walks a range of more keys than it looks up at once.

All sequences read the same pages, so that the cache stays small; the definition takes some of them."""
import numpy as np
import pytest

import gfd_amd
import paged_kv4_ref as ref4
import paged_kv_ref as ref
import test_gpu_paged_kv as gpu
from paged_kv_ref import BF16, FP16
from test_gpu_paged_kv import close

pytestmark = pytest.mark.gpu

KV = 4000


@pytest.fixture(autouse=True, scope="module")
def device():
    assert gfd_amd.device_count() > 0, "no GPU visible to libgfd_amd.so"
    assert gfd_amd.lib().gfd_set_device(0) == 0


@pytest.fixture(autouse=True)
def four_bits(monkeypatch):
    monkeypatch.setattr(gpu, "handle", ref4.handle)


def batch_of(rng, batch, q, hq, hk, d, dtype, lengths, **kw):
    """(pages, lengths of the sequences, the call); the first sequences' lengths are `lengths`."""
    pages = ref4.Pages4(rng, [KV], 16, hk, d, dtype, "heads")
    kv = rng.integers(1, KV + 1, batch).tolist()
    kv[:len(lengths)] = lengths
    pages.table = np.repeat(pages.table, batch, 0)
    return pages, kv, lambda: gpu.Attend(rng, pages, [q] * batch, kv, hq, dtype, **kw)


class Some:
    """Some of the first sequence's keys and values, for attention64."""

    def __init__(self, pages, j):
        self.heads = pages.heads
        self.k, self.v = [pages.k[0][j]], [pages.v[0][j]]


EDGES = [KV, 1, 1023, 1024, 1025, 1151, 1152, 1153, 2047, 2048, 2049, 2176, 2177, 2432, 2433, 3328, 3329, 3456, 3999]


# Two heads and 512 workgroups a round: ranges of 1152 and of 2432 keys, and whole contexts.
@pytest.mark.parametrize("batch", [1100, 2400, 5000])
@pytest.mark.parametrize("q,hq,d,dtype", [(1, 8, 64, BF16), (1, 8, 128, FP16), (2, 20, 128, BF16), (2, 20, 64, FP16),
                                          (1, 32, 256, BF16), (1, 64, 256, FP16)])
def test_ranges_of_several_pieces(batch, q, hq, d, dtype):
    """16 rows of a head, and 17 to 32."""
    rng = np.random.default_rng(90)
    window = 3000 if q == 2 else 0
    pages, kv, make = batch_of(rng, batch, q, hq, 2, d, dtype, EDGES, window=window)
    a = make()
    rows = ref.intervals([q] * batch, kv, window=window)
    pick = [t for t, r in enumerate(rows) if r[0] < (len(EDGES) if d == 64 else 12)]
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


FORMS = [(1, 8, 64, BF16), (1, 8, 128, FP16), (2, 20, 128, BF16), (1, 32, 256, FP16), (1, 64, 256, BF16)]


@pytest.mark.parametrize("at", [900, 1100, 2999])  # in the first and the second piece, and the last key
@pytest.mark.parametrize("q,hq,d,dtype", FORMS)
def test_a_group_that_reads_as_nan_in_a_piece(at, q, hq, d, dtype):
    """NaN in its 32 dims of the rows that see the key; the others' bits stay."""
    rng = np.random.default_rng(91)
    pages, kv, make = batch_of(rng, 2400, q, hq, 2, d, dtype, [3000, 901, 1101, 2000, 1100, 900])
    clean = pages.words.copy()
    group = d // 32 - 1
    pages.view(pages.table[0, at // 16], at % 16, "v_scales")[0, group] = 255
    a = make()
    out, lse = a.run()
    assert a.errors() == 0
    a.words.upload(clean)
    want, want_lse = a.run()
    assert (lse == want_lse).all() and np.isfinite(want).all()
    sees = np.array([lo <= at < hi for _, _, lo, hi in ref.intervals([q] * 2400, kv)])
    assert sees.any() and not sees.all()
    dims = slice(32 * group, 32 * group + 32)
    assert np.isnan(out[sees][:, :hq // 2, dims]).all()
    out[sees, :hq // 2, dims] = want[sees, :hq // 2, dims]
    assert (out == want).all()


@pytest.mark.parametrize("page", [20, 70, 187])  # keys 320 to 335, 1120 to 1135 and the last 8 of 3000
@pytest.mark.parametrize("q,hq,d,dtype", FORMS)
def test_a_bad_page_in_a_piece_is_reported_and_read_as_nothing(page, q, hq, d, dtype):
    rng = np.random.default_rng(92)
    pages, kv, make = batch_of(rng, 2400, q, hq, 2, d, dtype, [3000, 3000])
    pages.table[0, page] = pages.num_pages  # of the first sequence
    a = make()
    out, _ = a.run()
    assert a.errors() == gfd_amd.KV_ERR_PAGE
    for t, (b, _, lo, hi) in enumerate(ref.intervals([q] * 2, [3000] * 2)):
        j = np.arange(lo, hi)
        some = Some(pages, j[j // 16 != page] if b == 0 else j)
        want, _, tol, _ = ref.attention64(a.q[t:t + 1], some, [(0, 0, 0, len(some.k[0]))], dtype, float(np.float32(a.scale)))
        close(out[t:t + 1], want, tol, "row %d" % t)


@pytest.mark.parametrize("batch", [1100, 5000])
@pytest.mark.parametrize("hq,d,dtype", [(8, 64, FP16), (8, 128, BF16), (40, 128, FP16), (32, 256, BF16)])
def test_a_short_prefix_before_ranges_of_several_pieces(batch, hq, d, dtype):
    """The prefix's rows in a launch of their own."""
    rng = np.random.default_rng(93)
    prefix = 70
    pages = ref4.Pages4(rng, [KV], 16, 2, d, dtype, prefix=prefix)
    pages.table = np.repeat(pages.table, batch, 0)
    kv = (prefix + rng.integers(1, KV + 1, batch)).tolist()
    kv[:6] = [prefix + n for n in (KV, 1, 1024, 1025, 1153, 2177)]
    a = gpu.Attend(rng, pages, [1] * batch, kv, hq, dtype, prefix=prefix)
    rows = [(0, n - 1, 0, n) for n in kv[:12]]
    want, want_lse, tol, tol_lse = ref.attention64(a.q[:12], pages, rows, dtype, float(np.float32(a.scale)))
    out, lse = a.run()
    assert a.errors() == 0 and np.isfinite(out).all()
    close(out[:12], want, tol, "out")
    close(lse[:12], want_lse, tol_lse, "lse")


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("batch", [1, 9])
def test_a_shared_prefix_in_pieces(batch, d):
    """A prefix of 140800 keys whose table names the same ten pages again and again, with 64 heads: its ranges are of
    more than a piece where few rows share it."""
    rng = np.random.default_rng(94)
    heads, page, times = 64, 64, 220
    period = 10 * page
    prefix = period * times
    pages = ref4.Pages4(rng, [1] * batch, page, heads, d, BF16, prefix=period)
    pages.prefix_table = np.tile(pages.prefix_table, times)
    a = gpu.Attend(rng, pages, [1] * batch, [prefix + 1] * batch, heads, BF16, prefix=prefix)
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
