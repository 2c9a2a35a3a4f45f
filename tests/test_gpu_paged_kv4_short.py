"""Many short contexts in 4 bits, which a wave each takes: at most 128 keys, 512 sequences' heads and more.

All sequences read the same pages, so that the cache stays small."""
import numpy as np
import pytest

import gfd_amd
import paged_kv4_ref as ref4
import paged_kv_ref as ref
import test_gpu_paged_kv as gpu
from paged_kv_ref import BF16, FP16
from test_gpu_paged_kv import close
from test_gpu_paged_kv4_pieces import Some

pytestmark = pytest.mark.gpu

EDGES = [128, 1, 0, 31, 32, 33, 63, 64, 65, 95, 96, 97, 127, 2, 16, 17]


@pytest.fixture(autouse=True, scope="module")
def device():
    assert gfd_amd.device_count() > 0, "no GPU visible to libgfd_amd.so"
    assert gfd_amd.lib().gfd_set_device(0) == 0


@pytest.fixture(autouse=True)
def four_bits(monkeypatch):
    monkeypatch.setattr(gpu, "handle", ref4.handle)


def batch_of(rng, q, hq, hk, d, dtype, layout="block", page=16, batch=None, **kw):
    batch = -(-512 // hk) + 3 if batch is None else batch  # no multiple of 8
    pages = ref4.Pages4(rng, [128], page, hk, d, dtype, layout)
    kv = rng.integers(0, 129, batch).tolist()
    kv[:len(EDGES)] = EDGES
    pages.table = np.repeat(pages.table, batch, 0)

    def make():
        a = gpu.Attend(rng, pages, [q] * batch, kv, hq, dtype, **kw)
        assert batch * hk >= 512 and a.work_bytes == 0
        return a
    return pages, kv, make


def check(a, pages, rows, dtype, picked, **kw):
    """The picked sequences' rows; (out, lse) of all."""
    pick = [t for t, r in enumerate(rows) if r[0] in picked]
    want, want_lse, tol, tol_lse = ref.attention64(a.q[pick], pages, [(0,) + rows[t][1:] for t in pick], dtype,
                                                   float(np.float32(a.scale)), **kw)
    out, lse = a.run()
    none = np.isneginf(want_lse)
    close(out[pick], want, tol, "out")
    assert (np.isneginf(lse[pick]) == none).all()
    close(np.where(none, 0, lse[pick]), np.where(none, 0, want_lse), tol_lse, "lse")
    again, lse2 = a.run()
    assert (again == out)[np.isfinite(out)].all() and (lse2 == lse).all()
    return out, lse


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("q,hq,hk", [(1, 8, 8), (1, 32, 2), (1, 40, 2), (2, 16, 2), (5, 12, 2), (1, 7, 7)])
def test_lengths_around_tiles(q, hq, hk, d, dtype):
    """Up to 16 rows of a head, and 17 to 32."""
    rng = np.random.default_rng(50)
    pages, kv, make = batch_of(rng, q, hq, hk, d, dtype, "heads" if d == 128 else "block")
    a = make()
    rows = ref.intervals([q] * len(kv), kv)
    last = len(kv) - 1
    out, _ = check(a, pages, rows, dtype, set(range(len(EDGES))) | {last - 1, last})
    assert a.errors() == 0 and np.isfinite(out).all()


@pytest.mark.parametrize("page,layout", [(1, "block"), (5, "heads"), (24, "apart"), (64, "padded")])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_pages_and_layouts(d, page, layout):
    rng = np.random.default_rng(51)
    pages, kv, make = batch_of(rng, 1, 16, 4, d, BF16, layout, page)
    a = make()
    check(a, pages, ref.intervals([1] * len(kv), kv), BF16, set(range(len(EDGES))))
    assert a.errors() == 0


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("q", [1, 3])
@pytest.mark.parametrize("opts", [dict(softcap=5.0), dict(softcap=500.0), dict(slopes=True), dict(window=20),
                                  dict(window=1), dict(softcap=30.0, slopes=True, window=65)], ids=str)
def test_cap_bias_and_window(opts, q, d):
    rng = np.random.default_rng(52)
    opts = dict(opts)
    sl = np.float32(2.0 ** -np.linspace(0.5, 8, 16)).astype(float) if opts.pop("slopes", False) else None
    window = opts.pop("window", 0)
    pages, kv, make = batch_of(rng, q, 16, 2, d, FP16, window=window, slopes=sl, **opts)
    a = make()
    check(a, pages, ref.intervals([q] * len(kv), kv, window=window), FP16, set(range(len(EDGES))),
          softcap=opts.get("softcap", 0.0), slopes=sl)
    assert a.errors() == 0


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("dtype,byte", [(BF16, 255), (BF16, 253), (FP16, 255), (FP16, 141)])
@pytest.mark.parametrize("at", [0, 40, 127])
def test_a_group_that_reads_as_nan(at, dtype, byte, d):
    """In one value: NaN in its 32 dims of the sequences that see the key, no other bit of any."""
    rng = np.random.default_rng(53)
    pages, kv, make = batch_of(rng, 2, 8, 2, d, dtype)
    clean = pages.words.copy()
    group = d // 32 - 1
    pages.view(pages.table[0, at // 16], at % 16, "v_scales")[0, group] = byte
    a = make()
    out, lse = a.run()
    a.words.upload(clean)
    want, want_lse = a.run()
    assert (lse == want_lse).all() and np.isfinite(want).all()
    sees = np.array([lo <= at < hi for _, _, lo, hi in ref.intervals([2] * len(kv), kv)])
    assert sees.any() and not sees.all()
    dims = slice(32 * group, 32 * group + 32)
    assert np.isnan(out[sees][:, :4, dims]).all()
    out[sees, :4, dims] = want[sees, :4, dims]
    assert (out == want).all()


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("bad", [-1, -0x80000000, 0x7FFFFFFF])
def test_a_bad_page_is_reported_and_read_as_nothing(bad, d):
    rng = np.random.default_rng(54)
    pages, kv, make = batch_of(rng, 1, 8, 2, d, BF16)
    pages.table[0, 2] = pages.num_pages if bad == 0x7FFFFFFF else bad  # keys 32 to 47 of the first sequence, which has 128
    a = make()
    out, _ = a.run()
    assert a.errors() == gfd_amd.KV_ERR_PAGE
    for t, j in ((0, np.r_[0:32, 48:128]), (12, np.arange(127)), (4, np.arange(32))):
        some = Some(pages, j)
        want, _, tol, _ = ref.attention64(a.q[t:t + 1], some, [(0, 0, 0, len(j))], BF16, float(np.float32(a.scale)))
        close(out[t:t + 1], want, tol, "row %d" % t)


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("q,window", [(1, 127), (1, 30), (5, 100)])
def test_short_windows_of_long_contexts(q, window, d):
    rng = np.random.default_rng(55)
    batch = 259
    pages = ref4.Pages4(rng, [3000], 16, 2, d, BF16)
    pages.table = np.repeat(pages.table, batch, 0)
    kv = rng.integers(0, 3001, batch).tolist()
    kv[:8] = [3000, 0, 1, 2999, 128, 1024, 1025, window]
    a = gpu.Attend(rng, pages, [q] * batch, kv, 6, BF16, window=window)
    assert a.work_bytes == 0
    check(a, pages, ref.intervals([q] * batch, kv, window=window), BF16, set(range(16)) | {batch - 1})
    assert a.errors() == 0
