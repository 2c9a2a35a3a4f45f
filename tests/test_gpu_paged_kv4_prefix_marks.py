"""Groups that read as NaN and pages that are none, in a 4-bit prefix that sequences share, in every form that takes one:
few rows, a prefix of many with few rows behind it in one launch and in two, many rows."""
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

# tokens of each sequence, sequences, prefix, heads of the queries and of the cache, dims, type
FORMS = [(1, 3, 200, 8, 2, 128, BF16),        # 12 rows of a head
         (2, 4, 513, 12, 2, 64, FP16),        # 48: four waves of 32 rows, and few rows behind
         (1, 12, 200, 8, 2, 128, BF16),
         (1, 12, 200, 8, 2, 256, FP16),
         (1, 5, 12352, 1024, 32, 64, BF16),   # 160: eight waves in a launch of their own
         (40, 3, 200, 8, 2, 128, FP16)]       # blocks of many rows throughout


@pytest.fixture(autouse=True, scope="module")
def device():
    assert gfd_amd.device_count() > 0, "no GPU visible to libgfd_amd.so"
    assert gfd_amd.lib().gfd_set_device(0) == 0


@pytest.fixture(autouse=True)
def four_bits(monkeypatch):
    monkeypatch.setattr(gpu, "handle", ref4.handle)


@pytest.mark.parametrize("where", ["first", "middle", "last"])
@pytest.mark.parametrize("q,batch,prefix,hq,hk,d,dtype", FORMS)
def test_a_group_of_the_prefix_that_reads_as_nan(q, batch, prefix, hq, hk, d, dtype, where):
    """NaN in its 32 dims of the tokens that see the key, which a window keeps from others; no other bit changes."""
    rng = np.random.default_rng(70)
    own = (1 + q + 3 * np.arange(batch)).tolist()
    window = prefix - 20  # later sequences see less of the prefix
    pages = ref4.Pages4(rng, own, 16, hk, d, dtype, "heads", prefix=prefix)
    clean = pages.words.copy()
    kv = [prefix + n for n in own]
    rows = ref.intervals([q] * batch, kv, window=window)
    starts = sorted({lo for _, _, lo, _ in rows})
    at = {"first": starts[0], "middle": starts[len(starts) // 2], "last": prefix - 1}[where]
    group = d // 32 - 1
    pages.view(pages.prefix_table[at // 16], at % 16, "v_scales")[0, group] = 255
    a = gpu.Attend(rng, pages, [q] * batch, kv, hq, dtype, prefix=prefix, window=window)
    out, lse = a.run()
    assert a.errors() == 0
    a.words.upload(clean)
    want, want_lse = a.run()
    assert (lse == want_lse).all() and np.isfinite(want).all()
    sees = np.array([lo <= at < hi for _, _, lo, hi in rows])
    assert sees.any() and (where == "last" or not sees.all())
    dims = slice(32 * group, 32 * group + 32)
    assert np.isnan(out[sees][:, :hq // hk, dims]).all()
    out[sees, :hq // hk, dims] = want[sees, :hq // hk, dims]
    assert (out == want).all()


@pytest.mark.parametrize("bad", [-1, 0x7FFFFFFF])
@pytest.mark.parametrize("q,batch,prefix,hq,hk,d,dtype", FORMS)
def test_a_page_of_the_prefix_that_is_none(q, batch, prefix, hq, hk, d, dtype, bad):
    rng = np.random.default_rng(71)
    own = (q + rng.integers(0, 30, batch)).tolist()
    pages = ref4.Pages4(rng, own, 16, hk, d, dtype, prefix=prefix)
    page = len(pages.prefix_table) // 2
    pages.prefix_table[page] = bad
    kv = [prefix + n for n in own]
    a = gpu.Attend(rng, pages, [q] * batch, kv, hq, dtype, prefix=prefix)
    out, _ = a.run()
    assert a.errors() == gfd_amd.KV_ERR_PAGE
    rows = ref.intervals([q] * batch, kv)
    for t, h in [(0, 0), (len(rows) - 1, hq - 1)] + list(zip(rng.integers(0, len(rows), 12), rng.integers(0, hq, 12))):
        b, _, lo, hi = rows[t]
        j = np.arange(lo, hi)
        some = Some(ref4.OneHead(pages, b, h * hk // hq), j[(j // 16 != page) | (j >= prefix)])
        want, _, tol, _ = ref.attention64(a.q[t:t + 1, h:h + 1], some, [(0, 0, 0, len(some.k[0]))], dtype,
                                          float(np.float32(a.scale)))
        close(out[t:t + 1, h:h + 1], want, tol, "row %d, head %d" % (t, h))
