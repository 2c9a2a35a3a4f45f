"""Shared prefixes of a 4-bit cache so long that their blocks have 8 waves and a launch of their own, or come two to a
CU: some rows of each block against attention in 64 bits."""
import numpy as np
import pytest

import gfd_amd
import paged_kv4_ref as ref4
import paged_kv_ref as ref
import test_gpu_paged_kv as gpu
from paged_kv_ref import BF16, FP16
from test_gpu_paged_kv import close

pytestmark = pytest.mark.gpu

HK, HQ = 32, 1024  # 32 rows of a head for each token


@pytest.fixture(autouse=True, scope="module")
def device():
    assert gfd_amd.device_count() > 0, "no GPU visible to libgfd_amd.so"
    assert gfd_amd.lib().gfd_set_device(0) == 0


# Ranges of 1536 keys or more with two workgroups of 128 rows a CU: prefix * ceil(rows / 128) * 32 >= 1536 * 512.
@pytest.mark.parametrize("batch,prefix,d,dtype,layout,opts", [
    (5, 12352, 64, BF16, "heads", {}),                             # 160 rows: one block of 256
    (5, 12300, 128, FP16, "block", dict(softcap=30.0)),
    (8, 12288, 64, FP16, "apart", dict(window=12290)),             # 256 rows
    (14, 6200, 64, BF16, "heads", {}),                             # 448: two
    (3, 24640, 64, BF16, "heads", {}),                             # 96 rows: a block of 128
    (9, 8256, 64, BF16, "block", {}),                              # 288: three, as two of 256 would be 512
    (5, 12288, 256, BF16, "heads", {}),                            # 256 dims: two of 128
])
def test_a_long_shared_prefix(batch, prefix, d, dtype, layout, opts, monkeypatch):
    monkeypatch.setattr(gpu, "handle", ref4.handle)
    rng = np.random.default_rng(batch)
    q_lens, kv_lens = [1] * batch, [prefix + int(n) for n in rng.integers(0, 70, batch)]
    kv_lens[0] = prefix  # nothing of its own
    pages = ref4.Pages4(rng, [n - prefix for n in kv_lens], 32, HK, d, dtype, layout, prefix=prefix)
    a = gpu.Attend(rng, pages, q_lens, kv_lens, HQ, dtype, prefix=prefix, **opts)
    out, lse = a.run()
    assert a.errors() == 0
    rows = ref.intervals(q_lens, kv_lens, window=opts.get("window", 0))
    for t, h in zip([0, batch - 1, *rng.integers(0, batch, 30)], [0, HQ - 1, *rng.integers(0, HQ, 30)]):
        b, *interval = rows[t]
        one = ref4.OneHead(pages, b, h // 32)
        want, want_lse, tol, tol_lse = ref.attention64(a.q[t:t + 1, h:h + 1], one, [(0, *interval)], dtype,
                                                       np.float32(a.scale).astype(float), opts.get("softcap", 0.0))
        close(out[t:t + 1, h:h + 1], want, tol, "out %d %d" % (t, h))
        close(lse[t:t + 1, h:h + 1], want_lse, tol_lse, "lse %d %d" % (t, h))
    again, lse2 = a.run()
    assert (again == out).all() and (lse2 == lse).all()
