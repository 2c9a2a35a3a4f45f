"""Capped scores, softcap tanh(s / softcap), from caps that cut every score to caps so far above the scores
that they change nothing: right relative to the score, not to the cap."""
import numpy as np
import pytest

import gfd_amd
import paged_kv_ref as ref
from paged_kv_ref import BF16, E4M3, F32, FP16
from test_gpu_paged_kv import Attend, close

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True, scope="module")
def device():
    assert gfd_amd.device_count() > 0, "no GPU visible to libgfd_amd.so"
    assert gfd_amd.lib().gfd_set_device(0) == 0


def capped64(q, pages, rows, dtype, scale, softcap, slopes):
    """(out, lse, tol_out, tol_lse) from the formula in 64 bits.

    Off by, in steps F32 = 2^-24: a sum of d products in any order, d + 8 times the sum of their magnitudes (the cap's
    slope is at most 1); the cap's own operations 8 times the capped score; the bias 4 times itself and the
    score.  An error e of the scores is 2 e of a weight, and the exponent adds a few steps of its argument
    (below 28 for weights over 2^-40): 64.  Weights and output are rounded once to the 16-bit type."""
    T, hq, d = q.shape
    group = hq // pages.heads
    out, lse = np.zeros((T, hq, d)), np.zeros((T, hq))
    tol, tol_lse = np.zeros((T, hq, d)), np.zeros((T, hq))
    for t, (b, pos, lo, hi) in enumerate(rows):
        assert lo < hi
        far = np.abs(pos - np.arange(lo, hi))
        for h in range(hq):
            k, v = pages.k[b][lo:hi, h // group], pages.v[b][lo:hi, h // group]
            s = softcap * np.tanh(k @ q[t, h] * scale / softcap)
            err = (d + 8) * F32 * (np.abs(k) @ np.abs(q[t, h]) * scale) + 8 * F32 * np.abs(s)
            if slopes is not None:
                s = s - slopes[h] * far
                err = err + 4 * F32 * (slopes[h] * far + np.abs(s))
            m = s.max()
            w = np.exp(s - m)
            total, n = w.sum(), len(s)
            out[t, h], lse[t, h] = (w / total) @ v, m + np.log(total)
            rel = 2 * err.max() + 64 * F32
            tol[t, h] = ref.U[dtype] * np.abs(out[t, h]) + 1e-30 + \
                (1.01 * ref.U[dtype] + 1.01 * rel + 2 * n * F32) * ((w / total) @ np.abs(v))
            if dtype == FP16:  # steps no longer shrink below 2^-24
                tol[t, h] += 2.0 ** -25 + 2.0 ** -25 * np.abs(v).max() * n
            tol_lse[t, h] = err.max() + (16 + 2 * n) * F32 * (1 + abs(lse[t, h]))
    return out, lse, tol, tol_lse


def check(seed, q_lens, kv_lens, softcap, d=128, dtype=BF16, cache=None, prefix=0, slopes=False, scale=0.25):
    rng = np.random.default_rng(seed)
    pages = ref.Pages(rng, [n - prefix for n in kv_lens], 16, 2, d, dtype if cache is None else cache, prefix=prefix,
                      k_scale=1 / 32, v_scale=1 / 64, spread=20.0 if cache == E4M3 else 1.0)
    by = np.float32(2.0 ** -np.linspace(0.5, 8, 8)).astype(float) if slopes else None
    a = Attend(rng, pages, q_lens, kv_lens, 8, dtype, prefix=prefix, softcap=softcap, slopes=by, scale=scale)
    rows = ref.intervals(q_lens, kv_lens)
    want, want_lse, tol, tol_lse = capped64(a.q, pages, rows, dtype, scale, float(np.float32(softcap)), by)
    out, lse = a.run()
    assert a.errors() == 0
    close(lse, want_lse, tol_lse, "lse")
    close(out, want, tol, "out")


# Scores have a spread of some units: caps below, among, above and far above them.
CAPS = [1e-3, 0.5, 5.0, 12.0, 50.0, 1e3, 1e4, 1e6, 1e9, 1e20, 1e30, 1e38, 3.3e38]


@pytest.mark.parametrize("slopes", [False, True])
@pytest.mark.parametrize("softcap", CAPS)
@pytest.mark.parametrize("q,kv,prefix", [([1, 1, 1, 1], [1, 2, 5, 40], 0), ([34, 1], [34, 3], 0),
                                         ([1] * 17, list(range(21, 38)), 20)], ids=["few", "many", "both"])
def test_caps_of_every_size(q, kv, prefix, softcap, slopes):
    check(70, q, kv, softcap, prefix=prefix, slopes=slopes)


@pytest.mark.parametrize("softcap", [3.0, 40.0, 1e8])
@pytest.mark.parametrize("d,dtype,cache", [(64, FP16, None), (256, BF16, None), (128, FP16, E4M3), (256, BF16, E4M3)])
@pytest.mark.parametrize("q,kv", [([1, 2], [7, 33]), ([40], [40])], ids=["few", "many"])
def test_caps_of_every_type(q, kv, d, dtype, cache, softcap):
    check(71, q, kv, softcap, d=d, dtype=dtype, cache=cache)


@pytest.mark.parametrize("q,kv", [([1, 1], [40, 3]), ([40], [40])], ids=["few", "many"])
def test_the_smallest_cap_leaves_the_mean(q, kv):
    check(72, q, kv, 1e-40)


@pytest.mark.parametrize("slopes", [False, True])
@pytest.mark.parametrize("q,kv", [([1, 1], [40, 3]), ([40], [40])], ids=["few", "many"])
@pytest.mark.parametrize("scale", [2.0 ** -100, 2.0 ** -60])
def test_the_smallest_scales(q, kv, scale, slopes):
    check(73, q, kv, 1e4, slopes=slopes, scale=scale)
