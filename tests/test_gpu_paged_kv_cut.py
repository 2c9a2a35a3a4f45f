"""Lengths past the maxima that a call states: reported, keys past max_kv_len count as nothing and leave the others'
positions as they are, tokens past max_q_len are left alone."""
import numpy as np
import pytest

import gfd_amd
import paged_kv_ref as ref
from paged_kv_ref import BF16
from test_gpu_paged_kv import Attend, close

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True, scope="module")
def device():
    assert gfd_amd.device_count() > 0, "no GPU visible to libgfd_amd.so"
    assert gfd_amd.lib().gfd_set_device(0) == 0


OPTS = [dict(), dict(window=30), dict(slopes=True), dict(window=17, slopes=True)]


def check(q, kv, prefix=0, max_kv=None, max_q=None, window=0, slopes=False):
    rng = np.random.default_rng(100)
    pages = ref.Pages(rng, [n - prefix for n in kv], 16, 2, 128, BF16, prefix=prefix)
    by = np.float32(2.0 ** -np.linspace(0.5, 8, 8)).astype(float) if slopes else None
    a = Attend(rng, pages, q, kv, 8, BF16, prefix=prefix, window=window, slopes=by, max_kv=max_kv, max_q=max_q)
    rows = [(b, pos, lo, min(hi, max(kv) if max_kv is None else max_kv))
            for b, pos, lo, hi in ref.intervals(q, kv, window=window)]
    taken = np.concatenate([np.arange(n) < (n if max_q is None else max_q) for n in q])
    pick = np.flatnonzero(taken)
    want, want_lse, tol, tol_lse = ref.attention64(a.q[pick], pages, [rows[t] for t in pick], BF16,
                                                   float(np.float32(a.scale)), 0.0, by)
    out, lse = a.run()
    assert a.errors() == gfd_amd.KV_ERR_LENGTH
    close(out[pick], want, tol, "out")
    none = np.isneginf(want_lse)
    assert (np.isneginf(lse[pick]) == none).all()
    close(np.where(none, 0, lse[pick]), np.where(none, 0, want_lse), tol_lse, "lse")
    left = np.flatnonzero(~taken)
    assert (lse[left].view(np.uint32) == 0xA5A5A5A5).all()
    assert (out[left] == ref.decode(np.array([0xA5A5], np.uint16), BF16)[0]).all()


@pytest.mark.parametrize("opts", OPTS, ids=str)
@pytest.mark.parametrize("q,kv,prefix", [([1, 3], [90, 100], 0), ([80, 3], [100, 60], 0), ([100], [400], 0),
                                         ([1, 2], [100, 99], 64), ([1] * 17 + [4], [80] * 17 + [100], 64)], ids=str)
def test_keys_past_the_maximum_count_as_nothing(q, kv, prefix, opts):
    check(q, kv, prefix, max_kv=90 if max(kv) == 100 else 350, **opts)


@pytest.mark.parametrize("opts", OPTS, ids=str)
@pytest.mark.parametrize("q,kv,prefix,max_q", [([1, 5, 2], [90, 100, 7], 0, 2), ([80, 3], [100, 60], 0, 50),
                                               ([1, 4], [100, 99], 64, 3), ([1] * 17 + [4], [80] * 17 + [100], 64, 1)],
                         ids=str)
def test_tokens_past_the_maximum_are_left_alone(q, kv, prefix, max_q, opts):
    check(q, kv, prefix, max_q=max_q, **opts)


@pytest.mark.parametrize("window", [0, 0x7FFFFFFF])
@pytest.mark.parametrize("q", [[1], [40]], ids=str)
def test_the_largest_length_does_not_wrap(q, window):
    """A length of 2^31 - 1 and keys up to the maximum: far before the tokens, all of them visible."""
    rng = np.random.default_rng(101)
    pages = ref.Pages(rng, [70], 16, 2, 128, BF16)
    a = Attend(rng, pages, q, [70], 8, BF16, window=window)
    a.keep["kv_len"].upload(np.array([0x7FFFFFFF], np.int32))
    want, want_lse, tol, tol_lse = ref.attention64(a.q, pages, [(0, 0, 0, 70)] * q[0], BF16, float(np.float32(a.scale)))
    out, lse = a.run()
    assert a.errors() == gfd_amd.KV_ERR_LENGTH
    close(out, want, tol, "out")
    close(lse, want_lse, tol_lse, "lse")
