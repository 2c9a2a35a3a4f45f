"""Lists of more copies than a launch has workgroups, which then take several each."""
import numpy as np
import pytest

import gfd_amd
import paged_kv4_ref as ref4
import test_gpu_paged_kv as gpu
from paged_kv_ref import BF16, E4M3
from test_gpu_kv_pages import filled, parts
from test_gpu_paged_kv import up

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True, scope="module")
def device():
    assert gfd_amd.device_count() > 0, "no GPU visible to libgfd_amd.so"
    assert gfd_amd.lib().gfd_set_device(0) == 0


@pytest.mark.parametrize("cache,heads,page,layout", [(BF16, 2, 32, "heads"), (E4M3, 5, 64, "block"), (3, 3, 70, "heads"),
                                                     (3, 6, 128, "padded")])
@pytest.mark.parametrize("count", [None, 9500, 20000, 100])
def test_copies_past_a_launchs_workgroups(cache, heads, page, layout, count):
    """Pages that are a workgroup's work, or three times it; places that say nothing, refused ones and short copies
    among them; a count that ends in a later round, past the list and in the first round."""
    rng = np.random.default_rng(60)
    dim, n = 128, 20000
    x = filled(rng, 300, page, heads, dim, cache, layout)
    used = x.num_pages
    # Most of the list's places copy nothing, as a compaction's list past its count and a fork's without a part do.
    copies = np.full((n, 4), -1, np.int32)
    copies[:, 2:] = page, 0
    order = rng.permutation(used)
    half = used // 2
    places = np.sort(rng.choice(n, half, replace=False))
    places[:2], places[-2:] = (0, 1), (n - 2, n - 1)
    copies[places, 0], copies[places, 1] = order[:half], order[half:2 * half]
    copies[places[::3], 2] = rng.integers(0, page + 1, len(places[::3]))
    bad = np.setdiff1d(np.arange(0, n, 137), places)
    copies[bad] = [used, 0, page, 0]
    refused = np.setdiff1d(np.arange(5, n, 411), np.concatenate([places, bad]))
    copies[refused] = [0, 0, page + 1, 0]
    words, d_copies, error = up(x.words), up(copies), up(np.zeros(1, np.int32))
    handle = (ref4 if cache == 3 else gpu).handle(x, words)
    d_count = None if count is None else up(np.array([count], np.int32))
    gfd_amd.kv_copy_pages(handle, handle, d_copies.ptr, n, count=None if count is None else d_count.ptr,
                          error_flag=error.ptr)
    gfd_amd.synchronize()
    done = n if count is None else min(count, n)
    bits = gfd_amd.KV_ERR_PAGE * int((bad < done).any()) | gfd_amd.KV_ERR_LENGTH * int((refused < done).any())
    assert int(error.download(4).view(np.int32)[0]) == bits
    for at in places[places < done]:
        p, q, slots, _ = copies[at]
        for s in range(slots):
            for a, b in zip(parts(x, p, s), parts(x, q, s)):
                b[:] = a
    assert (words.download()[:x.words.nbytes] == x.words.view(np.uint8)).all()
