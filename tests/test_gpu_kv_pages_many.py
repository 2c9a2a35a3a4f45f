"""A fork of more items than the search for a page's item samples many times over, against the sequential model."""
import numpy as np
import pytest

import gfd_amd
from test_gpu_kv_pages import Pool

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True, scope="module")
def device():
    assert gfd_amd.device_count() > 0, "no GPU visible to libgfd_amd.so"
    assert gfd_amd.lib().gfd_set_device(0) == 0


@pytest.mark.parametrize("num,pages", [(70001, 200000), (70001, 60000), (1 << 17, 65536)])
def test_a_fork_of_very_many_items(num, pages):
    """Pages for all of them, and for some: the rest is -1.  Stretches of items that need nothing, skipped ones among them."""
    rng = np.random.default_rng(72)
    page, width = 4, 6
    table, refs = np.full((50, width), -5, np.int32), np.zeros(pages, np.int32)
    lens = rng.integers(1, 4 * width + 1, 50)
    place, used = rng.permutation(pages), 0
    for r, n in enumerate(lens):
        k = -(-n // page)
        table[r, :k] = place[used:used + k]
        refs[place[used:used + k]] = 1
        used += k
    p = Pool(refs, page, table, room=num)
    parent = rng.integers(-1, 50, num)
    length = np.where(parent < 0, 0, rng.integers(0, lens[np.maximum(parent, 0)] + 1))
    capacity = np.minimum(length + rng.integers(0, 9, num), page * width)
    child = rng.permutation(num)
    idle = np.arange(num) // 900 % 3 == 0  # need nothing
    parent[idle], length[idle], capacity[idle] = -1, 0, 0
    child[rng.random(num) < 0.05] = -1
    kids = np.full((num, width), -6, np.int32)
    _, errors = p.fork(parent, child, length, capacity, kids=kids)
    assert errors == (gfd_amd.KV_ERR_FULL if (p.refs != 0).all() else 0)
    p.free(child, capacity, kids)
    assert (p.refs == refs).all()
