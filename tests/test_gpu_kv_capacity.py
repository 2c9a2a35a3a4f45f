"""Rows whose pages were given for more tokens than are in them yet: brought together and let go of by their capacities,
they keep what was given to them, and lose it all."""
import numpy as np
import pytest

import gfd_amd
from test_gpu_kv_pages import Pool

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True, scope="module")
def device():
    assert gfd_amd.device_count() > 0, "no GPU visible to libgfd_amd.so"
    assert gfd_amd.lib().gfd_set_device(0) == 0


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("page", [1, 16])
def test_pages_given_ahead_are_moved_and_freed_with_the_capacity(page, in_place):
    p = Pool(np.zeros(64, np.int32), page, np.full((6, 8), -1, np.int32))
    capacity = np.array([8, 1, 5, 8, 3, 7]) * page
    assert p.fork([-1] * 6, list(range(6)), [0] * 6, capacity.tolist())[1] == 0
    p.free([0, 2], capacity[[0, 2]].tolist())
    length = capacity.copy()
    length[[0, 2]] = 0
    p.table[[0, 2]] = -1
    p.d_table.upload(p.table)
    moves, errors = p.compact(length.tolist(), in_place=in_place)
    assert errors == 0 and len(moves)
    if not in_place:
        return  # compact() has compared the new table and counts
    # Every row has as many pages as it was given, each its own, at the front.
    held = [p.table[r, :capacity[r] // page] for r in (1, 3, 4, 5)]
    assert sorted(np.concatenate(held)) == list(range(1 + 8 + 3 + 7)) and (p.refs[:19] == 1).all()
    p.free([1, 3, 4, 5], capacity[[1, 3, 4, 5]].tolist())
    assert not p.refs.any()
