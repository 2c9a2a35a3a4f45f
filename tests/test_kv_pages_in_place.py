"""Tables that a call on the cache's pages reads and writes in place, without a GPU: rows of two strides in one table would
lie across one another."""
import pytest

import gfd_amd
from test_paged_kv4 import M, compact, fork, needs_no_gpu, pool


@pytest.mark.parametrize("strides", [(10, 11), (11, 10), (10, 0)], ids=str)
def test_a_table_with_two_strides_is_refused(strides):
    with pytest.raises(gfd_amd.GfdError, match="gfd_kv_compact: table and new_table are one, with two strides"):
        gfd_amd.kv_compact(pool(), compact(table_stride=strides[0], new_stride=strides[1]), M, 1 << 20)
    with pytest.raises(gfd_amd.GfdError, match="gfd_kv_fork: table and child_table are one, with two strides"):
        gfd_amd.kv_fork(pool(), fork(table_stride=strides[0], child_stride=strides[1]), M, 1 << 20)


@needs_no_gpu
def test_two_tables_and_a_table_that_is_not_read_may_have_two_strides():
    for run in (lambda: gfd_amd.kv_compact(pool(), compact(new_table=2 * M, new_stride=11), M, 1 << 20),
                lambda: gfd_amd.kv_compact(pool(), compact(rows=0, new_stride=11), M, 1 << 20),
                lambda: gfd_amd.kv_fork(pool(), fork(child_table=2 * M, child_stride=11), M, 1 << 20),
                lambda: gfd_amd.kv_fork(pool(), fork(rows=0, child_stride=11), M, 1 << 20)):
        with pytest.raises(gfd_amd.GfdError, match="the launch failed"):
            run()
