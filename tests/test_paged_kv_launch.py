"""A call of the paged cache's operators whose launch fails says so (without a GPU every launch does)."""
import pytest

import gfd_amd
from test_paged_kv import cache, call, rows

needs_no_gpu = pytest.mark.skipif(gfd_amd.device_count() > 0, reason="the addresses are no memory: a launch has to fail")


@needs_no_gpu
def test_a_failed_launch_leaves_its_text_and_no_earlier_one():
    big = 1 << 40
    for name, run in (("gfd_kv_append", lambda: gfd_amd.kv_append(cache(), rows())),
                      ("gfd_paged_attention", lambda: gfd_amd.paged_attention(cache(), call(), 1 << 20, big)),
                      ("gfd_shared_prefix_attention",
                       lambda: gfd_amd.shared_prefix_attention(cache(), call(), 1 << 20, 16, 1 << 20, big))):
        with pytest.raises(gfd_amd.GfdError, match="negative num_tokens"):
            gfd_amd.kv_append(cache(), rows(num_tokens=-1))
        with pytest.raises(gfd_amd.GfdError, match=name + ": the launch failed: "):
            run()
