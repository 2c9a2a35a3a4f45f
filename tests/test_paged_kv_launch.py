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


# A launch has fewer than 2^32 threads along its grid: the largest call that is taken, and the next one.

@needs_no_gpu
def test_the_largest_append():
    largest = 4 * ((1 << 24) - 1)  # four tokens a workgroup of 256
    with pytest.raises(gfd_amd.GfdError, match="the launch failed"):
        gfd_amd.kv_append(cache(), rows(num_tokens=largest))
    for tokens in (largest + 1, 0x7FFFFFFF):
        with pytest.raises(gfd_amd.GfdError, match="gfd_kv_append: more work than one launch takes"):
            gfd_amd.kv_append(cache(), rows(num_tokens=tokens))


@needs_no_gpu
@pytest.mark.parametrize("prefix", [0, 160])
@pytest.mark.parametrize("sizes,largest", [(dict(max_kv_len=1000), (1 << 24) // 8 - 3),  # few rows: 256 threads a head and sequence
                                           # two blocks of 128 rows more: 64 tokens of 4 heads
                                           (dict(max_kv_len=1000, max_q_len=500), (1 << 24) // 8 - 5)])
def test_the_largest_batch(sizes, largest, prefix):
    """Two rounds of 8 workgroups may be filled up: so many sequences are one launch, and the next is refused."""
    for batch, why in ((largest - 40 * bool(prefix), "the launch failed"), (largest + 1, "more work than one launch takes")):
        c = call(batch=batch, num_tokens=64, **sizes)
        with pytest.raises(gfd_amd.GfdError, match=why):
            if prefix:
                gfd_amd.shared_prefix_attention(cache(), c, 1 << 20, prefix, 1 << 20, 1 << 60)
            else:
                gfd_amd.paged_attention(cache(), c, 1 << 20, 1 << 60)


def test_a_workspace_is_stated_only_for_calls_that_are_taken():
    with pytest.raises(gfd_amd.GfdError, match="more work than one launch takes"):
        gfd_amd.attention_workspace_bytes(cache(), call(batch=1 << 21, num_tokens=64, max_kv_len=1000))


@pytest.mark.parametrize("batch,heads", [(1 << 24, 65535), (1 << 24, 1 << 14), (1 << 20, 1 << 12), (1 << 24, 255), (1 << 11, 65535)])
@pytest.mark.parametrize("kv", [1, 129, 1 << 30])
@pytest.mark.parametrize("prefix,max_q", [(0, 1), (160, 1), (1 << 30, 1), (0, 1 << 24), (1 << 20, 500)])
def test_products_of_the_largest_sizes_do_not_wrap(batch, heads, kv, prefix, max_q):
    c = cache(num_heads=heads)
    k = call(batch=batch, num_tokens=1, max_q_len=max_q, max_kv_len=kv, num_q_heads=heads, table_stride=1 << 27)
    with pytest.raises(gfd_amd.GfdError, match="more work than one launch takes"):
        gfd_amd.attention_workspace_bytes(c, k, prefix)
