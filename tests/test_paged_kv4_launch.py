"""The largest calls of a 4-bit cache's attention and append that one launch takes, and failed launches' texts, without a
GPU (there every launch fails)."""
import pytest

import gfd_amd
from test_paged_kv import call, rows
from test_paged_kv4 import cache4

needs_no_gpu = pytest.mark.skipif(gfd_amd.device_count() > 0, reason="the addresses are no memory: a launch has to fail")


@needs_no_gpu
def test_a_failed_launch_leaves_its_text_and_no_earlier_one():
    big = 1 << 40
    pool = gfd_amd.KVPool(refs=1 << 20, num_pages=10, page_size=16)
    fork = gfd_amd.KVFork(table=1 << 20, child_table=1 << 20, table_stride=4, child_stride=4, rows=4, child_rows=4,
                          parent=1 << 20, child=1 << 20, len=1 << 20, copies=1 << 20, num=2)
    pages = gfd_amd.KVCompact(new_refs=1 << 20, table=1 << 20, new_table=1 << 20, table_stride=4, new_stride=4, len=1 << 20,
                              rows=4, copies=1 << 20, num_copies=1 << 20)
    read = gfd_amd.KVRead(k=1 << 20, v=1 << 20, k_stride=512, v_stride=512, slots=1 << 20, num_tokens=3, dtype=call().dtype)
    for name, run in (("gfd_kv4_append", lambda: gfd_amd.kv_append(cache4(), rows())),
                      ("gfd_kv4_read", lambda: gfd_amd.kv_read(cache4(), read)),
                      ("gfd_kv4_attention", lambda: gfd_amd.paged_attention(cache4(), call(), 1 << 20, big)),
                      ("gfd_kv4_shared_prefix_attention",
                       lambda: gfd_amd.shared_prefix_attention(cache4(), call(), 1 << 20, 16, 1 << 20, big)),
                      ("gfd_kv4_copy_pages", lambda: gfd_amd.kv_copy_pages(cache4(), cache4(), 1 << 20, 5)),
                      ("gfd_kv_fork", lambda: gfd_amd.kv_fork(pool, fork, 1 << 20, big)),
                      ("gfd_kv_free", lambda: gfd_amd.kv_free(pool, 1 << 20, 4, 4, 1 << 20, 1 << 20, 2)),
                      ("gfd_kv_compact", lambda: gfd_amd.kv_compact(pool, pages, 1 << 20, big))):
        with pytest.raises(gfd_amd.GfdError, match="negative num_tokens"):
            gfd_amd.kv_append(cache4(), rows(num_tokens=-1))
        with pytest.raises(gfd_amd.GfdError, match=name + ": the launch failed: "):
            run()


@needs_no_gpu
def test_the_largest_append():
    largest = 4 * ((1 << 24) - 1)  # four tokens a workgroup of 256
    with pytest.raises(gfd_amd.GfdError, match="the launch failed"):
        gfd_amd.kv_append(cache4(), rows(num_tokens=largest))
    for tokens in (largest + 1, 0x7FFFFFFF):
        with pytest.raises(gfd_amd.GfdError, match="gfd_kv4_append: more work than one launch takes"):
            gfd_amd.kv_append(cache4(), rows(num_tokens=tokens))


def test_batches_of_more_than_one_launch_are_refused():
    c = cache4()
    heads = c.num_heads
    # 256 threads a head and sequence, of fewer than 2^32; turns of 8 ranges' heads and two of 8 workgroups may be filled up.
    largest = ((1 << 24) - 1 - 16 - 16 * heads) // heads
    assert gfd_amd.attention_workspace_bytes(c, call(batch=largest, num_tokens=64, max_kv_len=1000)) >= 0
    for batch in (largest + 1, 1 << 24):
        with pytest.raises(gfd_amd.GfdError, match="more work than one launch takes"):
            gfd_amd.attention_workspace_bytes(c, call(batch=batch, num_tokens=64, max_kv_len=1000))


@pytest.mark.parametrize("batch,heads", [(1 << 24, 65535), (1 << 24, 1 << 14), (1 << 20, 1 << 12), (1 << 11, 65535)])
@pytest.mark.parametrize("kv", [1, 129, 1 << 30])
@pytest.mark.parametrize("prefix,max_q", [(0, 1), (160, 1), (1 << 30, 1), (0, 1 << 24), (1 << 20, 500)])
def test_products_of_the_largest_sizes_do_not_wrap(batch, heads, kv, prefix, max_q):
    k = call(batch=batch, num_tokens=1, max_q_len=max_q, max_kv_len=kv, num_q_heads=heads, table_stride=1 << 27)
    with pytest.raises(gfd_amd.GfdError, match="more work than one launch takes"):
        gfd_amd.attention_workspace_bytes(cache4(num_heads=heads), k, prefix)
