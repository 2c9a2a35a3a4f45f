"""Sizes of the paged cache's operators that no launch takes, and what their workspace depends on, without a GPU."""
import pytest

import gfd_amd
from test_paged_kv import cache, call


@pytest.mark.parametrize("bad", [
    dict(num_tokens=1 << 24, max_q_len=1 << 24, batch=1, num_q_heads=128),  # rows past 2^30
    dict(num_tokens=1 << 24, batch=1 << 24, max_kv_len=1 << 30, table_stride=1 << 30)], ids=str)
def test_more_than_one_launch_is_refused(bad):
    with pytest.raises(gfd_amd.GfdError, match="more work than one launch takes"):
        gfd_amd.paged_attention(cache(), call(**bad), 1 << 20, 1 << 60)
    with pytest.raises(gfd_amd.GfdError, match="more work than one launch takes"):
        gfd_amd.attention_workspace_bytes(cache(), call(**bad))


def test_no_size_that_is_taken_divides_by_zero():
    for batch in (0, 1, 7):
        for tokens in (0, 1, 500):
            for q in (0, 1, 500):
                for prefix in (0, 1, 1000):
                    for window in (0, 1, 0x7FFFFFFF):
                        n = gfd_amd.attention_workspace_bytes(
                            cache(), call(batch=batch, num_tokens=tokens, max_q_len=q, window=window), prefix)
                        assert 0 <= n < 1 << 30


def test_calls_that_split_keys_need_a_workspace_and_full_batches_need_none():
    rows = 32 * (128 + 2) * 4  # of one token: outputs, maximum and sum in 32 bits
    one = gfd_amd.attention_workspace_bytes(cache(), call(batch=1, num_tokens=1, max_kv_len=1000))
    assert one >= 2 * rows
    assert gfd_amd.attention_workspace_bytes(cache(), call(batch=1, num_tokens=1, max_kv_len=100)) == 0
    assert gfd_amd.attention_workspace_bytes(cache(), call(batch=1, num_tokens=8192, max_q_len=8192, max_kv_len=1000)) == 0
    assert gfd_amd.attention_workspace_bytes(cache(), call(batch=1, num_tokens=1, max_kv_len=100), 16) >= 2 * rows


@pytest.mark.parametrize("given", [(None, 1 << 40), (1 << 20, 100), ((1 << 20) + 8, 1 << 40)], ids=str)
def test_a_missing_small_or_misaligned_workspace_is_refused(given):
    with pytest.raises(gfd_amd.GfdError, match="workspace"):
        gfd_amd.paged_attention(cache(), call(), *given)
    with pytest.raises(gfd_amd.GfdError, match="workspace"):
        gfd_amd.shared_prefix_attention(cache(), call(), 1 << 20, 16, *given)
