"""Scales whose product leaves 32 bits are refused, on every side of both types, without a GPU."""
import pytest

import gfd_amd
from test_paged_kv import cache, call


@pytest.mark.parametrize("scale,k_scale,taken", [
    (0.1, 0.03, True), (2.0 ** -100, 1.0, True), (2.0 ** 100, 1.0, True), (1e-25, 1e25, True), (2.0 ** -60, 2.0 ** -40, True),
    (1e-30, 1e-30, False), (1e30, 1e30, False), (2.0 ** -101, 1.0, False), (2.0 ** 101, 1.0, False), (1e-45, 1.0, False),
    (2.0 ** -60, 2.0 ** -41, False)])
def test_scales_whose_product_is_out_of_range_are_refused(scale, k_scale, taken):
    c = cache(dtype=gfd_amd.E4M3, k_scale=k_scale)
    if taken:
        assert gfd_amd.attention_workspace_bytes(c, call(scale=scale)) >= 0
        return
    with pytest.raises(gfd_amd.GfdError, match="scale times k_scale"):
        gfd_amd.attention_workspace_bytes(c, call(scale=scale))
    with pytest.raises(gfd_amd.GfdError, match="scale times k_scale"):
        gfd_amd.paged_attention(c, call(scale=scale), 1 << 20, 1 << 40)


def test_the_scales_of_a_16_bit_cache_are_not_read():
    assert gfd_amd.attention_workspace_bytes(cache(k_scale=float("nan"), v_scale=0.0), call()) >= 0
    with pytest.raises(gfd_amd.GfdError, match="scale times k_scale"):
        gfd_amd.attention_workspace_bytes(cache(), call(scale=1e-31))
