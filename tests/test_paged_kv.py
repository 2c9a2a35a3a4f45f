"""The paged cache's operators without a GPU: what they refuse, and that a
refused or empty call launches nothing (on this side a launch would fail)."""
import ctypes

import numpy as np
import pytest

import gfd_amd
import paged_kv_ref as ref


def cache(**kw):
    a = dict(k=1 << 20, v=1 << 21, page_stride=32768, slot_stride=1024, head_stride=128, num_pages=8, page_size=16,
             num_heads=8, head_dim=128, dtype=gfd_amd.BF16, k_scale=1.0, v_scale=1.0)
    a.update(kw)
    return gfd_amd.KVCache(**a)


def rows(**kw):
    a = dict(q=1 << 20, k=1 << 20, v=1 << 20, q_out=1 << 20, q_stride=4096, k_stride=1024, v_stride=1024,
             q_out_stride=4096, positions=1 << 20, slots=1 << 20, inv_freq=1 << 20, num_tokens=4, num_q_heads=32,
             rotary_dim=128, interleaved=0, dtype=gfd_amd.BF16)
    a.update(kw)
    return gfd_amd.KVRows(**a)


def call(**kw):
    a = dict(q=1 << 20, out=1 << 20, lse=1 << 20, q_stride=4096, out_stride=4096, q_start=1 << 20, kv_len=1 << 20,
             block_table=1 << 20, table_stride=64, scale=0.1, batch=4, num_tokens=4, max_q_len=1, max_kv_len=1000,
             num_q_heads=32, dtype=gfd_amd.BF16)
    a.update(kw)
    return gfd_amd.Attention(**a)


def test_structs_are_laid_out_as_the_header_says():
    assert ctypes.sizeof(gfd_amd.KVCache) == 72
    assert ctypes.sizeof(gfd_amd.KVRows) == 112
    assert ctypes.sizeof(gfd_amd.Attention) == 136


BAD_CACHE = [dict(k=None), dict(v=None), dict(dtype=3), dict(num_pages=0), dict(page_size=0), dict(page_size=65537),
             dict(num_heads=0), dict(head_dim=96), dict(k=(1 << 20) + 8), dict(page_stride=32769),
             dict(head_stride=-128), dict(dtype=gfd_amd.E4M3, k_scale=0.0),
             dict(dtype=gfd_amd.E4M3, v_scale=float("inf")), dict(dtype=gfd_amd.E4M3, slot_stride=1032)]


@pytest.mark.parametrize("bad", BAD_CACHE, ids=str)
def test_a_bad_cache_is_refused(bad):
    with pytest.raises(gfd_amd.GfdError, match="gfd_kv_append: "):
        gfd_amd.kv_append(cache(**bad), rows())
    with pytest.raises(gfd_amd.GfdError, match="gfd_paged_attention: "):
        gfd_amd.paged_attention(cache(**bad), call())
    with pytest.raises(gfd_amd.GfdError, match="gfd_attention_workspace_bytes: "):
        gfd_amd.attention_workspace_bytes(cache(**bad), call())


@pytest.mark.parametrize("bad", [
    dict(dtype=gfd_amd.E4M3), dict(dtype=gfd_amd.FP16), dict(num_tokens=-1), dict(rotary_dim=130), dict(rotary_dim=63),
    dict(rotary_dim=-2), dict(q=None), dict(q_out=None), dict(num_q_heads=0), dict(q_stride=4097),
    dict(v_stride=1028), dict(k=(1 << 20) + 2), dict(k=None), dict(slots=None), dict(positions=None),
    dict(inv_freq=None)], ids=str)
def test_bad_rows_are_refused(bad):
    with pytest.raises(gfd_amd.GfdError, match="gfd_kv_append: "):
        gfd_amd.kv_append(cache(), rows(**bad))


@pytest.mark.parametrize("bad", [
    dict(dtype=gfd_amd.E4M3), dict(dtype=gfd_amd.FP16), dict(num_q_heads=12), dict(num_q_heads=0), dict(batch=-1),
    dict(num_tokens=-1), dict(max_q_len=-1), dict(max_kv_len=-1), dict(max_kv_len=(1 << 30) + 1), dict(scale=0.0),
    dict(scale=float("nan")), dict(softcap=-1.0), dict(softcap=float("inf")), dict(window=-1), dict(q_stride=4097),
    dict(out=(1 << 20) + 4), dict(table_stride=62), dict(q=None), dict(out=None), dict(q_start=None),
    dict(kv_len=None), dict(block_table=None)], ids=str)
def test_a_bad_call_is_refused(bad):
    with pytest.raises(gfd_amd.GfdError, match="gfd_paged_attention: "):
        gfd_amd.paged_attention(cache(), call(**bad), 1 << 20, 1 << 40)


def test_a_bad_prefix_is_refused():
    for table, n in ((1 << 20, -1), (None, 16)):
        with pytest.raises(gfd_amd.GfdError, match="gfd_shared_prefix_attention: "):
            gfd_amd.shared_prefix_attention(cache(), call(), table, n, 1 << 20, 1 << 40)
    with pytest.raises(gfd_amd.GfdError):
        gfd_amd.attention_workspace_bytes(cache(), call(), -1)


def test_a_missing_struct_is_refused():
    L = gfd_amd.lib()
    assert L.gfd_kv_append(None, rows(), None, None) != 0
    assert L.gfd_kv_append(cache(), None, None, None) != 0
    assert L.gfd_paged_attention(None, call(), None, 0, None, None) != 0
    assert L.gfd_paged_attention(cache(), None, None, 0, None, None) != 0
    assert L.gfd_attention_workspace_bytes(cache(), None, 0) == -1


def test_nothing_to_do_is_no_error():
    gfd_amd.kv_append(cache(), rows(num_tokens=0))
    gfd_amd.paged_attention(cache(), call(batch=0))
    gfd_amd.paged_attention(cache(), call(num_tokens=0))
    gfd_amd.paged_attention(cache(), call(max_q_len=0))
    assert gfd_amd.attention_workspace_bytes(cache(), call()) >= 0


# ------------------------------------------------------------ the oracle itself

def test_the_types_round_trip_and_round_to_nearest():
    for dtype, bits in ((ref.FP16, np.arange(0x7C00, dtype=np.uint16)), (ref.BF16, np.arange(0x7F80, dtype=np.uint16)),
                        (ref.E4M3, np.arange(127, dtype=np.uint8))):
        v = ref.decode(bits, dtype)
        assert (ref.encode(v, dtype) == bits).all() and (np.diff(v) > 0).all()
        mid = (v[:-1] + v[1:]) / 2
        even = bits[:-1] + (bits[:-1] & 1)
        assert (ref.encode(mid, dtype) == even).all()
    assert ref.decode(ref.encode(np.array([500.0, -1e9]), ref.E4M3), ref.E4M3).tolist() == [448.0, -448.0]


def test_the_oracle_agrees_with_a_whole_softmax():
    """attention64 of one sequence with nothing masked against the textbook form."""
    rng = np.random.default_rng(4)
    pages = ref.Pages(rng, [37], 5, 2, 64, ref.BF16, "heads", prefix=11)
    q = rng.standard_normal((3, 4, 64))
    rows_ = ref.intervals([3], [48], prefix_end=[48] * 3)
    out, lse, _, _ = ref.attention64(q, pages, rows_, ref.BF16, 0.125)
    k, v = (np.repeat(x, 2, axis=1) for x in (pages.k[0], pages.v[0]))
    s = np.einsum("thd,jhd->thj", q, k) * 0.125
    p = np.exp(s) / np.exp(s).sum(-1, keepdims=True)
    assert np.allclose(out, np.einsum("thj,jhd->thd", p, v)) and np.allclose(lse, np.log(np.exp(s).sum(-1)))


def test_a_rotation_by_a_whole_turn_changes_nothing_and_pairs_keep_their_length():
    rng = np.random.default_rng(5)
    x = rng.standard_normal((4, 2, 64))
    y, _ = ref.rotate64(x, np.array([0, 3, 70000, 1 << 20]), rng.random(16).astype(np.float32), False)
    assert (y[0] == x[0]).all() and (y[..., 32:] == x[..., 32:]).all()
    assert np.allclose(y[..., :16] ** 2 + y[..., 16:32] ** 2, x[..., :16] ** 2 + x[..., 16:32] ** 2)
