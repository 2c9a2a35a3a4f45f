"""The 4-bit cache, positions of several axes and the cache's pages without a GPU: what the calls refuse, that a refused
or empty call launches nothing, and the tests' own definitions."""
import ctypes

import numpy as np
import pytest

import gfd_amd
import kv_pages_ref as pages_ref
import paged_kv4_ref as ref4
import paged_kv_ref as ref
from paged_kv_ref import BF16, FP16
from test_paged_kv import cache, call, rows

M = 1 << 20
needs_no_gpu = pytest.mark.skipif(gfd_amd.device_count() > 0, reason="the addresses are no memory: a launch has to fail")


def cache4(**kw):
    a = dict(k=M, v=2 * M, k_scales=3 * M + 1, v_scales=4 * M + 3, page_stride=16384, slot_stride=512, head_stride=64,
             scale_page_stride=1024, num_pages=8, page_size=16, num_heads=8, head_dim=128)
    a.update(kw)
    return gfd_amd.KV4Cache(**a)


def axes(**kw):
    a = dict(positions=M, axis=M + 1, axis_stride=4, token_stride=1, num_axes=3)
    a.update(kw)
    return gfd_amd.RotaryAxes(**a)


def read(**kw):
    a = dict(k=M, v=M, k_stride=1024, v_stride=1024, slots=M, num_tokens=4, dtype=gfd_amd.BF16)
    a.update(kw)
    return gfd_amd.KVRead(**a)


def pool(**kw):
    a = dict(refs=M, num_pages=100, page_size=16)
    a.update(kw)
    return gfd_amd.KVPool(**a)


def fork(**kw):
    a = dict(table=M, child_table=M, table_stride=10, child_stride=10, rows=4, child_rows=4, parent=M, child=M, len=M,
             capacity=M, copies=M, num=3)
    a.update(kw)
    return gfd_amd.KVFork(**a)


def compact(**kw):
    a = dict(new_refs=M, table=M, new_table=M, table_stride=10, new_stride=10, len=M, rows=4, page_map=M, copies=M,
             num_copies=M)
    a.update(kw)
    return gfd_amd.KVCompact(**a)


def test_structs_are_laid_out_as_the_header_says():
    for name, size in (("KV4Cache", 80), ("RotaryAxes", 40), ("KVRead", 48), ("KVPool", 16), ("KVFork", 88),
                       ("KVCompact", 80)):
        assert ctypes.sizeof(getattr(gfd_amd, name)) == size, name
    assert gfd_amd.PAGE_COPY_DTYPE.itemsize == 16


BAD_CACHE = [dict(k=None), dict(v=None), dict(k_scales=None), dict(v_scales=None), dict(num_pages=0),
             dict(page_size=0), dict(page_size=65537), dict(num_heads=0), dict(num_heads=65536), dict(head_dim=96),
             dict(k=M + 8), dict(page_stride=16392), dict(slot_stride=520), dict(head_stride=-64),
             dict(scale_page_stride=-1), dict(page_stride=1 << 31), dict(scale_page_stride=1 << 31),
             dict(slot_stride=1 << 27, page_size=17)]


@pytest.mark.parametrize("bad", BAD_CACHE, ids=str)
def test_a_bad_cache_is_refused(bad):
    c = cache4(**bad)
    for name, run in (("gfd_kv4_append", lambda: gfd_amd.kv_append(c, rows())),
                      ("gfd_kv4_read", lambda: gfd_amd.kv_read(c, read())),
                      ("gfd_kv4_attention", lambda: gfd_amd.paged_attention(c, call())),
                      ("gfd_kv4_shared_prefix_attention",
                       lambda: gfd_amd.shared_prefix_attention(c, call(), M, 16, M, 1 << 40)),
                      ("gfd_kv4_attention_workspace_bytes", lambda: gfd_amd.attention_workspace_bytes(c, call())),
                      ("gfd_kv4_copy_pages", lambda: gfd_amd.kv_copy_pages(c, cache4(), M, 1)),
                      ("gfd_kv4_copy_pages", lambda: gfd_amd.kv_copy_pages(cache4(), c, M, 1))):
        with pytest.raises(gfd_amd.GfdError, match=name + ": "):
            run()


@needs_no_gpu
def test_the_largest_pages_are_taken():
    """Rows that end just within 2^31 bytes of their page's first (and one step further: refused above)."""
    with pytest.raises(gfd_amd.GfdError, match="the launch failed"):
        gfd_amd.kv_append(cache4(slot_stride=(1 << 27) - 64, page_size=17), rows())
    with pytest.raises(gfd_amd.GfdError, match="the launch failed"):
        gfd_amd.kv_append(cache4(page_stride=(1 << 31) - 16, scale_page_stride=(1 << 31) - 1), rows())


BAD_ROWS = [dict(dtype=gfd_amd.E4M3), dict(num_tokens=-1), dict(rotary_dim=130), dict(rotary_dim=63),
            dict(rotary_dim=-2), dict(q=None), dict(q_out=None), dict(num_q_heads=0), dict(q_stride=4097),
            dict(v_stride=1028), dict(k=M + 2), dict(k=None), dict(slots=None), dict(inv_freq=None),
            dict(num_tokens=0x7FFFFFFF)]


@pytest.mark.parametrize("bad", BAD_ROWS + [dict(positions=None)], ids=str)
def test_bad_rows_are_refused(bad):
    with pytest.raises(gfd_amd.GfdError, match="gfd_kv4_append: "):
        gfd_amd.kv_append(cache4(), rows(**bad))


@pytest.mark.parametrize("bad", [dict(positions=None), dict(axis=None), dict(num_axes=0), dict(num_axes=257)], ids=str)
def test_bad_axes_are_refused(bad):
    for c, name in ((cache(), "gfd_kv_append_axes"), (cache4(), "gfd_kv4_append")):
        with pytest.raises(gfd_amd.GfdError, match=name + ": "):
            gfd_amd.kv_append(c, rows(), axes=axes(**bad))


@pytest.mark.parametrize("bad", BAD_ROWS, ids=str)
def test_bad_rows_with_axes_are_refused(bad):
    for c, name in ((cache(), "gfd_kv_append_axes"), (cache4(), "gfd_kv4_append")):
        with pytest.raises(gfd_amd.GfdError, match=name + ": "):
            gfd_amd.kv_append(c, rows(**bad), axes=axes())


@pytest.mark.parametrize("bad", [dict(dtype=gfd_amd.E4M3), dict(num_tokens=-1), dict(k_stride=1028), dict(v=M + 8),
                                 dict(slots=None)], ids=str)
def test_bad_rows_to_read_are_refused(bad):
    for c, name in ((cache(), "gfd_kv_read"), (cache4(), "gfd_kv4_read")):
        with pytest.raises(gfd_amd.GfdError, match=name + ": "):
            gfd_amd.kv_read(c, read(**bad))
    with pytest.raises(gfd_amd.GfdError, match="gfd_kv_read: "):
        gfd_amd.kv_read(cache(), read(dtype=gfd_amd.FP16))


@pytest.mark.parametrize("bad", [
    dict(dtype=gfd_amd.E4M3), dict(num_q_heads=12), dict(batch=-1), dict(num_tokens=-1), dict(max_q_len=-1),
    dict(max_kv_len=(1 << 30) + 1), dict(scale=0.0), dict(scale=float("nan")), dict(scale=1e-31), dict(softcap=-1.0),
    dict(window=-1), dict(q_stride=4097), dict(out=M + 4), dict(table_stride=62), dict(q=None), dict(out=None),
    dict(q_start=None), dict(kv_len=None), dict(block_table=None)], ids=str)
def test_a_bad_call_is_refused(bad):
    with pytest.raises(gfd_amd.GfdError, match="gfd_kv4_attention: "):
        gfd_amd.paged_attention(cache4(), call(**bad), M, 1 << 40)


def test_a_bad_prefix_is_refused():
    for table, n in ((M, -1), (None, 16)):
        with pytest.raises(gfd_amd.GfdError, match="gfd_kv4_shared_prefix_attention: "):
            gfd_amd.shared_prefix_attention(cache4(), call(), table, n, M, 1 << 40)


@pytest.mark.parametrize("bad", [dict(refs=None), dict(num_pages=0), dict(num_pages=(1 << 24) + 1), dict(page_size=0),
                                 dict(page_size=65537)], ids=str)
def test_a_bad_pool_is_refused(bad):
    p = pool(**bad)
    for name, run in (("gfd_kv_fork", lambda: gfd_amd.kv_fork(p, fork(), M, 1 << 40)),
                      ("gfd_kv_free", lambda: gfd_amd.kv_free(p, M, 10, 4, M, M, 3)),
                      ("gfd_kv_compact", lambda: gfd_amd.kv_compact(p, compact(), M, 1 << 40)),
                      ("gfd_kv_pool_workspace_bytes", lambda: gfd_amd.kv_pool_workspace_bytes(p))):
        with pytest.raises(gfd_amd.GfdError, match=name + ": "):
            run()


@pytest.mark.parametrize("bad", [dict(num=-1), dict(num=(1 << 20) + 1), dict(table_stride=-1), dict(child_stride=-1),
                                 dict(rows=-1), dict(child_rows=-1), dict(parent=None), dict(child=None),
                                 dict(len=None), dict(child_table=None), dict(table=None), dict(copies=None),
                                 dict(copies=M + 8), dict(child_stride=(1 << 31) + 1)], ids=str)
def test_a_bad_fork_is_refused(bad):
    with pytest.raises(gfd_amd.GfdError, match="gfd_kv_fork: "):
        gfd_amd.kv_fork(pool(), fork(**bad), M, 1 << 40)


@pytest.mark.parametrize("bad", [dict(table_stride=-1), dict(new_stride=-1), dict(rows=-1), dict(rows=(1 << 20) + 1),
                                 dict(new_refs=None), dict(num_copies=None), dict(table=None), dict(new_table=None),
                                 dict(len=None), dict(copies=None), dict(copies=M + 4)], ids=str)
def test_a_bad_compaction_is_refused(bad):
    with pytest.raises(gfd_amd.GfdError, match="gfd_kv_compact: "):
        gfd_amd.kv_compact(pool(), compact(**bad), M, 1 << 40)


def test_a_bad_freeing_is_refused():
    for a in ((None, 10, 4, M, M, 3), (M, -1, 4, M, M, 3), (M, 10, -1, M, M, 3), (M, 10, 4, None, M, 3),
              (M, 10, 4, M, None, 3), (M, 10, 4, M, M, -1), (M, 10, 4, M, M, (1 << 20) + 1)):
        with pytest.raises(gfd_amd.GfdError, match="gfd_kv_free: "):
            gfd_amd.kv_free(pool(), *a)


def test_a_workspace_that_is_too_small_is_refused():
    need = gfd_amd.kv_pool_workspace_bytes(pool(), 3)
    for space, size in ((None, need), (M, need - 1), (M + 8, need)):
        with pytest.raises(gfd_amd.GfdError, match="gfd_kv_fork: workspace"):
            gfd_amd.kv_fork(pool(), fork(), space, size)
        with pytest.raises(gfd_amd.GfdError, match="gfd_kv_compact: workspace"):
            gfd_amd.kv_compact(pool(), compact(), space, size)
    for num in (-1, (1 << 20) + 1):
        with pytest.raises(gfd_amd.GfdError):
            gfd_amd.kv_pool_workspace_bytes(pool(), num)
    assert gfd_amd.kv_pool_workspace_bytes(pool(num_pages=1)) > 0


@pytest.mark.parametrize("bad", [dict(page_size=8), dict(num_heads=4), dict(head_dim=64)], ids=str)
def test_caches_of_other_sizes_are_refused(bad):
    for one, name in ((cache, "gfd_kv_copy_pages"), (cache4, "gfd_kv4_copy_pages")):
        with pytest.raises(gfd_amd.GfdError, match=name + ": "):
            gfd_amd.kv_copy_pages(one(), one(**bad), M, 1)


def test_copies_that_are_none_are_refused():
    for one in (cache, cache4):
        for copies, n in ((None, 1), (M + 8, 1), (M, -1)):
            with pytest.raises(gfd_amd.GfdError, match="copies"):
                gfd_amd.kv_copy_pages(one(), one(), copies, n)
    for bad in (dict(dtype=gfd_amd.FP16), dict(dtype=gfd_amd.E4M3)):
        with pytest.raises(gfd_amd.GfdError, match="types differ"):
            gfd_amd.kv_copy_pages(cache(), cache(**bad), M, 1)
    with pytest.raises(gfd_amd.GfdError, match="scales differ"):
        gfd_amd.kv_copy_pages(cache(dtype=gfd_amd.E4M3), cache(dtype=gfd_amd.E4M3, v_scale=2.0), M, 1)


def test_a_missing_struct_is_refused():
    L = gfd_amd.lib()
    for rc in (L.gfd_kv4_append(None, rows(), None, None, None), L.gfd_kv4_append(cache4(), None, None, None, None),
               L.gfd_kv_append_axes(None, rows(), axes(), None, None), L.gfd_kv4_attention(None, call(), None, 0, None, None),
               L.gfd_kv4_attention(cache4(), None, None, 0, None, None), L.gfd_kv_read(cache(), None, None, None),
               L.gfd_kv4_read(None, read(), None, None), L.gfd_kv_copy_pages(None, cache(), M, 1, None, None, None),
               L.gfd_kv4_copy_pages(cache4(), None, M, 1, None, None, None), L.gfd_kv_fork(None, fork(), M, M, None, None),
               L.gfd_kv_fork(pool(), None, M, M, None, None), L.gfd_kv_compact(pool(), None, M, M, None, None),
               L.gfd_kv_free(None, M, 1, 1, M, M, 1, None, None)):
        assert rc != 0
    assert L.gfd_kv4_attention_workspace_bytes(cache4(), None, 0) == -1
    assert L.gfd_kv_pool_workspace_bytes(None, 0) == -1


def test_nothing_to_do_is_no_error():
    for c in (cache(), cache4()):
        gfd_amd.kv_append(c, rows(num_tokens=0))
        gfd_amd.kv_append(c, rows(num_tokens=0), axes=axes())
        gfd_amd.kv_read(c, read(num_tokens=0))
        gfd_amd.kv_read(c, read(k=None, v=None))
        gfd_amd.kv_copy_pages(c, c, None, 0)
        gfd_amd.paged_attention(c, call(batch=0))
        gfd_amd.paged_attention(c, call(max_q_len=0))
    gfd_amd.kv_fork(pool(), fork(num=0), None, 0)
    gfd_amd.kv_free(pool(), M, 10, 4, M, M, 0)


@needs_no_gpu
def test_a_failed_launch_leaves_its_text():
    big = 1 << 60
    for name, run in (("gfd_kv4_append", lambda: gfd_amd.kv_append(cache4(), rows())),
                      ("gfd_kv_append_axes", lambda: gfd_amd.kv_append(cache(), rows(), axes=axes())),
                      ("gfd_kv4_read", lambda: gfd_amd.kv_read(cache4(), read())),
                      ("gfd_kv_read", lambda: gfd_amd.kv_read(cache(), read())),
                      ("gfd_kv4_attention", lambda: gfd_amd.paged_attention(cache4(), call(), M, big)),
                      ("gfd_kv4_shared_prefix_attention",
                       lambda: gfd_amd.shared_prefix_attention(cache4(), call(), M, 16, M, big)),
                      ("gfd_kv_copy_pages", lambda: gfd_amd.kv_copy_pages(cache(), cache(), M, 1)),
                      ("gfd_kv4_copy_pages", lambda: gfd_amd.kv_copy_pages(cache4(), cache4(), M, 1)),
                      ("gfd_kv_fork", lambda: gfd_amd.kv_fork(pool(), fork(), M, big)),
                      ("gfd_kv_fork", lambda: gfd_amd.kv_fork(pool(num_pages=1 << 24), fork(num=1 << 20), M, big)),
                      ("gfd_kv_free", lambda: gfd_amd.kv_free(pool(), M, 1 << 31, 4, M, M, 1 << 20)),
                      ("gfd_kv_compact", lambda: gfd_amd.kv_compact(pool(num_pages=1 << 24), compact(rows=1 << 20), M, big))):
        with pytest.raises(gfd_amd.GfdError, match=name + ": the launch failed: "):
            run()


@pytest.mark.parametrize("batch,heads", [(1 << 24, 65535), (1 << 20, 1 << 12), (1 << 11, 65535)])
@pytest.mark.parametrize("kv", [1, 129, 1 << 30])
@pytest.mark.parametrize("prefix,max_q", [(0, 1), (1 << 30, 1), (0, 1 << 24)])
def test_products_of_the_largest_sizes_do_not_wrap(batch, heads, kv, prefix, max_q):
    c = cache4(num_heads=heads)
    k = call(batch=batch, num_tokens=1, max_q_len=max_q, max_kv_len=kv, num_q_heads=heads, table_stride=1 << 27)
    with pytest.raises(gfd_amd.GfdError, match="more work than one launch takes"):
        gfd_amd.attention_workspace_bytes(c, k, prefix)


# ------------------------------------------------------------ the definitions themselves

def test_numbers_round_to_nearest_and_ties_to_even():
    byte = np.full((1, 1), 127, np.uint8)
    x = np.zeros((1, 32))
    x[0, :16] = [0.25, 0.2500001, 0.75, 0.7499999, 1.25, 1.75, 2.5, 3.5, 5, 5.0001, 7, 100, -0.25, -0.75, -5, -6]
    got = ref4.values(ref4.packed(ref4.codes(x, byte)), byte)[0, :16]
    assert got.tolist() == [0, 0.5, 1, 0.5, 1, 2, 2, 4, 4, 6, 6, 6, 0, -1, -4, -6]


@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_a_scale_is_the_least_power_of_which_the_largest_is_at_most_seven(dtype):
    rng = np.random.default_rng(0)
    lo, hi = ref4.SCALES[dtype]
    for top in np.concatenate([2.0 ** rng.uniform(-20, 15, 200), 7 * 2.0 ** np.arange(-10, 10), [0.0, 7e-30, 6.5e4]]):
        x = np.zeros((1, 32))
        x[0, 5] = -top
        e = float(ref4.scale_bytes(x, dtype)[0, 0]) - 127
        assert lo - 127 <= e <= hi - 127
        assert top <= 7 * 2.0 ** e or e == hi - 127
        assert top > 7 * 2.0 ** (e - 1) or e == lo - 127


def test_what_a_cache_holds_is_off_by_half_a_step():
    """Relative to its group's scale: a quarter under 2, a half under 4, one above, to 7."""
    x = np.random.default_rng(1).standard_normal((300, 64)) * 40
    numbers, byte = ref4.encode(x, BF16)
    unit = np.repeat(ref4.powers(byte), 32, -1)
    a = np.abs(x) / unit
    assert (np.abs(ref4.values(numbers, byte) - x) / unit <= np.where(a < 2, 0.25, np.where(a < 4, 0.5, 1))).all()


def test_a_group_with_an_infinity_or_a_nan_is_nan():
    x = np.ones((2, 64))
    x[0, 3], x[1, 40] = np.inf, np.nan
    v = ref4.values(*ref4.encode(x, BF16))
    assert np.isnan(v).tolist() == np.isnan(np.repeat([[np.nan, 1], [1, np.nan]], 32, 1)).tolist()


def test_pages_hold_what_they_say():
    for layout in ("block", "heads", "apart", "padded"):
        p = ref4.Pages4(np.random.default_rng(2), [11, 3], 4, 3, 64, layout=layout, prefix=5)
        for b, n in ((0, 16), (1, 8)):
            for j in range(n):
                table, at = (p.prefix_table, j) if j < 5 else (p.table[b], j - 5)
                for which in ("k", "v"):
                    bits = [p.view(table[at // 4], at % 4, w) for w in (which, which + "_scales")]
                    assert (ref4.values(*bits) == getattr(p, which)[b][j]).all()


def test_the_pool_keeps_count():
    """A walk of forks, freeings and compactions: counts are the tables' entries, no page is given away twice."""
    rng = np.random.default_rng(3)
    page, n = 4, 60
    refs, table = np.zeros(n, np.int32), np.full((8, 12), -9, np.int32)
    held = {}
    for step in range(300):
        rows_free = [r for r in range(8) if r not in held]
        if rows_free and rng.random() < 0.6:
            r = int(rng.choice(rows_free))
            parent = int(rng.choice(list(held))) if held and rng.random() < 0.6 else -1
            length = int(rng.integers(0, held[parent] + 1)) if parent >= 0 else 0
            room = min(48, length + int(rng.integers(0, 12)))
            copies, err = pages_ref.fork(refs, page, table, table, [parent], [r], [length], [room])
            if err:
                assert err == 16
                pages_ref.free(refs, page, table, [r], [room])
            else:
                held[r] = max(length, room)
                assert (copies[0, 0] >= 0) == (parent >= 0 and length % page != 0)
        elif held:
            r = int(rng.choice(list(held)))
            assert pages_ref.free(refs, page, table, [r], [held.pop(r)]) == 0
        if step % 20 == 19:
            lens = [held.get(r, 0) for r in range(8)]
            refs, page_map, copies, err = pages_ref.compact(refs, page, table, table, lens)
            assert err == 0 and (np.flatnonzero(refs) == np.arange((refs != 0).sum())).all()
        named = np.concatenate([table[r, :pages_ref.pages_of(m, page)] for r, m in held.items()] + [np.zeros(0, np.int32)])
        assert (np.bincount(named.astype(int), minlength=n) == refs).all()
