"""Reads of more units than one round of workgroups takes, past 2^32 elements of rows, and of slots outside the cache; appended rows
past 2^32 elements."""
import numpy as np
import pytest

import gfd_amd
import paged_kv4_ref as ref4
import paged_kv_ref as ref
import test_gpu_paged_kv as gpu
from paged_kv_ref import BF16, E4M3
from test_gpu_paged_kv import up

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True, scope="module")
def device():
    assert gfd_amd.device_count() > 0, "no GPU visible to libgfd_amd.so"
    assert gfd_amd.lib().gfd_set_device(0) == 0


@pytest.mark.parametrize("cache", [BF16, 3])
def test_more_rows_than_a_grid_takes_at_once(cache):
    """2^20 workgroups of 512 chunks of 8 values; the rows from the end of their first round on."""
    rng = np.random.default_rng(1)
    heads, d, page = 64, 64, 16
    tokens = (1 << 20) + 1500  # 2^20 of heads * d / 8 = 512 chunks are one round
    pages = (ref4.Pages4(rng, [page], page, heads, d, spare=0) if cache == 3 else
             ref.Pages(rng, [page], page, heads, d, cache, "block"))
    words, error = up(pages.words), up(np.zeros(1, np.int32))
    at = rng.integers(0, page, tokens)
    slots = up(pages.table[0, 0].astype(np.int64) * page + at)
    rows = gfd_amd.DeviceBuffer(tokens * heads * d * 2)
    tail = 1504  # rows
    first = (tokens - tail) * heads * d * 2
    gfd_amd.kv_read((ref4 if cache == 3 else gpu).handle(pages, words), gfd_amd.KVRead(
        k=rows.ptr, k_stride=heads * d, slots=slots.ptr, num_tokens=tokens, dtype=BF16), error_flag=error.ptr)
    gfd_amd.synchronize()
    assert not error.download(4).any()
    for offset, some in ((0, at[:tail]), (first, at[-tail:])):
        got = ref.decode(rows.download(tail * heads * d * 2, offset).view(np.uint16), BF16).reshape(tail, heads, d)
        assert (got == pages.k[0][some]).all()


@pytest.mark.parametrize("cache", [BF16, E4M3, 3])
@pytest.mark.parametrize("bad", [17 * 5, 17 * 5 + 1, 1 << 31, 1 << 40, (1 << 63) - 1])
def test_a_slot_outside_the_cache_is_reported_and_its_row_left(cache, bad):
    rng = np.random.default_rng(2)
    hk, d, page, tokens = 2, 64, 5, 12
    pages = (ref4.Pages4(rng, [tokens], page, hk, d, spare=14) if cache == 3 else
             ref.Pages(rng, [tokens], page, hk, d, cache, "block", k_scale=1 / 32, v_scale=1 / 64,
                       spread=20.0 if cache == E4M3 else 1.0))
    bad += (pages.num_pages - 17) * page if bad < 1 << 20 else 0  # the first two behind the last page
    words, error = up(pages.words), up(np.zeros(1, np.int32))
    slots = pages.table[0, np.arange(tokens) // page].astype(np.int64) * page + np.arange(tokens) % page
    slots[7], slots[9] = bad, -(1 << 62)
    keep = up(slots)
    bufs = [gfd_amd.DeviceBuffer(tokens * hk * d * 2) for _ in range(2)]
    for b in bufs:
        b.fill(0xA5)
    gfd_amd.kv_read((ref4 if cache == 3 else gpu).handle(pages, words), gfd_amd.KVRead(
        k=bufs[0].ptr, v=bufs[1].ptr, k_stride=hk * d, v_stride=hk * d, slots=keep.ptr, num_tokens=tokens, dtype=BF16),
        error_flag=error.ptr)
    gfd_amd.synchronize()
    assert int(error.download(4).view(np.int32)[0]) == gfd_amd.KV_ERR_PAGE
    for b, want in zip(bufs, (pages.k[0], pages.v[0])):
        bits = b.download().view(np.uint16).reshape(tokens, hk, d)
        assert (bits[[7, 9]] == 0xA5A5).all()
        live = np.setdiff1d(np.arange(tokens), [7, 9])
        off = np.abs(ref.decode(bits[live], BF16) - want[live])
        assert (off <= (ref.U[BF16] * 1.01 * np.abs(want[live]) if cache == E4M3 else 0)).all()


def test_appended_rows_past_32_bits_of_elements():
    """Rows of a stride of 2^27 + 8 elements, the last ones past 2^32: the same bits as close together."""
    rng = np.random.default_rng(3)
    hq, hk, d, page, tokens = 4, 2, 64, 8, 35
    width, stride = (hq + 2 * hk) * d, (1 << 27) + 8
    fused, _ = ref.quantised(rng, (tokens, width), BF16)
    far = gfd_amd.DeviceBuffer((tokens - 1) * stride * 2 + width * 2)
    near = up(fused)
    for t in range(tokens):
        far.upload(fused[t], t * stride * 2)
    d_positions, d_slots = up(np.arange(tokens, dtype=np.int32)), up(rng.permutation(tokens).astype(np.int64))
    inv, error = up((10000.0 ** (-np.arange(d // 2) / (d // 2))).astype(np.float32)), up(np.zeros(1, np.int32))
    results = []
    for rows, step in ((near, width), (far, stride)):
        pages = ref4.Pages4(np.random.default_rng(4), [0], page, hk, d, spare=5)
        words = up(pages.words)
        gfd_amd.kv_append(ref4.handle(pages, words), gfd_amd.KVRows(
            q=rows.ptr, k=rows.ptr + hq * d * 2, v=rows.ptr + (hq + hk) * d * 2, q_out=rows.ptr, q_stride=step, k_stride=step,
            v_stride=step, q_out_stride=step, positions=d_positions.ptr, slots=d_slots.ptr, inv_freq=inv.ptr,
            num_tokens=tokens, num_q_heads=hq, rotary_dim=d, dtype=BF16), error_flag=error.ptr)
        gfd_amd.synchronize()
        turned = [rows.download(hq * d * 2, t * step * 2) for t in range(tokens)]
        results.append(np.concatenate([words.download(), *turned]))
    assert not error.download(4).any() and (results[0] == results[1]).all()
