"""kv_append where four tokens share a workgroup (8192 and more), in every form: queries beside keys and values, in
place, pairs side by side, whole chunks apart and neither, every type and dim, slots that are skipped or outside."""
import numpy as np
import pytest

import gfd_amd
import paged_kv_ref as ref
from paged_kv_ref import BF16, E4M3, FP16
from test_gpu_paged_kv import close, up

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True, scope="module")
def device():
    assert gfd_amd.device_count() > 0, "no GPU visible to libgfd_amd.so"
    assert gfd_amd.lib().gfd_set_device(0) == 0


def rounded(y, off, dtype):
    """How far a value y, itself known to `off`, may lie from its rounding to the type."""
    if dtype == E4M3:  # a step of the lowest range is 2^-9; the division is one more 32-bit rounding
        return np.maximum(ref.U[E4M3] * np.abs(y), 2.0 ** -10) + 1.07 * off + 2 * ref.F32 * np.abs(y)
    return ref.U[dtype] * np.abs(y) + 1.01 * off + (2.0 ** -25 if dtype == FP16 else 0)


@pytest.mark.parametrize("tokens", [8192, 8193, 8195])
@pytest.mark.parametrize("d,rotary,pairs,hq,hk,dtype,cache,where,heads_first", [
    (64, 64, True, 3, 1, BF16, BF16, "apart", False),
    (64, 18, False, 3, 1, BF16, BF16, "in place", True),
    (128, 50, False, 2, 1, FP16, E4M3, "in place", False),
    (128, 128, False, 4, 2, BF16, E4M3, "apart", True),
    (128, 64, True, 1, 1, FP16, FP16, "in place", True),
    (128, 96, False, 2, 2, BF16, E4M3, "in place", False),
    (256, 256, False, 1, 1, FP16, FP16, "in place", False),
    (256, 34, False, 1, 1, BF16, BF16, "apart", True),
    (256, 64, True, 1, 1, BF16, E4M3, "none", False),
    (64, 0, False, 2, 1, FP16, E4M3, "apart", False)])
def test_every_form(tokens, d, rotary, pairs, hq, hk, dtype, cache, where, heads_first):
    rng = np.random.default_rng(tokens + d + rotary)
    page = 24
    pages = -(-tokens // page) + 2
    scales = (1 / 32, 1 / 64) if cache == E4M3 else (1.0, 1.0)
    size = 1 if cache == E4M3 else 2
    words = gfd_amd.DeviceBuffer(pages * 2 * page * hk * d * size)
    words.fill(0xA5)
    q_bits, q = ref.quantised(rng, (tokens, hq, d), dtype)
    k_bits, k = ref.quantised(rng, (tokens, hk, d), dtype)
    v_bits, v = ref.quantised(rng, (tokens, hk, d), dtype)
    fused = np.concatenate([x.reshape(tokens, -1) for x in (q_bits, k_bits, v_bits)], 1)
    width = fused.shape[1]
    slots = rng.permutation(pages * page)[:tokens].astype(np.int64)
    skipped = rng.random(tokens) < 0.1
    slots[skipped] = -1 - rng.integers(0, 5, skipped.sum())
    outside = ~skipped & (rng.random(tokens) < 0.01)
    slots[outside] = pages * page + rng.integers(0, 1 << 40, outside.sum())
    positions = rng.integers(0, 1 << 20, tokens).astype(np.int32)
    inv_freq = (10000.0 ** (-np.arange(rotary // 2) / max(rotary // 2, 1))).astype(np.float32)
    rows, q_out = up(fused), gfd_amd.DeviceBuffer(tokens * hq * d * 2 + 64)
    q_out.fill(0xA5)
    keep = [up(slots), up(positions), up(inv_freq), up(np.zeros(1, np.int32))]
    gfd_amd.kv_append(
        gfd_amd.KVCache(k=words.ptr, v=words.ptr + page * hk * d * size, page_stride=2 * page * hk * d,
                        slot_stride=d if heads_first else hk * d, head_stride=page * d if heads_first else d,
                        num_pages=pages, page_size=page, num_heads=hk, head_dim=d, dtype=cache, k_scale=scales[0],
                        v_scale=scales[1]),
        gfd_amd.KVRows(q=None if where == "none" else rows.ptr, k=rows.ptr + hq * d * 2,
                       v=rows.ptr + (hq + hk) * d * 2,
                       q_out=dict(none=None, apart=q_out.ptr).get(where, rows.ptr), q_stride=width, k_stride=width,
                       v_stride=width, q_out_stride=hq * d if where == "apart" else width, positions=keep[1].ptr,
                       slots=keep[0].ptr, inv_freq=keep[2].ptr, num_tokens=tokens, num_q_heads=hq, rotary_dim=rotary,
                       interleaved=int(pairs), dtype=dtype), error_flag=keep[3].ptr)
    gfd_amd.synchronize()
    assert int(keep[3].download(4).view(np.int32)[0]) == (gfd_amd.KV_ERR_PAGE if outside.any() else 0)
    after = words.download().view(np.uint8 if size == 1 else np.uint16)
    after = after.reshape((pages, 2, hk, page, d) if heads_first else (pages, 2, page, hk, d))
    if heads_first:
        after = after.transpose(0, 1, 3, 2, 4)
    there = ~skipped & ~outside
    kr, k_off = ref.rotate64(k, positions, inv_freq, pairs)
    at = slots[there]
    for i, (x, off) in enumerate(((kr, k_off), (v, 0 * v))):
        got = ref.decode(np.ascontiguousarray(after[at // page, i, at % page]), cache)
        y = x[there] / scales[i]
        if cache == E4M3:
            y = np.clip(y, -448, 448)
        close(got, y, rounded(y, off[there] / scales[i], cache), "keys" if i == 0 else "values")
    untouched = np.ones(pages * page, bool)
    untouched[at] = False
    flat = after.transpose(0, 2, 1, 3, 4).reshape(pages * page, -1)
    assert (flat[untouched] == (0xA5 if size == 1 else 0xA5A5)).all(), "written outside the tokens' slots"
    rows_after = rows.download().view(np.uint16)[:tokens * width].reshape(tokens, width)
    raw = q_out.download()
    assert (rows_after[:, hq * d:] == fused[:, hq * d:]).all()
    if where != "in place":
        assert (rows_after == fused).all()
    if where != "apart":
        assert (raw == 0xA5).all()
    assert (raw[tokens * hq * d * 2:] == 0xA5).all()
    if where == "none":
        return
    got = rows_after[:, :hq * d] if where == "in place" else raw[:tokens * hq * d * 2].view(np.uint16).reshape(tokens, -1)
    qr, q_off = ref.rotate64(q, positions, inv_freq, pairs)
    close(ref.decode(np.ascontiguousarray(got).reshape(tokens, hq, d), dtype), qr, rounded(qr, q_off, dtype), "q")
