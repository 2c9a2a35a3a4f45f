"""Every number of a 4-bit cache under every scale byte, bit for bit: read back as rows, and through attention where a
token sees one key, so that nothing is summed."""
import numpy as np
import pytest

import gfd_amd
import paged_kv4_ref as ref4
import paged_kv_ref as ref
import test_gpu_paged_kv as gpu
from paged_kv_ref import BF16, FP16
from test_gpu_paged_kv import up

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True, scope="module")
def device():
    assert gfd_amd.device_count() > 0, "no GPU visible to libgfd_amd.so"
    assert gfd_amd.lib().gfd_set_device(0) == 0


@pytest.fixture(autouse=True)
def four_bits(monkeypatch):
    monkeypatch.setattr(gpu, "handle", ref4.handle)


def pages_of_all(dim, dtype, order):
    """256 slots: slot s has the scale byte order[s] throughout, and all 16 numbers twice in each group, each group in an
    order of its own.  The values are what the bits stand for, NaN past the scales that an append writes."""
    rng = np.random.default_rng(dim)
    pages = ref4.Pages4(rng, [256], 16, 2, dim, dtype)
    for which in ("k", "v"):
        for s in range(256):
            codes = np.stack([np.concatenate([rng.permutation(32) % 16 for _ in range(dim // 32)]) for _ in range(2)])
            numbers = ref4.packed(codes.astype(np.uint8))
            scales = np.full((2, dim // 32), order[s], np.uint8)
            at = pages.table[0, s // 16], s % 16
            pages.view(*at, which)[:] = numbers
            pages.view(*at, which + "_scales")[:] = scales
            getattr(pages, which)[0][s] = ref4.values(numbers, scales) if order[s] <= ref4.SCALES[dtype][1] else np.nan
    return pages


def compare(got, want, dtype):
    """Exact in bf16, as its small numbers hold them all; below 2^-14 in fp16 the nearest multiple of 2^-24, ties to even."""
    assert (np.isnan(got) == np.isnan(want)).all()
    there = ~np.isnan(want)
    assert (got[there] == ref.decode(ref.encode(want[there], dtype), dtype)).all()
    assert dtype == FP16 or (got[there] == want[there]).all()


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_rows_read_back(dim, dtype):
    pages = pages_of_all(dim, dtype, np.arange(256))
    words = up(pages.words)
    slots = up(pages.table[0][np.arange(256) // 16].astype(np.int64) * 16 + np.arange(256) % 16)
    out = [gfd_amd.DeviceBuffer(256 * 2 * dim * 2) for _ in range(2)]
    error = up(np.zeros(1, np.int32))
    gfd_amd.kv_read(ref4.handle(pages, words), gfd_amd.KVRead(
        k=out[0].ptr, v=out[1].ptr, k_stride=2 * dim, v_stride=2 * dim, slots=slots.ptr, num_tokens=256, dtype=dtype),
        error_flag=error.ptr)
    gfd_amd.synchronize()
    assert int(error.download(4).view(np.int32)[0]) == 0
    for b, want in zip(out, (pages.k[0], pages.v[0])):
        bits = b.download(256 * 2 * dim * 2).view(np.uint16).reshape(256, 2, dim)
        compare(ref.decode(np.ascontiguousarray(bits), dtype), want, dtype)


@pytest.mark.parametrize("form", ["few rows", "few rows, a wave each", "many rows"])
@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_values_through_attention(form, dim, dtype):
    """A weight of one times a value is the value, next to keys of every other byte that are not seen."""
    rng = np.random.default_rng(3)
    pages = pages_of_all(dim, dtype, rng.permutation(256).astype(np.uint8))
    for s in range(256):  # ordinary scores
        pages.view(pages.table[0, s // 16], s % 16, "k_scales")[:] = 127
    seen = np.arange(256)
    if form == "many rows":
        q_lens, kv_lens = [256], [256]
    else:
        q_lens, kv_lens = [1] * 256, seen + 1
        pages.table = np.repeat(pages.table, 256, 0)
        if form != "few rows":  # contexts of at most 128 keys: the second half of the sequences have the second half of the pages
            kv_lens = seen % 128 + 1
            pages.table[128:, :8] = pages.table[128:, 8:]
    a = gpu.Attend(rng, pages, q_lens, list(kv_lens), 4, dtype, window=1)
    out, lse = a.run()
    assert a.errors() == 0 and np.isfinite(lse).all()
    compare(out, np.repeat(pages.v[0][seen], 2, 1), dtype)
