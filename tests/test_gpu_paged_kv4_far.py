"""A 4-bit cache whose pages lie far apart, past 32 bits of bytes: the same bits as of one in a few kilobytes."""
import numpy as np
import pytest

import gfd_amd
import paged_kv4_ref as ref4
import paged_kv_ref as ref
import test_gpu_paged_kv as gpu
from paged_kv_ref import BF16
from test_gpu_kv4_append import Step
from test_gpu_paged_kv import up

pytestmark = pytest.mark.gpu

STRIDE = (1 << 30) + (1 << 20) + 16  # 23 pages: 25 GB


@pytest.fixture(autouse=True, scope="module")
def device():
    assert gfd_amd.device_count() > 0, "no GPU visible to libgfd_amd.so"
    assert gfd_amd.lib().gfd_set_device(0) == 0


@pytest.fixture(scope="module")
def far():
    return gfd_amd.DeviceBuffer(22 * STRIDE + (1 << 20))


def spread(near, far):
    """The descriptor of the same pages, far apart."""
    first = min(near.k, near.v, near.k_scales, near.v_scales)
    names = ("k", "v", "k_scales", "v_scales")
    sizes = {n: getattr(near, n) for n in ("slot_stride", "head_stride", "num_pages", "page_size", "num_heads", "head_dim")}
    return gfd_amd.KV4Cache(**{n: far.ptr + getattr(near, n) - first for n in names}, page_stride=STRIDE,
                            scale_page_stride=STRIDE, **sizes)


def copies(n):
    return up(np.array([(p, p, 16, 0) for p in range(n)], np.int32))


@pytest.mark.parametrize("q_lens,kv_lens,prefix", [([1, 1], [150, 70], 0), ([60], [200], 0), ([1, 2], [120, 130], 100),
                                                   ([40, 9], [150, 140], 100)], ids=str)
def test_attention_and_copies(q_lens, kv_lens, prefix, far, monkeypatch):
    monkeypatch.setattr(gpu, "handle", ref4.handle)
    rng = np.random.default_rng(1)
    own = sum(-(-(n - prefix) // 16) for n in kv_lens) + -(-prefix // 16)
    pages = ref4.Pages4(rng, [n - prefix for n in kv_lens], 16, 2, 128, layout="heads", prefix=prefix, spare=23 - own)
    a = gpu.Attend(rng, pages, q_lens, kv_lens, 8, BF16, prefix=prefix)
    want, want_lse = a.run()
    near, a.cache = a.cache, spread(a.cache, far)
    gfd_amd.kv_copy_pages(a.cache, near, copies(23).ptr, 23, error_flag=a.error.ptr)
    out, lse = a.run()
    assert a.errors() == 0
    assert (out == want).all() and (lse == want_lse).all()
    # And back.
    a.words.fill(0)
    gfd_amd.kv_copy_pages(near, a.cache, copies(23).ptr, 23, error_flag=a.error.ptr)
    a.cache = near
    out, lse = a.run()
    assert a.errors() == 0 and (out == want).all() and (lse == want_lse).all()


def test_append_and_read(far):
    rng = np.random.default_rng(2)
    pages = ref4.Pages4(rng, [0], 16, 2, 128, layout="block", spare=23)
    words = up(pages.words)
    near = ref4.handle(pages, words)
    s = Step(rng, 70, 6, 2, 128, BF16, 128, 23 * 16 // 5)
    got = []
    for cache in (near, spread(near, far)):
        s.append(cache)
        k, v = (gfd_amd.DeviceBuffer(70 * 2 * 128 * 2) for _ in range(2))
        k.fill(0)
        v.fill(0)
        gfd_amd.kv_read(cache, gfd_amd.KVRead(k=k.ptr, v=v.ptr, k_stride=256, v_stride=256, slots=s.buffers["slots"].ptr,
                                              num_tokens=70, dtype=BF16), error_flag=s.buffers["error"].ptr)
        gfd_amd.synchronize()
        assert s.errors() == 0
        got.append(np.concatenate([x.download() for x in (k, v, s.q_out)]))
    assert s.slots.max() // 16 * STRIDE > 1 << 32 and (got[0] == got[1]).all()
    assert np.isfinite(ref.decode(got[0][:70 * 256 * 4].view(np.uint16), BF16)).all()
