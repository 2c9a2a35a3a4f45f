"""What a call of the paged cache's operators reports is its own: an earlier call's error is not."""
import ctypes

import numpy as np
import pytest

import gfd_amd
import paged_kv_ref as ref
from paged_kv_ref import BF16
from test_gpu_paged_kv import Attend, close, up

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True, scope="module")
def device():
    assert gfd_amd.device_count() > 0, "no GPU visible to libgfd_amd.so"
    assert gfd_amd.lib().gfd_set_device(0) == 0


@pytest.fixture
def fail_elsewhere():
    """Some other HIP call of the program fails, on the host, and its error is left to be asked for."""
    hip = ctypes.CDLL(None)

    def fail():
        assert hip.hipSetDevice(1 << 20) != 0

    yield fail
    assert hip.hipGetLastError() != 0  # the program's own, still there



@pytest.mark.parametrize("q,kv,prefix", [([1], [3000], 0), ([70], [150], 0), ([1] * 9, [610] * 9, 600)], ids=str)
def test_attention_after_a_failed_call(q, kv, prefix, fail_elsewhere):
    rng = np.random.default_rng(95)
    pages = ref.Pages(rng, [n - prefix for n in kv], 16, 2, 128, BF16, prefix=prefix)
    a = Attend(rng, pages, q, kv, 8, BF16, prefix=prefix)
    want, want_lse = a.run()
    a.out.fill(0xA5)
    a.lse.fill(0xA5)
    fail_elsewhere()
    a.launch()
    gfd_amd.synchronize()
    out, lse = a.read()
    assert (out == want).all() and (lse == want_lse).all()


def test_append_after_a_failed_call(fail_elsewhere):
    rng = np.random.default_rng(96)
    pages = ref.Pages(rng, [0], 16, 2, 128, BF16, spare=2)
    words = up(pages.words)
    rows, slots = up(np.full((3, 2, 128), 0x3F80, np.uint16)), up(np.array([3, 7, 31], np.int64))
    k = dict(page_stride=pages.strides[0], slot_stride=pages.strides[1], head_stride=pages.strides[2])
    cache = gfd_amd.KVCache(k=words.ptr, v=words.ptr + pages.v_offset * 2, num_pages=pages.num_pages, page_size=16,
                            num_heads=2, head_dim=128, dtype=BF16, **k)
    fail_elsewhere()
    gfd_amd.kv_append(cache, gfd_amd.KVRows(k=rows.ptr, v=rows.ptr, k_stride=256, v_stride=256, slots=slots.ptr,
                                            num_tokens=3, dtype=BF16))
    gfd_amd.synchronize()
    assert (words.download().view(np.uint16) == 0x3F80).sum() == 3 * 2 * 256


def test_the_largest_batch_is_one_launch():
    """2^24 - 24 workgroups of 256 threads, all but a few of sequences without tokens."""
    rng = np.random.default_rng(97)
    batch, kv = (1 << 21) - 3, 200
    pages = ref.Pages(rng, [kv], 256, 8, 64, BF16, spare=0)
    pages.table = np.zeros((batch, 1), np.int32)
    a = Attend(rng, pages, [1] * 3, [kv] * 3, 8, BF16)
    starts = np.zeros(batch + 1, np.int32)
    lengths = np.zeros(batch, np.int32)
    for i, b in enumerate((0, batch // 2, batch - 1)):  # the sequences with a token
        starts[b + 1:] = i + 1
        lengths[b] = kv
    keep = up(starts), up(lengths)
    a.call.q_start, a.call.kv_len, a.call.batch = keep[0].ptr, keep[1].ptr, batch
    assert gfd_amd.attention_workspace_bytes(a.cache, a.call) == 0
    want, want_lse, tol, tol_lse = ref.attention64(a.q, pages, [(0, kv - 1, 0, kv)] * 3, BF16, float(np.float32(a.scale)))
    out, lse = a.run()
    close(out, want, tol, "out")
    close(lse, want_lse, tol_lse, "lse")
    a.call.batch = batch + 1
    with pytest.raises(gfd_amd.GfdError, match="more work than one launch takes"):
        a.launch()
