"""The paged cache's operators on two streams at once, each with its own workspace: the bits of the same calls one after
the other, run eagerly and out of two graphs that replay side by side."""
import ctypes

import numpy as np
import pytest

import gfd_amd
import paged_kv4_ref as ref4
import test_gpu_paged_kv as gpu
from paged_kv_ref import BF16
from test_gpu_kv4_append import Step
from test_gpu_paged_kv import up

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True, scope="module")
def device():
    assert gfd_amd.device_count() > 0, "no GPU visible to libgfd_amd.so"
    assert gfd_amd.lib().gfd_set_device(0) == 0


class Work:
    """A batch's attention over a 4-bit cache; rows appended to another; pages of a pool forked, brought together, freed."""

    def __init__(self, seed, q_lens, kv_lens, prefix):
        rng = self.rng = np.random.default_rng(seed)
        pages = ref4.Pages4(rng, [n - prefix for n in kv_lens], 16, 2, 128, prefix=prefix)
        self.attend = gpu.Attend(rng, pages, q_lens, kv_lens, 8, BF16, prefix=prefix)
        to = ref4.Pages4(rng, [0], 16, 2, 128, spare=40)
        self.words = up(to.words)
        self.cache = ref4.handle(to, self.words)
        self.step = Step(rng, 90, 6, 2, 128, BF16, 128, 40 * 16 // 5)
        n = 3000
        self.table = np.full((16, 64), -1, np.int32)
        self.table[:8] = rng.permutation(n)[:512].reshape(8, 64)
        self.refs = np.bincount(self.table[:8].reshape(-1), minlength=n).astype(np.int32)
        lens = rng.integers(1, 1000, 8).astype(np.int32)
        i32 = lambda x: up(np.asarray(x, np.int32))
        self.d = dict(refs=i32(self.refs), table=i32(self.table), new_refs=i32(self.refs), new_table=i32(self.table),
                      parent=i32(rng.integers(0, 8, 8)), child=i32(np.arange(8, 16)), len=i32(lens), room=i32(lens + 20),
                      copies=i32(np.zeros((8, 4))), moves=i32(np.zeros((n // 2, 4))), count=i32([0]), error=i32([0]),
                      all=i32(np.full(16, 1024)))
        p = {k: b.ptr for k, b in self.d.items()}
        self.pool = gfd_amd.KVPool(refs=p["refs"], num_pages=n, page_size=16)
        self.need = gfd_amd.kv_pool_workspace_bytes(self.pool, 8)
        self.space = gfd_amd.DeviceBuffer(self.need)
        self.fork = gfd_amd.KVFork(table=p["table"], child_table=p["table"], table_stride=64, child_stride=64, rows=16,
                                   child_rows=16, parent=p["parent"], child=p["child"], len=p["len"], capacity=p["room"],
                                   copies=p["copies"], num=8)
        self.together = gfd_amd.KVCompact(new_refs=p["new_refs"], table=p["table"], new_table=p["new_table"],
                                          table_stride=64, new_stride=64, len=p["all"], rows=8, copies=p["moves"],
                                          num_copies=p["count"])
        self.p = p
        self.stream, self.graph, self.exe = ctypes.c_void_p(), ctypes.c_void_p(), ctypes.c_void_p()
        assert gfd_amd.lib().gfd_stream_create(ctypes.byref(self.stream)) == 0

    def reset(self):
        for name, x in (("refs", self.refs), ("table", self.table), ("new_refs", self.refs), ("new_table", self.table)):
            self.d[name].upload(x)
        self.attend.out.fill(0xA5)
        self.attend.lse.fill(0xA5)
        self.words.fill(0xFF)

    def launch(self):
        more = dict(error_flag=self.p["error"], stream=self.stream)
        gfd_amd.kv_fork(self.pool, self.fork, self.space.ptr, self.need, **more)
        self.attend.launch(self.stream)
        gfd_amd.kv_compact(self.pool, self.together, self.space.ptr, self.need, **more)
        gfd_amd.kv_append(self.cache, self.step.rows, **more)
        gfd_amd.kv_free(self.pool, self.p["table"], 64, 16, self.p["child"], self.p["room"], 8, **more)

    def wait(self):
        assert gfd_amd.lib().gfd_stream_synchronize(self.stream) == 0

    def result(self):
        names = ("refs", "table", "copies", "moves", "new_refs", "new_table", "count", "error")
        return [self.d[k].download() for k in names] + [self.words.download(), *self.attend.read()]


def test_two_streams_at_once(monkeypatch):
    monkeypatch.setattr(gpu, "handle", ref4.handle)
    hip = ctypes.CDLL(None)  # the HIP runtime that the library has loaded
    works = [Work(60, [1, 1, 1], [2300, 40, 900], 0), Work(61, [1, 2], [1600, 1610], 1590)]
    want = []
    for w in works:
        w.reset()
        w.launch()
        w.wait()
        want.append(w.result())
        assert not w.d["error"].download(4).any() and w.attend.errors() == 0
    same = lambda: all((a == b).all() for w, x in zip(works, want) for a, b in zip(w.result(), x))
    for _ in range(5):
        for w in works:
            w.reset()
        gfd_amd.synchronize()
        for w in works:
            w.launch()
        for w in works:
            w.wait()
        assert same()
    for w in works:
        assert hip.hipStreamBeginCapture(w.stream, 2) == 0
        w.launch()
        assert hip.hipStreamEndCapture(w.stream, ctypes.byref(w.graph)) == 0
        assert hip.hipGraphInstantiate(ctypes.byref(w.exe), w.graph, None, None, ctypes.c_size_t(0)) == 0
    for _ in range(5):
        for w in works:
            w.reset()
        gfd_amd.synchronize()
        for w in works:
            assert hip.hipGraphLaunch(w.exe, w.stream) == 0
        for w in works:
            w.wait()
        assert same()
    for w in works:
        assert hip.hipGraphExecDestroy(w.exe) == 0 and hip.hipGraphDestroy(w.graph) == 0
        gfd_amd.lib().gfd_stream_destroy(w.stream)
