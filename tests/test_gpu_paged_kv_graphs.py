"""A decode step, append and attention, captured once and replayed as the contexts grow: new keys, values and
queries, positions, slots, lengths and pages between the replays, each replay against the same step run eagerly."""
import ctypes

import numpy as np
import pytest

import gfd_amd
import paged_kv_ref as ref
from paged_kv_ref import BF16, E4M3
from test_gpu_paged_kv import up

pytestmark = pytest.mark.gpu

PAGE, HEADS, DIM, HQ = 16, 2, 128, 8


@pytest.fixture(autouse=True, scope="module")
def device():
    assert gfd_amd.device_count() > 0, "no GPU visible to libgfd_amd.so"
    assert gfd_amd.lib().gfd_set_device(0) == 0


class Steps:
    """A batch whose contexts grow by `q` tokens a step, in a cache of its own."""

    def __init__(self, rng, starts, q, cache_type, prefix):
        self.rng, self.q, self.prefix, self.batch = rng, q, prefix, len(starts)
        self.lengths = np.array(starts)
        self.own_pages = 1 + (max(starts) - prefix + 8 * q) // PAGE
        shared = -(-prefix // PAGE)
        pages = shared + self.batch * self.own_pages
        size = 1 if cache_type == E4M3 else 2
        bits, _ = ref.quantised(rng, (pages * 2 * PAGE * HEADS * DIM,), cache_type, 20.0 if cache_type == E4M3 else 1.0)
        self.words = up(bits)
        self.cache = gfd_amd.KVCache(
            k=self.words.ptr, v=self.words.ptr + PAGE * HEADS * DIM * size, page_stride=2 * PAGE * HEADS * DIM,
            slot_stride=HEADS * DIM, head_stride=DIM, num_pages=pages, page_size=PAGE, num_heads=HEADS, head_dim=DIM,
            dtype=cache_type, k_scale=1 / 32, v_scale=1 / 64)
        place = rng.permutation(pages).astype(np.int32)
        self.table = place[shared:].reshape(self.batch, -1)
        tokens, width = self.batch * q, (HQ + 2 * HEADS) * DIM
        self.tokens = tokens
        self.d = dict(rows=gfd_amd.DeviceBuffer(tokens * width * 2), positions=gfd_amd.DeviceBuffer(tokens * 4),
                      slots=gfd_amd.DeviceBuffer(tokens * 8), kv_len=gfd_amd.DeviceBuffer(self.batch * 4),
                      table=gfd_amd.DeviceBuffer(self.table.nbytes), prefix=up(place[:shared]),
                      inv_freq=up((10000.0 ** (-np.arange(DIM // 2) / (DIM // 2))).astype(np.float32)),
                      q_start=up(np.arange(0, tokens + 1, q, dtype=np.int32)), error=up(np.zeros(1, np.int32)),
                      out=gfd_amd.DeviceBuffer(tokens * HQ * DIM * 2), lse=gfd_amd.DeviceBuffer(tokens * HQ * 4))
        p = {k: b.ptr for k, b in self.d.items()}
        self.rows = gfd_amd.KVRows(
            q=p["rows"], k=p["rows"] + HQ * DIM * 2, v=p["rows"] + (HQ + HEADS) * DIM * 2, q_out=p["rows"],
            q_stride=width, k_stride=width, v_stride=width, q_out_stride=width, positions=p["positions"],
            slots=p["slots"], inv_freq=p["inv_freq"], num_tokens=tokens, num_q_heads=HQ, rotary_dim=DIM, dtype=BF16)
        self.call = gfd_amd.Attention(
            q=p["rows"], out=p["out"], lse=p["lse"], q_stride=width, out_stride=HQ * DIM, q_start=p["q_start"],
            kv_len=p["kv_len"], block_table=p["table"], table_stride=self.own_pages, scale=DIM ** -0.5,
            batch=self.batch, num_tokens=tokens, max_q_len=q, max_kv_len=prefix + self.own_pages * PAGE,
            num_q_heads=HQ, dtype=BF16)
        self.need = gfd_amd.attention_workspace_bytes(self.cache, self.call, prefix)
        self.workspace = gfd_amd.DeviceBuffer(max(self.need, 16))
        self.workspace.fill(0xFF)

    def grow(self):
        """The next step's inputs, and one sequence's pages in another order; returns the fused rows."""
        self.lengths += self.q
        fused, _ = ref.quantised(self.rng, (self.tokens, (HQ + 2 * HEADS) * DIM), BF16)
        at = (self.lengths[:, None] - self.q + np.arange(self.q)).reshape(-1)
        b = int(self.rng.integers(self.batch))
        self.table[b] = self.rng.permutation(self.table[b])
        own = at - self.prefix
        seq = np.repeat(np.arange(self.batch), self.q)
        slots = self.table[seq, own // PAGE].astype(np.int64) * PAGE + own % PAGE
        for name, x in (("positions", at.astype(np.int32)), ("slots", slots), ("kv_len", self.lengths.astype(np.int32)),
                        ("table", self.table)):
            self.d[name].upload(x)
        return fused

    def launch(self, stream=None):
        gfd_amd.kv_append(self.cache, self.rows, error_flag=self.d["error"].ptr, stream=stream)
        more = dict(workspace=self.workspace.ptr, workspace_bytes=self.need, error_flag=self.d["error"].ptr, stream=stream)
        if self.prefix:
            gfd_amd.shared_prefix_attention(self.cache, self.call, self.d["prefix"].ptr, self.prefix, **more)
        else:
            gfd_amd.paged_attention(self.cache, self.call, **more)

    def result(self):
        assert int(self.d["error"].download(4).view(np.int32)[0]) == 0
        return [self.d[x].download() for x in ("rows", "out", "lse")] + [self.words.download()]


@pytest.mark.parametrize("cache_type", [BF16, E4M3])
@pytest.mark.parametrize("starts,q,prefix", [([300, 40, 900], 1, 0), ([33, 150], 30, 0), ([600, 610, 597], 2, 590),
                                             ([140] * 20, 3, 128)], ids=str)
def test_a_captured_step_replays_over_new_lengths_pages_and_slots(starts, q, prefix, cache_type):
    hip = ctypes.CDLL(None)  # the HIP runtime that the library has loaded
    s = Steps(np.random.default_rng(110), starts, q, cache_type, prefix)
    stream, graph, exe = ctypes.c_void_p(), ctypes.c_void_p(), ctypes.c_void_p()
    assert gfd_amd.lib().gfd_stream_create(ctypes.byref(stream)) == 0
    assert hip.hipStreamBeginCapture(stream, 2) == 0
    s.launch(stream)
    assert hip.hipStreamEndCapture(stream, ctypes.byref(graph)) == 0
    assert hip.hipGraphInstantiate(ctypes.byref(exe), graph, None, None, ctypes.c_size_t(0)) == 0
    seen = []
    for _ in range(6):
        fused, before = s.grow(), s.words.download()
        s.d["rows"].upload(fused)
        s.launch()
        gfd_amd.synchronize()
        want = s.result()
        s.words.upload(before)
        s.d["rows"].upload(fused)  # the queries were turned in place
        s.d["out"].fill(0xA5)
        s.d["lse"].fill(0xA5)
        s.workspace.fill(0xFF)
        assert hip.hipGraphLaunch(exe, stream) == 0
        assert gfd_amd.lib().gfd_stream_synchronize(stream) == 0
        got = s.result()
        assert all((x == y).all() for x, y in zip(got, want))
        assert (got[3] != before).any()
        seen.append(got[1])
    assert not any((x == y).all() for i, x in enumerate(seen) for y in seen[:i])
    assert hip.hipGraphExecDestroy(exe) == 0 and hip.hipGraphDestroy(graph) == 0
    gfd_amd.lib().gfd_stream_destroy(stream)
