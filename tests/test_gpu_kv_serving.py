"""The paged cache's operators as a serving program calls them: prompts about images appended to a 4-bit cache, samples
forked from them, each decoded for some steps, some dropped, the cache brought together, and decoding goes on.  All steps
run on one stream without waits.  Every step's attention is compared with the definition over what the cache holds, read
out of it, and the keys and values of every token with what was appended."""
import ctypes

import numpy as np
import pytest

import gfd_amd
import kv_pages_ref as model
import paged_kv4_ref as ref4
import paged_kv_ref as ref
from paged_kv_ref import BF16
from test_gpu_kv4_append import held
from test_gpu_paged_kv import close, up

pytestmark = pytest.mark.gpu

PAGE, HQ, HK, D, PAGES, WIDTH, ROWS = 8, 6, 2, 128, 90, 14, 10
SECTIONS = np.repeat(np.arange(3), [16, 24, 24]).astype(np.uint8)


@pytest.fixture(autouse=True, scope="module")
def device():
    assert gfd_amd.device_count() > 0, "no GPU visible to libgfd_amd.so"
    assert gfd_amd.lib().gfd_set_device(0) == 0


class Values:
    """Sequences' keys and values, for attention64."""

    heads = HK

    def __init__(self, k, v):
        self.k, self.v = k, v


class Server:
    def __init__(self, layers):
        self.rng = np.random.default_rng(50)
        self.refs, self.table = np.zeros(PAGES, np.int32), np.full((ROWS, WIDTH), -1, np.int32)
        self.d_refs, self.d_table = up(self.refs), up(self.table)
        self.layers = [ref4.Pages4(self.rng, [0], PAGE, HK, D, BF16, layout, spare=PAGES) for layout in layers]
        self.words = [up(p.words) for p in self.layers]
        self.caches = [ref4.handle(p, w) for p, w in zip(self.layers, self.words)]
        self.pool = gfd_amd.KVPool(refs=self.d_refs.ptr, num_pages=PAGES, page_size=PAGE)
        self.need = gfd_amd.kv_pool_workspace_bytes(self.pool, ROWS)
        self.space = gfd_amd.DeviceBuffer(self.need)
        self.error = up(np.zeros(1, np.int32))
        self.inv_freq = (10000.0 ** (-np.arange(D // 2) / (D // 2))).astype(np.float32)
        self.fixed = dict(inv=up(self.inv_freq), axis=up(SECTIONS))
        self.length = {}  # row -> tokens
        # layer -> row -> [keys, how far off, values] as appended
        self.tokens = [{} for _ in layers]
        self.keep = []
        self.stream = ctypes.c_void_p()
        assert gfd_amd.lib().gfd_stream_create(ctypes.byref(self.stream)) == 0
        self.more = dict(error_flag=self.error.ptr, stream=self.stream)

    def up(self, x):
        """Input of a call that may still run when this returns."""
        self.keep.append(up(x))
        return self.keep[-1].ptr

    def wait(self):
        assert gfd_amd.lib().gfd_stream_synchronize(self.stream) == 0
        assert int(self.error.download(4).view(np.int32)[0]) == 0
        self.keep.clear()
        n = ROWS * WIDTH
        assert (self.d_refs.download()[:4 * PAGES].view(np.int32) == self.refs).all()
        assert (self.d_table.download()[:4 * n].view(np.int32).reshape(ROWS, WIDTH) == self.table).all()

    def fork(self, parent, child, length, capacity):
        copies = gfd_amd.DeviceBuffer(16 * len(child))
        self.keep.append(copies)
        args = [self.up(np.array(x, np.int32)) for x in (parent, child, length, capacity)]
        gfd_amd.kv_fork(self.pool, gfd_amd.KVFork(
            table=self.d_table.ptr, child_table=self.d_table.ptr, table_stride=WIDTH, child_stride=WIDTH, rows=ROWS,
            child_rows=ROWS, parent=args[0], child=args[1], len=args[2], capacity=args[3], copies=copies.ptr,
            num=len(child)), self.space.ptr, self.need, **self.more)
        for c in self.caches:
            gfd_amd.kv_copy_pages(c, c, copies.ptr, len(child), **self.more)
        assert model.fork(self.refs, PAGE, self.table, self.table, parent, child, length, capacity)[1] == 0
        for p, c, n in zip(parent, child, length):
            self.length[c] = n if p >= 0 else self.length.get(c, 0)  # a row that grows: n is the room that it has
            for layer in self.tokens:
                layer[c] = [x[:n] for x in layer[p]] if p >= 0 else layer.get(c, [np.zeros((0, HK, D))] * 3)

    def drop(self, rows, room):
        gfd_amd.kv_free(self.pool, self.d_table.ptr, WIDTH, ROWS, self.up(np.array(rows, np.int32)),
                        self.up(np.array(room, np.int32)), len(rows), **self.more)
        assert model.free(self.refs, PAGE, self.table, rows, room) == 0
        for r in rows:
            del self.length[r]

    def compact(self, room):
        lens = np.array([room.get(r, 0) for r in range(ROWS)], np.int32)
        moves, count = gfd_amd.DeviceBuffer(16 * (PAGES // 2)), gfd_amd.DeviceBuffer(16)
        self.keep += [moves, count]
        gfd_amd.kv_compact(self.pool, gfd_amd.KVCompact(
            new_refs=self.d_refs.ptr, table=self.d_table.ptr, new_table=self.d_table.ptr, table_stride=WIDTH,
            new_stride=WIDTH, len=self.up(lens), rows=ROWS, copies=moves.ptr, num_copies=count.ptr), self.space.ptr,
            self.need, **self.more)
        for c in self.caches:
            gfd_amd.kv_copy_pages(c, c, moves.ptr, PAGES // 2, count=count.ptr, **self.more)
        self.refs, _, _, err = model.compact(self.refs, PAGE, self.table, self.table, lens)
        assert err == 0

    def step(self, new):
        """Rows' next tokens ({row: how many}) appended to every layer, and their attention; a check behind it."""
        rows, q_lens = list(new), list(new.values())
        seq = np.repeat(rows, q_lens)
        at = np.concatenate([np.arange(self.length[r], self.length[r] + n) for r, n in new.items()])
        for r, n in new.items():
            self.length[r] += n
        T, width = len(seq), (HQ + 2 * HK) * D
        positions = np.stack([at // 5, at % 5, at * 2 % 7]).astype(np.int32)
        slots = self.table[seq, at // PAGE].astype(np.int64) * PAGE + at % PAGE
        kv = np.array([self.length[r] for r in rows], np.int32)
        d_table, d_slots, d_pos = self.up(self.table[rows]), self.up(slots), self.up(positions)
        d_kv, d_start = self.up(kv), self.up(np.concatenate([[0], np.cumsum(q_lens)]).astype(np.int32))
        results = []
        for layer, cache in zip(self.tokens, self.caches):
            bits, x = ref.quantised(self.rng, (T, HQ + 2 * HK, D), BF16, 1.5)
            p = self.up(bits.reshape(T, -1))
            out, q_out = gfd_amd.DeviceBuffer(T * HQ * D * 2), gfd_amd.DeviceBuffer(T * HQ * D * 2)
            gfd_amd.kv_append(cache, gfd_amd.KVRows(
                q=p, k=p + HQ * D * 2, v=p + (HQ + HK) * D * 2, q_out=q_out.ptr, q_stride=width, k_stride=width,
                v_stride=width, q_out_stride=HQ * D, slots=d_slots, inv_freq=self.fixed["inv"].ptr, num_tokens=T,
                num_q_heads=HQ, rotary_dim=D, dtype=BF16), axes=gfd_amd.RotaryAxes(
                    positions=d_pos, axis=self.fixed["axis"].ptr, axis_stride=T, token_stride=1, num_axes=3), **self.more)
            call = gfd_amd.Attention(q=q_out.ptr, out=out.ptr, q_stride=HQ * D, out_stride=HQ * D, q_start=d_start,
                                     kv_len=d_kv, block_table=d_table, table_stride=WIDTH, scale=D ** -0.5,
                                     batch=len(rows), num_tokens=T, max_q_len=max(q_lens), max_kv_len=int(kv.max()),
                                     num_q_heads=HQ, dtype=BF16)
            need = gfd_amd.attention_workspace_bytes(cache, call)
            work = gfd_amd.DeviceBuffer(max(need, 16))
            gfd_amd.paged_attention(cache, call, work.ptr, need, **self.more)
            self.keep += [out, q_out, work]
            k, off = ref4.rotated(x[:, HQ:HQ + HK], positions, self.inv_freq, False, SECTIONS)
            v = x[:, HQ + HK:]
            for r in rows:
                layer[r] = [np.concatenate([old, new_[seq == r]]) for old, new_ in zip(layer[r], (k, off, v))]
            results.append((out, q_out))
        # All sequences' tokens back out of the cache: rows of (row, position).
        where = [(r, j) for r in rows for j in range(self.length[r])]
        every = np.array([self.table[r, j // PAGE] * PAGE + j % PAGE for r, j in where], np.int64)
        read = []
        for cache in self.caches:
            back = [gfd_amd.DeviceBuffer(len(every) * HK * D * 2) for _ in range(2)]
            gfd_amd.kv_read(cache, gfd_amd.KVRead(k=back[0].ptr, v=back[1].ptr, k_stride=HK * D, v_stride=HK * D,
                                                  slots=self.up(every), num_tokens=len(every), dtype=BF16), **self.more)
            read.append(back)
        table = self.table.copy()
        self.wait()
        owner = np.array([r for r, _ in where])
        for number, (layer, (out, q_out), back, pages, words) in enumerate(
                zip(self.tokens, results, read, self.layers, self.words)):
            k, v = (ref.decode(b.download().view(np.uint16), BF16).reshape(len(every), HK, D) for b in back)
            pages.words = words.download()[:len(pages.words)]
            for r in rows:
                scales = [np.stack([pages.view(table[r, j // PAGE], j % PAGE, w) for j in range(self.length[r])])
                          for w in ("k_scales", "v_scales")]
                want_k, off, want_v = layer[r]
                held(k[owner == r], scales[0], want_k, off, BF16, "layer %d keys" % number)
                held(v[owner == r], scales[1], want_v, np.zeros_like(want_v), BF16, "layer %d values" % number)
            q = ref.decode(q_out.download().view(np.uint16), BF16).reshape(T, HQ, D)
            got = ref.decode(out.download().view(np.uint16), BF16).reshape(T, HQ, D)
            values = Values([k[owner == r] for r in rows], [v[owner == r] for r in rows])
            want, _, tol, _ = ref.attention64(q, values, ref.intervals(q_lens, kv.tolist()), BF16,
                                              float(np.float32(D ** -0.5)))
            close(got, want, tol, "layer %d" % number)


def test_a_server():
    s = Server(["heads", "block"])
    # Two prompts, and one that shares the first 19 tokens of the first.
    s.fork([-1, -1], [0, 1], [0, 0], [40, 33])
    s.step({0: 37, 1: 30})
    s.fork([0], [2], [19], [30])
    s.step({2: 6, 1: 1})
    # Samples: three of the first prompt, two of the second, one of the sample.
    s.fork([0, 0, 0, 1, 1, 2], [3, 4, 5, 6, 7, 8], [37, 37, 32, 31, 31, 25], [50, 50, 50, 44, 44, 40])
    for _ in range(3):
        s.step({r: 1 for r in (3, 4, 5, 6, 7, 8)})
    # Some are dropped, the prompts too; what is left keeps what it shares.
    s.drop([0, 1, 4, 7], [40, 33, 50, 44])
    s.compact({2: 30, 3: 50, 5: 50, 6: 44, 8: 40})
    assert (np.flatnonzero(s.refs) == np.arange((s.refs != 0).sum())).all()
    s.step({3: 1, 5: 2, 6: 1, 8: 1})
    # A sample grows past its room, another begins from it, and drafts are verified.
    s.fork([-1], [3], [50], [80])
    s.fork([3], [9], [41], [60])
    s.step({3: 9, 9: 2, 2: 1})
    s.drop([2, 3, 5, 6, 8, 9], [30, 80, 50, 44, 40, 60])
    assert not s.refs.any()
    s.wait()
    gfd_amd.lib().gfd_stream_destroy(s.stream)
