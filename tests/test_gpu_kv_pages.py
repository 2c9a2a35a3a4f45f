"""Pages copied, forked, freed and brought together on the GPU against the pool in plain Python (kv_pages_ref)."""
import ctypes

import numpy as np
import pytest

import gfd_amd
import kv_pages_ref as model
import paged_kv4_ref as ref4
import paged_kv_ref as ref
import test_gpu_paged_kv as gpu
from paged_kv_ref import BF16, E4M3, FP16
from test_gpu_paged_kv import up

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True, scope="module")
def device():
    assert gfd_amd.device_count() > 0, "no GPU visible to libgfd_amd.so"
    assert gfd_amd.lib().gfd_set_device(0) == 0


def ints(buffer, shape):
    n = int(np.prod(shape))
    return buffer.download(4 * n).view(np.int32).reshape(shape).copy() if n else np.zeros(shape, np.int32)


class Pool:
    """Counts and a table on the device, and the same in plain Python."""

    def __init__(self, refs, page, table, room=64):
        self.refs, self.page, self.table, self.room = refs.astype(np.int32), page, table.astype(np.int32), room
        self.d_refs, self.d_table = up(self.refs), up(self.table)
        self.pool = gfd_amd.KVPool(refs=self.d_refs.ptr, num_pages=len(refs), page_size=page)
        self.need = gfd_amd.kv_pool_workspace_bytes(self.pool, room)
        self.workspace = gfd_amd.DeviceBuffer(self.need + 64)
        self.workspace.fill(0xFF)
        self.error = up(np.zeros(1, np.int32))

    def errors(self):
        gfd_amd.synchronize()
        got = int(self.error.download(4).view(np.int32)[0])
        self.error.fill(0)
        assert (self.workspace.download(64, self.need) == 0xFF).all(), "written past the workspace"
        return got

    def more(self, stream=None):
        return dict(error_flag=self.error.ptr, stream=stream)

    def fork(self, parent, child, length, capacity=None, kids=None):
        """kids: another table for the children; returns (copies, errors) after comparing everything."""
        num = len(child)
        child_table = self.table if kids is None else kids
        d_kids = self.d_table if kids is None else up(kids)
        d = [up(np.array(x, np.int32)) for x in (parent, child, length)]
        d_room = None if capacity is None else up(np.array(capacity, np.int32))
        copies = gfd_amd.DeviceBuffer(16 * num + 64)
        copies.fill(0xA5)
        call = gfd_amd.KVFork(table=self.d_table.ptr, child_table=d_kids.ptr, table_stride=self.table.shape[1],
                              child_stride=child_table.shape[1], rows=len(self.table), child_rows=len(child_table),
                              parent=d[0].ptr, child=d[1].ptr, len=d[2].ptr,
                              capacity=None if capacity is None else d_room.ptr, copies=copies.ptr, num=num)
        gfd_amd.kv_fork(self.pool, call, self.workspace.ptr, self.need, **self.more())
        got_errors = self.errors()
        want, errors = model.fork(self.refs, self.page, self.table, child_table, parent, child, length, capacity)
        assert got_errors == errors
        assert (ints(copies, (num, 4)) == want).all()
        assert (copies.download(64, 16 * num) == 0xA5).all(), "written past the copies"
        assert (ints(d_kids, child_table.shape) == child_table).all()
        assert (ints(self.d_refs, self.refs.shape) == self.refs).all()
        return want, errors

    def free(self, row, length, table=None):
        table = self.table if table is None else table
        d = [up(np.array(x, np.int32)) for x in (row, length)]
        d_table = up(table)
        gfd_amd.kv_free(self.pool, d_table.ptr, table.shape[1], len(table), d[0].ptr, d[1].ptr, len(row), **self.more())
        got = self.errors()
        assert got == model.free(self.refs, self.page, table, row, length)
        assert (ints(self.d_refs, self.refs.shape) == self.refs).all()
        return got

    def compact(self, length, in_place=True, with_map=True, width=None):
        n, half = len(self.refs), len(self.refs) // 2
        new = self.table.copy() if in_place else np.full((len(self.table), width or self.table.shape[1]), -77, np.int32)
        d_new, d_refs = (self.d_table, self.d_refs) if in_place else (up(new), up(np.full(n, -78, np.int32)))
        d_len, page_map = up(np.array(length, np.int32)), up(np.full(n, -79, np.int32))
        copies, count = gfd_amd.DeviceBuffer(16 * half + 64), up(np.full(1, -1, np.int32))
        copies.fill(0xA5)
        call = gfd_amd.KVCompact(new_refs=d_refs.ptr, table=self.d_table.ptr, new_table=d_new.ptr,
                                 table_stride=self.table.shape[1], new_stride=new.shape[1], len=d_len.ptr,
                                 rows=len(self.table), page_map=page_map.ptr if with_map else None, copies=copies.ptr,
                                 num_copies=count.ptr)
        gfd_amd.kv_compact(self.pool, call, self.workspace.ptr, self.need, **self.more())
        got_errors = self.errors()
        refs, where, moves, errors = model.compact(self.refs, self.page, self.table, new, length)
        assert got_errors == errors
        assert int(ints(count, (1,))[0]) == len(moves)
        assert (ints(copies, (len(moves), 4)) == moves).all()
        assert (copies.download()[16 * len(moves):] == 0xA5).all(), "written past the copies"
        assert (ints(d_new, new.shape) == new).all()
        assert (ints(d_refs, refs.shape) == refs).all()
        assert (ints(page_map, (n,)) == (where if with_map else -79)).all()
        if not in_place:
            assert (ints(self.d_refs, self.refs.shape) == self.refs).all()
            assert (ints(self.d_table, self.table.shape) == self.table).all()
        else:
            self.refs, self.table = refs, new
        return moves, errors


def family(seed, pages, page, rows, width, lengths):
    """A pool whose rows have pages of their own, anywhere."""
    rng = np.random.default_rng(seed)
    table, refs = np.full((rows, width), -5, np.int32), np.zeros(pages, np.int32)
    place, used = rng.permutation(pages), 0
    for r, n in enumerate(lengths):
        k = -(-n // page)
        table[r, :k] = place[used:used + k]
        refs[place[used:used + k]] = 1
        used += k
    return Pool(refs, page, table)


# ------------------------------------------------------------ fork and free

@pytest.mark.parametrize("page", [1, 5, 16, 64])
@pytest.mark.parametrize("pages", [40, 1024, 1025, 5000])
def test_sequences_that_go_on_from_others(page, pages):
    p = family(1, pages, page, 12, 30, [7 * page, 3 * page + page // 2, 1])
    n = 3 * page + page // 2
    p.fork([0, 1, 1, 2, 0], [4, 5, 6, 7, 8], [7 * page, n, n, 1, 2 * page + (page > 1)],
           [7 * page + 1, n, n + 4 * page, 1, 0])
    p.free([4, 5, 0], [7 * page + 1, n, 7 * page])
    p.fork([6, -1], [9, 10], [n + page, 0], [n + page, 5 * page])
    p.free([6, 7, 8, 9, 10], [n + 4 * page, 1, 2 * page + (page > 1), n + page, 5 * page])
    p.free([1, 2], [n, 1])
    assert not p.refs.any()


def test_no_capacity_is_the_length():
    p = family(2, 50, 16, 6, 10, [100, 40])
    p.fork([0, 1, -1, 0], [2, 3, 4, 5], [100, 32, 33, 0])


def test_rows_that_grow_and_begin():
    p = family(3, 60, 16, 4, 12, [100, 40])
    p.fork([-1, -1, -1, -1], [0, 1, 2, 3], [100, 40, 0, 0], [150, 48, 17, 0])
    assert p.refs.sum() == 10 + 3 + 2


def test_a_row_without_tokens_and_items_that_are_skipped():
    p = family(4, 60, 16, 6, 12, [100])
    p.fork([0, 0, 3, -1], [-1, 2, -7, -1], [100, 0, 5, 9], [190, 0, 50, 20])
    assert p.refs.sum() == 7


@pytest.mark.parametrize("bad", [dict(parent=12), dict(parent=-2), dict(child=12), dict(child=0x7FFFFFFF),
                                 dict(length=-1), dict(length=16 * 13), dict(capacity=16 * 12 + 1),
                                 dict(capacity=0x7FFFFFFF), dict(length=0x7FFFFFFF)], ids=str)
def test_an_item_of_no_row_is_skipped_and_takes_no_page(bad):
    p = family(5, 60, 16, 12, 12, [100, 40])
    one = dict(parent=0, child=5, length=50, capacity=60)
    one.update(bad)
    _, errors = p.fork([1, one["parent"], 0], [4, one["child"], 6], [40, one["length"], 99],
                       [50, one["capacity"], 120])
    assert errors == gfd_amd.KV_ERR_ROW


@pytest.mark.parametrize("pages", [7, 8, 10, 11, 12, 13])
def test_a_pool_that_runs_out(pages):
    """Seven pages are held, six are asked for: what is missing is -1, in the items' order."""
    p = family(6, 13, 16, 8, 12, [100])
    if pages < 13:
        p.refs[np.flatnonzero(p.refs == 0)[:13 - pages]] = 3
        p.d_refs.upload(p.refs)
    _, errors = p.fork([0, 0, -1, 0], [1, 2, 3, 4], [33, 20, 0, 16], [33, 48, 32, 17])
    assert errors == (gfd_amd.KV_ERR_FULL if pages < 13 else 0)
    p.free([1, 2, 3, 4], [33, 48, 32, 17])


@pytest.mark.parametrize("held", [0, 3, 4096])
def test_needs_of_more_than_all_pages_leave_the_rest_without(held):
    p = Pool(np.r_[np.ones(held, int), np.zeros(70, int)], 1, np.full((5, 100), -3))
    _, errors = p.fork([-1] * 4, [0, 1, 2, 3], [0] * 4, [30, 60, 100, 1])
    assert errors == gfd_amd.KV_ERR_FULL


def test_a_bad_page_of_a_parent_is_passed_on_as_none():
    p = family(7, 60, 16, 8, 12, [100, 40])
    for at, bad in ((1, 60), (2, -1), (3, -0x80000000)):
        p.table[0, at] = bad
    p.table[1, 2] = 1 << 20
    p.d_table.upload(p.table)
    copies, errors = p.fork([0, 1], [3, 4], [100, 40], [100, 60])
    assert errors == gfd_amd.KV_ERR_PAGE and (copies[1] == model.NONE).all() and copies[0, 0] >= 0


def test_children_in_another_table():
    p = family(8, 200, 16, 3, 12, [100, 40, 180])
    kids = np.full((9, 20), -6, np.int32)
    p.fork([2, 0, 0, 1], [8, 0, 3, 4], [170, 99, 96, 5], [310, 0, 97, 80], kids=kids)
    assert p.free([8, 0, 3, 4], [310, 99, 97, 80], kids) == 0
    assert p.refs.sum() == 7 + 3 + 12


@pytest.mark.parametrize("num,pages", [(700, 3000), (2500, 20000), (60, 65536), (60, 65537), (3000, 90000), (1025, 400000)])
def test_many_items_over_many_chunks(num, pages):
    """More items than places in the search's first step, pages of several workgroups."""
    rng = np.random.default_rng(9)
    page, width = 4, 40
    lens = rng.integers(1, 150, 20)
    table, refs = np.full((20, width), -5, np.int32), np.zeros(pages, np.int32)
    place, used = rng.permutation(pages), 0
    for r, n in enumerate(lens):
        k = -(-n // page)
        table[r, :k] = place[used:used + k]
        refs[place[used:used + k]] = 1
        used += k
    p = Pool(refs, page, table, room=num)
    parent = rng.integers(-1, 20, num)
    length = np.where(parent < 0, 0, [rng.integers(0, lens[r] + 1) for r in parent])
    capacity = length + rng.integers(0, 9, num)
    kids = np.full((num + 5, width), -6, np.int32)
    child = rng.permutation(num + 5)[:num]
    _, errors = p.fork(parent, child, length, capacity, kids=kids)
    assert errors in (0, gfd_amd.KV_ERR_FULL)
    p.free(child, capacity, kids)
    assert (p.refs == refs).all()


def test_a_page_freed_too_often_stays_free():
    p = family(10, 60, 16, 4, 12, [100])
    assert p.free([0, 0, 0], [40, 100, 16]) == gfd_amd.KV_ERR_REFS
    assert not p.refs.any()


def test_freeing_of_rows_and_entries_that_are_none():
    p = family(11, 60, 16, 4, 12, [100])
    p.table[0, 1], p.table[0, 2] = -1, -9
    assert p.free([-1, 0, -5], [50, 100, -3]) == 0
    assert p.free([4, 0, 0], [1, -1, 16 * 12 + 1]) == gfd_amd.KV_ERR_ROW
    p.table[0, 3] = 60
    assert p.free([0], [64]) == gfd_amd.KV_ERR_PAGE | gfd_amd.KV_ERR_REFS


def test_long_rows_of_few_sequences():
    p = family(12, 50000, 1, 4, 20000, [19999, 1])
    p.fork([0, -1], [2, 1], [19999, 1], [20000, 9000])
    p.free([2, 0], [20000, 19999])


# ------------------------------------------------------------ compact

@pytest.mark.parametrize("pages,share", [(1, 1.0), (1, 0.0), (2, 0.5), (7, 0.6), (64, 0.4), (1023, 0.3), (1024, 0.5),
                                         (1025, 0.9), (5000, 0.02), (5000, 0.5), (20000, 0.7),
                                         (65536, 0.4), (65537, 0.4), (300000, 0.6)])
@pytest.mark.parametrize("in_place", [True, False])
def test_pages_brought_together(pages, share, in_place):
    rng = np.random.default_rng(pages)
    refs = np.where(rng.random(pages) < share, rng.integers(1, 5, pages), 0)
    live = np.flatnonzero(refs)
    width = max(1, min(64, len(live)))
    table = np.full((6, width + 3), -4)
    lens = []
    for r in range(6):
        n = int(rng.integers(0, width + 1)) if len(live) else 0
        table[r, :n] = rng.choice(live, n) if n else []
        lens.append(max(0, n * 8 - int(rng.integers(0, 8))) if n else 0)
    p = Pool(refs, 8, table)
    p.compact(lens, in_place, with_map=pages % 2 == 0, width=width + 9)
    if in_place:
        moves, _ = p.compact(lens, in_place)
        assert len(moves) == 0


def test_used_pages_at_the_front_or_the_back():
    for refs in (np.r_[np.ones(3000), np.zeros(3000)], np.r_[np.zeros(3000), np.ones(3000)],
                 np.r_[np.ones(1024), np.zeros(1024), np.ones(1024)], np.zeros(2048), np.ones(2048)):
        p = Pool(refs, 16, np.zeros((1, 4)))
        p.compact([0], False)


def test_entries_of_free_pages_and_of_none():
    p = family(13, 60, 16, 4, 12, [100, 60, 30])
    p.free([1], [60])
    p.table[0, 2], p.table[2, 0] = -1, 1 << 30
    p.d_table.upload(p.table)
    _, errors = p.compact([100, 60, 30, 0], False)  # row 1's pages are free
    assert errors == gfd_amd.KV_ERR_PAGE
    _, errors = p.compact([-1, 0, 0, 16 * 12 + 1], False)
    assert errors == gfd_amd.KV_ERR_ROW


def test_no_rows():
    refs = np.zeros(100)
    refs[90:] = 2
    p = Pool(refs, 16, np.zeros((0, 4)))
    p.compact([], False)


# ------------------------------------------------------------ copies

def filled(rng, pages, page, heads, d, cache, layout):
    x = (ref4.Pages4(rng, [0], page, heads, d, BF16, layout, spare=pages) if cache == 3 else
         ref.Pages(rng, [0], page, heads, d, cache, layout, k_scale=0.5, v_scale=0.25, spare=pages))
    x.words = rng.integers(0, 1 << 16, len(x.words)).astype(x.words.dtype)
    return x


def parts(x, page, slot):
    """The views of what a slot has."""
    if isinstance(x, ref4.Pages4):
        return [x.view(page, slot, w) for w in ("k", "v", "k_scales", "v_scales")]
    return [x.view(page, slot), x.view(page, slot, x.v_offset)]


@pytest.mark.parametrize("cache", [BF16, FP16, E4M3, 3])
@pytest.mark.parametrize("d,heads,page", [(64, 1, 1), (64, 3, 5), (128, 8, 16), (256, 2, 24), (128, 5, 70)])
@pytest.mark.parametrize("from_,to", [("block", "block"), ("heads", "block"), ("apart", "heads"), ("padded", "apart"),
                                      ("block", "padded")])
def test_pages_copied_between_caches(cache, d, heads, page, from_, to):
    rng = np.random.default_rng(30)
    src, dst = (filled(rng, n, page, heads, d, cache, layout) for n, layout in ((9, from_), (12, to)))
    a, b = rng.permutation(9)[:7], rng.permutation(12)[:7]
    copies = np.stack([a, b, rng.integers(0, page + 1, 7), np.full(7, 99)], 1).astype(np.int32)
    copies[2, 2], copies[3, 0], copies[4, 1] = page, -1, -1
    d_src, d_dst, d_copies, error = up(src.words), up(dst.words), up(copies), up(np.zeros(1, np.int32))
    handle = ref4.handle if cache == 3 else gpu.handle
    for count in (None, 3, 0, 100, -2):
        d_dst.upload(dst.words)
        d_count = None if count is None else up(np.array([count], np.int32))
        gfd_amd.kv_copy_pages(handle(dst, d_dst), handle(src, d_src), d_copies.ptr, 7,
                              count=None if count is None else d_count.ptr, error_flag=error.ptr)
        gfd_amd.synchronize()
        assert int(error.download(4).view(np.int32)[0]) == 0
        want = dst.words.copy()
        for p, q, slots, _ in copies[:7 if count is None else min(max(count, 0), 7)]:
            if p < 0 or q < 0:
                continue
            for s in range(slots):
                before, dst.words = dst.words, want
                for x, y in zip(parts(src, p, s), parts(dst, q, s)):
                    y[:] = x
                dst.words = before
        assert (d_dst.download()[:want.nbytes] == want.view(np.uint8)).all()
    assert (d_src.download()[:src.words.nbytes] == src.words.view(np.uint8)).all()


@pytest.mark.parametrize("cache", [BF16, 3])
@pytest.mark.parametrize("bad,error_bit", [((17, 0, 4), 1), ((0, 17, 4), 1), ((0x7FFFFFFF, 1, 4), 1), ((0, 1, 18), 2),
                                           ((0, 1, -1), 2)], ids=str)
def test_a_bad_copy_is_reported_and_the_others_are_made(cache, bad, error_bit):
    rng = np.random.default_rng(31)
    x = filled(rng, 17, 16, 2, 128, cache, "block")
    assert x.num_pages == 17
    words, error = up(x.words), up(np.zeros(1, np.int32))
    handle = (ref4 if cache == 3 else gpu).handle(x, words)
    copies = up(np.array([(2, 3, 16, 0), bad + (0,), (4, 5, 16, 0)], np.int32))
    gfd_amd.kv_copy_pages(handle, handle, copies.ptr, 3, error_flag=error.ptr)
    gfd_amd.synchronize()
    assert int(error.download(4).view(np.int32)[0]) == error_bit
    for p, q in ((2, 3), (4, 5)):
        for s in range(16):
            for a, b in zip(parts(x, p, s), parts(x, q, s)):
                b[:] = a
    assert (words.download()[:x.words.nbytes] == x.words.view(np.uint8)).all()


def test_many_copies():
    rng = np.random.default_rng(32)
    x = filled(rng, 20000, 1, 1, 64, BF16, "block")
    order = rng.permutation(x.num_pages)
    copies = np.stack([order[:9000], order[9000:18000], np.ones(9000), np.zeros(9000)], 1).astype(np.int32)
    words, d_copies = up(x.words), up(copies)
    handle = gpu.handle(x, words)
    gfd_amd.kv_copy_pages(handle, handle, d_copies.ptr, 9000)
    gfd_amd.synchronize()
    want = x.words.reshape(x.num_pages, -1).copy()
    want[copies[:, 1]] = want[copies[:, 0]]
    assert (words.download()[:want.nbytes].view(np.uint16) == want.reshape(-1)).all()


# ------------------------------------------------------------ a graph

def test_a_captured_fork_copy_and_freeing_replay():
    """Over changed parents, lengths and counts, against the same calls run eagerly."""
    hip = ctypes.CDLL(None)  # the HIP runtime that the library has loaded
    rng = np.random.default_rng(33)
    page, n = 16, 300
    x = filled(rng, n - 3, page, 2, 64, 3, "heads")
    n = x.num_pages
    words = up(x.words)
    cache = ref4.handle(x, words)
    table = np.full((12, 20), -1, np.int32)
    table[:6] = rng.permutation(n)[:120].reshape(6, 20)
    refs = np.bincount(table[:6].reshape(-1), minlength=n).astype(np.int32)
    d = dict(refs=up(refs), table=up(table), parent=up(np.zeros(6, np.int32)), child=up(np.arange(6, 12, dtype=np.int32)),
             len=up(np.zeros(6, np.int32)), room=up(np.zeros(6, np.int32)), copies=up(np.zeros((6, 4), np.int32)),
             error=up(np.zeros(1, np.int32)), count=up(np.zeros(1, np.int32)), moves=up(np.zeros((n // 2, 4), np.int32)),
             new_refs=up(refs), new_table=up(table), lens=up(np.full(12, 320, np.int32)))
    p = {k: b.ptr for k, b in d.items()}
    pool = gfd_amd.KVPool(refs=p["refs"], num_pages=n, page_size=page)
    need = gfd_amd.kv_pool_workspace_bytes(pool, 6)
    space = gfd_amd.DeviceBuffer(need)
    call = gfd_amd.KVFork(table=p["table"], child_table=p["table"], table_stride=20, child_stride=20, rows=12,
                          child_rows=12, parent=p["parent"], child=p["child"], len=p["len"], capacity=p["room"],
                          copies=p["copies"], num=6)
    together = gfd_amd.KVCompact(new_refs=p["new_refs"], table=p["table"], new_table=p["new_table"], table_stride=20,
                                 new_stride=20, len=p["lens"], rows=6, copies=p["moves"], num_copies=p["count"])

    def step(stream=None):
        more = dict(error_flag=p["error"], stream=stream)
        gfd_amd.kv_fork(pool, call, space.ptr, need, **more)
        gfd_amd.kv_copy_pages(cache, cache, p["copies"], 6, **more)
        gfd_amd.kv_compact(pool, together, space.ptr, need, **more)
        gfd_amd.kv_copy_pages(cache, cache, p["moves"], n // 2, count=p["count"], **more)
        gfd_amd.kv_free(pool, p["table"], 20, 12, p["child"], p["room"], 6, **more)

    def state():
        names = ("refs", "table", "copies", "moves", "new_refs", "new_table")
        return [d[k].download() for k in names] + [d[k].download(4) for k in ("count", "error")] + [words.download()]

    stream, graph, exe = ctypes.c_void_p(), ctypes.c_void_p(), ctypes.c_void_p()
    assert gfd_amd.lib().gfd_stream_create(ctypes.byref(stream)) == 0
    assert hip.hipStreamBeginCapture(stream, 2) == 0
    step(stream)
    assert hip.hipStreamEndCapture(stream, ctypes.byref(graph)) == 0
    assert hip.hipGraphInstantiate(ctypes.byref(exe), graph, None, None, ctypes.c_size_t(0)) == 0
    for _ in range(4):
        length = rng.integers(0, 301, 6).astype(np.int32)
        for name, v in (("parent", rng.integers(0, 6, 6)), ("len", length), ("room", length + rng.integers(0, 20, 6))):
            d[name].upload(v.astype(np.int32))
        results = []
        for run in ("eager", "replayed"):
            words.upload(x.words)
            for name, v in (("refs", refs), ("table", table), ("new_refs", refs), ("new_table", table)):
                d[name].upload(v)
            for name in ("copies", "count", "moves"):
                d[name].fill(0)
            if run == "eager":
                step()
                gfd_amd.synchronize()
            else:
                assert hip.hipGraphLaunch(exe, stream) == 0
                assert gfd_amd.lib().gfd_stream_synchronize(stream) == 0
            results.append(state())
        assert all((a == b).all() for a, b in zip(*results))
        assert (results[0][0].view(np.int32)[:n] == refs).all() and not results[0][7].any()
    assert hip.hipGraphExecDestroy(exe) == 0 and hip.hipGraphDestroy(graph) == 0
    gfd_amd.lib().gfd_stream_destroy(stream)
