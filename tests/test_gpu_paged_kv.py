"""kv_append, paged_attention and shared_prefix_attention on the GPU against
their definitions in 64 bits (paged_kv_ref), at the sizes, layouts and masks where they
can go wrong: lengths of zero and one, pages that end inside a tile, pages of
one token, heads that share keys in odd groups, rows that see nothing, NaN in
every slot and page that no token sees, tables whose unused entries are no pages."""
import ctypes

import numpy as np
import pytest

import gfd_amd
import paged_kv_ref as ref
from paged_kv_ref import BF16, E4M3, FP16

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True, scope="module")
def device():
    assert gfd_amd.device_count() > 0, "no GPU visible to libgfd_amd.so"
    assert gfd_amd.lib().gfd_set_device(0) == 0


def up(arr):
    arr = np.ascontiguousarray(arr)
    b = gfd_amd.DeviceBuffer(max(arr.nbytes, 16))
    if arr.nbytes:
        b.upload(arr.view(np.uint8).reshape(-1))
    return b


def handle(pages, words):
    size = pages.words.itemsize
    return gfd_amd.KVCache(k=words.ptr, v=words.ptr + pages.v_offset * size, page_stride=pages.strides[0],
                           slot_stride=pages.strides[1], head_stride=pages.strides[2], num_pages=pages.num_pages,
                           page_size=pages.page_size, num_heads=pages.heads, head_dim=pages.dim, dtype=pages.dtype,
                           k_scale=pages.k_scale, v_scale=pages.v_scale)


class Attend:
    """One call's device side; run() returns (out, lse) as values."""

    def __init__(self, rng, pages, q_lens, kv_lens, hq, dtype, prefix=0, scale=None, softcap=0.0, slopes=None,
                 window=0, doc_start=None, prefix_end=None, q_pad=0, max_kv=None, max_q=None, out_pad=0):
        self.T, self.hq, self.d, self.dtype = sum(q_lens), hq, pages.dim, dtype
        self.q_bits, q = ref.quantised(rng, (self.T, hq, pages.dim), dtype, 1.5)
        self.q = q
        wide = np.full((self.T, hq * pages.dim + q_pad), 0x7FFF, np.uint16)
        wide[:, :hq * pages.dim] = self.q_bits.reshape(self.T, -1)
        self.out_stride = hq * pages.dim + out_pad
        self.words = up(pages.words)
        self.cache = handle(pages, self.words)
        self.keep = dict(q=up(wide), q_start=up(np.concatenate([[0], np.cumsum(q_lens)]).astype(np.int32)),
                         kv_len=up(np.array(kv_lens, np.int32)), table=up(pages.table), pre=up(pages.prefix_table))
        for name, v in (("doc_start", doc_start), ("prefix_end", prefix_end)):
            if v is not None:
                self.keep[name] = up(np.array(v, np.int32))
        if slopes is not None:
            self.keep["slopes"] = up(np.asarray(slopes, np.float32))
        ptr = {k: b.ptr for k, b in self.keep.items()}
        self.out, self.lse = gfd_amd.DeviceBuffer(self.T * self.out_stride * 2 + 64), gfd_amd.DeviceBuffer(self.T * hq * 4 + 64)
        self.error = up(np.zeros(1, np.int32))
        self.prefix = prefix
        self.scale = pages.dim ** -0.5 if scale is None else scale
        self.call = gfd_amd.Attention(
            q=ptr["q"], out=self.out.ptr, lse=self.lse.ptr, q_stride=wide.shape[1], out_stride=self.out_stride,
            q_start=ptr["q_start"], kv_len=ptr["kv_len"], block_table=ptr["table"], table_stride=pages.table.shape[1],
            doc_start=ptr.get("doc_start"), prefix_end=ptr.get("prefix_end"), slopes=ptr.get("slopes"),
            scale=self.scale, softcap=softcap, window=window, batch=len(q_lens), num_tokens=self.T,
            max_q_len=max(q_lens) if max_q is None else max_q, max_kv_len=max(kv_lens) if max_kv is None else max_kv,
            num_q_heads=hq, dtype=dtype)
        n = gfd_amd.attention_workspace_bytes(self.cache, self.call, prefix)
        self.work_bytes = n
        self.workspace = gfd_amd.DeviceBuffer(n + 64)
        self.workspace.fill(0xFF)  # what it holds before a call does not matter

    def launch(self, stream=None):
        more = dict(workspace=self.workspace.ptr, workspace_bytes=self.work_bytes, error_flag=self.error.ptr,
                    stream=stream)
        if self.prefix:
            gfd_amd.shared_prefix_attention(self.cache, self.call, self.keep["pre"].ptr, self.prefix, **more)
        else:
            gfd_amd.paged_attention(self.cache, self.call, **more)

    def read(self):
        n = self.T * self.out_stride
        raw = self.out.download()
        assert (raw[n * 2:] == 0xA5).all(), "written past the output"
        bits = raw[:n * 2].view(np.uint16).reshape(self.T, self.out_stride)
        assert (bits[:, self.hq * self.d:] == 0xA5A5).all(), "written between the output's rows"
        lse = self.lse.download()
        assert (lse[self.T * self.hq * 4:] == 0xA5).all(), "written past lse"
        out = ref.decode(np.ascontiguousarray(bits[:, :self.hq * self.d]), self.dtype)
        return out.reshape(self.T, self.hq, self.d), lse[:self.T * self.hq * 4].view(np.float32).reshape(self.T, self.hq)

    def run(self):
        self.out.fill(0xA5)
        self.lse.fill(0xA5)
        self.launch()
        gfd_amd.synchronize()
        tail = self.workspace.download(64, self.work_bytes)
        assert (tail == 0xFF).all(), "written past the workspace"
        return self.read()

    def errors(self):
        return int(self.error.download(4).view(np.int32)[0])


def close(got, want, tol, what):
    off = np.abs(got - want)
    bad = ~(off <= tol)
    assert not bad.any(), "%s: %d of %d off, worst %.3g of tolerance %.3g at %s: %r for %r" % (
        what, bad.sum(), bad.size, off[bad].max() if np.isfinite(off[bad]).any() else np.nan, tol[bad].max(),
        np.argwhere(bad)[0], got[bad][0], want[bad][0])


def check(a, pages, q_lens, kv_lens, softcap=0.0, slopes=None, **masks):
    rows = ref.intervals(q_lens, kv_lens, **masks)
    want, want_lse, tol, tol_lse = ref.attention64(a.q, pages, rows, a.dtype, np.float32(a.scale).astype(float), softcap,
                                                   slopes)
    out, lse = a.run()
    assert a.errors() == 0
    close(out, want, tol, "out")
    none = np.isneginf(want_lse)
    assert (np.isneginf(lse) == none).all()
    close(np.where(none, 0, lse), np.where(none, 0, want_lse), tol_lse, "lse")
    again, lse2 = a.run()  # the same call again gives the same bits
    assert (again == out).all() and (lse2 == lse).all()


def case(seed, q_lens, kv_lens, hq=8, hk=2, d=128, page=16, dtype=BF16, cache=None, layout="block", prefix=0,
         softcap=0.0, slopes=False, window=0, doc_start=None, prefix_end=None, **kw):
    rng = np.random.default_rng(seed)
    pages = ref.Pages(rng, [n - prefix for n in kv_lens], page, hk, d, dtype if cache is None else cache, layout,
                      prefix=prefix, k_scale=1 / 32, v_scale=1 / 64, spread=20.0 if cache == E4M3 else 1.0)
    sl = np.float32(2.0 ** -np.linspace(0.5, 8, hq)).astype(float) if slopes else None
    a = Attend(rng, pages, q_lens, kv_lens, hq, dtype, prefix=prefix, softcap=softcap, slopes=sl, window=window,
               doc_start=doc_start, prefix_end=prefix_end, **kw)
    check(a, pages, q_lens, kv_lens, softcap=softcap, slopes=sl, window=window, doc_start=doc_start,
          prefix_end=prefix_end)
    return a


# ------------------------------------------------------------ single tokens

@pytest.mark.parametrize("kv", [[1], [15, 16, 17], [31, 32, 33, 64], [127, 128, 129, 1, 2], [500, 3, 1025]], ids=str)
@pytest.mark.parametrize("page", [1, 5, 16, 24, 64])
def test_single_tokens_at_lengths_around_pages_and_tiles(kv, page):
    case(1, [1] * len(kv), kv, page=page)


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("hq,hk", [(4, 4), (8, 1), (14, 2), (32, 2), (40, 1), (1, 1)])
def test_single_tokens_of_every_head_grouping(d, hq, hk):
    case(2, [1, 1], [70, 201], hq=hq, hk=hk, d=d, page=8)


@pytest.mark.parametrize("layout", ["block", "heads", "apart", "padded"])
@pytest.mark.parametrize("dtype,cache", [(BF16, None), (FP16, None), (BF16, E4M3), (FP16, E4M3)])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_single_tokens_of_every_type_and_layout(layout, dtype, cache, d):
    case(3, [1, 1, 1], [33, 150, 300], dtype=dtype, cache=cache, layout=layout, page=16, d=d)


@pytest.mark.parametrize("opts", [dict(softcap=5.0), dict(slopes=True), dict(window=20), dict(window=1),
                                  dict(softcap=30.0, slopes=True, window=65)], ids=str)
def test_single_tokens_with_cap_bias_and_window(opts):
    case(4, [1, 1, 1, 1], [1, 64, 190, 333], hq=6, hk=3, **opts)


def test_single_tokens_far_in_a_long_context_over_many_splits():
    case(5, [1, 1], [9001, 4100], hq=4, hk=1, page=32)


def test_many_sequences_of_odd_lengths():
    rng = np.random.default_rng(11)
    kv = rng.integers(1, 200, 70).tolist()
    case(6, [1] * 70, kv, hq=4, hk=2, d=64, page=16)


def test_tokens_without_any_key_and_sequences_without_tokens():
    case(7, [1, 0, 1, 2, 0], [0, 5, 1, 1, 0])  # the fourth's first token lies before all keys


# ------------------------------------------------------------ several tokens

@pytest.mark.parametrize("q,kv", [([2], [2]), ([3, 5], [40, 5]), ([9], [300]), ([17, 1, 30], [17, 64, 100]),
                                  ([64], [64]), ([65], [129]), ([130, 3], [130, 260]), ([200], [700])], ids=str)
@pytest.mark.parametrize("hq,hk", [(4, 4), (8, 2), (7, 1)])
def test_prompts_and_chunks(q, kv, hq, hk):
    case(8, q, kv, hq=hq, hk=hk)


@pytest.mark.parametrize("dtype,cache", [(BF16, None), (FP16, None), (BF16, E4M3), (FP16, E4M3)])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("page,layout", [(16, "block"), (5, "heads"), (64, "padded"), (1, "block"), (32, "heads")])
def test_prompts_of_every_type_dim_and_page(dtype, cache, d, page, layout):
    case(9, [90, 41], [150, 41], dtype=dtype, cache=cache, d=d, page=page, layout=layout, hq=4, hk=2)


def _documents(q_lens, kv_lens, seed):
    """(doc_start, prefix_end) per token: packed documents, some with a prefix that all of their tokens see."""
    rng = np.random.default_rng(seed)
    start, end = [], []
    for n, kv in zip(q_lens, kv_lens):
        cuts = np.unique(np.concatenate([[0], rng.integers(0, kv, 3)]))
        lens = np.diff(np.append(cuts, kv))
        seen = [int(rng.integers(0, x + 1)) for x in lens]
        for pos in range(kv - n, kv):
            at = np.searchsorted(cuts, pos, side="right") - 1
            start.append(int(cuts[at]))
            end.append(int(cuts[at]) + seen[at])
    return start, end


@pytest.mark.parametrize("seed", [0, 1, 2])
@pytest.mark.parametrize("q,kv", [([1, 3], [80, 50]), ([150], [150]), ([90, 64], [200, 64])], ids=str)
def test_documents_and_prefixes(seed, q, kv):
    start, end = _documents(q, kv, seed)
    case(10, q, kv, doc_start=start)
    case(11, q, kv, prefix_end=end, softcap=20.0)
    case(12, q, kv, doc_start=start, prefix_end=end, slopes=True, d=64)


@pytest.mark.parametrize("q,kv", [([4], [40]), ([120], [260])], ids=str)
def test_rows_that_see_nothing_between_rows_that_do(q, kv):
    rng = np.random.default_rng(3)
    start = np.where(rng.random(sum(q)) < 0.3, 0x7FFFFFFF, 0)
    start[0] = 0x7FFFFFFF
    case(13, q, kv, doc_start=start)
    case(14, q, kv, doc_start=np.full(sum(q), 0x7FFFFFFF))  # nobody sees anything


@pytest.mark.parametrize("q,kv", [([1], [500]), ([5], [500]), ([140], [500])], ids=str)
def test_windows(q, kv):
    for window in (1, 30, 64, 499, 4000):
        case(15, q, kv, window=window)


def test_prefix_ends_past_the_keys_are_cut():
    case(16, [5, 70], [9, 70], prefix_end=[0x7FFFFFFF] * 75)


@pytest.mark.parametrize("q,kv", [([1, 1], [100, 257]), ([100], [130])], ids=str)
@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_large_scores(q, kv, dtype):
    """Scores of some hundreds: the maximum has to be taken off before exp."""
    case(17, q, kv, dtype=dtype, scale=4.0)


@pytest.mark.parametrize("q,kv,window", [([1], [300], 40), ([3], [300], 40)], ids=str)
def test_nan_and_infinity_before_the_window_change_nothing(q, kv, window):
    rng = np.random.default_rng(18)
    pages = ref.Pages(rng, kv, 16, 2, 128, BF16)
    dead = kv[0] - q[0] + 1 - window  # keys below: seen by no token
    for j in range(dead):
        for at in (0, pages.v_offset):
            pages.view(pages.table[0, j // 16], j % 16, at)[:] = (0x7FC0, 0x7F80, 0xFF80)[j % 3]
    a = Attend(rng, pages, q, kv, 8, BF16, window=window)
    check(a, pages, q, kv, window=window)


@pytest.mark.parametrize("q,kv", [([40], [40]), ([150], [150])], ids=str)
def test_nan_in_one_document_stays_there(q, kv):
    """Documents whose border lies inside a tile: NaN and infinite values of the first reach no token of the second."""
    rng = np.random.default_rng(19)
    pages = ref.Pages(rng, kv, 16, 2, 128, BF16)
    cut = kv[0] // 2 + 3
    for j in range(0, cut, 2):
        for at in (0, pages.v_offset):
            pages.view(pages.table[0, j // 16], j % 16, at)[:] = (0x7FC0, 0x7F80)[j // 2 % 2]
    start = np.where(np.arange(q[0]) < cut, 0, cut)
    a = Attend(rng, pages, q, kv, 8, BF16, doc_start=start)
    want, _, tol, _ = ref.attention64(a.q, pages, ref.intervals(q, kv, doc_start=start), BF16, a.scale)
    out, lse = a.run()
    close(out[cut:], want[cut:], tol[cut:], "the second document")
    assert np.isnan(out[:cut]).all()


def test_strided_queries_and_outputs():
    case(20, [1, 40, 2], [9, 77, 300], q_pad=64, out_pad=8)


def test_no_lse():
    rng = np.random.default_rng(21)
    for q, kv in (([1, 1], [300, 40]), ([70], [99])):
        pages = ref.Pages(rng, kv, 16, 2, 128, BF16)
        a = Attend(rng, pages, q, kv, 8, BF16)
        want, _ = a.run()
        a.call.lse = None
        out, lse = a.run()
        assert (out == want).all() and (lse.view(np.uint32) == 0xA5A5A5A5).all()


def test_larger_maxima_than_needed_change_nothing():
    rng = np.random.default_rng(22)
    pages = ref.Pages(rng, [50, 130], 16, 2, 128, BF16)
    pages.table = np.pad(pages.table, ((0, 0), (0, 300)), constant_values=0x7FFFFFF0)
    a = Attend(rng, pages, [1, 1], [50, 130], 8, BF16, max_kv=4000, max_q=7)
    check(a, pages, [1, 1], [50, 130])


@pytest.mark.parametrize("q", [[1, 1], [80, 3]], ids=str)
def test_lengths_past_the_maximum_are_cut_and_reported(q):
    rng = np.random.default_rng(23)
    pages = ref.Pages(rng, [90, 100], 16, 2, 128, BF16)
    a = Attend(rng, pages, q, [90, 100], 8, BF16, max_kv=90)
    a.run()
    assert a.errors() == gfd_amd.KV_ERR_LENGTH


@pytest.mark.parametrize("q", [[1], [70]], ids=str)
@pytest.mark.parametrize("bad", [-1, -0x80000000, 0x7FFFFFFF])
def test_a_bad_page_is_reported_and_read_as_nothing(q, bad):
    rng = np.random.default_rng(24)
    pages = ref.Pages(rng, [100], 16, 2, 128, BF16)
    pages.table[0, 2] = pages.num_pages if bad == 0x7FFFFFFF else bad
    a = Attend(rng, pages, q, [100], 8, BF16)
    out, lse = a.run()
    assert a.errors() == gfd_amd.KV_ERR_PAGE
    # The same without those keys: their weight is zero.
    keep = np.r_[0:32, 48:100]
    rows = ref.intervals(q, [100])
    for t, (b, pos, lo, hi) in enumerate(rows):
        j = keep[(keep >= lo) & (keep < hi)]
        for h in range(8):
            s = pages.k[0][j, h // 4] @ a.q[t, h] * a.scale
            w = np.exp(s - s.max())
            v = pages.v[0][j, h // 4]
            tol = 2.1 * 2.0 ** -8 * (w / w.sum() @ np.abs(v)) + 1e-3 * 2.0 ** -8
            close(out[t, h], w / w.sum() @ v, tol, "row %d" % t)


# ------------------------------------------------------------ shared prefix

@pytest.mark.parametrize("page", [1, 16, 24])
@pytest.mark.parametrize("prefix", [1, 16, 100, 513])
def test_a_shared_prefix_and_what_follows(prefix, page):
    case(30, [1, 1, 1], [prefix + 1, prefix + 20, prefix + 150], prefix=prefix, page=page)


@pytest.mark.parametrize("dtype,cache", [(BF16, None), (FP16, None), (BF16, E4M3), (FP16, E4M3)])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("hq,hk", [(4, 4), (8, 1), (14, 2)])
def test_a_shared_prefix_of_every_type_and_grouping(dtype, cache, d, hq, hk):
    case(31, [1, 3, 1, 2], [310, 303, 300, 420], prefix=300, dtype=dtype, cache=cache, d=d, hq=hq, hk=hk)


@pytest.mark.parametrize("batch,q", [(1, 1), (40, 1), (70, 1), (9, 5), (3, 80)])
def test_a_shared_prefix_of_batches_of_every_size(batch, q):
    rng = np.random.default_rng(batch)
    q_lens = [q] + rng.integers(0, q + 1, batch - 1).tolist()
    kv = [200 + n + int(rng.integers(0, 40)) for n in q_lens]
    case(32, q_lens, kv, prefix=200, hq=4, hk=2)


def test_a_long_shared_prefix_over_many_splits():
    case(33, [1] * 5, [6001, 6002, 6100, 6033, 6001], prefix=6000, hq=8, hk=2, page=32)


@pytest.mark.parametrize("opts", [dict(softcap=5.0), dict(slopes=True), dict(window=70), dict(window=5),
                                  dict(softcap=30.0, slopes=True, window=130)], ids=str)
def test_a_shared_prefix_with_cap_bias_and_window(opts):
    case(34, [1, 4, 1, 2], [129, 200, 140, 330], prefix=128, **opts)


def test_a_shared_prefix_with_documents():
    q, kv = [30, 2, 1], [150, 180, 161]
    start, end = _documents(q, kv, 6)
    case(35, q, kv, prefix=120, doc_start=start, prefix_end=end)
    start[0] = start[31] = 0x7FFFFFFF
    case(36, q, kv, prefix=120, doc_start=start)


def test_a_prefix_that_is_all_there_is():
    """Tokens whose own keys lie in the prefix: nothing follows it."""
    case(37, [1, 2], [64, 64], prefix=64)


# ------------------------------------------------------------ append

@pytest.mark.parametrize("layout", ["block", "heads", "apart", "padded"])
@pytest.mark.parametrize("dtype,cache", [(BF16, BF16), (FP16, FP16), (BF16, E4M3), (FP16, E4M3)])
@pytest.mark.parametrize("d,rotary,pairs", [(128, 128, False), (128, 64, True), (64, 18, False), (256, 256, True),
                                            (256, 0, False), (64, 2, True), (128, 96, False)])
def test_append(layout, dtype, cache, d, rotary, pairs):
    _append(1, layout, dtype, cache, d, rotary, pairs, 13)


@pytest.mark.parametrize("tokens", [1, 2, 64, 300, 1000])
@pytest.mark.parametrize("with_q", [True, False])
def test_append_of_few_and_many_tokens(tokens, with_q):
    _append(2, "block", BF16, BF16, 128, 128, False, tokens, with_q=with_q)


@pytest.mark.parametrize("hq,hk", [(1, 1), (7, 7), (28, 4), (64, 8)])
@pytest.mark.parametrize("cache", [BF16, E4M3])
def test_append_of_every_head_count(hq, hk, cache):
    _append(3, "heads", BF16, cache, 64, 64, False, 21, hq=hq, hk=hk)


def test_append_turns_queries_in_place():
    _append(4, "block", FP16, FP16, 128, 128, False, 9, in_place=True)
    _append(4, "block", FP16, FP16, 128, 128, True, 9, in_place=True)
    _append(4, "block", FP16, FP16, 128, 50, False, 9, in_place=True)


def test_append_with_infinities_nan_and_overflow():
    _append(5, "block", BF16, E4M3, 128, 0, False, 6, special=True)
    _append(5, "block", BF16, BF16, 128, 0, False, 6, special=True)


def _append(seed, layout, dtype, cache, d, rotary, pairs, tokens, hq=6, hk=2, with_q=True, in_place=False,
            special=False):
    rng = np.random.default_rng(seed)
    page = 5
    pages = ref.Pages(rng, [0], page, hk, d, cache, layout, k_scale=1 / 32, v_scale=1 / 64,
                      spare=2 * -(-tokens // page) + 1)
    before = pages.words.copy()
    q_bits, q = ref.quantised(rng, (tokens, hq, d), dtype)
    k_bits, k = ref.quantised(rng, (tokens, hk, d), dtype)
    v_bits, v = ref.quantised(rng, (tokens, hk, d), dtype)
    if special:
        odd = np.array([np.inf, -np.inf, np.nan, 3e4, -3e4, 0.0, -0.0, 2.0 ** -14])
        k_bits[0, 0, :8] = v_bits[0, 0, :8] = ref.encode(odd, dtype)
        k, v = ref.decode(k_bits, dtype), ref.decode(v_bits, dtype)
    fused = np.concatenate([q_bits.reshape(tokens, -1), k_bits.reshape(tokens, -1), v_bits.reshape(tokens, -1)], 1)
    slots = rng.permutation(pages.num_pages * page)[:tokens].astype(np.int64)
    positions = rng.integers(0, 1 << 20, tokens).astype(np.int32)
    positions[0] = 0
    if tokens > 3:
        slots[2] = -1
        positions[3] = 0x7FFFFFFF
    inv_freq = (10000.0 ** (-np.arange(rotary // 2) / max(rotary // 2, 1))).astype(np.float32)
    words, rows_d = up(pages.words), up(fused)
    keep = dict(slots=up(slots), positions=up(positions), inv_freq=up(inv_freq))
    q_out = gfd_amd.DeviceBuffer(tokens * hq * d * 2 + 64)
    q_out.fill(0xA5)
    error = up(np.zeros(1, np.int32))
    width = fused.shape[1]
    gfd_amd.kv_append(handle(pages, words), gfd_amd.KVRows(
        q=rows_d.ptr if with_q else None, k=rows_d.ptr + hq * d * 2, v=rows_d.ptr + (hq + hk) * d * 2,
        q_out=None if not with_q else rows_d.ptr if in_place else q_out.ptr, q_stride=width, k_stride=width,
        v_stride=width, q_out_stride=width if in_place else hq * d, positions=keep["positions"].ptr,
        slots=keep["slots"].ptr, inv_freq=keep["inv_freq"].ptr, num_tokens=tokens, num_q_heads=hq, rotary_dim=rotary,
        interleaved=int(pairs), dtype=dtype), error_flag=error.ptr)
    gfd_amd.synchronize()
    assert int(error.download(4).view(np.int32)[0]) == 0
    kr, k_off = ref.rotate64(k, positions, inv_freq, pairs)
    after = words.download().view(pages.words.dtype)[:len(before)]
    touched = np.zeros(len(before), bool)
    mask = pages.words
    for which, at, x, off, scale in ((0, 0, kr, k_off, pages.k_scale), (1, pages.v_offset, v, 0 * v, pages.v_scale)):
        for t in range(tokens):
            if slots[t] < 0:
                continue
            pages.words = after
            got = ref.decode(pages.view(slots[t] // page, slots[t] % page, at).copy(), cache)
            pages.words = touched.view(np.uint8)
            pages.view(slots[t] // page, slots[t] % page, at)[:] = 1
            y, o = x[t] / scale, off[t] / scale
            if cache == E4M3:
                y = np.clip(y, -448, 448)
                # A step of the lowest range is 2^-9; the division is one more 32-bit rounding.
                tol = np.maximum(ref.U[E4M3] * np.abs(y), 2.0 ** -10) + 1.07 * o + 2 * ref.F32 * np.abs(y)
            else:
                tol = ref.U[cache] * np.abs(y) + 1.01 * o + (2.0 ** -25 if cache == FP16 else 0)
            same = (got == y) | (np.isnan(got) & np.isnan(y))
            close(np.where(same, 0, got), np.where(same, 0, y), np.where(same, 0, tol), "cache %d token %d" % (which, t))
    pages.words = mask
    assert (after[~touched] == before[~touched]).all(), "written outside the tokens' slots"
    qr, q_off = ref.rotate64(q, positions, inv_freq, pairs)
    raw = q_out.download()
    assert (raw[tokens * hq * d * 2:] == 0xA5).all()
    rows_after = rows_d.download().view(np.uint16).reshape(tokens, width)
    if in_place:
        got = rows_after[:, :hq * d].copy()
        assert (rows_after[:, hq * d:] == fused[:, hq * d:]).all()
    else:
        got = raw[:tokens * hq * d * 2].view(np.uint16)
        assert (rows_after == fused).all()
    if not with_q:
        assert (got == 0xA5A5).all()
        return
    close(ref.decode(got.reshape(tokens, hq, d), dtype), qr, ref.U[dtype] * np.abs(qr) + 1.01 * q_off +
          (2.0 ** -25 if dtype == FP16 else 0), "q")


def test_append_reports_a_slot_outside_the_cache_and_writes_the_others():
    rng = np.random.default_rng(6)
    pages = ref.Pages(rng, [0], 16, 2, 128, BF16, spare=2)
    words = up(pages.words)
    rows = up(np.full((3, 2, 128), 0x3F80, np.uint16))
    for bad in (32, 1 << 40, 0x7FFFFFFFFFFFFFFF):
        error, slots = up(np.zeros(1, np.int32)), up(np.array([3, bad, 31], np.int64))
        gfd_amd.kv_append(handle(pages, words), gfd_amd.KVRows(
            k=rows.ptr, v=rows.ptr, k_stride=256, v_stride=256, slots=slots.ptr, num_tokens=3, dtype=BF16),
            error_flag=error.ptr)
        gfd_amd.synchronize()
        assert int(error.download(4).view(np.int32)[0]) == gfd_amd.KV_ERR_PAGE
        after = words.download().view(np.uint16)
        assert (after == 0x3F80).sum() == 2 * 2 * 256


# ------------------------------------------------------------ together, and the caller's side

def test_append_then_attend_on_a_stream_of_its_own():
    """A step as a program runs it: append on a stream, attend on the same one, no waits between."""
    rng = np.random.default_rng(40)
    q_lens, kv_lens, hq, hk, d = [1, 5, 1], [40, 70, 129], 8, 2, 128
    pages = ref.Pages(rng, kv_lens, 16, hk, d, BF16)
    tokens = sum(q_lens)
    a = Attend(rng, pages, q_lens, kv_lens, hq, BF16)
    want, want_lse = a.run()
    # Take the last tokens' keys and values out of the cache and append them.
    at = [(b, kv - n + i) for b, (n, kv) in enumerate(zip(q_lens, kv_lens)) for i in range(n)]
    slots = np.array([int(pages.table[b, j // 16]) * 16 + j % 16 for b, j in at], np.int64)
    kb = np.stack([pages.view(s // 16, s % 16).copy() for s in slots])
    vb = np.stack([pages.view(s // 16, s % 16, pages.v_offset).copy() for s in slots])
    for s in slots:
        pages.view(s // 16, s % 16)[:] = pages.view(s // 16, s % 16, pages.v_offset)[:] = 0x7FC0
    a.words.upload(pages.words)
    keep = [up(kb), up(vb), up(slots)]
    stream = ctypes.c_void_p()
    assert gfd_amd.lib().gfd_stream_create(ctypes.byref(stream)) == 0
    a.out.fill(0xA5)
    a.lse.fill(0xA5)
    gfd_amd.kv_append(a.cache, gfd_amd.KVRows(k=keep[0].ptr, v=keep[1].ptr, k_stride=hk * d, v_stride=hk * d,
                                              slots=keep[2].ptr, num_tokens=tokens, dtype=BF16), stream=stream)
    a.launch(stream)
    assert gfd_amd.lib().gfd_stream_synchronize(stream) == 0
    gfd_amd.lib().gfd_stream_destroy(stream)
    out, lse = a.read()
    assert (out == want).all() and (lse == want_lse).all()


def test_a_workspace_that_is_too_small_is_refused():
    rng = np.random.default_rng(41)
    pages = ref.Pages(rng, [5000], 16, 1, 128, BF16)
    a = Attend(rng, pages, [1], [5000], 4, BF16)
    if a.work_bytes:
        with pytest.raises(gfd_amd.GfdError, match="workspace"):
            gfd_amd.paged_attention(a.cache, a.call, a.workspace.ptr, a.work_bytes - 1)
        with pytest.raises(gfd_amd.GfdError, match="workspace"):
            gfd_amd.paged_attention(a.cache, a.call, None, 1 << 40)


def test_a_captured_step_replays():
    """Append and attend in a graph, replayed over changed inputs, against eager calls."""
    hip = ctypes.CDLL(None)  # the HIP runtime that the library has loaded
    rng = np.random.default_rng(42)
    for q_lens, kv_lens, prefix in (([1, 1, 1], [300, 40, 900], 0), ([70], [150], 0), ([1, 2], [600, 610], 590)):
        pages = ref.Pages(rng, [n - prefix for n in kv_lens], 16, 2, 128, BF16, prefix=prefix)
        a = Attend(rng, pages, q_lens, kv_lens, 8, BF16, prefix=prefix)
        a.run()
        stream, graph, exe = ctypes.c_void_p(), ctypes.c_void_p(), ctypes.c_void_p()
        assert gfd_amd.lib().gfd_stream_create(ctypes.byref(stream)) == 0
        assert hip.hipStreamBeginCapture(stream, 2) == 0
        a.launch(stream)
        assert hip.hipStreamEndCapture(stream, ctypes.byref(graph)) == 0
        assert hip.hipGraphInstantiate(ctypes.byref(exe), graph, None, None, ctypes.c_size_t(0)) == 0
        for _ in range(4):
            bits = ref.encode(rng.standard_normal((a.T, 8 * 128)), BF16)
            a.keep["q"].upload(bits)
            want, want_lse = a.run()
            a.out.fill(0xA5)
            a.lse.fill(0xA5)
            assert hip.hipGraphLaunch(exe, stream) == 0
            assert gfd_amd.lib().gfd_stream_synchronize(stream) == 0
            out, lse = a.read()
            assert (out == want).all() and (lse == want_lse).all()
        assert hip.hipGraphExecDestroy(exe) == 0 and hip.hipGraphDestroy(graph) == 0
        gfd_amd.lib().gfd_stream_destroy(stream)
