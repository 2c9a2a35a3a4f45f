"""Attention over a 4-bit cache on the GPU against its definition in 64 bits, at the sizes, layouts and masks where it
can go wrong.  The cache's numbers are exact in the rows' type, so the tolerances are those of a 16-bit cache."""
import ctypes

import numpy as np
import pytest

import gfd_amd
import paged_kv4_ref as ref4
import paged_kv_ref as ref
import test_gpu_paged_kv as gpu
from paged_kv_ref import BF16, FP16
from test_gpu_paged_kv import _documents, check, close, up

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True, scope="module")
def device():
    assert gfd_amd.device_count() > 0, "no GPU visible to libgfd_amd.so"
    assert gfd_amd.lib().gfd_set_device(0) == 0


@pytest.fixture(autouse=True)
def four_bits(monkeypatch):
    """The calls' device side is the other caches', but for the descriptor."""
    monkeypatch.setattr(gpu, "handle", ref4.handle)


def case(seed, q_lens, kv_lens, hq=8, hk=2, d=128, page=16, dtype=BF16, layout="block", prefix=0, softcap=0.0,
         slopes=False, window=0, doc_start=None, prefix_end=None, **kw):
    rng = np.random.default_rng(seed)
    pages = ref4.Pages4(rng, [n - prefix for n in kv_lens], page, hk, d, dtype, layout, prefix=prefix)
    sl = np.float32(2.0 ** -np.linspace(0.5, 8, hq)).astype(float) if slopes else None
    a = gpu.Attend(rng, pages, q_lens, kv_lens, hq, dtype, prefix=prefix, softcap=softcap, slopes=sl, window=window,
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
@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_single_tokens_of_every_type_and_layout(layout, dtype, d):
    case(3, [1, 1, 1], [33, 150, 300], dtype=dtype, layout=layout, page=16, d=d)


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("opts", [dict(softcap=5.0), dict(softcap=500.0), dict(slopes=True), dict(window=20),
                                  dict(window=1), dict(softcap=30.0, slopes=True, window=65)], ids=str)
def test_single_tokens_with_cap_bias_and_window(opts, d):
    case(4, [1, 1, 1, 1], [1, 64, 190, 333], hq=6, hk=3, d=d, **opts)


@pytest.mark.parametrize("d,layout", [(64, "heads"), (128, "block"), (128, "apart"), (256, "heads")])
def test_single_tokens_far_in_a_long_context_over_many_splits(d, layout):
    case(5, [1, 1], [9001, 4100], hq=4, hk=1, d=d, page=32, layout=layout)


@pytest.mark.parametrize("d,hq,hk", [(64, 4, 2), (128, 32, 8), (256, 3, 3)])
def test_many_sequences_of_odd_lengths(d, hq, hk):
    kv = np.random.default_rng(11).integers(1, 200, 70).tolist()
    case(6, [1] * 70, kv, hq=hq, hk=hk, d=d, page=16)


def test_tokens_without_any_key_and_sequences_without_tokens():
    case(7, [1, 0, 1, 2, 0], [0, 5, 1, 1, 0])  # the fourth's first token lies before all keys


def test_ranges_walked_in_pieces():
    """A full card's ranges of more than 1024 keys: 512 sequences, few of them long."""
    rng = np.random.default_rng(8)
    kv = [2500, 2100, 1025, 1024] + [40] * 508
    pages = ref4.Pages4(rng, kv, 64, 1, 64)
    pages.table = np.pad(pages.table, ((0, 0), (0, 700)), constant_values=0x7FFFFFF0)
    a = gpu.Attend(rng, pages, [1] * 512, kv, 2, BF16, max_kv=40_000)
    check(a, pages, [1] * 512, kv)


# ------------------------------------------------------------ several tokens

@pytest.mark.parametrize("q,kv", [([2], [2]), ([3, 5], [40, 5]), ([9], [300]), ([17, 1, 30], [17, 64, 100]),
                                  ([64], [64]), ([65], [129]), ([130, 3], [130, 260]), ([200], [700])], ids=str)
@pytest.mark.parametrize("hq,hk", [(4, 4), (8, 2), (7, 1)])
def test_prompts_and_chunks(q, kv, hq, hk):
    case(10, q, kv, hq=hq, hk=hk)


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("page,layout", [(16, "block"), (5, "heads"), (64, "padded"), (1, "block"), (32, "apart")])
def test_prompts_of_every_type_dim_and_page(dtype, d, page, layout):
    case(11, [90, 41], [150, 41], dtype=dtype, d=d, page=page, layout=layout, hq=4, hk=2)


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("d", [64, 128])
def test_a_prompt_of_many_rows(d, dtype):
    """Blocks of 256 rows: 512 tokens of 256 heads, some of their rows looked at."""
    rng = np.random.default_rng(12)
    pages = ref4.Pages4(rng, [530], 32, 64, d, dtype, "heads")
    a = gpu.Attend(rng, pages, [512], [530], 256, dtype)
    out, lse = a.run()
    assert a.errors() == 0
    for t, h in zip(rng.integers(0, 512, 150).tolist() + [0, 511], rng.integers(0, 256, 150).tolist() + [0, 255]):
        one = ref4.OneHead(pages, 0, h // 4)
        want, want_lse, tol, tol_lse = ref.attention64(a.q[t:t + 1, h:h + 1], one, [ref.intervals([512], [530])[t]],
                                                       dtype, np.float32(a.scale).astype(float))
        close(out[t:t + 1, h:h + 1], want, tol, "out %d %d" % (t, h))
        close(lse[t:t + 1, h:h + 1], want_lse, tol_lse, "lse %d %d" % (t, h))


@pytest.mark.parametrize("seed", [0, 1])
@pytest.mark.parametrize("q,kv", [([1, 3], [80, 50]), ([150], [150]), ([90, 64], [200, 64])], ids=str)
def test_documents_and_prefixes(seed, q, kv):
    start, end = _documents(q, kv, seed)
    case(13, q, kv, doc_start=start)
    case(14, q, kv, prefix_end=end, softcap=20.0)
    case(15, q, kv, doc_start=start, prefix_end=end, slopes=True, d=64)


@pytest.mark.parametrize("q,kv", [([4], [40]), ([120], [260])], ids=str)
def test_rows_that_see_nothing_between_rows_that_do(q, kv):
    start = np.where(np.random.default_rng(3).random(sum(q)) < 0.3, 0x7FFFFFFF, 0)
    start[0] = 0x7FFFFFFF
    case(16, q, kv, doc_start=start)
    case(17, q, kv, doc_start=np.full(sum(q), 0x7FFFFFFF))  # nobody sees anything


@pytest.mark.parametrize("q,kv", [([1], [500]), ([5], [500]), ([140], [500])], ids=str)
def test_windows(q, kv):
    for window in (1, 30, 64, 499, 4000):
        case(18, q, kv, window=window)


def test_strided_queries_and_outputs():
    case(20, [1, 40, 2], [9, 77, 300], q_pad=64, out_pad=8)


@pytest.mark.parametrize("q,kv", [([1, 1], [100, 257]), ([100], [130])], ids=str)
@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_large_scores(q, kv, dtype):
    case(21, q, kv, dtype=dtype, scale=4.0)


# ------------------------------------------------------------ scales

@pytest.mark.parametrize("q,kv,window", [([1], [300], 40), ([3], [300], 40), ([1], [70], 9)], ids=str)
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("dtype,bytes_", [(BF16, (253, 254, 255)), (FP16, (141, 200, 255))])
def test_nan_before_the_window_changes_nothing(q, kv, window, d, dtype, bytes_):
    rng = np.random.default_rng(22)
    pages = ref4.Pages4(rng, kv, 16, 2, d, dtype)
    for j in range(kv[0] - q[0] + 1 - window):  # seen by no token
        for which in ("k_scales", "v_scales"):
            pages.view(pages.table[0, j // 16], j % 16, which)[:] = bytes_[j % 3]
    a = gpu.Attend(rng, pages, q, kv, 8, dtype, window=window)
    check(a, pages, q, kv, window=window)


@pytest.mark.parametrize("q", [1, 3, 40, 150])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("dtype,byte", [(BF16, 255), (BF16, 253), (FP16, 255), (FP16, 141)])
def test_a_group_beyond_the_scales_reads_as_nan_and_only_where_it_is_seen(q, d, dtype, byte):
    """One group of one value: NaN in its 32 dims of the rows that see it, and in no other dim or row."""
    rng = np.random.default_rng(23)
    kv = max(q, 30) + 7
    pages = ref4.Pages4(rng, [kv], 16, 1, d, dtype)
    at = kv - q + q // 2  # the rows from q // 2 on see it
    clean = pages.words.copy()
    group = d // 32 - 1
    pages.view(pages.table[0, at // 16], at % 16, "v_scales")[0, group] = byte
    a = gpu.Attend(rng, pages, [q], [kv], 4, dtype)
    out, lse = a.run()
    a.words.upload(clean)
    want, want_lse = a.run()
    assert (lse == want_lse).all()
    dims = slice(32 * group, 32 * group + 32)
    assert np.isnan(out[q // 2:, :, dims]).all()
    out[q // 2:, :, dims] = want[q // 2:, :, dims]
    # The other rows' products are the same ones, of the same weights.
    assert (out == want).all()


@pytest.mark.parametrize("q", [1, 100])
def test_a_nan_key_reaches_the_rows_that_see_it(q):
    rng = np.random.default_rng(24)
    kv = q + 60
    pages = ref4.Pages4(rng, [kv], 16, 2, 128, BF16)
    at = kv - q + q // 2
    pages.view(pages.table[0, at // 16], at % 16, "k_scales")[:, 1] = 255
    a = gpu.Attend(rng, pages, [q], [kv], 4, BF16)
    out, lse = a.run()
    assert np.isnan(out[q // 2:]).all() and np.isnan(lse[q // 2:]).all()
    # Against the definition: rows of a wave take a larger maximum at the same tiles, and one that is NaN may lead to more
    # of them, so the bits are not those of a call without it.
    rows = ref.intervals([q], [kv])[:q // 2]
    want, want_lse, tol, tol_lse = ref.attention64(a.q[:q // 2], pages, rows, BF16, np.float32(a.scale).astype(float))
    close(out[:q // 2], want, tol, "out")
    close(lse[:q // 2], want_lse, tol_lse, "lse")


@pytest.mark.parametrize("q", [1, 50])
@pytest.mark.parametrize("dtype,byte", [(BF16, 0), (BF16, 1), (BF16, 60), (BF16, 190), (BF16, 240), (FP16, 104),
                                        (FP16, 90), (FP16, 140)])
def test_values_of_the_scales_ends(q, dtype, byte):
    """All values of one scale: the output is that of the scale 1 times it, as the rows' type holds both."""
    rng = np.random.default_rng(25)
    kv = q + 33
    pages = ref4.Pages4(rng, [kv], 16, 1, 128, dtype)
    for j in range(kv):
        pages.view(pages.table[0, j // 16], j % 16, "v_scales")[:] = byte
    numbers = np.stack([pages.view(pages.table[0, j // 16], j % 16, "v").copy() for j in range(kv)])
    exact = ref4.values(numbers, np.full((kv, 1, 4), byte, np.uint8))
    held = exact if dtype == BF16 else exact.astype(np.float16).astype(np.float64)
    pages.v[0] = held
    a = gpu.Attend(rng, pages, [q], [kv], 4, dtype)
    rows = ref.intervals([q], [kv])
    want, want_lse, tol, tol_lse = ref.attention64(a.q, pages, rows, dtype, np.float32(a.scale).astype(float))
    out, lse = a.run()
    assert a.errors() == 0
    if dtype == BF16:
        # Products and sums under 2^-126 may be taken for zeros, and so may what is rounded to the type there.
        tol = tol + 2.0 ** -126 * (kv + 2)
    close(out, want, tol, "out")
    close(lse, want_lse, tol_lse, "lse")


# ------------------------------------------------------------ lengths and pages that are none

@pytest.mark.parametrize("q", [[1, 1], [80, 3]], ids=str)
def test_lengths_past_the_maximum_are_cut_and_reported(q):
    rng = np.random.default_rng(26)
    pages = ref4.Pages4(rng, [90, 100], 16, 2, 128)
    a = gpu.Attend(rng, pages, q, [90, 100], 8, BF16, max_kv=90)
    a.run()
    assert a.errors() == gfd_amd.KV_ERR_LENGTH


@pytest.mark.parametrize("q", [[1], [70]], ids=str)
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("bad", [-1, -0x80000000, 0x7FFFFFFF])
def test_a_bad_page_is_reported_and_read_as_nothing(q, d, bad):
    rng = np.random.default_rng(27)
    pages = ref4.Pages4(rng, [100], 16, 2, d)
    pages.table[0, 2] = pages.num_pages if bad == 0x7FFFFFFF else bad
    a = gpu.Attend(rng, pages, q, [100], 8, BF16)
    out, lse = a.run()
    assert a.errors() == gfd_amd.KV_ERR_PAGE
    keep = np.r_[0:32, 48:100]  # the same without those keys: their weight is zero
    for t, (b, pos, lo, hi) in enumerate(ref.intervals(q, [100])):
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


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("hq,hk", [(4, 4), (8, 1), (14, 2)])
def test_a_shared_prefix_of_every_type_and_grouping(dtype, d, hq, hk):
    case(31, [1, 3, 1, 2], [310, 303, 300, 420], prefix=300, dtype=dtype, d=d, hq=hq, hk=hk)


@pytest.mark.parametrize("batch,q", [(1, 1), (40, 1), (70, 1), (9, 5), (3, 80)])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_a_shared_prefix_of_batches_of_every_size(batch, q, d):
    rng = np.random.default_rng(batch)
    q_lens = [q] + rng.integers(0, q + 1, batch - 1).tolist()
    kv = [200 + n + int(rng.integers(0, 40)) for n in q_lens]
    case(32, q_lens, kv, prefix=200, hq=4, hk=2, d=d, layout="heads")


def test_a_long_shared_prefix_over_many_splits():
    case(33, [1] * 5, [6001, 6002, 6100, 6033, 6001], prefix=6000, hq=8, hk=2, page=32)


@pytest.mark.parametrize("opts", [dict(softcap=5.0), dict(slopes=True), dict(window=70), dict(window=5),
                                  dict(softcap=30.0, slopes=True, window=130)], ids=str)
def test_a_shared_prefix_with_cap_bias_and_window(opts):
    case(34, [1, 4, 1, 2], [129, 200, 140, 330], prefix=128, **opts)


def test_a_prefix_that_is_all_there_is():
    case(37, [1, 2], [64, 64], prefix=64)


# ------------------------------------------------------------ the caller's side

def test_a_workspace_that_is_too_small_is_refused():
    rng = np.random.default_rng(41)
    pages = ref4.Pages4(rng, [5000], 16, 1, 128)
    a = gpu.Attend(rng, pages, [1], [5000], 4, BF16)
    assert a.work_bytes
    for space, size in ((a.workspace.ptr, a.work_bytes - 1), (None, 1 << 40), (a.workspace.ptr + 8, 1 << 40)):
        with pytest.raises(gfd_amd.GfdError, match="gfd_kv4_attention: workspace"):
            gfd_amd.paged_attention(a.cache, a.call, space, size)


def test_a_captured_step_replays():
    hip = ctypes.CDLL(None)  # the HIP runtime that the library has loaded
    rng = np.random.default_rng(42)
    for q_lens, kv_lens, prefix in (([1, 1, 1], [300, 40, 900], 0), ([70], [150], 0), ([1, 2], [600, 610], 590)):
        pages = ref4.Pages4(rng, [n - prefix for n in kv_lens], 16, 2, 128, prefix=prefix)
        a = gpu.Attend(rng, pages, q_lens, kv_lens, 8, BF16, prefix=prefix)
        a.run()
        stream, graph, exe = ctypes.c_void_p(), ctypes.c_void_p(), ctypes.c_void_p()
        assert gfd_amd.lib().gfd_stream_create(ctypes.byref(stream)) == 0
        assert hip.hipStreamBeginCapture(stream, 2) == 0
        a.launch(stream)
        assert hip.hipStreamEndCapture(stream, ctypes.byref(graph)) == 0
        assert hip.hipGraphInstantiate(ctypes.byref(exe), graph, None, None, ctypes.c_size_t(0)) == 0
        for _ in range(4):
            a.keep["q"].upload(ref.encode(rng.standard_normal((a.T, 8 * 128)), BF16))
            want, want_lse = a.run()
            a.out.fill(0xA5)
            a.lse.fill(0xA5)
            assert hip.hipGraphLaunch(exe, stream) == 0
            assert gfd_amd.lib().gfd_stream_synchronize(stream) == 0
            out, lse = a.read()
            assert (out == want).all() and (lse == want_lse).all()
        assert hip.hipGraphExecDestroy(exe) == 0 and hip.hipGraphDestroy(graph) == 0
        gfd_amd.lib().gfd_stream_destroy(stream)
