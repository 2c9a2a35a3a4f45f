"""The paged cache's operators where a call is cut into more than one piece: blocks of
256 rows, batches past a wave's lanes and past the sampled starts, long keys split
over workgroups, a prefix and what follows in one launch; values that are no numbers where
some rows see them and others do not; lengths and windows at the ends of their types."""
import importlib.util
import os

import numpy as np
import pytest

import gfd_amd
import paged_kv_ref as ref
from paged_kv_ref import BF16, E4M3, FP16
from test_gpu_paged_kv import Attend, case, close

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True, scope="module")
def device():
    assert gfd_amd.device_count() > 0, "no GPU visible to libgfd_amd.so"
    assert gfd_amd.lib().gfd_set_device(0) == 0


def check_some(a, pages, q_lens, kv_lens, sequences, softcap=0.0, slopes=None, **masks):
    """check() of test_gpu_paged_kv over some sequences' rows only: the oracle goes row by row."""
    rows = ref.intervals(q_lens, kv_lens, **masks)
    pick = [t for t, r in enumerate(rows) if r[0] in sequences]
    want, want_lse, tol, tol_lse = ref.attention64(a.q[pick], pages, [rows[t] for t in pick], a.dtype,
                                                   np.float32(a.scale).astype(float), softcap, slopes)
    out, lse = a.run()
    assert a.errors() == 0
    close(out[pick], want, tol, "out")
    none = np.isneginf(want_lse)
    assert (np.isneginf(lse[pick]) == none).all() and np.isfinite(out).all()
    close(np.where(none, 0, lse[pick]), np.where(none, 0, want_lse), tol_lse, "lse")


@pytest.mark.parametrize("opts", [dict(), dict(softcap=8.0), dict(slopes=True), dict(softcap=20.0, slopes=True),
                                  dict(window=21), dict(prefix=48)], ids=str)
@pytest.mark.parametrize("d,dtype,cache", [(64, BF16, None), (128, FP16, None), (128, BF16, E4M3)])
def test_blocks_of_256_rows(d, dtype, cache, opts):
    rng = np.random.default_rng(50)
    opts = dict(opts)
    prefix, window = opts.pop("prefix", 0), opts.get("window", 0)
    hq, hk, n = 64, 8, 36
    q = [64] * (n - 4) + [63, 1, 0, 64]
    kv = [prefix + int(x) + int(rng.integers(0, 100)) for x in q]
    pages = ref.Pages(rng, [x - prefix for x in kv], 16, hk, d, dtype if cache is None else cache, "heads", prefix=prefix,
                      k_scale=1 / 32, v_scale=1 / 64, spread=20.0 if cache == E4M3 else 1.0)
    slopes = np.float32(2.0 ** -np.linspace(0.5, 8, hq)).astype(float) if opts.pop("slopes", False) else None
    a = Attend(rng, pages, q, kv, hq, dtype, prefix=prefix, slopes=slopes, softcap=opts.get("softcap", 0.0), window=window)
    assert a.T * hq >= 2 * 256 * 256  # enough rows for blocks of 256
    check_some(a, pages, q, kv, (0, 17, n - 3, n - 1), opts.get("softcap", 0.0), slopes, window=window)


def test_more_sequences_than_a_wave_has_lanes():
    rng = np.random.default_rng(51)
    q = rng.integers(0, 31, 150).tolist()
    kv = [n + int(rng.integers(0, 50)) for n in q]
    case(52, q, kv, hq=16, hk=8, d=64)
    pages = ref.Pages(rng, kv, 16, 2, 64, FP16)
    check_some(Attend(rng, pages, q, kv, 16, FP16), pages, q, kv, (0, 63, 64, 127, 128, 149))


@pytest.mark.parametrize("batch", [20, 700, 1100])
def test_a_prefix_for_more_sequences_than_starts_are_sampled(batch):
    rng = np.random.default_rng(53)
    q = rng.integers(0, 3, batch).tolist()
    kv = [20 + n + int(rng.integers(0, 9)) for n in q]
    case(54, q, kv, prefix=20, hq=4, hk=2, d=64, page=8)


@pytest.mark.parametrize("opts", [dict(), dict(softcap=5.0, slopes=True), dict(window=19)], ids=str)
@pytest.mark.parametrize("d,dtype,cache", [(64, FP16, None), (128, BF16, None), (128, BF16, E4M3), (256, BF16, None),
                                           (256, FP16, E4M3)])
@pytest.mark.parametrize("q", [1, 3])  # 16 and 32 rows of a wave
def test_many_short_contexts(q, d, dtype, cache, opts):
    rng = np.random.default_rng(64)
    q_lens = rng.integers(0, q + 1, 260).tolist()
    kv = rng.integers(0, 129, 260).tolist()
    kv[:6] = [1, 31, 32, 33, 128, 0]
    assert max(q_lens) == q and len(kv) * 2 >= 512  # enough for a wave each
    case(65, q_lens, kv, hq=12, hk=2, d=d, dtype=dtype, cache=cache, **opts)


@pytest.mark.parametrize("bits", [0x7FC0, 0x7F80])
def test_values_that_are_no_numbers_in_many_short_contexts(bits):
    rng = np.random.default_rng(66)
    q, kv = [2] * 256, [50] * 256
    pages = ref.Pages(rng, kv, 16, 2, 128, BF16)
    for b in range(0, 256, 2):  # the last key: the second token sees it, the first does not
        pages.view(pages.table[b, 49 // 16], 49 % 16, pages.v_offset)[:, 3] = bits
    a = Attend(rng, pages, q, kv, 8, BF16)
    want, _, tol, _ = ref.attention64(a.q, pages, ref.intervals(q, kv), BF16, a.scale)
    out, _ = a.run()
    odd = np.zeros(out.shape, bool)
    odd[1::4, :, 3] = True
    close(out[~odd], want[~odd], tol[~odd], "what sees none")
    assert np.isnan(out[odd]).all() if bits == 0x7FC0 else (out[odd] == np.inf).all()


@pytest.mark.parametrize("q,kv", [([70], [5000]), ([40, 1, 33], [2900, 3000, 33])], ids=str)
@pytest.mark.parametrize("dtype,cache", [(BF16, None), (BF16, E4M3)])
@pytest.mark.parametrize("d", [64, 256])
def test_prompts_over_keys_that_are_split(q, kv, d, dtype, cache):
    case(55, q, kv, hq=4, hk=2, d=d, dtype=dtype, cache=cache, page=24)


@pytest.mark.parametrize("opts", [dict(), dict(softcap=5.0), dict(slopes=True), dict(window=700),
                                  dict(softcap=30.0, slopes=True)], ids=str)
@pytest.mark.parametrize("d,dtype,cache", [(64, FP16, None), (128, BF16, None), (128, FP16, E4M3), (256, BF16, None)])
def test_a_long_prefix_of_many_rows_and_few_that_follow(d, dtype, cache, opts):
    case(56, [1, 2, 1, 4, 1, 1, 3, 1], [1301, 1500, 1310, 1304, 1400, 1301, 1333, 1370], prefix=1300, hq=12, hk=2, d=d,
         dtype=dtype, cache=cache, page=32, layout="heads", **opts)


@pytest.mark.parametrize("q,kv", [([6], [3]), ([3], [6]), ([60], [20]), ([70, 2], [100, 1])], ids=str)
def test_the_widest_window_is_none(q, kv):
    case(57, q, kv, window=0x7FFFFFFF, prefix_end=[0x7FFFFFFF] * sum(q))
    case(58, q, kv, window=0x7FFFFFFF)


@pytest.mark.parametrize("q", [[1, 2], [60, 2]], ids=str)
@pytest.mark.parametrize("length", [-1, -0x80000000])
def test_negative_lengths_are_none(q, length):
    rng = np.random.default_rng(59)
    kv = [70, 90]
    pages = ref.Pages(rng, kv, 16, 2, 128, BF16)
    a = Attend(rng, pages, q, kv, 8, BF16)
    a.keep["kv_len"].upload(np.array([length, 90], np.int32))
    out, lse = a.run()
    assert (out[:q[0]] == 0).all() and np.isneginf(lse[:q[0]]).all()
    rows = ref.intervals(q, kv)
    want, want_lse, tol, tol_lse = ref.attention64(a.q[q[0]:], pages, rows[q[0]:], BF16, a.scale)
    close(out[q[0]:], want, tol, "out")
    close(lse[q[0]:], want_lse, tol_lse, "lse")


@pytest.mark.parametrize("batch", [4, 40])  # few rows over the prefix, and many
@pytest.mark.parametrize("bits,value", [(0x7FC0, np.nan), (0x7F80, np.inf), (0xFF80, -np.inf)], ids=str)
def test_a_shared_value_that_is_no_number_reaches_those_that_see_it(batch, bits, value):
    """A key of the prefix that lies in some tokens' windows and before others'."""
    rng = np.random.default_rng(60)
    prefix, window, at = 300, 100, 250
    kv = [prefix + 1 + int(x) for x in np.linspace(0, 90, batch)]
    pages = ref.Pages(rng, [n - prefix for n in kv], 16, 2, 128, BF16, prefix=prefix)
    pages.view(pages.prefix_table[at // 16], at % 16, pages.v_offset)[:, 5] = bits
    a = Attend(rng, pages, [1] * batch, kv, 8, BF16, prefix=prefix, window=window)
    rows = ref.intervals([1] * batch, kv, window=window)
    want, _, tol, _ = ref.attention64(a.q, pages, rows, BF16, a.scale)
    out, lse = a.run()
    sees = np.array([lo <= at for _, _, lo, _ in rows])
    assert sees.any() and not sees.all() and np.isfinite(lse).all()
    close(out[~sees], want[~sees], tol[~sees], "tokens that do not see it")
    others = np.arange(128) != 5
    close(out[sees][..., others], want[sees][..., others], tol[sees][..., others], "other dims")
    got = out[sees][..., 5]
    assert np.isnan(got).all() if np.isnan(value) else (got == value).all()


@pytest.mark.parametrize("q,kv", [([40], [40]), ([150], [150])], ids=str)
def test_infinite_values_in_one_document_keep_their_sign(q, kv):
    rng = np.random.default_rng(61)
    pages = ref.Pages(rng, kv, 16, 2, 128, FP16)
    cut = kv[0] // 2 + 3
    pages.view(pages.table[0, 0], 0, pages.v_offset)[:, 7] = 0x7C00
    pages.view(pages.table[0, 0], 0, pages.v_offset)[:, 9] = 0xFC00
    start = np.where(np.arange(q[0]) < cut, 0, cut)
    a = Attend(rng, pages, q, kv, 8, FP16, doc_start=start, scale=0.01)
    want, _, tol, _ = ref.attention64(a.q, pages, ref.intervals(q, kv, doc_start=start), FP16, a.scale)
    out, _ = a.run()
    close(out[cut:], want[cut:], tol[cut:], "the second document")
    assert (out[:cut, :, 7] == np.inf).all() and (out[:cut, :, 9] == -np.inf).all()


@pytest.mark.parametrize("batch", [3, 40])
@pytest.mark.parametrize("bad", [-1, 0x7FFFFFFF])
def test_a_bad_page_of_the_prefix_is_reported_and_read_as_nothing(batch, bad):
    rng = np.random.default_rng(62)
    prefix = 100
    kv = [prefix + 1 + int(x) for x in rng.integers(0, 30, batch)]
    pages = ref.Pages(rng, [n - prefix for n in kv], 16, 2, 64, BF16, prefix=prefix)
    pages.prefix_table[2] = bad
    a = Attend(rng, pages, [1] * batch, kv, 8, BF16, prefix=prefix)
    out, lse = a.run()
    assert a.errors() == gfd_amd.KV_ERR_PAGE
    for t in range(batch):
        j = np.r_[0:32, 48:kv[t]]
        for h in range(8):
            k, v = pages.k[t][j, h // 4], pages.v[t][j, h // 4]
            s = k @ a.q[t, h] * a.scale
            w = np.exp(s - s.max())
            # Weights and the output are rounded once, 2^-8 relative; 32-bit sums are far below a tenth of that.
            close(out[t, h], w / w.sum() @ v, 2.1 * 2.0 ** -8 * (w / w.sum() @ np.abs(v)) + 1e-3 * 2.0 ** -8, "row %d" % t)


@pytest.mark.parametrize("tokens", [8192, 8193, 9001])
def test_append_of_steps_whose_tokens_share_workgroups(tokens):
    """Small heads, so that the oracle's part stays short: whole rows compared at once."""
    rng = np.random.default_rng(63)
    page, hk, d = 64, 1, 64
    pages = -(-tokens // page) + 1
    blocks = gfd_amd.DeviceBuffer(pages * 2 * page * d * 2)
    blocks.fill(0xFF)
    k_bits, k = ref.quantised(rng, (tokens, hk, d), BF16)
    v_bits, _ = ref.quantised(rng, (tokens, hk, d), BF16)
    slots = rng.permutation(pages * page)[:tokens].astype(np.int64)
    positions = rng.integers(0, 1 << 20, tokens).astype(np.int32)
    inv_freq = (10000.0 ** (-np.arange(16) / 16)).astype(np.float32)

    def up(x):
        b = gfd_amd.DeviceBuffer(x.nbytes)
        b.upload(np.ascontiguousarray(x).view(np.uint8).reshape(-1))
        return b

    keep = [up(x) for x in (k_bits, v_bits, slots, positions, inv_freq)]
    gfd_amd.kv_append(
        gfd_amd.KVCache(k=blocks.ptr, v=blocks.ptr + page * d * 2, page_stride=2 * page * d, slot_stride=d, head_stride=d,
                        num_pages=pages, page_size=page, num_heads=hk, head_dim=d, dtype=BF16),
        gfd_amd.KVRows(k=keep[0].ptr, v=keep[1].ptr, k_stride=d, v_stride=d, slots=keep[2].ptr, positions=keep[3].ptr,
                       inv_freq=keep[4].ptr, num_tokens=tokens, rotary_dim=32, dtype=BF16))
    gfd_amd.synchronize()
    after = blocks.download().view(np.uint16).reshape(pages, 2, page, d)
    got_k, got_v = (after[slots // page, i, slots % page] for i in (0, 1))
    assert (got_v == v_bits[:, 0]).all()
    want, off = ref.rotate64(k, positions, inv_freq, False)
    close(ref.decode(got_k, BF16), want[:, 0], ref.U[BF16] * np.abs(want[:, 0]) + 1.01 * off[:, 0], "keys")
    untouched = np.ones(pages * page, bool)
    untouched[slots] = False
    assert (after.transpose(0, 2, 1, 3).reshape(pages * page, -1)[untouched] == 0xFFFF).all()


def test_the_example_decodes():
    at = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "paged_decode.py")
    spec = importlib.util.spec_from_file_location("paged_decode", at)
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    assert example.main(chats=5, prompt=160, steps=19) > 0
