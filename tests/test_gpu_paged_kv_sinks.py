"""Many keys far below one that outweighs each of them: their weights together are not lost in 16 bits.

The first key's score is `gap` and its value zero, all others' scores are zero and their values V, so a token
that sees n others gets V n w / (1 + n w), w = e^-gap."""
import numpy as np
import pytest

import gfd_amd
import paged_kv_ref as ref
from paged_kv_ref import BF16, E4M3, F32, FP16
from test_gpu_paged_kv import Attend, close

pytestmark = pytest.mark.gpu

V = 256.0


@pytest.fixture(autouse=True, scope="module")
def device():
    assert gfd_amd.device_count() > 0, "no GPU visible to libgfd_amd.so"
    assert gfd_amd.lib().gfd_set_device(0) == 0


@pytest.mark.parametrize("dtype,cache", [(FP16, FP16), (FP16, E4M3), (BF16, BF16)])
@pytest.mark.parametrize("gap", [9.0, 16.90625, 17.1875, 17.5, 18.0])  # nats; 16 bits hold them
@pytest.mark.parametrize("batch,q,kv,hq,hk,prefix", [(600, 1, 600, 8, 2, 0), (600, 1, 120, 8, 2, 0), (1, 300, 2000, 64, 64, 0),
                                                     (64, 1, 700, 8, 2, 600)], ids=["few", "short", "many", "both"])
def test_keys_far_below_one_count(batch, q, kv, hq, hk, prefix, gap, dtype, cache):
    d = 64
    rng = np.random.default_rng(80)
    pages = ref.Pages(rng, [kv - prefix], 16, hk, d, cache, prefix=prefix)
    for words, at, value in ((ref.encode(0.0, cache), 0, 0.0), (ref.encode(V, cache), pages.v_offset, V)):
        for j in range(kv):
            page = pages.prefix_table[j // 16] if j < prefix else pages.table[0, (j - prefix) // 16]
            slot = (j if j < prefix else j - prefix) % 16
            pages.view(page, slot, at)[:] = words
    first = pages.prefix_table[0] if prefix else pages.table[0, 0]
    pages.view(first, 0)[:, :32] = ref.encode(1.0, cache)  # the first key: 32 ones; q: gap / 32 there
    pages.view(first, 0, pages.v_offset)[:] = ref.encode(0.0, cache)
    pages.table = np.repeat(pages.table, batch, 0)  # all sequences read the same pages
    q_lens, kv_lens = [q] * batch, [kv] * batch
    a = Attend(rng, pages, q_lens, kv_lens, hq, dtype, prefix=prefix, scale=1.0)
    unit = np.zeros((a.T, hq, d))
    unit[..., :32] = gap / 32
    bits = ref.encode(unit, dtype)
    gap = float(ref.decode(bits, dtype)[0, 0, 0] * 32)  # bf16 holds it to 2^-8
    a.keep["q"].upload(bits)
    out, lse = a.run()
    n = np.array([pos for _, pos, _, _ in ref.intervals(q_lens, kv_lens)], float)
    mass = n * np.exp(-gap)
    want, want_lse = V * mass / (1 + mass), gap + np.log1p(mass)
    # Off by: the scores' sum, (d + 8) steps of the score, twice; the exponent, 64 steps; the sums over keys; weights
    # and output rounded once.  FP16: the output's steps no longer shrink below 2^-24, and what a key loses of its weight
    # once it is below 2^-28 of the largest is at most 2^-39 of that one.
    tol = (2.02 * ref.U[dtype] + 2 * (d + 8) * F32 * gap + (64 + 2 * kv) * F32) * want
    if dtype == FP16:
        tol = tol + 2.0 ** -25 + 2.0 ** -39 * V * n
    shape = (a.T, hq, d)
    close(out, np.broadcast_to(want[:, None, None], shape), np.broadcast_to(tol[:, None, None], shape), "out")
    tol_lse = (d + 8) * F32 * gap + (16 + 2 * kv) * F32 * (1 + want_lse)
    close(lse, np.broadcast_to(want_lse[:, None], lse.shape), np.broadcast_to(tol_lse[:, None], lse.shape), "lse")
