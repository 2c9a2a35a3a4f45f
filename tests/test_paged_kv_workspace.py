"""How much workspace attention asks for, over sizes up to the largest, without a GPU."""
import random

import pytest

import gfd_amd
from test_paged_kv import cache, call


def need(batch, max_q, kv, q_heads=32, heads=8, dim=128, prefix=0, tokens=None, **kw):
    c = cache(num_heads=heads, head_dim=dim, head_stride=dim, slot_stride=heads * dim, page_stride=32 * heads * dim)
    n = gfd_amd.attention_workspace_bytes(
        c, call(batch=batch, num_tokens=batch * max_q if tokens is None else tokens, max_q_len=max_q, max_kv_len=kv,
                num_q_heads=q_heads, q_stride=q_heads * dim, out_stride=q_heads * dim, table_stride=1 << 27, **kw), prefix)
    assert n >= 0
    return n


def bound(batch, max_q, q_heads, heads, dim, prefix, tokens):
    """Of the header: a row's ranges times 4 (dim + 2) bytes, and a word for each block of rows and head."""
    group = q_heads // heads
    ranges = 1 + 8192 / (batch * heads)
    if prefix:
        ranges += 1 + (8192 if tokens * group <= 32 else 256) / heads
    return 4 * (dim + 2) * q_heads * tokens * ranges + 4 * heads * (batch + tokens * group / 128)


@pytest.mark.parametrize("batch,kv", [(512, 131072), (2048, 131072), (2048, 1 << 20), (64, 1 << 20), (8192, 1 << 20)])
def test_a_full_card_needs_little(batch, kv):
    assert need(batch, 1, kv) <= 4 * 130 * 32 * (batch + 1024) + 32 * batch


def test_batches_that_fill_the_card_many_times_need_none():
    for kv in (1000, 131072, 1 << 20):
        assert need(1024, 1, kv) == 0 or kv * 8192 > 1 << 27
        assert need(4096, 1, kv) == 0


def test_no_size_needs_more_than_the_bound():
    rng = random.Random(7)
    for _ in range(4000):
        heads, group = rng.choice([1, 2, 4, 8, 12, 40]), rng.choice([1, 4, 7, 8, 16, 40])
        dim = rng.choice([64, 128, 256])
        batch, q = int(2 ** rng.uniform(0, 11)), rng.choice([1, 1, 2, 5, 8, 33, 500])
        tokens = rng.randint(q, batch * q)
        if tokens * heads * group > 1 << 30:
            continue  # refused
        prefix = rng.choice([0, 0, 1, int(2 ** rng.uniform(4, 20))])
        kv = prefix + int(2 ** rng.uniform(0, 20))
        extra = rng.choice([{}, dict(window=int(2 ** rng.uniform(0, 14)))])
        n = need(batch, q, kv, heads * group, heads, dim, prefix, tokens, **extra)
        assert n <= bound(batch, q, heads * group, heads, dim, prefix, tokens), (batch, q, kv, heads, group, dim, prefix, tokens)


@pytest.mark.parametrize("q_len,kv,rows", [(100, 4196, 128), (1, 8000, 16)])
def test_ranges_of_256_dims_fill_the_card_once(q_len, kv, rows):
    """One workgroup of 256 dims fits a CU, two of 128: ranges times blocks times heads are at most as many."""
    for dim, fit in ((128, 2), (256, 1)):
        blocks = -(-q_len * 4 // rows)
        ranges = need(1, q_len, kv, dim=dim) // (4 * (dim + 2) * 32 * q_len)
        assert 128 * fit < ranges * blocks * 8 <= 256 * fit
