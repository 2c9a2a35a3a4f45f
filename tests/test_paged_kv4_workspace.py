"""How much workspace attention over a 4-bit cache asks for, over sizes up to the largest, without a GPU."""
import random

import gfd_amd
from test_paged_kv import call
from test_paged_kv4 import cache4


def test_no_size_needs_more_than_the_bound():
    """Of the header: a row's ranges times 4 (dim + 2) bytes, and a word for each block of rows and head."""
    rng = random.Random(8)
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
        c = cache4(num_heads=heads, head_dim=dim, head_stride=dim // 2, slot_stride=heads * dim // 2,
                   page_stride=17 * heads * dim, scale_page_stride=17 * heads * dim)
        k = call(batch=batch, num_tokens=tokens, max_q_len=q, max_kv_len=kv, num_q_heads=heads * group,
                 q_stride=heads * group * dim, out_stride=heads * group * dim, table_stride=1 << 27, **extra)
        n = gfd_amd.attention_workspace_bytes(c, k, prefix)
        ranges = 1 + 8192 / (batch * heads)
        if prefix:
            ranges += 1 + (8192 if tokens * group <= 32 else 512) / heads
        most = 4 * (dim + 2) * heads * group * tokens * ranges + 4 * heads * (batch + tokens * group / 128)
        assert 0 <= n <= most, (batch, q, kv, heads, group, dim, prefix, tokens)
