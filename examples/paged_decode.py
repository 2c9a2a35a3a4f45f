#!/usr/bin/env python3
"""Chats on one system prompt, decoded from a KV cache that was offloaded to the host.

1. The system prompt's pages lie scattered in pinned host memory; one zero-copy
   gather brings them into the cache's first pages, where they are shared.
2. Each chat's own tokens are appended to its own pages, rotated to their positions.
3. Every decode step appends one token per chat and attends: over the shared
   prompt, read once for all chats, and over each chat's own pages.

python examples/paged_decode.py [chats] [prompt tokens] [steps]
"""
import os
import sys
import time

import numpy as np

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
import gfd_amd  # noqa: E402

PAGE, HEADS, DIM, Q_HEADS = 16, 8, 128, 32  # a page: 16 tokens' keys, then their values, 64 KiB in bf16
SLOT = HEADS * DIM
PAGE_ELEMS = 2 * PAGE * SLOT


def bf16(x):
    u = np.ascontiguousarray(x, np.float32).view(np.uint32)
    return ((u + 0x7FFF + ((u >> 16) & 1)) >> 16).astype(np.uint16)


def f32(bits):
    return (bits.astype(np.uint32) << 16).view(np.float32)


def up(a):
    a = np.ascontiguousarray(a)
    b = gfd_amd.DeviceBuffer(max(a.nbytes, 16))
    b.upload(a.view(np.uint8).reshape(-1))
    return b


def main(chats=8, prompt=1024, steps=4, seed=0):
    assert prompt % PAGE == 0
    rng = np.random.default_rng(seed)
    shared, own = prompt // PAGE, -(-steps // PAGE)
    num_pages = shared + chats * own
    blocks = gfd_amd.DeviceBuffer(num_pages * PAGE_ELEMS * 2)
    blocks.fill(0)
    cache = gfd_amd.KVCache(k=blocks.ptr, v=blocks.ptr + PAGE * SLOT * 2, page_stride=PAGE_ELEMS, slot_stride=SLOT,
                            head_stride=DIM, num_pages=num_pages, page_size=PAGE, num_heads=HEADS, head_dim=DIM,
                            dtype=gfd_amd.BF16)

    # The prompt's pages come back from host memory, in the order of the table.
    host = gfd_amd.HostBuffer(2 * shared * PAGE_ELEMS * 2)
    pages = host.array.view(np.uint16).reshape(2 * shared, PAGE_ELEMS)
    for p in pages:
        p[:] = bf16(rng.standard_normal(PAGE_ELEMS))
    order = rng.permutation(2 * shared)[:shared]
    addresses = up(np.uint64(host.ptr) + order.astype(np.uint64) * np.uint64(PAGE_ELEMS * 2))
    gfd_amd.zero_copy_gather_tokens(addresses.ptr, blocks.ptr, PAGE_ELEMS * 2, shared)
    prefix_table = up(np.arange(shared, dtype=np.int32))
    table_host = shared + np.arange(chats * own, dtype=np.int32).reshape(chats, own)
    table = up(table_host)

    inv_freq = up((10000.0 ** (-np.arange(DIM // 2) / (DIM // 2))).astype(np.float32))
    q_start = up(np.arange(chats + 1, dtype=np.int32))
    width = (Q_HEADS + 2 * HEADS) * DIM
    rows = gfd_amd.DeviceBuffer(chats * width * 2)  # a projection's output: q, k and v of a token side by side
    positions, slots, kv_len = (gfd_amd.DeviceBuffer(chats * n) for n in (4, 8, 4))
    out = gfd_amd.DeviceBuffer(chats * Q_HEADS * DIM * 2)
    error = up(np.zeros(1, np.int32))
    step_rows = gfd_amd.KVRows(q=rows.ptr, k=rows.ptr + Q_HEADS * DIM * 2, v=rows.ptr + (Q_HEADS + HEADS) * DIM * 2,
                               q_out=rows.ptr, q_stride=width, k_stride=width, v_stride=width, q_out_stride=width,
                               positions=positions.ptr, slots=slots.ptr, inv_freq=inv_freq.ptr, num_tokens=chats,
                               num_q_heads=Q_HEADS, rotary_dim=DIM, dtype=gfd_amd.BF16)
    call = gfd_amd.Attention(q=rows.ptr, out=out.ptr, q_stride=width, out_stride=Q_HEADS * DIM, q_start=q_start.ptr,
                             kv_len=kv_len.ptr, block_table=table.ptr, table_stride=own, scale=DIM ** -0.5, batch=chats,
                             num_tokens=chats, max_q_len=1, max_kv_len=prompt + steps, num_q_heads=Q_HEADS,
                             dtype=gfd_amd.BF16)
    need = gfd_amd.attention_workspace_bytes(cache, call, prompt)  # once, for the largest call
    workspace = gfd_amd.DeviceBuffer(max(need, 16))

    for step in range(steps):
        rows.upload(bf16(rng.standard_normal((chats, width))))
        positions.upload(np.full(chats, prompt + step, np.int32))
        slots.upload((table_host[:, step // PAGE] * PAGE + step % PAGE).astype(np.int64))
        kv_len.upload(np.full(chats, prompt + step + 1, np.int32))
        gfd_amd.synchronize()
        t0 = time.perf_counter()
        gfd_amd.kv_append(cache, step_rows, error_flag=error.ptr)
        gfd_amd.shared_prefix_attention(cache, call, prefix_table.ptr, prompt, workspace.ptr, need, error.ptr)
        gfd_amd.synchronize()
        us = (time.perf_counter() - t0) * 1e6
    assert int(error.download(4).view(np.int32)[0]) == 0, "a slot or page was out of range"

    # The last step's first and last chat against numpy, from what the cache holds.
    held = f32(blocks.download().view(np.uint16)[:num_pages * PAGE_ELEMS]).reshape(num_pages, 2, PAGE, HEADS, DIM)
    q = f32(rows.download().view(np.uint16)[:chats * width]).reshape(chats, width)[:, :Q_HEADS * DIM]
    got = f32(out.download().view(np.uint16)[:chats * Q_HEADS * DIM]).reshape(chats, Q_HEADS, DIM)
    assert (held[:shared].reshape(shared, -1) == f32(pages[order])).all(), "the gathered pages differ"
    worst = 0.0
    for chat in (0, chats - 1):
        at = np.concatenate([np.arange(shared), table_host[chat]])
        k, v = (held[at, i].reshape(-1, HEADS, DIM)[:prompt + steps].astype(np.float64) for i in (0, 1))
        for h in range(Q_HEADS):
            s = k[:, h * HEADS // Q_HEADS] @ q[chat, h * DIM:(h + 1) * DIM].astype(np.float64) * np.float32(DIM ** -0.5)
            w = np.exp(s - s.max())
            want = (w / w.sum()) @ v[:, h * HEADS // Q_HEADS]
            # One rounding of the output and one of each weight, 2^-8 relative, and room for the 32-bit sums.
            tol = 2 ** -8 * np.abs(want) + 1.1 * 2 ** -8 * ((w / w.sum()) @ np.abs(v[:, h * HEADS // Q_HEADS]))
            worst = max(worst, float((np.abs(got[chat, h] - want) / tol).max()))
    assert worst <= 1, worst
    print("%d chats on %d shared tokens: last step %.1f us, worst error %.2f of the tolerance" % (chats, prompt, us, worst))
    return us


if __name__ == "__main__":
    main(*(int(x) for x in sys.argv[1:4]))
