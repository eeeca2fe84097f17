"""Pages of 8 bits, their scales and kept tokens past 2^32 bytes of a pool: on the GPU, bit for bit what a small pool with the same contents gives."""
from __future__ import annotations

import numpy as np
import pytest

from test_gpu_page_sight import dev, tokens_of

pytestmark = pytest.mark.gpu


def test_offsets_past_32_bits(e2c, torch_cuda):
    torch = torch_cuda
    KV, D, page, far = 8, 128, 32, 140_000  # 32 KB of codes a page: 4.6 GB each of k and v
    if torch.cuda.mem_get_info()[0] < 16 << 30:
        pytest.skip("needs 16 GB")
    H, lens, rows = 16, [700, 333, 64], 5
    need = sum(-(-x // page) for x in lens)
    caches = []
    for n_pages in (need, far):
        cache = e2c.PageCache.new(1, n_pages, page, KV, D, 3, 30, torch.int8)
        at = n_pages - need
        for i, x in enumerate(lens):
            blocks = -(-x // page)
            cache.table[i, :blocks] = torch.arange(at, at + blocks, dtype=torch.int32, device="cuda")
            cache.refs[at:at + blocks] = 1
            at += blocks
        cache.length.copy_(dev(torch, lens))
        caches.append(cache)
    g = torch.Generator(device="cuda").manual_seed(4)
    T = sum(lens)
    q, k, v = (torch.randn(T, h, D, generator=g, device="cuda").bfloat16() for h in (H, KV, KV))
    cos, sin = e2c.rope_table(1024, D)
    seqs, starts = dev(torch, range(3)), dev(torch, np.concatenate([[0], np.cumsum(lens)]))
    few = dev(torch, range(0, 3 * rows + 1, rows))
    parents = dev(torch, [-1, 0, 0, 2, -1] * 3)
    got = []
    for cache in caches:
        x = cache.store(0, q, k, v, cos, sin, seqs, starts)
        many = cache.attention(0, x, seqs, starts, max(lens), window=200, sinks=4)
        last = torch.cat([x[int(b) - rows:int(b)] for b in starts[1:]])
        tree, _ = cache.tree(parents, seqs, few, rows)
        some = cache.attention(0, last, seqs, few, rows, tree=tree)
        one = cache.attention(0, last[::rows].contiguous(), seqs, dev(torch, range(4)), 1)
        loaded = cache.load(0, seqs, starts, T)
        cache.keep(seqs, few, dev(torch, [0, 2, 3, 0, 0] * 3), dev(torch, [3, 2, 0]))
        e2c.check()
        held = [y for s, n in enumerate([698, 330, 59]) for y in tokens_of(cache, s, n)]
        got.append([x, many, some, one, *loaded, cache.length.clone(), *held])
    assert got[1][6].tolist() == [698, 330, 59]
    for a, b in zip(*got):
        assert torch.equal(a, b)
