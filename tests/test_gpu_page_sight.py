"""Attention over pages with sinks, over trees of drafted tokens and over pages of 8 bits; the store into such pages and
their reading back; trees and what is kept of them: on the GPU, against plain 64-bit forms.

Tolerances are those of test_gpu_prompt_cache.py, with u the unit roundoff of q's type, and for pages of 8 bits, whose second
product has fp16 operands whatever q's type:
  attention  besides u |out| for the result, 2^-11 sum p|v| each for the exponential (times its token's scale, where that is
             applied there) and for v = code * scale where that becomes an operand; an exponential below 2^-14 of the row's
             largest (times its scale) loses 2^-25 of that absolutely, so that a row is off by 2^-25 of the largest |v| a key.
             Logits are the same 32-bit sums of products, and one product more for the key's scale
  codes      a head's values are within half a step (scale / 2) of the 64-bit rotation, and 2^-22 of the largest magnitude for
             the rotation, the scale and the quotient in 32 bits; equal to the 32-bit arithmetic written out
  read back  code * scale in fp32 (2^-24), rounded once to the output type
  bits, positions, lengths, counts and moved rows are exact.
"""
from __future__ import annotations

import math

import numpy as np
import pytest

from test_gpu_prompt_cache import CASES, DT, UNIT, assert_attention, make_batch, turn64

pytestmark = pytest.mark.gpu


def dev(torch, v):
    return torch.tensor(np.asarray(v), dtype=torch.int32, device="cuda")


def random_parents(rng, rows):
    """Chains with side branches, several roots: a row's parent is one before it, or -1."""
    return [-1 if r == 0 or rng.random() < 0.1 else r - 1 if rng.random() < 0.6 else int(rng.integers(-1, r)) for r in range(rows)]


def tree_mask(parents):
    n = len(parents)
    m = np.zeros((n, n), bool)
    for r, p in enumerate(parents):
        if p >= 0:
            m[r] = m[p]
        m[r, r] = True
    return m


def tree_words(masks, words):
    """[T][words] int32 of entries' bit matrices."""
    out = []
    for m in masks:
        for row in m:
            w = np.zeros(words, np.uint32)
            for i in np.flatnonzero(row):
                w[i // 32] |= np.uint32(1 << (i % 32))
            out.append(w)
    return np.array(out, np.uint32).reshape(-1, words).view(np.int32)


def held64(cache, name, layer, pages):
    """A sequence's keys or values in 64 bits, page by page: [pages][page][kv][dim]."""
    x = getattr(cache, name)[layer][pages].double()
    s = getattr(cache, name + "_scale")
    return x if s is None else x * s[layer][pages].double().transpose(-1, -2)[..., None]


def sight64(torch, cache, layer, q, seqs, q_start, causal, window, scale, sinks=0, masks=None):
    """out, sum p|v|, lse and the largest |logit| in 64 bits, a sequence at a time. masks: entries' bits among their rows."""
    T, H, D = q.shape
    page, KV = cache.k.shape[2], cache.k.shape[3]
    out = torch.zeros(T, H, D, dtype=torch.float64, device="cuda")
    mag, lse = torch.zeros_like(out), torch.full((T, H), -math.inf, dtype=torch.float64, device="cuda")
    big = torch.zeros(T, H, dtype=torch.float64, device="cuda")
    qs = q_start.tolist()
    for i, s in enumerate(seqs.tolist()):
        L, a, b = int(cache.length[s]), qs[i], qs[i + 1]
        if L == 0 or a == b:
            continue
        pages = cache.table[s, :-(-L // page)].long()
        k, v = (held64(cache, name, layer, pages).flatten(0, 1)[:L].repeat_interleave(H // KV, 1) for name in "kv")
        own = L - (b - a)
        j = torch.arange(L, device="cuda")[None]
        if masks is None:
            p = torch.arange(own, L, device="cuda")[:, None]
            sees = torch.ones(b - a, L, dtype=torch.bool, device="cuda")
            if causal:
                sees &= j <= p
        else:
            bits = torch.tensor(masks[i], device="cuda")
            p = (own + bits.sum(1) - 1)[:, None]
            sees = (j < own).expand(b - a, L).clone()
        if window >= 0:
            sees &= ((j - p).abs() <= window) | (j < sinks)
        if masks is not None:
            at = max(own, 0)
            sees[:, at:] = bits[:, at - own:]
        x = torch.einsum("thd,jhd->htj", q[a:b].double(), k) * scale
        x = x.masked_fill(~sees, -math.inf)
        r = torch.logsumexp(x, -1)
        w = torch.exp(x - r[..., None]).masked_fill(~sees, 0.0)
        out[a:b] = torch.einsum("htj,jhd->thd", w, v)
        mag[a:b] = torch.einsum("htj,jhd->thd", w, v.abs())
        lse[a:b] = r.T
        big[a:b] = x.abs().masked_fill(~sees, 0).amax(-1).T
    return out, mag, lse, big


def assert_codes(torch, got, lse, want, name, keys, largest):
    """assert_attention for pages of 8 bits whose values are at most `largest`."""
    out, mag, ref, big = want
    logit = 2.0 ** -18 * (1 + big)
    tol = UNIT[name] * out.abs() + (2.02 * 2.0 ** -11 + 2 * logit[..., None]) * mag + 2.0 ** -25 * (1 + keys * largest) + 1e-7
    assert not torch.isnan(got).any()
    assert ((got.double() - out).abs() - tol).max().item() <= 0
    empty = torch.isinf(ref)
    assert torch.equal(torch.isinf(lse), empty) and (lse[empty] < 0).all()
    assert ((lse.double() - ref).abs() - logit)[~empty].max().item() <= 0


# ------------------------------------------------------------------------------------------ sinks
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("causal,window,sinks", [(True, 0, 1), (True, 130, 4), (False, 37, 200), (True, 300, 128), (True, 20, 10 ** 6),
                                                 (False, 0, 129)])
@pytest.mark.parametrize("case", list(CASES))
def test_sinks(e2c, torch_cuda, case, causal, window, sinks, dtype):
    torch = torch_cuda
    lens, queries, shared, H, KV, D, page = CASES[case]
    cache, q, seqs, q_start, max_q = make_batch(e2c, torch, 12, lens, queries, shared, H, KV, D, page, dtype)
    out, lse = cache.attention(0, q, seqs, q_start, max_q, shared=shared, causal=causal, window=window, sinks=sinks, lse=True)
    e2c.check()
    assert_attention(torch, out, lse, sight64(torch, cache, 0, q, seqs, q_start, causal, window, D ** -0.5, sinks), dtype, max(lens))
    again = cache.attention(0, q, seqs, q_start, max_q, shared=shared, causal=causal, window=window, sinks=sinks)
    assert torch.equal(again, out), "two calls differ"


def test_sinks_without_a_window_change_nothing(e2c, torch_cuda):
    torch = torch_cuda
    cache, q, seqs, q_start, max_q = make_batch(e2c, torch, 5, [700, 90, 3], [4, 90, 1], 0, 4, 2, 128, 16, "bf16")
    a = cache.attention(0, q, seqs, q_start, max_q)
    assert torch.equal(a, cache.attention(0, q, seqs, q_start, max_q, sinks=8))
    e2c.check()


def test_tiles_between_sinks_and_window_are_not_read(e2c, torch_cuda):
    """NaN keys and values there reach no result, and a table that points anywhere there is not followed."""
    torch = torch_cuda
    for D, page in ((64, 8), (128, 32), (256, 64)):
        cache, q, seqs, q_start, max_q = make_batch(e2c, torch, 6, [2000, 1999], [3, 200], 0, 4, 2, D, page, "bf16")
        first, last = 128 // page, (2000 - 200 - 100) // 128 * 128 // page
        want = sight64(torch, cache, 0, q, seqs, q_start, True, 100, D ** -0.5, 7)
        for s in range(2):
            pages = cache.table[s, first:last].long()
            cache.k[:, pages] = float("nan")
            cache.v[:, pages] = float("nan")
        cache.table[:2, first:last] = -5
        out, lse = cache.attention(0, q, seqs, q_start, max_q, window=100, sinks=7, lse=True)
        e2c.check()
        assert_attention(torch, out, lse, want, "bf16", 2000)


# ------------------------------------------------------------------------------------------ trees
@pytest.mark.parametrize("rows", [[1], [31, 1, 0, 32], [33, 64, 7], [200, 3], [5] * 70])
def test_tree_bits_and_positions(e2c, torch_cuda, rows):
    torch = torch_cuda
    rng = np.random.default_rng(sum(rows))
    lens = [r + int(rng.integers(0, 300)) for r in rows]
    cache, q, seqs, q_start, max_q = make_batch(e2c, torch, 1, lens, rows, 0, 2, 1, 64, 16, "f16")
    parents = [random_parents(rng, rows[s]) for s in seqs.tolist()]
    tree, pos = cache.tree(dev(torch, sum(parents, [])), seqs, q_start, max_q)
    e2c.check()
    masks = [tree_mask(p) for p in parents]
    assert np.array_equal(tree.cpu().numpy(), tree_words(masks, tree.shape[1]))
    want = np.concatenate([lens[s] - rows[s] + m.sum(1) - 1 for s, m in zip(seqs.tolist(), masks)])
    assert np.array_equal(pos.cpu().numpy(), want)


def test_tree_parents_that_are_not_before_are_reported(e2c, torch_cuda):
    torch = torch_cuda
    cache, q, seqs, q_start, max_q = make_batch(e2c, torch, 1, [40], [5], 0, 2, 1, 64, 16, "f16")
    tree, pos = cache.tree(dev(torch, [-1, 1, 7, -2, 2 ** 31 - 1]), seqs, q_start, 5)
    with pytest.raises(e2c.E2CudaError, match="outside the cache"):
        e2c.check()
    assert tree[:, 0].tolist() == [1, 2, 4, 8, 16] and pos.tolist() == [35] * 5


TREES = {
    # lens, rows, shared, H, KV, D, page
    "one": ([1], [1], 0, 1, 1, 64, 8),
    "no text": ([9, 64], [9, 64], 0, 4, 2, 128, 16),
    "few": ([300, 20, 131, 33], [11, 4, 3, 1], 0, 16, 4, 128, 16),
    "two tiles of drafts": ([400, 777], [200, 150], 0, 4, 2, 64, 32),
    "several row tiles": ([1000, 130], [65, 70], 0, 8, 1, 256, 64),
    "verify": ([500 + 37 * i for i in range(40)], [31 - i % 9 for i in range(40)], 0, 8, 2, 128, 32),
    "behind a document": ([640 + 24 + 3 * (i % 60) for i in range(220)], [24 - i % 7 for i in range(220)], 640, 4, 2, 256, 32),
    "drafts in the prefix": ([640 + i % 4 for i in range(200)], [6] * 200, 640, 4, 2, 128, 64),
    "odd group": ([190, 77], [33, 77], 64, 7, 1, 128, 64),
    "more rows than tokens": ([3, 60], [7, 5], 0, 4, 2, 64, 16),
}


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("window,sinks", [(-1, 0), (0, 0), (40, 3), (200, 140)])
@pytest.mark.parametrize("case", list(TREES))
def test_tree_attention(e2c, torch_cuda, case, window, sinks, dtype):
    torch = torch_cuda
    lens, rows, shared, H, KV, D, page = TREES[case]
    rng = np.random.default_rng(len(case))
    cache, q, seqs, q_start, max_q = make_batch(e2c, torch, 13, lens, rows, shared, H, KV, D, page, dtype)
    parents = [random_parents(rng, rows[s]) for s in seqs.tolist()]
    tree, _ = cache.tree(dev(torch, sum(parents, [])), seqs, q_start, max_q)
    out, lse = cache.attention(0, q, seqs, q_start, max_q, shared=shared, window=window, sinks=sinks, tree=tree, lse=True)
    e2c.check()
    masks = [tree_mask(p) for p in parents]
    assert_attention(torch, out, lse, sight64(torch, cache, 0, q, seqs, q_start, True, window, D ** -0.5, sinks, masks), dtype, max(lens))


@pytest.mark.parametrize("words", [4, 9])
def test_masks_of_the_callers(e2c, torch_cuda, words):
    """Any bits: rows without their own, rows without any (which, without text, see nothing), bits past the rows."""
    torch = torch_cuda
    rng = np.random.default_rng(words)
    lens, rows = [128, 100, 333], [128, 100, 97]
    cache, q, seqs, q_start, max_q = make_batch(e2c, torch, 2, lens, rows, 0, 4, 4, 64, 16, "f16")
    masks = [rng.random((rows[s], rows[s])) < 0.2 for s in seqs.tolist()]
    for m in masks:
        m[::7] = False
    bits = tree_words(masks, words)
    for i, s in enumerate(seqs.tolist()):  # what lies past an entry's rows says nothing
        past = np.zeros(words * 32, bool)
        past[rows[s]:] = True
        bits[q_start[i].item():q_start[i + 1].item()] |= tree_words([past[None]], words)[0]
    out, lse = cache.attention(0, q, seqs, q_start, max_q, tree=torch.tensor(bits, device="cuda"), lse=True)
    e2c.check()
    want = sight64(torch, cache, 0, q, seqs, q_start, True, -1, 0.125, 0, masks)
    assert_attention(torch, out, lse, want, "f16", 333)
    assert torch.isinf(want[2]).any() and (out[torch.isinf(lse)] == 0).all()


def test_chain_is_causal(e2c, torch_cuda):
    """A tree that is one chain sees what causal rows see, bit for bit."""
    torch = torch_cuda
    for D, shared in ((64, 0), (128, 256), (256, 0)):
        lens, rows = [300 + 9 * i for i in range(60)], [1 + i % 9 for i in range(60)]
        cache, q, seqs, q_start, max_q = make_batch(e2c, torch, 3, lens, rows, shared, 4, 2, D, 32, "bf16")
        parents = dev(torch, sum([list(range(-1, rows[s] - 1)) for s in seqs.tolist()], []))
        tree, pos = cache.tree(parents, seqs, q_start, max_q)
        a = cache.attention(0, q, seqs, q_start, max_q, shared=shared, tree=tree)
        b = cache.attention(0, q, seqs, q_start, max_q, shared=shared)
        e2c.check()
        assert torch.equal(a, b)


# ------------------------------------------------------------------------------------------ what is kept of a tree
def tagged(e2c, torch, dtype, layers, n_pages, page, kv, D, max_seqs, max_blocks, seed):
    cache = e2c.PageCache.new(layers, n_pages, page, kv, D, max_seqs, max_blocks, getattr(torch, dtype))
    g = torch.Generator(device="cuda").manual_seed(seed)
    for x in (cache.k, cache.v):
        x.copy_(torch.randint(-127, 128, x.shape, generator=g, device="cuda"))
    for x in (cache.k_scale, cache.v_scale):
        if x is not None:
            x.copy_(torch.rand(x.shape, generator=g, device="cuda"))
    return cache


def tokens_of(cache, s, count):
    """Everything the cache holds of a sequence's first tokens."""
    page = cache.k.shape[2]
    import torch

    at = torch.arange(count, device="cuda")
    p, slot = cache.table[s, at // page].long(), at % page
    got = [cache.k[:, p, slot], cache.v[:, p, slot]]
    if cache.k_scale is not None:
        got += [cache.k_scale[:, p, :, slot], cache.v_scale[:, p, :, slot]]
    return got


@pytest.mark.parametrize("dtype,layers,page,kv,D", [("bfloat16", 1, 8, 1, 64), ("int8", 3, 16, 2, 128), ("float16", 2, 32, 33, 256),
                                                    ("int8", 2, 64, 3, 64), ("bfloat16", 5, 16, 130, 128)])
def test_keep(e2c, torch_cuda, dtype, layers, page, kv, D):
    torch = torch_cuda
    rng = np.random.default_rng(page + kv)
    n, texts, rows = 6, [0, 5, page, 3 * page - 1, 40, 17], [9, 1, 2 * page + 3, 12, 0, 31]
    cache = tagged(e2c, torch, dtype, layers, 96, page, kv, D, n, 24, page)
    cache.append(dev(torch, range(n)), dev(torch, texts))
    cache.append(dev(torch, range(n)), dev(torch, rows))
    e2c.check()
    kept = [sorted(rng.permutation(r)[:int(rng.integers(0, r + 1))].tolist()) for r in rows]
    kept[0], kept[2] = [], list(range(rows[2]))  # none of a sequence without text, all of another
    order = rng.permutation(n)
    before = [tokens_of(cache, s, texts[s] + rows[s]) for s in range(n)]
    table, others = cache.table.clone(), cache.refs.clone()
    q_start = np.concatenate([[0], np.cumsum([rows[s] for s in order])])
    flat = sum([kept[s] + [-7] * (rows[s] - len(kept[s])) for s in order], [])
    cache.keep(dev(torch, order), dev(torch, q_start), dev(torch, flat), dev(torch, [len(kept[s]) for s in order]))
    e2c.check()
    assert torch.equal(cache.table, table)
    for s in range(n):
        now = texts[s] + len(kept[s])
        assert int(cache.length[s]) == now
        at = torch.tensor(list(range(texts[s])) + [texts[s] + r for r in kept[s]], device="cuda", dtype=torch.long)
        for x, y in zip(tokens_of(cache, s, now), before[s]):
            assert torch.equal(x, y.transpose(0, 1)[at].transpose(0, 1) if x.dim() == y.dim() and x.shape[0] == layers else y[at])
        others[table[s, -(-now // page):-(-(texts[s] + rows[s]) // page)].long()] -= 1
    assert torch.equal(cache.refs, others)


def test_keep_refuses_bad_lists_and_shared_pages(e2c, torch_cuda):
    """Such entries are left as they are and reported, the others are done."""
    torch = torch_cuda
    cache = tagged(e2c, torch, "int8", 2, 64, 16, 2, 64, 9, 8, 1)
    cache.append(dev(torch, range(7)), dev(torch, [20] * 7))
    cache.fork(dev(torch, [6]), dev(torch, [7]))
    state = [x.clone() for x in (cache.k, cache.v, cache.length, cache.refs)]
    # descending, past the rows, negative, twice the same, more than the rows, a page that others map; then one that is right
    lists = [[3, 1], [0, 4], [-1, 2], [2, 2], [0, 1], [1, 2], [0, 2]]
    counts = [2, 2, 2, 2, 5, 2, 2]
    seqs = [0, 1, 2, 3, 4, 6, 5]
    flat = sum([x + [0, 0] for x in lists], [])
    cache.keep(dev(torch, seqs), dev(torch, range(0, 29, 4)), dev(torch, flat), dev(torch, counts))
    with pytest.raises(e2c.E2CudaError, match="outside the cache"):
        e2c.check()
    assert cache.length.tolist() == [20, 20, 20, 20, 20, 18, 20, 20, 0]
    assert torch.equal(cache.refs, state[3])
    own = cache.table[5, 1].long()
    for x, y in ((cache.k, state[0]), (cache.v, state[1])):
        same = x == y
        same[:, own, 1] = x[:, own, 1] == y[:, own, 2]
        assert same.all()
    # sequences that are not there
    cache.keep(dev(torch, [-1, 9]), dev(torch, [0, 2, 4]), dev(torch, [0, 1, 0, 1]), dev(torch, [2, 2]))
    with pytest.raises(e2c.E2CudaError, match="outside the cache"):
        e2c.check()


# ------------------------------------------------------------------------------------------ rotary positions of their own
@pytest.mark.parametrize("dtype", ["bfloat16", "int8"])
def test_store_at_positions(e2c, torch_cuda, dtype):
    torch = torch_cuda
    cache = e2c.PageCache.new(1, 20, 16, 2, 64, 3, 8, getattr(torch, dtype))
    cache.append(dev(torch, [1, 2]), dev(torch, [30, 50]))
    cos, sin = e2c.rope_table(64, 64)
    q, k, v = (torch.randn(9, h, 64, device="cuda").bfloat16() for h in (4, 2, 2))
    pos = dev(torch, [26, 27, 27, 28, 63, 0, 64, -1, 46])  # one past the table, one before it
    seqs, qs = dev(torch, [1, 2]), dev(torch, [0, 4, 9])
    out = torch.full_like(q, 7.0)
    cache.store(0, q, k, v, cos, sin, seqs, qs, pos=pos, out=out)
    with pytest.raises(e2c.E2CudaError, match="position outside"):
        e2c.check()
    good = [0, 1, 2, 3, 4, 5, 8]
    want, mag = turn64(torch, q[good], cos, sin, pos[good], False, False)
    assert ((out[good].double() - want).abs() <= UNIT["bf16"] * want.abs() + 4 * 2.0 ** -24 * mag).all()
    assert (out[[6, 7]] == 7.0).all()
    k2, _ = cache.load(0, seqs, qs, 9, dtype=torch.float32)
    e2c.check()
    want, _ = turn64(torch, k[good], cos, sin, pos[good], False, False)
    step = want.abs().amax(-1, keepdim=True) * (2.0 ** -8 if dtype == "bfloat16" else 0.5 / 127)
    assert ((k2[good].double() - want).abs() <= step * (1 + 2.0 ** -10)).all()


# ------------------------------------------------------------------------------------------ pages of 8 bits
def quantised(torch, x):
    """Codes and scales of heads, in the 32-bit arithmetic of the engine's activation quantiser."""
    amax = x.float().abs().amax(-1, keepdim=True)
    some = amax > 0
    # one division, rounded once: torch takes 127.0 / amax as a reciprocal times 127
    codes = (x.float() * torch.where(some, torch.full_like(amax, 127.0) / amax, 1.0)).round().to(torch.int8)
    return codes, torch.where(some, amax * float(np.float32(1 / 127)), 1.0)[..., 0]


def make_codes(e2c, torch, seed, lens, queries, shared, H, KV, D, page, dtype, spread=1.0, layers=1):
    """make_batch's cache in 8 bits; tokens' sizes differ by e^spread, and scales are NaN wherever nothing is held."""
    cache, q, seqs, q_start, max_q = make_batch(e2c, torch, seed, lens, queries, shared, H, KV, D, page, dtype, layers=layers)
    g = torch.Generator(device="cuda").manual_seed(seed + 1)
    parts = []
    for x in (cache.k, cache.v):
        held = ~torch.isnan(x[..., 0])
        size = (torch.randn(held.shape, generator=g, device="cuda") * spread).exp()
        codes, scale = quantised(torch, torch.nan_to_num(x).float() * size[..., None])
        wild = torch.randint(-128, 128, codes.shape, generator=g, device="cuda").to(torch.int8)
        parts.append((torch.where(held[..., None], codes, wild), torch.where(held, scale, float("nan")).transpose(-1, -2).contiguous()))
    (k, ks), (v, vs) = parts
    return e2c.PageCache(k, v, cache.table, cache.length, cache.refs, ks, vs), q, seqs, q_start, max_q


def largest(cache):
    return 127.0 * cache.v_scale.nan_to_num().abs().max().item()


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("causal,window,sinks", [(True, -1, 0), (False, 37, 0), (True, 130, 4), (False, 0, 129)])
@pytest.mark.parametrize("case", list(CASES))
def test_codes_attention(e2c, torch_cuda, case, causal, window, sinks, dtype):
    torch = torch_cuda
    lens, queries, shared, H, KV, D, page = CASES[case]
    cache, q, seqs, q_start, max_q = make_codes(e2c, torch, 14, lens, queries, shared, H, KV, D, page, dtype, spread=0.3)
    out, lse = cache.attention(0, q, seqs, q_start, max_q, shared=shared, causal=causal, window=window, sinks=sinks, lse=True)
    e2c.check()
    want = sight64(torch, cache, 0, q, seqs, q_start, causal, window, D ** -0.5, sinks)
    assert_codes(torch, out, lse, want, dtype, max(lens), largest(cache))
    again = cache.attention(0, q, seqs, q_start, max_q, shared=shared, causal=causal, window=window, sinks=sinks)
    assert torch.equal(again, out), "two calls differ"


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("case", list(TREES))
def test_codes_tree_attention(e2c, torch_cuda, case, dtype):
    torch = torch_cuda
    lens, rows, shared, H, KV, D, page = TREES[case]
    rng = np.random.default_rng(len(case))
    cache, q, seqs, q_start, max_q = make_codes(e2c, torch, 15, lens, rows, shared, H, KV, D, page, dtype, spread=0.3)
    parents = [random_parents(rng, rows[s]) for s in seqs.tolist()]
    tree, _ = cache.tree(dev(torch, sum(parents, [])), seqs, q_start, max_q)
    for window, sinks in ((-1, 0), (40, 3)):
        out, lse = cache.attention(0, q, seqs, q_start, max_q, shared=shared, window=window, sinks=sinks, tree=tree, lse=True)
        e2c.check()
        want = sight64(torch, cache, 0, q, seqs, q_start, True, window, D ** -0.5, sinks, [tree_mask(p) for p in parents])
        assert_codes(torch, out, lse, want, dtype, max(lens), largest(cache))


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("src,dtype", [("bf16", "bf16"), ("f32", "f16"), ("f16", "bf16")])
@pytest.mark.parametrize("lens,queries,H,KV,D,page,rot,pad", [([5], [5], 1, 1, 64, 8, 64, 0), ([1, 40, 17], [1, 1, 1], 8, 2, 128, 16, 128, 8),
                                                              ([70, 33], [70, 20], 10, 5, 256, 32, 96, 8), ([19, 64], [3, 64], 4, 2, 64, 16, 20, 3)])
def test_codes_store_and_load(e2c, torch_cuda, lens, queries, H, KV, D, page, rot, pad, src, dtype, interleaved):
    """Codes and scales against the 32-bit arithmetic and against 64 bits, what is read back, and all else left as it was."""
    torch = torch_cuda
    cache, _, seqs, q_start, _ = make_codes(e2c, torch, 21, lens, queries, 0, H, KV, D, page, "f16", layers=2)
    T = int(q_start[-1])
    rows = torch.randn(T, (H + 2 * KV) * D + pad, device="cuda").to(getattr(torch, DT[src]))[:, pad:]  # an odd pad: no 16-byte accesses
    q, k, v = rows.unflatten(1, (H + 2 * KV, D)).split([H, KV, KV], 1)
    v[0] = 0  # an all-zero head
    cos, sin = e2c.rope_table(max(lens), rot)
    before = [x.clone() for x in (cache.k, cache.v, cache.k_scale, cache.v_scale)]
    out = cache.store(1, q, k, v, cos, sin, seqs, q_start, interleaved=interleaved, dtype=getattr(torch, DT[dtype]))
    e2c.check()
    pos = torch.cat([torch.arange(lens[s] - queries[s], lens[s]) for s in seqs.tolist()]).cuda()
    owner = torch.cat([torch.full((queries[s],), s) for s in seqs.tolist()]).cuda()
    want, mag = turn64(torch, q, cos, sin, pos, interleaved, False)
    assert ((out.double() - want).abs() <= UNIT[dtype] * want.abs() + 2.0 ** -25 + 4 * 2.0 ** -24 * mag).all()
    p, slot = cache.table[owner, pos // page].long(), pos % page
    turned, mag = turn64(torch, k, cos, sin, pos, interleaved, False)
    for x, s, exact, err in ((cache.k, cache.k_scale, turned, 4 * 2.0 ** -24 * mag), (cache.v, cache.v_scale, v.double(), torch.zeros_like(mag))):
        codes, scale = x[1][p, slot], s[1][p, :, slot]
        amax = exact.abs().amax(-1, keepdim=True)
        step = torch.where(amax > 0, amax / 127, 1.0)
        assert ((scale.double() - step[..., 0]).abs() <= 2.0 ** -22 * step[..., 0]).all()
        assert ((codes.double() * step - exact).abs() <= step * (0.5 + 127 * 2.0 ** -21) + err).all()
        assert codes.abs().max() <= 127 and (codes[0].abs().amax(-1) == 127).sum() == (amax[0] > 0).sum()
    assert torch.equal(cache.v[1][p, slot], quantised(torch, v)[0]) and torch.equal(cache.v_scale[1][p, :, slot], quantised(torch, v)[1])
    for name in ("bfloat16", "float32", "float16"):
        t = getattr(torch, name)
        got = cache.load(1, seqs, q_start, T, dtype=t)
        e2c.check()
        for y, x, s in zip(got, (cache.k, cache.v), (cache.k_scale, cache.v_scale)):
            assert torch.equal(y, (x[1][p, slot].float() * s[1][p, :, slot][..., None]).to(t))
    for x, y in zip((cache.k, cache.v), before[:2]):  # the other layer, and tokens that are not the batch's
        keep = torch.ones_like(x[..., 0, 0], dtype=torch.bool)
        keep[1, p, slot] = False
        assert torch.equal(x[keep], y[keep])


def test_load_first_and_rows_that_are_not_there(e2c, torch_cuda):
    torch = torch_cuda
    for dtype in ("f16", "bf16"):
        cache, _, seqs, _, _ = make_batch(e2c, torch, 4, [50, 20, 9], [1, 1, 1], 0, 2, 2, 64, 8, dtype)
        order = dev(torch, [2, 0, 1])
        k, v = cache.load(0, order, dev(torch, [0, 4, 10, 12]), 12, first=dev(torch, [5, 13, 18]))
        e2c.check()
        for i, (s, t) in enumerate([(2, j) for j in range(5, 9)] + [(0, j) for j in range(13, 19)] + [(1, 18), (1, 19)]):
            assert torch.equal(k[i], cache.k[0, cache.table[s, t // 8].long(), t % 8]) and torch.equal(v[i], cache.v[0, cache.table[s, t // 8].long(), t % 8])
        # before the first token, past the last, a sequence that is not there
        k, _ = cache.load(0, dev(torch, [2, 0, 77]), dev(torch, [0, 2, 4, 5]), 5, first=dev(torch, [-1, 49, 0]))
        with pytest.raises(e2c.E2CudaError, match="outside the cache"):
            e2c.check()
        assert torch.equal(k[1], cache.k[0, cache.table[2, 0].long(), 0]) and torch.equal(k[2], cache.k[0, cache.table[0, 6].long(), 1])


def test_heads_that_are_not_finite_or_tiny(e2c, torch_cuda):
    """Such a head stands for NaN, one below 2^-100 for zeros; a row that sees the key is NaN, and others are as before."""
    torch = torch_cuda
    cache = e2c.PageCache.new(1, 40, 16, 2, 64, 2, 16, torch.int8)
    seqs, qs = dev(torch, [0]), dev(torch, [0, 200])
    cache.append(seqs, dev(torch, [200]))
    cos, sin = e2c.rope_table(256, 64)
    q, k, v = (torch.randn(200, h, 64, device="cuda") for h in (4, 2, 2))
    k[150, 0, 3], k[160, 0, 5], k[10, 1], v[170, 1, 7] = float("nan"), float("inf"), 1e-35, float("-inf")
    x = cache.store(0, q, k, v, cos, sin, seqs, qs)
    k2, v2 = cache.load(0, seqs, qs, 200)
    e2c.check()
    assert x.dtype == torch.bfloat16
    assert torch.isnan(k2[[150, 160], 0]).all() and not torch.isnan(k2[[150, 160], 1]).any() and (k2[10, 1] == 0).all()
    assert torch.isnan(v2[170, 1]).all() and torch.isnan(v2).sum() == 64
    for rows in (200, 3):  # the form of many rows and of few: the last tokens
        out, lse = cache.attention(0, x[200 - rows:].contiguous(), seqs, dev(torch, [0, rows]), rows, lse=True)
        e2c.check()
        at = torch.arange(200 - rows, 200, device="cuda")
        assert torch.equal(torch.isnan(out[:, :2]).all(-1).all(-1), at >= 150) and torch.equal(torch.isnan(lse[:, 0]), at >= 150)
        assert torch.isnan(out[at >= 170][:, 2:]).all() and not torch.isnan(lse[:, 2:]).any()


def test_page_operations_move_scales(e2c, torch_cuda):
    torch = torch_cuda
    cache = tagged(e2c, torch, "int8", 3, 40, 16, 2, 64, 6, 8, 3)
    cache.append(dev(torch, [0, 1, 2]), dev(torch, [30, 50, 10]))
    e2c.check()
    parent = [x.clone() for x in tokens_of(cache, 0, 30)]
    other = [x.clone() for x in tokens_of(cache, 2, 10)]
    cache.fork(dev(torch, [0]), dev(torch, [4]))
    cache.append(dev(torch, [4]), dev(torch, [1]))  # copies the partly filled page
    cache.free(dev(torch, [1]))
    cache.compact()
    e2c.check()
    assert cache.table[0, 1] != cache.table[4, 1]
    for s, want in ((0, parent), (4, parent), (2, other)):
        for x, y in zip(tokens_of(cache, s, want[0].shape[1] if s != 2 else 10), want):
            assert torch.equal(x, y)


def test_refusals_of_tensors(e2c, torch_cuda):
    torch = torch_cuda
    cache, q, seqs, q_start, max_q = make_codes(e2c, torch, 2, [40, 20], [3, 2], 0, 4, 2, 64, 16, "f16")
    good = (cache.k, cache.v, cache.table, cache.length, cache.refs)
    for scales in ((), (cache.k_scale, None), (cache.k_scale, cache.v_scale.half()), (cache.k_scale, cache.v_scale[..., :-1]), (cache.k_scale.cpu(), cache.v_scale)):
        with pytest.raises(e2c.E2CudaError, match="PageCache"):
            e2c.PageCache(*good, *scales)
    plain = make_batch(e2c, torch, 2, [40], [3], 0, 4, 2, 64, 16, "f16")[0]
    with pytest.raises(e2c.E2CudaError, match="only there"):
        e2c.PageCache(plain.k, plain.v, plain.table, plain.length, plain.refs, cache.k_scale, cache.v_scale)
    with pytest.raises(e2c.E2CudaError, match="attention: q"):
        cache.attention(0, q.float(), seqs, q_start, max_q)
    for tree in (torch.zeros(5, 1, dtype=torch.int32), torch.zeros(4, 1, dtype=torch.int32, device="cuda"),
                 torch.zeros(5, 1, dtype=torch.int64, device="cuda"), torch.zeros(5, 2, dtype=torch.int32, device="cuda")[:, :1]):
        with pytest.raises(e2c.E2CudaError, match="tree"):
            cache.attention(0, q, seqs, q_start, max_q, tree=tree)
    with pytest.raises(e2c.E2CudaError, match="sinks"):
        cache.attention(0, q, seqs, q_start, max_q, window=3, sinks=-1)
    with pytest.raises(e2c.E2CudaError):
        cache.tree(torch.zeros(5, dtype=torch.int32), seqs, q_start, max_q)
    with pytest.raises(e2c.E2CudaError):
        cache.keep(seqs, q_start, torch.zeros(5, dtype=torch.int32, device="cuda"), torch.zeros(3, dtype=torch.int32, device="cuda"))
    with pytest.raises(e2c.E2CudaError):
        cache.store(0, q, q[:, :2], q[:, :2], *e2c.rope_table(64, 64), seqs, q_start, pos=torch.zeros(5, dtype=torch.int64, device="cuda"))


@pytest.mark.parametrize("dtype", ["int8", "bfloat16"])
def test_drafting_steps_in_a_graph(e2c, torch_cuda, dtype):
    """Steps of append, tree, store, attention and keep as a program runs them, captured on another stream and replayed,
    against the same steps of a cache whose accepted tokens were all that was ever stored."""
    torch = torch_cuda
    rng = np.random.default_rng(7)
    n, m, steps, H, KV, D, page = 3, 6, 5, 4, 2, 128, 16
    cos, sin = e2c.rope_table(256, D)
    g = torch.Generator(device="cuda").manual_seed(9)

    def new():
        cache = e2c.PageCache.new(1, 64, page, KV, D, n, 12, getattr(torch, dtype))
        cache.append(dev(torch, range(n)), dev(torch, [21] * n))
        return cache

    text = [torch.randn(21 * n, h, D, generator=g, device="cuda").bfloat16() for h in (H, KV, KV)]
    seqs, grow, qs = dev(torch, range(n)), dev(torch, [m] * n), dev(torch, range(0, n * m + 1, m))
    cache, plain = new(), new()
    for c in (cache, plain):
        c.store(0, *text, cos, sin, seqs, dev(torch, range(0, 21 * n + 1, 21)))
    q, k, v = (torch.zeros(n * m, h, D, device="cuda", dtype=torch.bfloat16) for h in (H, KV, KV))
    parents, kept, counts = (torch.zeros(s, dtype=torch.int32, device="cuda") for s in (n * m, n * m, n))
    out = torch.zeros_like(q)

    def step(stream=None):
        cache.append(seqs, grow, stream=stream)
        tree, pos = cache.tree(parents, seqs, qs, m, stream=stream)
        x = cache.store(0, q, k, v, cos, sin, seqs, qs, pos=pos, stream=stream)
        cache.attention(0, x, seqs, qs, m, tree=tree, out=out, stream=stream)
        cache.keep(seqs, qs, kept, counts, stream=stream)

    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    graph, drafts = None, []
    for i in range(steps):
        trees = [random_parents(rng, m) for _ in range(n)]
        paths = []
        for t in trees:
            path, r = [], int(rng.integers(0, m))
            while r >= 0:
                path.append(r)
                r = t[r]
            paths.append(path[::-1])
        with torch.cuda.stream(stream):
            for x in (q, k, v):
                x.copy_(torch.randn(x.shape, generator=g, device="cuda"))
            parents.copy_(dev(torch, sum(trees, [])))
            kept.copy_(dev(torch, sum([p + [0] * (m - len(p)) for p in paths], [])))
            counts.copy_(dev(torch, [len(p) for p in paths]))
            if i < 2:
                step()
            else:
                if graph is None:
                    torch.cuda.synchronize()
                    graph = torch.cuda.CUDAGraph()
                    with torch.cuda.graph(graph, stream=stream):
                        step()
                graph.replay()
        torch.cuda.synchronize()
        e2c.check()
        # the accepted path as it would have been decoded: causal rows behind the same text
        sizes = [len(p) for p in paths]
        rows = torch.tensor([s * m + r for s in range(n) for r in paths[s]], device="cuda")
        plain.append(seqs, dev(torch, sizes))
        starts = dev(torch, np.concatenate([[0], np.cumsum(sizes)]))
        x = plain.store(0, q[rows], k[rows], v[rows], cos, sin, seqs, starts)
        want = plain.attention(0, x, seqs, starts, max(sizes))
        e2c.check()
        assert torch.equal(cache.length, plain.length)
        for a, b in zip(cache.load(0, seqs, starts, len(rows)), plain.load(0, seqs, starts, len(rows))):
            assert torch.equal(a, b)
        # keys in another order in the sums, and other tiles: both are rounded from the same 32-bit sums within bf16's half steps
        assert (out[rows].float() - want.float()).abs().max() <= 2.0 ** -6 * want.float().abs().max()
    assert int((cache.refs > 0).sum()) == sum(-(-int(x) // page) for x in cache.length)


def test_two_streams_with_workspaces_of_their_own(e2c, torch_cuda):
    torch = torch_cuda
    cache, q, seqs, q_start, max_q = make_codes(e2c, torch, 8, [900, 1000, 1100] * 20, [2] * 60, 0, 8, 4, 128, 16, "bf16")
    big, qb, seqb, startb, maxb = make_batch(e2c, torch, 8, [3000, 2500], [300, 200], 0, 8, 2, 64, 32, "f16")
    want = cache.attention(0, q, seqs, q_start, max_q), big.attention(0, qb, seqb, startb, maxb, window=300, sinks=5)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for _ in range(10):
        got.append((cache.attention(0, q, seqs, q_start, max_q, stream=streams[0]), big.attention(0, qb, seqb, startb, maxb, window=300, sinks=5, stream=streams[1])))
        got.append((cache.attention(0, q, seqs, q_start, max_q, stream=streams[1]), big.attention(0, qb, seqb, startb, maxb, window=300, sinks=5, stream=streams[0])))
    torch.cuda.synchronize()
    e2c.check()
    for a, b in got:
        assert torch.equal(a, want[0]) and torch.equal(b, want[1])
