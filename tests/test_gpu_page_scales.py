"""Attention over pages of 8 bits whose heads of v differ in size by many powers of two: heads of zeros, tokens that outweigh
their neighbours in and out of sight, the largest and the smallest scales that a store leaves. On the GPU, against the 64-bit form
of test_gpu_page_sight.py, in the forms for few rows, for many, and behind a packed prefix.

A row's tolerance comes from what it sees alone (u: unit roundoff of q's type; p: its 64-bit weights; s: scales of v):
  result      u |out|, and in fp16 2^-25 for a subnormal
  operands    an exponential times its token's scale is rounded to fp16: 2^-11 of it, or 2^-25 of the row's largest such product
              where it is below 2^-14 of that, so 2^-25 127 (keys seen) max p s; a scale below 2^-96 counts as 2^-96 in this
              maximum, and heads of zeros, which have no products, count as no more
  exponents   2 * 2^-18 (1 + the largest |logit|) for the logits' 32-bit sums, as there, and 2^-18 for an exponent of up to 128
  sums        exponentials are held 2^16 above their size relative to the row's largest product, from 2^-126 on, so that a row whose
              largest product has the scale 2^e loses keys of weights below 2^(e - 142): (keys seen) 2^(e - 142), and 2^-20 for sums
              in 32 bits
  lse         the logits' error, the sums', and four roundings of numbers of up to 256
"""
from __future__ import annotations

import numpy as np
import pytest

from test_gpu_page_sight import UNIT, dev, make_codes, random_parents, sight64, tree_mask
from test_gpu_prompt_cache import CASES, TINY

pytestmark = pytest.mark.gpu


def peaks64(torch, cache, q, seqs, q_start, causal, window, scale, lse, sinks=0, masks=None):
    """Each row's keys seen, its largest p s (heads of zeros aside, s at least 2^-96) and the s of that."""
    T, H, _ = q.shape
    KV = cache.k.shape[3]
    seen, peak, at = (torch.zeros(T, H, dtype=torch.float64, device="cuda") for _ in range(3))
    # the same form again, over values that are one number a token: all of its head's are alike
    qs = q_start.tolist()
    page = cache.k.shape[2]
    for i, s in enumerate(seqs.tolist()):
        L, a, b = int(cache.length[s]), qs[i], qs[i + 1]
        if L == 0 or a == b:
            continue
        pages = cache.table[s, :-(-L // page)].long()
        ks = cache.k_scale[0][pages].double().transpose(-1, -2).flatten(0, 1)[:L]
        vs = cache.v_scale[0][pages].double().transpose(-1, -2).flatten(0, 1)[:L]
        k = cache.k[0][pages].double().flatten(0, 1)[:L] * ks[..., None]
        some = (cache.v[0][pages] != 0).any(-1).flatten(0, 1)[:L]
        vs = torch.where(some, vs, 0.0).clamp_min(2.0 ** -96).repeat_interleave(H // KV, 1)
        own = L - (b - a)
        j = torch.arange(L, device="cuda")[None]
        if masks is None:
            p = torch.arange(own, L, device="cuda")[:, None]
            sees = (j <= p) if causal else torch.ones(b - a, L, dtype=torch.bool, device="cuda")
        else:
            bits = torch.tensor(masks[i], device="cuda")
            p = (own + bits.sum(1) - 1)[:, None]
            sees = (j < own).expand(b - a, L).clone()
        if window >= 0:
            sees = sees & (((j - p).abs() <= window) | (j < sinks))
        if masks is not None:
            sees[:, max(own, 0):] = bits[:, max(own, 0) - own:]
        x = torch.einsum("thd,jhd->thj", q[a:b].double(), k.repeat_interleave(H // KV, 1)) * scale
        w = torch.exp(x - lse[a:b][..., None]).masked_fill(~sees[:, None], 0.0) * vs.T[None]
        peak[a:b], arg = w.max(-1)
        at[a:b] = vs.T[None].expand(b - a, H, L).gather(-1, arg[..., None])[..., 0]
        seen[a:b] = sees.sum(-1)[:, None].double()
    return seen, peak, at


def assert_scaled(torch, cache, got, q, seqs, q_start, causal, window, scale, name, sinks=0, masks=None):
    out, mag, ref, big = sight64(torch, cache, 0, q, seqs, q_start, causal, window, scale, sinks, masks)
    seen, peak, at = peaks64(torch, cache, q, seqs, q_start, causal, window, scale, ref, sinks, masks)
    sums = seen * at * 2.0 ** -142 + 2.0 ** -20
    logit = 2.0 ** -18 * (1 + big)
    rel = 2.0 ** -11 * 1.01 + 2 * logit + 2.0 ** -18 + sums
    tol = UNIT[name] * 1.01 * out.abs() + TINY[name] + rel[..., None] * mag + (2.0 ** -25 * 127 * seen * peak)[..., None]
    y, lse = got
    assert not torch.isnan(y).any()
    off = (y.double() - out).abs() - tol
    worst = ((y.double() - out).norm(dim=-1) / out.norm(dim=-1).clamp_min(1e-300)).max().item()
    assert off.max().item() <= 0, f"a row is off by {worst:.3g} of its size"
    empty = torch.isinf(ref)
    assert torch.equal(torch.isinf(lse), empty) and (lse[empty] < 0).all()
    assert ((lse.double() - ref).abs() - logit - sums - 4 * 2.0 ** -24 * 256)[~empty].max().item() <= 0


def random_scales(torch, cache, g, low, high):
    """v's scales of held tokens times 2^x, x from low to high."""
    cache.v_scale.mul_(torch.exp2(low + (high - low) * torch.rand(cache.v_scale.shape, generator=g, device="cuda")))


def some_heads(torch, cache, g, part):
    """[layers][n_pages][kv][page] truth values; the tokens' own order, for codes, is its transpose."""
    return torch.rand(cache.v_scale.shape, generator=g, device="cuda") < part


def zero_heads(torch, cache, heads):
    """As a store leaves heads of zeros."""
    cache.v.masked_fill_(heads.transpose(-1, -2)[..., None], 0)
    cache.v_scale.masked_fill_(heads, 1.0)


def outliers(torch, cache, g, low, high, part=0.01):
    heads = some_heads(torch, cache, g, part)
    up = torch.exp2(low + (high - low) * torch.rand(cache.v_scale.shape, generator=g, device="cuda"))
    cache.v_scale.copy_(torch.where(heads, cache.v_scale * up, cache.v_scale))
    return heads


def light_outliers(torch, cache, g, q):
    """Large tokens that every row sees with a weight of about e^-60."""
    q.copy_(q.abs())
    heads = outliers(torch, cache, g, 20, 50)
    D = q.shape[-1]
    cache.k.masked_fill_(heads.transpose(-1, -2)[..., None], -127)
    # the sum of |2 randn| over D dimensions is 1.6 D
    cache.k_scale.masked_fill_(heads & ~torch.isnan(cache.k_scale), 60 * D ** 0.5 / (127 * 1.6 * D))


SPREADS = {
    "wide": lambda t, c, g, q: random_scales(t, c, g, -10, 10),
    "zeros": lambda t, c, g, q: (random_scales(t, c, g, -9, -8), zero_heads(t, c, some_heads(t, c, g, 0.1))),
    "zeros among tiny ones": lambda t, c, g, q: (random_scales(t, c, g, -26, -25), zero_heads(t, c, some_heads(t, c, g, 0.02))),
    "ones": lambda t, c, g, q: c.v_scale.masked_fill_(~t.isnan(c.v_scale), 1.0),  # of heads that are not zeros
    "outliers": lambda t, c, g, q: outliers(t, c, g, 20, 60),
    "light outliers": lambda t, c, g, q: light_outliers(t, c, g, q),
}
FORMS = ["one token", "ragged decode", "long", "odd group", "prompts", "one key head each", "group of 48", "prompts behind a prefix", "packed prefix",
         "packed prefix, heads of 128", "packed prefix, small heads", "packed prefix, queries reach into it"]


@pytest.mark.parametrize("causal,window,sinks", [(True, -1, 0), (False, 37, 0), (True, 20, 3)])
@pytest.mark.parametrize("case", FORMS)
@pytest.mark.parametrize("spread", list(SPREADS))
def test_scales_of_many_sizes(e2c, torch_cuda, spread, case, causal, window, sinks):
    torch = torch_cuda
    lens, queries, shared, H, KV, D, page = CASES[case]
    cache, q, seqs, q_start, max_q = make_codes(e2c, torch, 31, lens, queries, shared, H, KV, D, page, "bf16", spread=0.3)
    SPREADS[spread](torch, cache, torch.Generator(device="cuda").manual_seed(len(case)), q)
    got = cache.attention(0, q, seqs, q_start, max_q, shared=shared, causal=causal, window=window, sinks=sinks, lse=True)
    e2c.check()
    assert_scaled(torch, cache, got, q, seqs, q_start, causal, window, D ** -0.5, "bf16", sinks)


@pytest.mark.parametrize("rows,H,KV,D", [(4, 8, 2, 128), (9, 8, 2, 128), (40, 4, 2, 64), (30, 2, 1, 256), (3, 2, 2, 64)])
@pytest.mark.parametrize("spread", ["zeros", "outliers"])
def test_scales_of_many_sizes_in_trees(e2c, torch_cuda, spread, rows, H, KV, D):
    """Large tokens on other branches, and zeros."""
    torch = torch_cuda
    rng = np.random.default_rng(rows)
    lens = [rows + x for x in (0, 70, 1000)]
    cache, q, seqs, q_start, max_q = make_codes(e2c, torch, 32, lens, [rows] * 3, 0, H, KV, D, 16, "f16", spread=0.3)
    g = torch.Generator(device="cuda").manual_seed(rows)
    if spread == "zeros":
        random_scales(torch, cache, g, -6, -5)  # fp16's result keeps its bits
        zero_heads(torch, cache, some_heads(torch, cache, g, 0.2))
    else:
        outliers(torch, cache, g, 5, 8, 0.1)
    parents = [random_parents(rng, rows) for _ in lens]
    tree, _ = cache.tree(dev(torch, sum(parents, [])), seqs, q_start, max_q)
    got = cache.attention(0, q, seqs, q_start, max_q, tree=tree, lse=True)
    e2c.check()
    assert_scaled(torch, cache, got, q, seqs, q_start, True, -1, D ** -0.5, "f16", 0, [tree_mask(p) for p in parents])


@pytest.mark.parametrize("rows", [2, 100])
def test_a_large_token_out_of_sight_changes_nothing(e2c, torch_cuda, rows):
    """The last token of all, which only the last row sees."""
    torch = torch_cuda
    cache, q, seqs, q_start, max_q = make_codes(e2c, torch, 33, [300], [rows], 0, 4, 2, 128, 16, "bf16", spread=0.3)
    was, lse0 = cache.attention(0, q, seqs, q_start, max_q, lse=True)
    cache.v_scale[0, cache.table[0, 299 // 16].long(), :, 299 % 16] *= 2.0 ** 40
    now, lse = cache.attention(0, q, seqs, q_start, max_q, lse=True)
    e2c.check()
    assert torch.equal(now[:-1], was[:-1]) and torch.equal(lse[:-1], lse0[:-1])
    assert not torch.equal(now[-1], was[-1])


@pytest.mark.parametrize("rows", [1, 64])
def test_stored_zeros_beside_small_values(e2c, torch_cuda, rows):
    """From the store on: a first token whose value is zero and which draws half of the weight."""
    torch = torch_cuda
    H, KV, D, L = 4, 2, 128, 700
    cache = e2c.PageCache.new(1, 50, 16, KV, D, 1, 50, torch.int8)
    seqs = dev(torch, [0])
    cache.append(seqs, dev(torch, [L]))
    g = torch.Generator(device="cuda").manual_seed(rows)
    q, k, v = (torch.randn(L, h, D, generator=g, device="cuda") for h in (H, KV, KV))
    v *= 1e-3
    q[..., 0], k[..., 0], k[0], v[0] = 8.0, 0.0, 0.0, 0.0
    k[0, :, 0] = 11.0
    ones, none = torch.ones(L, 1, device="cuda"), torch.zeros(L, 1, device="cuda")  # no rotation
    x = cache.store(0, q.bfloat16(), k.bfloat16(), v.bfloat16(), ones, none, seqs, dev(torch, [0, L]))
    assert (cache.v_scale[0, cache.table[0, 0].long(), :, 0] == 1).all()
    x, starts = x[L - rows:].contiguous(), dev(torch, [0, rows])
    got = cache.attention(0, x, seqs, starts, rows, lse=True)
    e2c.check()
    assert_scaled(torch, cache, got, x, seqs, starts, True, -1, D ** -0.5, "bf16")


@pytest.mark.parametrize("low,high,part", [(100, 118, 1.0), (116, 118, 0.02), (-104, -100, 1.0), (-104, -90, 1.0), (-100, 100, 1.0)])
@pytest.mark.parametrize("rows,H,KV,D", [(1, 8, 2, 128), (16, 1, 1, 64), (3, 8, 4, 256), (60, 4, 2, 64), (100, 2, 1, 256), (33, 4, 1, 128)])
def test_largest_and_smallest_scales(e2c, torch_cuda, low, high, part, rows, H, KV, D):
    torch = torch_cuda
    cache, q, seqs, q_start, max_q = make_codes(e2c, torch, 34, [300, 45], [rows, min(rows, 45)], 0, H, KV, D, 16, "bf16", spread=0.0)
    g = torch.Generator(device="cuda").manual_seed(rows)
    cache.v_scale.mul_(32)  # about 1: a head's largest of D normal values is 2.5 to 3
    if part == 1.0:
        random_scales(torch, cache, g, low, high)
    else:
        outliers(torch, cache, g, low, high, part)
    got = cache.attention(0, q, seqs, q_start, max_q, lse=True)
    e2c.check()
    assert_scaled(torch, cache, got, q, seqs, q_start, True, -1, D ** -0.5, "bf16")


@pytest.mark.parametrize("rows,H,KV,D", [(1, 8, 2, 128), (2, 8, 1, 64), (3, 8, 4, 256), (60, 4, 2, 64), (100, 2, 1, 256), (33, 4, 1, 128)])
@pytest.mark.parametrize("up", [False, True])
def test_scales_in_steps(e2c, torch_cuda, up, rows, H, KV, D):
    """Runs of tokens whose values are 2^180 times the others': the weights of the small ones count all the same."""
    torch = torch_cuda
    cache, q, seqs, q_start, max_q = make_codes(e2c, torch, 35, [900], [rows], 0, H, KV, D, 16, "bf16", spread=0.0)
    t = torch.arange(900, device="cuda")
    at = torch.where((t // 150 % 2 == 1) == up, 90.0, -90.0)
    pages = cache.table[0, :57].long()
    size = torch.exp2(torch.nn.functional.pad(at, (0, 912 - 900))).view(57, 1, 16)
    cache.v_scale[0, pages] *= size
    got = cache.attention(0, q, seqs, q_start, max_q, lse=True)
    e2c.check()
    assert_scaled(torch, cache, got, q, seqs, q_start, True, -1, D ** -0.5, "bf16")


@pytest.mark.parametrize("rows,H,KV,D", [(1, 8, 1, 128), (2, 16, 2, 64), (3, 10, 2, 256), (40, 4, 2, 128)])
@pytest.mark.parametrize("by", [2.0 ** 60, 1e38, 2.0 ** -60])
def test_a_query_of_another_size_changes_no_other(e2c, torch_cuda, by, rows, H, KV, D):
    """Rows of one product, whose queries are heads of very different sizes."""
    torch = torch_cuda
    cache, q, seqs, q_start, max_q = make_codes(e2c, torch, 36, [500, 70], [rows] * 2, 0, H, KV, D, 16, "bf16", spread=0.3)
    was, lse0 = cache.attention(0, q, seqs, q_start, max_q, lse=True)
    odd = q.clone()
    odd[rows - 1, 1] *= by
    now, lse = cache.attention(0, odd, seqs, q_start, max_q, lse=True)
    e2c.check()
    same = torch.ones(2 * rows, H, dtype=torch.bool, device="cuda")
    same[rows - 1, 1] = False
    assert torch.equal(now[same], was[same]) and torch.equal(lse[same], lse0[same])
    assert not torch.equal(now[~same], was[~same])
