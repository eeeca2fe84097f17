"""Rotary positions, the paged cache and attention over it on the GPU, against plain 64-bit forms.

Tolerances, from the arithmetic (u: unit roundoff of the type, 2^-p for its p significant
bits: 2^-8 bf16, 2^-11 fp16, 2^-24 fp32):
  rope       two products and a sum in fp32: 4 * 2^-24 (|a| + |b|), and one rounding to the output type
  attention  the probabilities are rounded to the 16-bit type before the second product, the result is
             rounded once: u sum p|v| + u |out|, with p and the sums in fp32 (relative 2^-20 covers
             exp2's approximation and a logit's fp32 accumulation); fp16 probabilities below 2^-14 of
             the largest lose 2^-25 absolutely each
  lse        fp32: the largest logit's accumulation error and a logarithm
  page operations are exact.
"""
from __future__ import annotations

import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

DT = {"bf16": "bfloat16", "f16": "float16", "f32": "float32"}
UNIT = {"bf16": 2.0 ** -8, "f16": 2.0 ** -11, "f32": 2.0 ** -24}
TINY = {"bf16": 0.0, "f16": 2.0 ** -25, "f32": 0.0}  # half the smallest step of a subnormal


def turn64(torch, x, cos, sin, pos, interleaved, transpose):
    """The rotation of each pair in 64 bits, and the sum of magnitudes each result is made of."""
    x, half = x.double(), cos.shape[1]
    c, s = cos.double()[pos.long()][:, None], sin.double()[pos.long()][:, None]
    if transpose:
        s = -s
    at = torch.arange(half, device=x.device)
    i, j = (2 * at, 2 * at + 1) if interleaved else (at, at + half)
    y, mag = x.clone(), x.abs().clone()
    y[..., i], y[..., j] = x[..., i] * c - x[..., j] * s, x[..., j] * c + x[..., i] * s
    mag[..., i] = mag[..., j] = (x[..., i].abs() + x[..., j].abs()) * torch.maximum(c.abs(), s.abs())
    return y, mag


def assert_rope(got, want, mag, name):
    tol = UNIT[name] * want.abs() + TINY[name] + 4 * 2.0 ** -24 * mag
    off = (got.double() - want).abs() - tol
    assert off.max().item() <= 0, f"off by {off.max().item():.3g} past the tolerance"


# ------------------------------------------------------------------------------------------ rotary positions
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("backward", [False, True])
@pytest.mark.parametrize("xt,yt", [("bf16", "bf16"), ("f16", "f16"), ("f32", "f32"), ("f32", "bf16"), ("f32", "f16")])
@pytest.mark.parametrize("T,H,D,rot", [(1, 1, 64, 64), (7, 5, 128, 32), (33, 12, 256, 256), (130, 3, 80, 80), (5, 2, 34, 6),
                                       (3, 9, 2, 2), (61, 4, 96, 24)])
def test_rope(e2c, torch_cuda, T, H, D, rot, xt, yt, backward, interleaved):
    torch = torch_cuda
    g = torch.Generator(device="cuda").manual_seed(T * H + D)
    cos, sin = e2c.rope_table(500, rot)
    x = torch.randn(T, H, D, generator=g, device="cuda").to(getattr(torch, DT[xt]))
    pos = torch.randint(0, 500, (T,), generator=g, device="cuda", dtype=torch.int32)
    y = e2c.rope(x, cos, sin, pos, interleaved=interleaved, backward=backward, dtype=getattr(torch, DT[yt]))
    e2c.check()
    assert_rope(y, *turn64(torch, x, cos, sin, pos, interleaved, backward), yt)


@pytest.mark.parametrize("interleaved", [False, True])
def test_rope_strides_and_in_place(e2c, torch_cuda, interleaved):
    """Rows of a wider matrix, at aligned and odd offsets, in place; the columns beside them stay."""
    torch = torch_cuda
    cos, sin = e2c.rope_table(64, 32)
    for width, at in ((4 * 64 + 24, 8), (4 * 64 + 3, 1)):
        rows = torch.randn(19, width, device="cuda").bfloat16()
        before = rows.clone()
        x = rows[:, at:at + 256].unflatten(1, (4, 64))
        want, mag = turn64(torch, x, cos, sin, torch.arange(19, device="cuda"), interleaved, False)
        e2c.rope(x, cos, sin, interleaved=interleaved, out=x)
        e2c.check()
        assert_rope(x, want, mag, "bf16")
        assert torch.equal(rows[:, :at], before[:, :at]) and torch.equal(rows[:, at + 256:], before[:, at + 256:])


def test_rope_gradient_against_differences(e2c, torch_cuda):
    """<g, R(x + h d) - R(x)> / h == <R^T g, d>: the map is linear, so the difference is exact up to fp32."""
    torch = torch_cuda
    g = torch.Generator(device="cuda").manual_seed(5)
    cos, sin = e2c.rope_table(100, 48, scaling=e2c.RopeScaling(e2c.ROPE_BY_PAIRS, 32, 8.0, 0, 0, 0))
    for inter in (False, True):
        x, d, w = (torch.randn(20, 3, 64, generator=g, device="cuda") for _ in range(3))
        step = e2c.rope(x + d, cos, sin, interleaved=inter).double() - e2c.rope(x, cos, sin, interleaved=inter).double()
        left = (w.double() * step).sum().item()
        right = (e2c.rope(w, cos, sin, interleaved=inter, backward=True).double() * d.double()).sum().item()
        scale = (w.double().abs() * (x.abs() + d.abs()).double()).sum().item()
        assert abs(left - right) <= 16 * 2.0 ** -24 * scale


def test_rope_position_outside_the_table(e2c, torch_cuda):
    """Taken as position 0 (no rotation) and reported; the other rows are right."""
    torch = torch_cuda
    cos, sin = e2c.rope_table(10, 64)
    x = torch.randn(4, 2, 64, device="cuda")
    pos = torch.tensor([3, 10, -1, 2 ** 31 - 1], dtype=torch.int32, device="cuda")
    y = e2c.rope(x, cos, sin, pos)
    with pytest.raises(e2c.E2CudaError, match="position outside"):
        e2c.check()
    assert torch.equal(y[1:], x[1:])
    assert_rope(y[:1], *turn64(torch, x[:1], cos, sin, pos[:1], False, False), "f32")


def table64(rot, theta, kind, factor=1.0, original=0, fast=0.0, slow=0.0, gain=0.0):
    """The scaled frequencies and the gain, written from the definitions."""
    i = np.arange(rot // 2)
    f = theta ** (-2.0 * i / rot)
    if kind == "linear":
        f = f / factor
    if kind == "ntk":
        f = (theta * factor ** (rot / (rot - 2.0))) ** (-2.0 * i / rot)
    if kind == "rotations":
        turns = original * f / (2 * math.pi)
        keep = np.clip((turns - (slow or 1.0)) / ((fast or 4.0) - (slow or 1.0)), 0, 1)
        f = keep * f + (1 - keep) * f / factor
    if kind == "pairs":
        def pair(t):
            return rot * math.log(original / (t * 2 * math.pi)) / (2 * math.log(theta))
        a, b = max(math.floor(pair(fast or 32.0)), 0), min(math.ceil(pair(slow or 1.0)), rot - 1)
        ramp = np.clip((i - a) / max(b - a, 1e-3), 0, 1)
        f = f / factor * ramp + f * (1 - ramp)
        gain = gain or 0.1 * math.log(factor) + 1.0
    return f, gain or 1.0


@pytest.mark.parametrize("rot,theta", [(64, 1e4), (256, 1e6), (2, 1e4), (512, 5e5)])
@pytest.mark.parametrize("kind,extra", [("plain", {}), ("linear", dict(factor=4.0)), ("ntk", dict(factor=8.0)),
                                        ("rotations", dict(factor=8.0, original=8192)),
                                        ("rotations", dict(factor=2.0, original=512, fast=16.0, slow=2.0)),
                                        ("pairs", dict(factor=16.0, original=4096)),
                                        ("pairs", dict(factor=4.0, original=2048, gain=1.5))])
def test_rope_table(e2c, torch_cuda, rot, theta, kind, extra):
    """Every entry within fp32 rounding of the 64-bit value, at positions up to 300000."""
    if kind == "ntk" and rot == 2:
        pytest.skip("rot / (rot - 2)")
    kinds = dict(plain=0, linear=1, ntk=2, rotations=3, pairs=4)
    s = e2c.RopeScaling(kind=kinds[kind], **extra)
    P = 300001
    cos, sin = e2c.rope_table(P, rot, theta, s)
    e2c.check()
    f, gain = table64(rot, float(np.float32(theta)), kind, **extra)
    for at in (0, 1, 77, 4095, 131072, P - 1):
        a = at * f
        # fp32 rounding, and 64-bit rounding of an angle up to 3e5
        tol = abs(gain) * (2.0 ** -24 + 1e-9)
        assert np.abs(cos[at].cpu().numpy() - gain * np.cos(a)).max() <= tol
        assert np.abs(sin[at].cpu().numpy() - gain * np.sin(a)).max() <= tol


# ------------------------------------------------------------------------------------------ page operations
class Model:
    """The cache's rules, one sequence at a time on the host: values are (layer, page, slot) tags."""

    def __init__(self, n_pages, page, max_seqs, max_blocks):
        self.page, self.max_blocks = page, max_blocks
        self.table = np.zeros((max_seqs, max_blocks), np.int64)
        self.len, self.refs = np.zeros(max_seqs, np.int64), np.zeros(n_pages, np.int64)
        self.data = np.arange(n_pages)  # what each page holds

    def blocks(self, s):
        return -(-self.len[s] // self.page)

    def fork(self, parents, children):
        for a, c in zip(parents, children):
            b = self.blocks(a)
            self.table[c, :b] = self.table[a, :b]
            np.add.at(self.refs, self.table[a, :b], 1)
            self.len[c] = self.len[a]

    def append(self, seqs, counts):
        """False (and nothing done) when there are too few pages."""
        refs, plan, need = self.refs.copy(), [], 0
        for s, c in zip(seqs, counts):
            b0, b1 = self.blocks(s), -(-(self.len[s] + c) // self.page)
            cow = c > 0 and self.len[s] % self.page != 0 and refs[self.table[s, b0 - 1]] > 1
            plan.append((s, c, b0, b1, cow))
            need += b1 - b0 + cow
        free = np.flatnonzero(refs == 0)
        if need > len(free):
            return False
        at = 0
        for s, c, b0, b1, cow in plan:
            if cow:
                old, new = self.table[s, b0 - 1], free[at]
                at += 1
                self.data[new] = self.data[old]
                self.refs[old] -= 1
                self.refs[new] = 1
                self.table[s, b0 - 1] = new
            k = b1 - b0
            self.table[s, b0:b1] = free[at:at + k]
            self.refs[free[at:at + k]] = 1
            at += k
            self.len[s] += c
        return True

    def free(self, seqs):
        for s in seqs:
            np.add.at(self.refs, self.table[s, :self.blocks(s)], -1)
            self.len[s] = 0

    def compact(self):
        used = int((self.refs > 0).sum())
        src, dst = np.flatnonzero(self.refs[used:] > 0) + used, np.flatnonzero(self.refs[:used] == 0)
        to = np.arange(len(self.refs))
        to[src] = dst
        self.data[dst], self.refs[dst], self.refs[src] = self.data[src], self.refs[src], 0
        for s in range(len(self.len)):
            b = self.blocks(s)
            self.table[s, :b] = to[self.table[s, :b]]
        return used


def same_state(cache, m, tags=None):
    assert np.array_equal(cache.length.cpu().numpy(), m.len)
    assert np.array_equal(cache.refs.cpu().numpy(), m.refs)
    t = cache.table.cpu().numpy()
    for s in range(len(m.len)):
        assert np.array_equal(t[s, :m.blocks(s)], m.table[s, :m.blocks(s)]), s
    if tags is not None:  # every element of a page carries the page's first content
        import torch

        for x, shift in ((cache.k, 0), (cache.v, 7)):
            want = tags[torch.as_tensor(m.data, device=x.device)]
            for layer in range(x.shape[0]):
                assert torch.equal(x[layer].flatten(1), (want + layer + shift).to(x.dtype)[:, None].expand(-1, x[layer, 0].numel()))


def tagged(e2c, torch, layers, n_pages, page, kv, dim, max_seqs, max_blocks, dtype):
    cache = e2c.PageCache.new(layers, n_pages, page, kv, dim, max_seqs, max_blocks, getattr(torch, DT[dtype]))
    tags = torch.arange(n_pages, device="cuda") % 190  # exact in bf16 with the layer added
    for x, shift in ((cache.k, 0), (cache.v, 7)):
        for layer in range(layers):
            x[layer].copy_((tags + layer + shift).to(x.dtype)[:, None, None, None].expand(x[layer].shape))
    return cache, tags


@pytest.mark.parametrize("n_pages,page,kv,dim,layers,max_seqs,dtype", [(40, 8, 1, 64, 1, 6, "bf16"), (333, 16, 2, 128, 3, 40, "f16"),
                                                                      (5001, 32, 1, 64, 2, 1500, "bf16"),
                                                                      (97, 64, 3, 256, 5, 9, "bf16"), (20, 1024, 1, 64, 1, 4, "f16")])
def test_page_operations_follow_the_rules(e2c, torch_cuda, n_pages, page, kv, dim, layers, max_seqs, dtype):
    """Random forks, appends (some too large for the pool), frees, compactions: tables, counts and every
    page's contents equal the host model's after each."""
    torch = torch_cuda
    rng = np.random.default_rng(n_pages)
    max_blocks = 12
    cache, tags = tagged(e2c, torch, layers, n_pages, page, kv, dim, max_seqs, max_blocks, dtype)
    m = Model(n_pages, page, max_seqs, max_blocks)

    def dev(v):
        return torch.tensor(np.asarray(v), dtype=torch.int32, device="cuda")

    for step in range(40):
        live, idle = np.flatnonzero(m.len > 0), np.flatnonzero(m.len == 0)
        op = rng.choice(["append", "append", "fork", "free", "compact"])
        if op == "append":
            seqs = rng.permutation(max_seqs)[:rng.integers(1, max_seqs + 1)]
            room = max_blocks * page - m.len[seqs]
            counts = np.minimum(rng.integers(0, 2 * page + 2, len(seqs)), room)
            cache.append(dev(seqs), dev(counts))
            if not m.append(seqs, counts):
                with pytest.raises(e2c.E2CudaError, match="not enough free pages"):
                    e2c.check()
        elif op == "fork" and len(live) and len(idle):
            k = rng.integers(1, len(idle) + 1)
            parents, children = rng.choice(live, k), rng.permutation(idle)[:k]
            cache.fork(dev(parents), dev(children))
            m.fork(parents, children)
        elif op == "free":
            seqs = rng.permutation(max_seqs)[:rng.integers(1, max_seqs // 2 + 2)]
            cache.free(dev(seqs))
            m.free(seqs)
        elif op == "compact":
            used = torch.full((1,), -1, dtype=torch.int32, device="cuda")
            cache.compact(used)
            assert used.item() == m.compact()
        e2c.check()
        same_state(cache, m, tags)
    assert (m.refs >= 0).all()


def test_sharers_growing_in_one_call_each_get_a_copy(e2c, torch_cuda):
    torch = torch_cuda
    cache, tags = tagged(e2c, torch, 2, 16, 16, 2, 64, 4, 4, "bf16")
    m = Model(16, 16, 4, 4)

    def dev(v):
        return torch.tensor(v, dtype=torch.int32, device="cuda")

    for op, a, b in (("append", [0], [21]), ("fork", [0, 0, 0], [1, 2, 3]), ("append", [3, 1, 0, 2], [1, 12, 1, 0])):
        getattr(cache, op)(dev(a), dev(b))
        assert getattr(m, op)(a, b) in (True, None)
    e2c.check()
    same_state(cache, m, tags)


def test_bad_entries_are_left_out_and_reported(e2c, torch_cuda):
    torch = torch_cuda
    cache, tags = tagged(e2c, torch, 1, 32, 8, 1, 64, 5, 3, "bf16")
    m = Model(32, 8, 5, 3)

    def dev(v):
        return torch.tensor(v, dtype=torch.int32, device="cuda")

    def reported(match):
        with pytest.raises(e2c.E2CudaError, match=match):
            e2c.check()

    # outside the cache, a negative count, more tokens than the table has room for
    cache.append(dev([7, 0, -1, 1, 2]), dev([1, 9, 1, -3, 25]))
    m.append([0], [9])
    reported("outside the cache")
    same_state(cache, m, tags)
    # a child in use, a child outside, a parent outside, a sequence that is its own child
    cache.append(dev([1]), dev([4]))
    m.append([1], [4])
    cache.fork(dev([0, 0, 9, 2]), dev([1, 5, 2, 2]))
    reported("outside the cache")
    same_state(cache, m, tags)
    cache.fork(dev([0]), dev([3]))
    m.fork([0], [3])
    cache.free(dev([-4, 0, 5]))
    m.free([0])
    reported("outside the cache")
    same_state(cache, m, tags)
    cache.copy(dev([31, 40, 2, -1]), dev([30, 4, -2, 7]))  # 31 -> 30 is right, -1 asks for nothing
    m.data[30] = m.data[31]
    reported("outside the cache")
    same_state(cache, m, tags)


def test_append_refuses_more_than_the_pool_and_leaves_it(e2c, torch_cuda):
    torch = torch_cuda
    cache, tags = tagged(e2c, torch, 1, 5, 8, 1, 64, 3, 8, "f16")
    m = Model(5, 8, 3, 8)

    def dev(v):
        return torch.tensor(v, dtype=torch.int32, device="cuda")

    cache.append(dev([0, 1]), dev([17, 16]))
    m.append([0, 1], [17, 16])
    e2c.check()
    same_state(cache, m, tags)
    cache.append(dev([2]), dev([1]))
    with pytest.raises(e2c.E2CudaError, match="not enough free pages"):
        e2c.check()
    same_state(cache, m, tags)
    cache.append(dev([0, 1]), dev([7, 0]))  # room in the last page
    m.append([0, 1], [7, 0])
    e2c.check()
    same_state(cache, m, tags)


# ------------------------------------------------------------------------------------------ a batch over the cache
def make_batch(e2c, torch, seed, lens, queries, shared, H, KV, D, page, dtype, layers=1, spare=5, poison=float("nan")):
    """A cache whose sequences share their first `shared` tokens, with NaN wherever nothing is held, table
    entries past a sequence's pages that point anywhere, and the batch in another order than the cache."""
    rng = np.random.default_rng(seed)
    dt = getattr(torch, DT[dtype])
    n = len(lens)
    g = torch.Generator(device="cuda").manual_seed(seed)
    tails = [max(0, L - shared) for L in lens]
    own = [-(-t // page) for t in tails]
    n_pages = shared // page + sum(own) + spare
    max_blocks = max(1, shared // page + max(own, default=0)) + 2
    cache = e2c.PageCache.new(layers, n_pages, page, KV, D, n + 1, max_blocks, dt)
    order = rng.permutation(n_pages)
    wild = np.array([-1, n_pages, 2 ** 31 - 1, -2 ** 31, 0])
    table = wild[rng.integers(0, len(wild), (n + 1, max_blocks))]
    refs = np.zeros(n_pages, np.int64)
    at = shared // page
    for i, (L, b) in enumerate(zip(lens, own)):
        s = min(-(-L // page), shared // page)
        table[i, :s] = order[:s]
        table[i, shared // page:shared // page + b] = order[at:at + b]
        np.add.at(refs, table[i, :-(-L // page)], 1)
        at += b
    cache.table.copy_(torch.tensor(table, dtype=torch.int32))
    cache.length[:n] = torch.tensor(lens, dtype=torch.int32, device="cuda")
    cache.refs.copy_(torch.tensor(refs, dtype=torch.int32))
    for x in (cache.k, cache.v):
        x.copy_(torch.randn(x.shape, generator=g, device="cuda"))
        held = torch.zeros(n_pages, page, dtype=torch.bool)
        for i, L in enumerate(lens):
            for b in range(-(-L // page)):
                held[table[i, b], :min(page, L - b * page)] = True
        x.masked_fill_(~held.cuda()[None, :, :, None, None], poison)
    seqs = rng.permutation(n)
    q_start = np.concatenate([[0], np.cumsum([queries[s] for s in seqs])])
    T = int(q_start[-1])
    q = (2.0 * torch.randn(T, H, D, generator=g, device="cuda")).to(dt)

    def dev(v):
        return torch.tensor(np.asarray(v), dtype=torch.int32, device="cuda")

    return cache, q, dev(seqs), dev(q_start), max(1, max(queries))


def attention64(torch, cache, layer, q, seqs, q_start, causal, window, scale):
    """out, sum p|v|, lse and the largest |logit| in 64 bits, a sequence at a time."""
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
        k = cache.k[layer][pages].flatten(0, 1)[:L].double().repeat_interleave(H // KV, 1)
        v = cache.v[layer][pages].flatten(0, 1)[:L].double().repeat_interleave(H // KV, 1)
        p = torch.arange(L - (b - a), L, device="cuda")[:, None]
        j = torch.arange(L, device="cuda")[None]
        sees = torch.ones(b - a, L, dtype=torch.bool, device="cuda")
        if causal:
            sees &= j <= p
        if window >= 0:
            sees &= (j - p).abs() <= window
        x = torch.einsum("thd,jhd->htj", q[a:b].double(), k) * scale
        x = x.masked_fill(~sees, -math.inf)
        r = torch.logsumexp(x, -1)
        w = torch.exp(x - r[..., None]).masked_fill(~sees, 0.0)
        out[a:b] = torch.einsum("htj,jhd->thd", w, v)
        mag[a:b] = torch.einsum("htj,jhd->thd", w, v.abs())
        lse[a:b] = r.T
        big[a:b] = x.abs().masked_fill(~sees, 0).amax(-1).T
    return out, mag, lse, big


def assert_attention(torch, got, lse, want, name, keys):
    out, mag, ref, big = want
    u = UNIT[name]
    # a logit's error: D products in fp32, here at most 2^-18 of its size and of the terms' (~|q||k|)
    eps = 2.0 ** -18 * (1 + big)[..., None]
    # sum p|v| covers |out| too; the two roundings may both go the same way
    tol = 2.02 * u * mag + TINY[name] * (1 + keys * 6.0) + 2 * eps * mag + 1e-7
    off = (got.double() - out).abs() - tol
    assert not torch.isnan(got).any()
    assert off.max().item() <= 0, f"off by {off.max().item():.3g} past the tolerance, error {(got.double() - out).abs().max().item():.3g}"
    if lse is not None:
        empty = torch.isinf(ref)
        assert torch.equal(torch.isinf(lse), empty) and (lse[empty] < 0).all()
        assert ((lse.double() - ref).abs() - 2.0 ** -18 * (1 + big))[~empty].max().item() <= 0


CASES = {
    # lens, queries, shared, H, KV, D, page
    "one token": ([1], [1], 0, 1, 1, 64, 8),
    "one query": ([300], [1], 0, 8, 2, 128, 16),
    "long": ([20011], [1], 0, 4, 1, 128, 32),
    "ragged decode": ([1, 5, 17, 128, 129, 700, 64, 31], [1] * 8, 0, 8, 2, 128, 16),
    "empty ones": ([0, 40, 0, 1, 128], [1, 1, 0, 0, 2], 0, 6, 2, 64, 8),
    "more queries than tokens": ([3, 60], [7, 5], 0, 4, 2, 64, 16),
    "prefix decode": ([512 + x for x in (0, 1, 16, 33, 200)], [1] * 5, 512, 8, 2, 128, 16),
    "prefix, few tokens past it": ([256] * 3 + [257] * 40, [1] * 43, 256, 10, 2, 64, 64),
    "prefix, many rows": ([640 + 3 * i for i in range(70)], [1 + i % 3 for i in range(70)], 640, 4, 1, 256, 32),
    "queries reach into the prefix": ([130, 128, 150], [9, 5, 30], 128, 4, 2, 128, 16),
    "long prefix": ([8192 + 77, 8192 + 5], [1, 2], 8192, 8, 8, 64, 128),
    "shorter than the prefix": ([64, 10, 200], [1, 1, 3], 128, 4, 2, 64, 32),
    "prompts": ([257, 100, 513], [257, 100, 300], 0, 4, 2, 256, 64),
    "prompts behind a prefix": ([1024 + 200, 1024 + 131], [200, 100], 1024, 8, 4, 128, 128),
    "odd group": ([190, 77], [33, 77], 64, 7, 1, 128, 64),
    "wide group": ([140, 300], [3, 1], 0, 128, 1, 64, 16),
    "group of 48": ([513, 40], [4, 9], 0, 96, 2, 128, 8),
    "one key head each": ([600], [600], 0, 12, 12, 64, 256),
    "large pages": ([1500, 1024, 2048], [5, 1, 64], 1024, 4, 2, 64, 1024),
    # as many sequences as make the shared tokens worth one pass for the batch
    "packed prefix": ([640 + 3 * (i % 90) for i in range(220)], [1 + i % 3 for i in range(220)], 640, 4, 2, 256, 32),
    "packed prefix, heads of 128": ([512 + (7 * i) % 130 for i in range(160)], [1 + (i % 5 == 0) for i in range(160)], 512, 10, 5, 128, 16),
    "packed prefix, small heads": ([1024 + i for i in range(70)], [2] * 70, 1024, 8, 4, 64, 128),
    "packed prefix, more row tiles than blocks": ([256 + i % 9 for i in range(500)], [1] * 500, 256, 64, 8, 64, 64),
    "packed prefix, shorter sequences": ([384, 100, 0, 390] * 90, [1] * 360, 384, 4, 2, 128, 128),
    "packed prefix, queries reach into it": ([640 + i % 4 for i in range(200)], [6] * 200, 640, 4, 2, 128, 64),
    "one item a block": ([33] * 150, [1] * 150, 0, 8, 2, 256, 32),
    "short tails, heads of 128": ([1 + (i * 11) % 300 for i in range(190)], [1 + i % 2 for i in range(190)], 0, 8, 2, 128, 8),
    "short tails, heads of 256": ([1 + (i * 13) % 400 for i in range(140)], [1 + i % 3 for i in range(140)], 0, 4, 2, 256, 16),
    "many sequences": ([1 + (i * 37) % 90 for i in range(700)], [1] * 700, 0, 2, 1, 64, 8),
}


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("causal,window", [(True, -1), (False, -1), (True, 0), (False, 37), (True, 130), (False, 0)])
@pytest.mark.parametrize("case", list(CASES))
def test_attention(e2c, torch_cuda, case, causal, window, dtype):
    """Every shape under every mask; NaN where the cache holds nothing must reach no result."""
    torch = torch_cuda
    lens, queries, shared, H, KV, D, page = CASES[case]
    cache, q, seqs, q_start, max_q = make_batch(e2c, torch, 11, lens, queries, shared, H, KV, D, page, dtype)
    scale = 1.0 / math.sqrt(D)
    out, lse = cache.attention(0, q, seqs, q_start, max_q, shared=shared, causal=causal, window=window, lse=True)
    e2c.check()
    assert_attention(torch, out, lse, attention64(torch, cache, 0, q, seqs, q_start, causal, window, scale), dtype, max(lens))
    again = cache.attention(0, q, seqs, q_start, max_q, shared=shared, causal=causal, window=window)
    assert torch.equal(again, out), "two calls differ"


@pytest.mark.parametrize("poison", [float("inf"), -float("inf"), 65504.0])
def test_attention_ignores_what_is_past_the_length(e2c, torch_cuda, poison):
    torch = torch_cuda
    for D, page in ((64, 8), (128, 64), (256, 16)):
        cache, q, seqs, q_start, max_q = make_batch(e2c, torch, 3, [70, 9, 129, 33], [1, 2, 5, 33], 0, 4, 2, D, page, "f16", poison=poison)
        out, lse = cache.attention(0, q, seqs, q_start, max_q, lse=True, causal=False)
        e2c.check()
        assert_attention(torch, out, lse, attention64(torch, cache, 0, q, seqs, q_start, False, -1, D ** -0.5), "f16", 129)


@pytest.mark.parametrize("scale", [0.0, -0.3, 4.0])
def test_attention_scales(e2c, torch_cuda, scale):
    """No scale, a negative one, and one that leaves a single key: logits in the hundreds."""
    torch = torch_cuda
    cache, q, seqs, q_start, max_q = make_batch(e2c, torch, 4, [300 + 5 * i for i in range(9)], [4] * 9, 256, 4, 2, 128, 32, "bf16")
    out, lse = cache.attention(0, q, seqs, q_start, max_q, shared=256, scale=scale, lse=True)
    e2c.check()
    assert_attention(torch, out, lse, attention64(torch, cache, 0, q, seqs, q_start, True, -1, scale), "bf16", 400)


def same_where_not_finite(torch, got, lse, want, big, name, keys):
    """NaN and infinite sums exactly where the 64-bit form has them; every other row within the tolerance."""
    out, mag, ref, _ = want
    lost = torch.isnan(out)
    assert torch.equal(torch.isnan(got), lost)
    assert torch.equal(torch.isnan(lse), torch.isnan(ref)) and torch.equal(torch.isinf(lse), torch.isinf(ref))
    endless = torch.isinf(ref)
    assert torch.equal(lse[endless] > 0, ref[endless] > 0)

    def settled(x):
        return x.masked_fill(lost, 0.0)

    fill = 0.0 if ref.isnan().any() or endless.any() else None
    sums = [x if fill is None else x.masked_fill(~torch.isfinite(ref), fill) for x in (lse, ref)]
    assert_attention(torch, settled(got), sums[0], (settled(out), settled(mag), sums[1], big), name, keys)


UNSETTLED = {
    # lens, queries, shared, KV: every item in one block; items that blocks share; a prefix read for the batch
    "undivided": ([384] * 148, [2] * 148, 0, 1),
    "divided": ([20011, 15000, 9000], [1, 3, 2], 0, 2),
    "prefix": ([512 + (7 * i) % 130 + 2 for i in range(160)], [1 + (i % 5 == 0) for i in range(160)], 512, 5),
}


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("what", ["q nan", "k nan", "k inf", "v nan"])
@pytest.mark.parametrize("form", list(UNSETTLED))
def test_attention_keeps_nan_and_infinity(e2c, torch_cuda, form, what, D, dtype):
    """A NaN in a query, a key or a value in sight, and the NaN of an infinite logit, reach the result, in
    whatever column of a tile the key lies; rows that do not see them are right."""
    torch = torch_cuda
    lens, queries, shared, KV = UNSETTLED[form]
    H = 2 * KV
    cache, q, seqs, q_start, max_q = make_batch(e2c, torch, 31, lens, queries, shared, H, KV, D, 16, dtype)
    big = attention64(torch, cache, 0, q, seqs, q_start, False, -1, D ** -0.5)[3]
    rng = np.random.default_rng(D)
    if what == "q nan":
        for t in range(0, q.shape[0], 3):
            q[t, t % H, t * 5 % D] = float("nan")
    else:
        x = cache.v if what == "v nan" else cache.k
        value = float("nan") if what.endswith("nan") else float("inf")
        for i in range(1, len(lens), 2):  # one key head of every second sequence, at every column of a tile
            j = shared + (37 * i) % (lens[i] - shared)
            x[0, int(cache.table[i, j // 16]), j % 16, i % KV, rng.integers(D)] = value
        if form == "prefix":  # and of one token that all share, in one key head
            x[0, int(cache.table[0, 300 // 16]), 300 % 16, 2, 5] = value
    out, lse = cache.attention(0, q, seqs, q_start, max_q, shared=shared, causal=False, lse=True)
    e2c.check()
    want = attention64(torch, cache, 0, q, seqs, q_start, False, -1, D ** -0.5)
    assert torch.isnan(want[0]).any() and not torch.isnan(want[0]).all()
    same_where_not_finite(torch, out, lse, want, big, dtype, max(lens))


@pytest.mark.parametrize("at", range(0, 128, 3))
def test_attention_keeps_a_nan_of_every_column(e2c, torch_cuda, at):
    """One NaN key in the first, whole tile of 300 keys."""
    torch = torch_cuda
    cache, q, seqs, q_start, max_q = make_batch(e2c, torch, 32, [300], [3], 0, 4, 2, 128, 64, "bf16")
    cache.k[0, int(cache.table[0, at // 64]), at % 64, 1, 0] = float("nan")
    out, lse = cache.attention(0, q, seqs, q_start, max_q, lse=True)
    e2c.check()
    assert torch.isnan(out[:, 2:]).all() and torch.isnan(lse[:, 2:]).all()
    assert torch.isfinite(out[:, :2]).all() and torch.isfinite(lse[:, :2]).all()


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("form", list(UNSETTLED))
def test_attention_of_infinite_logits_only(e2c, torch_cuda, form, D):
    """Every key infinite in one dimension: logits of +infinity (q > 0 there) or -infinity. No softmax of either
    exists, the sums are what they are; a row without a key in sight still gets zeros."""
    torch = torch_cuda
    lens, queries, shared, KV = UNSETTLED[form]
    lens = [0 if i == 1 and form != "prefix" else n for i, n in enumerate(lens)]
    cache, q, seqs, q_start, max_q = make_batch(e2c, torch, 33, lens, queries, shared, 2 * KV, KV, D, 16, "f16")
    cache.k[..., 0] = float("inf")
    q[..., 0] = 1.0
    q[:, 1::2, 0] = -1.0
    out, lse = cache.attention(0, q, seqs, q_start, max_q, shared=shared, causal=False, lse=True)
    e2c.check()
    counts = q_start.long().diff()
    sees = torch.repeat_interleave(cache.length[seqs.long()] > 0, counts)
    assert torch.isnan(out[sees]).all() and (out[~sees] == 0).all()
    assert (lse[sees][:, 0::2] == math.inf).all() and (lse[sees][:, 1::2] == -math.inf).all() and (lse[~sees] == -math.inf).all()


def test_attention_hides_nan_keys_out_of_sight(e2c, torch_cuda):
    """A NaN key that a row's mask leaves out does not reach it."""
    torch = torch_cuda
    for D, shared in ((64, 0), (128, 256), (256, 0)):
        cache, q, seqs, q_start, max_q = make_batch(e2c, torch, 34, [300] * 150, [4] * 150, shared, 2, 1, D, 32, "bf16")
        for i in range(150):
            cache.k[0, int(cache.table[i, 298 // 32]), 298 % 32] = float("nan")
        out, lse = cache.attention(0, q, seqs, q_start, max_q, shared=shared, lse=True)
        e2c.check()
        seen = torch.arange(600, device="cuda") % 4 >= 2  # positions 298 and 299
        assert torch.isnan(out[seen]).all() and torch.isnan(lse[seen]).all()
        assert torch.isfinite(out[~seen]).all() and torch.isfinite(lse[~seen]).all()


def test_attention_strided_rows_and_layers(e2c, torch_cuda):
    """q and out as columns of wider rows, the second layer of the cache; what lies beside out stays."""
    torch = torch_cuda
    cache, q, seqs, q_start, max_q = make_batch(e2c, torch, 5, [100, 257, 3], [2, 40, 1], 0, 6, 2, 64, 16, "bf16", layers=3)
    T = q.shape[0]
    rows = torch.randn(T, 6 * 64 + 72, device="cuda").bfloat16()
    rows[:, 8:8 + 384] = q.flatten(1)
    wide = torch.full((T, 512), 3.0, device="cuda").bfloat16()
    out = wide[:, 64:64 + 384].unflatten(1, (6, 64))
    cache.attention(1, rows[:, 8:8 + 384].unflatten(1, (6, 64)), seqs, q_start, max_q, out=out)
    e2c.check()
    assert_attention(torch, out, None, attention64(torch, cache, 1, q, seqs, q_start, True, -1, 0.125), "bf16", 257)
    assert (wide[:, :64] == 3).all() and (wide[:, 448:] == 3).all()


def test_attention_sequence_outside_the_cache(e2c, torch_cuda):
    """Its rows see nothing (zeros), it is reported, and the other entries are right."""
    torch = torch_cuda
    cache, q, seqs, q_start, max_q = make_batch(e2c, torch, 6, [50, 60, 70], [1, 1, 1], 0, 4, 2, 64, 16, "bf16")
    seqs[1] = 99
    out, lse = cache.attention(0, q, seqs, q_start, max_q, lse=True)
    with pytest.raises(e2c.E2CudaError, match="outside the cache"):
        e2c.check()
    assert (out[1] == 0).all() and torch.isinf(lse[1]).all()
    keep = torch.tensor([0, 2], device="cuda")
    want = attention64(torch, cache, 0, q[keep], seqs[keep], torch.tensor([0, 1, 2]), True, -1, 0.125)
    assert_attention(torch, out[keep], lse[keep], want, "bf16", 70)


def test_attention_refuses_too_many_heads_for_a_key_head(e2c, torch_cuda):
    torch = torch_cuda
    cache = e2c.PageCache.new(1, 4, 16, 1, 64, 2, 4, torch.bfloat16)
    q = torch.zeros(1, 129, 64, device="cuda", dtype=torch.bfloat16)
    seqs, q_start = torch.tensor([0], device="cuda").int(), torch.tensor([0, 1], device="cuda").int()
    with pytest.raises(e2c.E2CudaError, match="heads 129 over 1"):
        cache.attention(0, q, seqs, q_start, 1)
    e2c.check()


def test_host_tensors_are_refused(e2c, torch_cuda):
    """Refused on the host, whichever argument it is; and nothing of such a call is kept."""
    torch = torch_cuda
    cache, q, seqs, q_start, max_q = make_batch(e2c, torch, 41, [50, 60], [1, 2], 0, 4, 2, 64, 16, "bf16")
    k, (cos, sin) = q[:, :2].contiguous(), e2c.rope_table(64, 64)
    want = cache.attention(0, q, seqs, q_start, max_q)
    pos, out = torch.zeros(3, dtype=torch.int32, device="cuda"), torch.empty_like(q)
    calls = ((e2c.rope, [q, cos, sin], dict(pos=pos, out=out)), (cache.store, [0, q, k, k, cos, sin, seqs, q_start], dict(out=out)),
             (cache.attention, [0, q, seqs, q_start, max_q], dict(out=out)), (cache.fork, [seqs, seqs], {}),
             (cache.append, [seqs, seqs], {}), (cache.free, [seqs], {}), (cache.copy, [seqs, seqs], {}), (cache.compact, [seqs[:1]], {}))
    cache._scratch.clear()
    for f, args, kw in calls:
        for at in [*range(len(args)), *kw]:
            a, b = list(args), dict(kw)
            where = b if at in b else a
            if not torch.is_tensor(where[at]):
                continue
            where[at] = where[at].cpu()
            with pytest.raises(e2c.E2CudaError, match="cuda:0, got cpu"):
                f(*a, **b)
    assert torch.equal(cache.attention(0, q, seqs, q_start, max_q), want)
    e2c.check()


@pytest.mark.parametrize("case", ["ragged decode", "prefix decode", "packed prefix, small heads", "prompts"])
def test_attention_bound_above_the_rows(e2c, torch_cuda, case):
    """max_q is an upper bound: one above an entry's rows, and above all rows there are, gives the same."""
    torch = torch_cuda
    lens, queries, shared, H, KV, D, page = CASES[case]
    cache, q, seqs, q_start, max_q = make_batch(e2c, torch, 12, lens, queries, shared, H, KV, D, page, "bf16")
    want = attention64(torch, cache, 0, q, seqs, q_start, True, -1, D ** -0.5)
    for bound in (max_q + 1, q.shape[0], q.shape[0] + 1, 1 << 20):
        out, lse = cache.attention(0, q, seqs, q_start, bound, shared=shared, lse=True)
        e2c.check()
        assert_attention(torch, out, lse, want, "bf16", max(lens))


@pytest.mark.parametrize("wild", [-1, 1 << 20, 2 ** 31 - 1])
@pytest.mark.parametrize("D,shared", [(64, 0), (128, 0), (256, 0), (128, 512)])
def test_attention_page_outside_the_pool(e2c, torch_cuda, D, shared, wild):
    """A page that a sequence holds but the pool does not is reported, and other sequences are right."""
    torch = torch_cuda
    n = 160
    cache, q, seqs, q_start, max_q = make_batch(e2c, torch, 42, [shared + 90 + i for i in range(n)], [1] * n, shared, 8, 4, D, 16, "bf16")
    for x in (cache.k, cache.v):
        x.nan_to_num_(0.0)
    bad = int(seqs[5])
    cache.table[bad, shared // 16 + 2] = wild
    out, lse = cache.attention(0, q, seqs, q_start, max_q, shared=shared, lse=True)
    with pytest.raises(e2c.E2CudaError, match="page outside the cache"):
        e2c.check()
    keep = torch.tensor([i for i in range(n) if i != 5], device="cuda")
    starts = torch.arange(n, device="cuda")
    want = attention64(torch, cache, 0, q[keep], seqs[keep], starts, True, -1, D ** -0.5)
    assert_attention(torch, out[keep], lse[keep], want, "bf16", shared + 90 + n)


@pytest.mark.parametrize("window", [2 ** 31 - 1, 2 ** 31, 2 ** 32, 2 ** 63 - 1, -2 ** 32])
def test_attention_window_wider_than_any_sequence(e2c, torch_cuda, window):
    torch = torch_cuda
    cache, q, seqs, q_start, max_q = make_batch(e2c, torch, 43, [300, 70], [5, 40], 0, 4, 2, 64, 16, "bf16")
    for causal in (False, True):
        want = cache.attention(0, q, seqs, q_start, max_q, causal=causal)
        assert torch.equal(cache.attention(0, q, seqs, q_start, max_q, causal=causal, window=window), want)
    e2c.check()


def test_attention_past_32_bit_offsets(e2c, torch_cuda):
    """A pool of over 2^32 bytes in one layer: pages at its end are read."""
    torch = torch_cuda
    page, KV, D, n_pages = 64, 4, 256, 36000
    cache = e2c.PageCache.new(1, n_pages, page, KV, D, 2, 8, torch.bfloat16)
    for x in (cache.k, cache.v):
        x[0, -9:].normal_()
    cache.table[0, :5] = torch.arange(n_pages - 5, n_pages, device="cuda").int()
    cache.length[0] = 5 * page - 7
    cache.refs[-5:] = 1
    q = torch.randn(3, 8, D, device="cuda").bfloat16()
    seqs, q_start = torch.tensor([0], device="cuda").int(), torch.tensor([0, 3], device="cuda").int()
    out, lse = cache.attention(0, q, seqs, q_start, 3, lse=True)
    e2c.check()
    assert_attention(torch, out, lse, attention64(torch, cache, 0, q, seqs, q_start, True, -1, D ** -0.5), "bf16", 320)


def test_attention_of_one_long_prompt(e2c, torch_cuda):
    """131072 tokens in one call, over 2^24 tiles: rows at its ends and between, against 64 bits."""
    torch = torch_cuda
    T, H, KV, D = 131072, 32, 2, 64
    cache, q, seqs, q_start, max_q = make_batch(e2c, torch, 5, [T], [T], 0, H, KV, D, 128, "bf16", spare=0)
    out, lse = cache.attention(0, q, seqs, q_start, max_q, lse=True)
    e2c.check()
    for t in (0, 127, 128, 77777, T - 1):
        cache.length[0] = t + 1
        row = torch.tensor([0, 1], device="cuda").int()
        want = attention64(torch, cache, 0, q[t:t + 1], seqs, row, True, -1, D ** -0.5)
        assert_attention(torch, out[t:t + 1], lse[t:t + 1], want, "bf16", t + 1)


@pytest.mark.parametrize("n,each,shared", [(1, 16384, 0), (1536, 1, 1 << 14)])
def test_attention_of_too_large_a_batch_does_nothing(e2c, torch_cuda, n, each, shared):
    """Lengths of 2^24 make over 2^30 tiles; the call is reported and leaves the output as it was."""
    torch = torch_cuda
    cache = e2c.PageCache.new(1, 4, 128, 8, 64, n, 1 << 17, torch.bfloat16)
    cache.length.fill_(1 << 24)
    q = torch.zeros(n * each, 128, 64, device="cuda", dtype=torch.bfloat16)
    out = torch.full_like(q, 7)
    seqs = torch.arange(n, device="cuda").int()
    q_start = torch.arange(0, n * each + 1, each, device="cuda").int()
    cache.attention(0, q, seqs, q_start, each, shared=shared, causal=False, out=out)
    with pytest.raises(e2c.E2CudaError, match="too large"):
        e2c.check()
    assert (out == 7).all()
    e2c.check()


# ------------------------------------------------------------------------------------------ the cache write
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("src,dtype", [("bf16", "bf16"), ("f32", "bf16"), ("f16", "f16"), ("f32", "f16")])
@pytest.mark.parametrize("lens,queries,H,KV,D,page,rot", [([5], [5], 1, 1, 64, 8, 64), ([1, 40, 17], [1, 1, 1], 8, 2, 128, 16, 128),
                                                          ([300, 7, 129], [200, 7, 100], 6, 3, 64, 32, 16),
                                                          ([33, 64], [33, 0], 4, 2, 256, 64, 256), ([12, 9], [4, 9], 5, 5, 128, 8, 6)])
def test_store(e2c, torch_cuda, lens, queries, H, KV, D, page, rot, src, dtype, interleaved):
    """q, k rotated at their positions; k and v in their places; every other slot untouched."""
    torch = torch_cuda
    cache, _, seqs, q_start, _ = make_batch(e2c, torch, 21, lens, queries, 0, H, KV, D, page, dtype, layers=2, poison=5.0)
    T = int(q_start[-1])
    cos, sin = e2c.rope_table(512, rot)
    for pad, at in ((64, 16), (7, 3)):  # aligned rows and odd ones
        rows = torch.randn(T, (H + 2 * KV) * D + pad, device="cuda").to(getattr(torch, DT[src]))
        x = rows[:, at:at + (H + 2 * KV) * D].unflatten(1, (H + 2 * KV, D))
        q, k, v = x.split([H, KV, KV], 1)
        before = cache.k.clone(), cache.v.clone()
        got = cache.store(1, q, k, v, cos, sin, seqs, q_start, interleaved=interleaved)
        e2c.check()
        qs, place = q_start.tolist(), []
        for i, s in enumerate(seqs.tolist()):
            place += [(s, int(cache.length[s]) - (qs[i + 1] - t)) for t in range(qs[i], qs[i + 1])]
        pos = torch.tensor([p for _, p in place], device="cuda")
        assert_rope(got, *turn64(torch, q, cos, sin, pos, interleaved, False), dtype)
        page_of = torch.tensor([int(cache.table[s, p // page]) for s, p in place], device="cuda")
        slot = pos % page
        assert_rope(cache.k[1, page_of, slot], *turn64(torch, k, cos, sin, pos, interleaved, False), dtype)
        assert torch.equal(cache.v[1, page_of, slot], v.to(cache.v.dtype))
        after_k, after_v = cache.k.clone(), cache.v.clone()
        after_k[1, page_of, slot], after_v[1, page_of, slot] = before[0][1, page_of, slot], before[1][1, page_of, slot]
        assert torch.equal(after_k, before[0]) and torch.equal(after_v, before[1])


def test_store_rows_without_a_place_are_left_out(e2c, torch_cuda):
    """A sequence outside the cache, more queries than tokens, a position past the rotary table."""
    torch = torch_cuda
    cache, _, _, _, _ = make_batch(e2c, torch, 22, [4, 40], [1, 1], 0, 2, 1, 64, 8, "bf16", poison=5.0)
    cos, sin = e2c.rope_table(39, 64)

    def dev(v):
        return torch.tensor(v, dtype=torch.int32, device="cuda")

    for seqs, q_start, match in (([8], [0, 1], "outside the cache"), ([0], [0, 6], "outside the cache"),
                                 ([1], [0, 1], "position outside")):
        T, before = q_start[-1], (cache.k.clone(), cache.v.clone())
        q, kv = torch.randn(T, 2, 64, device="cuda").bfloat16(), torch.randn(T, 1, 64, device="cuda").bfloat16()
        cache.store(0, q, kv, kv, cos, sin, dev(seqs), dev(q_start))
        with pytest.raises(e2c.E2CudaError, match=match):
            e2c.check()
        if q_start[-1] == 1:
            assert torch.equal(cache.k, before[0]) and torch.equal(cache.v, before[1])


# ------------------------------------------------------------------------------------------ used together
def test_fork_append_store_attend_in_a_graph_and_on_another_stream(e2c, torch_cuda):
    """A prompt stored once, forked, each branch decoded a few tokens: eager, replayed as a graph, and on a
    second stream, all equal; and equal to each branch's prompt and tokens stored and attended alone."""
    torch = torch_cuda
    H, KV, D, page, n, steps, prompt = 4, 2, 64, 16, 3, 20, 37
    g = torch.Generator(device="cuda").manual_seed(9)
    cos, sin = e2c.rope_table(128, D)
    first = torch.randn(prompt, H + 2 * KV, D, generator=g, device="cuda")
    later = torch.randn(steps, n, H + 2 * KV, D, generator=g, device="cuda")

    def dev(v):
        return torch.tensor(v, dtype=torch.int32, device="cuda")

    children, starts, ones = dev([2, 1, 3]), dev([0, 1, 2, 3]), dev([1, 1, 1])

    def begin():
        cache = e2c.PageCache.new(1, 32, page, KV, D, 4, 8, torch.bfloat16)
        cache.append(dev([0]), dev([prompt]))
        cache.store(0, *first.split([H, KV, KV], 1), cos, sin, dev([0]), dev([0, prompt]))
        cache.fork(dev([0, 0, 0]), children)
        return cache

    def step(cache, x, stream=None):
        cache.append(children, ones, stream=stream)
        q = cache.store(0, *x.split([H, KV, KV], 1), cos, sin, children, starts, stream=stream)
        return cache.attention(0, q, children, starts, 1, shared=32, stream=stream)

    cache = begin()
    want = [step(cache, later[i]).clone() for i in range(steps)]
    e2c.check()

    other = begin()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = [step(other, later[i], side).clone() for i in range(steps)]
    e2c.check(side)
    assert all(torch.equal(a, b) for a, b in zip(want, got))

    graphed = begin()
    x = later[0].clone()
    step(graphed, x)  # the workspace is made before the capture
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = step(graphed, x)
    for i in range(1, steps):
        x.copy_(later[i])
        graph.replay()
        assert torch.equal(y, want[i])
    e2c.check()

    # each branch by itself, its tokens stored in one go
    alone = e2c.PageCache.new(1, 32, page, KV, D, 1, 8, torch.bfloat16)
    for b in range(n):
        rows = torch.cat([first, later[:, b]])
        alone.append(dev([0]), dev([prompt + steps]))
        q = alone.store(0, *rows.split([H, KV, KV], 1), cos, sin, dev([0]), dev([0, prompt + steps]))
        ref = attention64(torch, alone, 0, q, dev([0]), dev([0, prompt + steps]), True, -1, D ** -0.5)
        got = torch.stack([w[b] for w in want])
        assert_attention(torch, got, None, [r[prompt:] for r in ref], "bf16", prompt + steps)
        alone.free(dev([0]))


def test_graph_survives_a_larger_call(e2c, torch_cuda):
    """A captured call's workspace is not given back when a later call needs a larger one."""
    torch = torch_cuda
    n = 300
    cache, q, seqs, q_start, max_q = make_batch(e2c, torch, 8, [3029] * n, [1] * n, 3024, 8, 2, 128, 16, "bf16")
    few = q[:2], seqs[:2], q_start[:3], 1
    torch.cuda.synchronize()
    st = torch.cuda.Stream()
    with torch.cuda.stream(st):
        want = cache.attention(0, *few)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=st):
            got = cache.attention(0, *few)
        (before, _), = cache._scratch.values()
        cache.attention(0, q, seqs, q_start, max_q, shared=3024)
        (after, _), = cache._scratch.values()
        assert after.numel() > before.numel()
        del before
        held = [torch.full((1 << 20,), 7, device="cuda", dtype=torch.uint8) for _ in range(200)]  # what was given back
        got.zero_()
        graph.replay()
    torch.cuda.synchronize()
    e2c.check()
    assert torch.equal(got, want)
    assert all((x == 7).all() for x in held)


def test_results_belong_to_their_stream(e2c, torch_cuda):
    """Memory freed on torch's stream, where a kernel may still use it, is not what another stream's call writes."""
    torch = torch_cuda
    cos, sin = e2c.rope_table(64, 64)
    x = torch.randn(4096, 16, 64, device="cuda").bfloat16()
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    gone = torch.empty_like(x)
    at = gone.data_ptr()
    del gone
    assert torch.empty_like(x).data_ptr() == at  # torch's stream would get it again
    pos = torch.zeros(4096, device="cuda", dtype=torch.int32)
    y = e2c.rope(x, cos, sin, pos, stream=st)
    assert y.data_ptr() != at
    torch.cuda.synchronize()
    e2c.check()


def test_example_shared_and_recomputed_agree(e2c, torch_cuda):
    """The example's two ways to the same embeddings. Both round activations to int8 and attention operands to
    bf16; the difference is bf16's in attention (2^-8 of a row) carried through two layers, far below
    the 1e-3 asked of the cosine."""
    import importlib.util
    from pathlib import Path

    path = Path(__file__).resolve().parent.parent / "examples" / "prompt_cache.py"
    spec = importlib.util.spec_from_file_location("prompt_cache_example", path)
    ex = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(ex)
    for texts, instruction, text in ((5, 70, 9), (90, 1030, 12)):
        one, other, _ = ex.embed(e2c, texts, instruction, text, 2)
        assert torch_cuda.isfinite(one).all()
        assert (one * other).sum(1).min().item() > 0.999
