"""The prompt-cache operators (rotary positions, a paged key/value cache, attention over its pages with a
shared prefix): the cases they are measured on, their plain forms and their definitions in 64 bits.

A case is a dict of plain values. ``prepare`` makes what a serving program has in hand, ``run`` makes one pass:
the operators' plain form in 32-bit torch where ``own`` is false, this repository's entry points where it
is true. ``exact`` evaluates the definition in 64 bits.

Kinds:
    rotate   rotary positions on the heads of token rows (and their transpose, the gradient)
    store    rotary positions on q and k, k and v written into the pages of their sequences
    branch   fork one cached prompt, grow every branch (copying the partly filled page), free the branches
    copy     copy listed pages of every layer
    compact  move the pages in use to the low end of the pool
    attend   queries against the cached keys of their sequences, whose first ``shared`` tokens are in common
"""
import importlib.util
import math
import sys
from pathlib import Path

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
SIZE = {"bf16": 2, "f16": 2, "f32": 4}


def listed():
    return [
        # one decode step of 16 sequences: latency counts
        dict(name="rotate decode", kind="rotate", dtype="bf16", tokens=16, heads=40, dim=128, rot=128, interleaved=False,
             backward=False, positions=32768),
        # a quarter of each head rotated, pairs interleaved, an odd number of tokens with strided rows
        dict(name="rotate partial", kind="rotate", dtype="f16", tokens=20011, heads=24, dim=64, rot=16, interleaved=True,
             backward=False, positions=131072),
        # the gradient of the rotation over a training batch's q and k in 32 bits
        dict(name="rotate gradient", kind="rotate", dtype="f32", tokens=16384, heads=40, dim=128, rot=128,
             interleaved=False, backward=True, positions=8192),
        # one decode step of 64 sequences into 16-token pages
        dict(name="store decode", kind="store", dtype="bf16", source="bf16", n=64, queries=1, held=900, heads=32,
             kv_heads=8, dim=128, rot=128, page=16, interleaved=False),
        # prompts of this framework's own head shape (4 heads of 256, 2 key/value heads) from a 32-bit projection
        dict(name="store prompts", kind="store", dtype="bf16", source="f32", n=24, queries=1000, held=0, heads=4, kv_heads=2,
             dim=256, rot=256, page=64, interleaved=False),
        # 32 continuations of one prompt, each given its own copy of the partly filled page
        dict(name="branch", kind="branch", dtype="bf16", n=32, held=1003, grow=5, layers=8, kv_heads=2, dim=256, page=16,
             pool=16384),
        # pages swapped between two places of the pool
        dict(name="copy pages", kind="copy", dtype="f16", count=1021, layers=16, kv_heads=8, dim=128, page=16, pool=4096),
        # a pool with one page in three free: what lies past the used count moves down
        dict(name="compact", kind="compact", dtype="bf16", n=128, held=509, layers=12, kv_heads=4, dim=128, page=32,
             pool=4096),
        # one token for each of 4 short sequences: latency counts
        dict(name="attend few", kind="attend", dtype="bf16", n=4, queries=1, shared=256, own=100, heads=16, kv_heads=4,
             dim=128, page=16, causal=True, window=-1),
        # one token for each of 128 sequences behind one long instruction
        dict(name="attend decode", kind="attend", dtype="bf16", n=128, queries=1, shared=16384, own=700, heads=32,
             kv_heads=8, dim=128, page=32, causal=True, window=-1),
        # 48 candidates of 61 tokens scored against one document, this framework's head shape
        dict(name="attend candidates", kind="attend", dtype="f16", n=48, queries=61, shared=6144, own=61, heads=4,
             kv_heads=2, dim=256, page=64, causal=True, window=-1),
        # whole prompts of ragged lengths, a sliding window in both directions, small heads
        dict(name="attend prompts", kind="attend", dtype="bf16", n=12, queries=2500, shared=0, own=2500, heads=12,
             kv_heads=12, dim=64, page=128, causal=False, window=512),
    ]


def _log(rng, lo, hi):
    """A whole number of [lo, hi], spread over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["rotate", "store", "branch", "copy", "compact", "attend", "attend", "attend"])
    dtype = rng.choice(["bf16", "f16"])
    while True:
        dim = rng.choice([64, 128, 256])
        kv = rng.choice([1, 2, 4, 8])
        heads = kv * rng.choice([1, 2, 4, 5, 7, 8])
        page = rng.choice([8, 16, 32, 64, 128])
        if kind == "rotate":
            rot = rng.choice([dim, dim // 2, dim // 4])
            c = dict(kind=kind, dtype=rng.choice(["bf16", "f16", "f32"]), tokens=_log(rng, 1, 16384), heads=heads, dim=dim,
                     rot=rot, interleaved=rng.random() < 0.5, backward=rng.random() < 0.5, positions=_log(rng, 1024, 262144))
        elif kind == "store":
            c = dict(kind=kind, dtype=dtype, source=rng.choice([dtype, "f32"]), n=_log(rng, 1, 256), queries=_log(rng, 1, 2048),
                     held=_log(rng, 1, 4096), heads=heads, kv_heads=kv, dim=dim, rot=rng.choice([dim, dim // 2]), page=page,
                     interleaved=rng.random() < 0.5)
        elif kind == "branch":
            c = dict(kind=kind, dtype=dtype, n=_log(rng, 1, 128), held=_log(rng, 1, 4096), grow=_log(rng, 1, 64),
                     layers=_log(rng, 1, 24), kv_heads=kv, dim=dim, page=page, pool=_log(rng, 256, 32768))
        elif kind == "copy":
            pool = _log(rng, 64, 4096)
            c = dict(kind=kind, dtype=dtype, count=_log(rng, 1, pool // 2), layers=_log(rng, 1, 24), kv_heads=kv, dim=dim,
                     page=page, pool=pool)
        elif kind == "compact":
            c = dict(kind=kind, dtype=dtype, n=_log(rng, 2, 256), held=_log(rng, 2, 1024), layers=_log(rng, 1, 16), kv_heads=kv,
                     dim=dim, page=page, pool=_log(rng, 64, 8192))
        else:
            queries = 1 if rng.random() < 0.5 else _log(rng, 2, 512)
            shared = rng.choice([0, 1, 1]) * _log(rng, 1, 16384) // page * page
            c = dict(kind=kind, dtype=dtype, n=_log(rng, 1, 256), queries=queries, shared=shared,
                     own=queries + rng.choice([0, 1, 1]) * _log(rng, 1, 2048), heads=heads, kv_heads=kv, dim=dim, page=page,
                     causal=rng.random() < 0.7, window=rng.choice([-1, -1, _log(rng, 16, 1024)]))
        if _fits(c):
            return c


def _pool_bytes(c):
    return 2 * c.get("layers", 1) * _pool(c) * c["page"] * c["kv_heads"] * c["dim"] * 2


def _pool(c):
    """Pages of the case's pool."""
    if c["kind"] == "attend":
        return (c["shared"] + c["n"] * _ceil(c["own"], c["page"]) * c["page"]) // c["page"] + 7
    if c["kind"] == "store":
        return c["n"] * _ceil(c["held"] + c["queries"], c["page"]) + 5
    return c["pool"]


def _fits(c):
    """Whether a drawn case is possible and costs no more than the largest listed ones."""
    if c["kind"] == "branch" and _ceil(c["held"], c["page"]) + c["n"] * (2 + _ceil(c["grow"], c["page"])) > c["pool"]:
        return False
    if c["kind"] == "compact" and 2 * c["n"] * _ceil(c["held"], c["page"]) > c["pool"]:
        return False
    if c["kind"] == "attend":
        span = c["shared"] + c["own"]
        if c["n"] * c["queries"] * c["heads"] * span > 6e8 or c["n"] * span * c["kv_heads"] * c["dim"] > 2.5e9:
            return False  # the plain form holds every score and every gathered key in 32 bits
    if c["kind"] != "rotate" and _pool_bytes(c) > 4e9:
        return False
    w = work(c)
    return w["bytes"] < 2e9 and w["flops"] < 5e11


def _ceil(a, b):
    return -(-a // b)


def _lengths(c):
    """Tokens of each sequence past the shared ones, and its queries: ragged, as a batch's are."""
    n = c["n"]
    if c["kind"] == "attend":
        own_len = [max(1, c["own"] - (i * 7919 % max(1, c["own"] // 3 + 1)) * (i > 0)) for i in range(n)]
        q = [min(o, max(1, c["queries"] - (i * 31 % max(1, c["queries"] // 4 + 1)) * (i > 0))) for i, o in enumerate(own_len)]
        return own_len, q
    q = [max(1, c["queries"] - (i * 31 % max(1, c["queries"] // 4 + 1)) * (i > 0)) for i in range(n)]
    return [c["held"] + x for x in q], q


def _tables(positions, rot, dev):
    """cos and sin of every position's rot / 2 angles (theta 1e4), in 32 bits from 64."""
    f = 1e4 ** (-torch.arange(0, rot, 2, dtype=torch.float64, device=dev) / rot)
    a = torch.arange(positions, dtype=torch.float64, device=dev)[:, None] * f
    return a.cos().float(), a.sin().float()


def prepare(case, seed):
    c, dev = case, torch.device("cuda")
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    s = {"case": c}

    def normal(*shape, dtype, scale=1.0):
        return (torch.randn(*shape, generator=g, device=dev, dtype=torch.float32) * scale).to(dtype)

    def ints(v):
        return torch.tensor(v, dtype=torch.int32, device=dev)

    def pool_values(*shape, dtype):
        """Values of a cache that has been in use: random in blocks of 16 Mi, made in the cache's type."""
        t = torch.empty(*shape, device=dev, dtype=dtype)
        flat = t.view(-1)
        block = normal(min(flat.numel(), 1 << 24), dtype=dtype)
        for at in range(0, flat.numel(), block.numel()):
            part = flat[at:at + block.numel()]
            part.copy_(block[:part.numel()].roll(at // block.numel() * 4099))
        return t

    if c["kind"] == "rotate":
        dt = DTYPES[c["dtype"]]
        s["cos"], s["sin"] = _tables(c["positions"], c["rot"], dev)
        # q and k as the first columns of a fused projection's rows
        rows = normal(c["tokens"], c["heads"] * c["dim"] + 64, dtype=dt)
        s["x"] = rows[:, :c["heads"] * c["dim"]].unflatten(1, (c["heads"], c["dim"]))
        s["pos"] = torch.randint(0, c["positions"], (c["tokens"],), generator=g, device=dev, dtype=torch.int32)
        return s

    dt, pool, ps, kv, d = DTYPES[c["dtype"]], _pool(c), c["page"], c["kv_heads"], c["dim"]
    order = torch.randperm(pool, generator=g, device=dev).int()  # pages are handed out in no order
    shape = (c.get("layers", 1), pool, ps, kv, d)
    s["k"], s["v"] = pool_values(*shape, dtype=dt), pool_values(*shape, dtype=dt)
    refs = torch.zeros(pool, dtype=torch.int32, device=dev)

    if c["kind"] in ("attend", "store"):
        n = c["n"]
        shared = c.get("shared", 0)
        tail, q = _lengths(c)
        blocks = [_ceil(t, ps) for t in tail]
        width = shared // ps + max(blocks)
        table = torch.zeros(n, width, dtype=torch.int32)
        perm, at, used = order.cpu(), shared // ps, torch.zeros(pool, dtype=torch.int32)
        table[:, :at] = perm[:at]
        used[perm[:at].long()] = n
        for i, b in enumerate(blocks):
            table[i, shared // ps:shared // ps + b] = perm[at:at + b]
            used[perm[at:at + b].long()] = 1
            at += b
        s["table"], s["refs"] = table.to(dev), used.to(dev)
        s["len"] = ints([shared + t for t in tail])
        s["seqs"] = torch.randperm(n, generator=g, device=dev).int()  # the batch's order is not the cache's
        counts = torch.tensor(q)[s["seqs"].cpu().long()]
        s["q_start"] = torch.cat([torch.zeros(1, dtype=torch.int64), counts.cumsum(0)]).int().to(dev)
        s["tokens"], s["max_q"] = int(counts.sum()), max(q)
        if c["kind"] == "attend":
            s["q"] = normal(s["tokens"], c["heads"], d, dtype=dt, scale=2.0)
            s["scale"] = 1.0 / math.sqrt(d)
            return s
        src = DTYPES[c["source"]]
        # q, k and v side by side in the rows of one projection that go on past them
        rows = normal(s["tokens"], (c["heads"] + 2 * kv) * d + 64, dtype=src)[:, :-64]
        s["q_in"], s["k_in"], s["v_in"] = rows.unflatten(1, (c["heads"] + 2 * kv, d)).split([c["heads"], kv, kv], 1)
        s["cos"], s["sin"] = _tables(c["held"] + c["queries"], c["rot"], dev)
        return s

    if c["kind"] == "branch":
        n, b = c["n"], _ceil(c["held"], ps)
        width = _ceil(c["held"] + c["grow"], ps) + 1
        s["table"] = torch.zeros(n + 1, width, dtype=torch.int32, device=dev)
        s["table"][0, :b] = order[:b]
        # other sequences hold half of what is left; the free pages are scattered among theirs
        rest = order[b:]
        spare = n * (2 + _ceil(c["grow"], ps))
        refs[rest[spare:].long()] = torch.randint(0, 2, (max(0, len(rest) - spare),), generator=g, device=dev, dtype=torch.int32)
        refs[order[:b].long()] = 1
        s["refs"] = refs
        s["len"] = torch.zeros(n + 1, dtype=torch.int32, device=dev)
        s["len"][0] = c["held"]
        s["parents"], s["children"] = ints([0] * n), ints(range(1, n + 1))
        s["grow"] = ints([max(1, c["grow"] - i % 3) for i in range(n)])
        return s

    if c["kind"] == "copy":
        s["src"], s["dst"] = order[:c["count"]].contiguous(), order[c["count"]:2 * c["count"]].contiguous()
        s["table"] = torch.zeros(1, 1, dtype=torch.int32, device=dev)
        s["len"], s["refs"] = torch.zeros(1, dtype=torch.int32, device=dev), refs
        return s

    # compact: the sequences' pages lie anywhere in the pool, every third sequence is a fork of the one before it
    n, b = c["n"], _ceil(c["held"], ps)
    spots = order[:n * b].view(n, b)
    forks = torch.arange(2, n, 3, device=dev)
    spots[forks] = spots[forks - 1].clone()
    s["table"] = spots.clone()
    s["len"] = torch.full((n,), c["held"], dtype=torch.int32, device=dev)
    refs.index_add_(0, spots.reshape(-1).long(), torch.ones(n * b, dtype=torch.int32, device=dev))
    s["refs"] = refs
    s["found"] = [s["table"].clone(), s["refs"].clone()]  # the pool as a pass finds it
    return s


# ------------------------------------------------------------------------------------- this repository's operators
def _package():
    if "e2c_b200" not in sys.modules:
        pkg = Path("e2.c_b200").resolve()
        spec = importlib.util.spec_from_file_location("e2c_b200", pkg / "__init__.py", submodule_search_locations=[str(pkg)])
        mod = importlib.util.module_from_spec(spec)
        sys.modules["e2c_b200"] = mod
        spec.loader.exec_module(mod)
    return sys.modules["e2c_b200"]


def _run_own(s):
    c, e2c = s["case"], _package()
    if c["kind"] == "rotate":
        return e2c.rope(s["x"], s["cos"], s["sin"], s["pos"], interleaved=c["interleaved"], backward=c["backward"])
    if "cache" not in s:  # the handle that a program keeps: pointers and sizes, no data
        s["cache"] = e2c.PageCache(s["k"], s["v"], s["table"], s["len"], s["refs"])
    cache = s["cache"]
    if c["kind"] == "store":
        q = cache.store(0, s["q_in"], s["k_in"], s["v_in"], s["cos"], s["sin"], s["seqs"], s["q_start"],
                        interleaved=c["interleaved"])
        return {"q": q, "k": s["k"], "v": s["v"]}
    if c["kind"] == "branch":
        cache.fork(s["parents"], s["children"])
        cache.append(s["children"], s["grow"])
        grown = s["table"].clone(), s["len"].clone(), s["refs"].clone()
        cache.free(s["children"])
        return {"table": grown[0], "len": grown[1], "grown": grown[2], "refs": s["refs"], "k": s["k"], "v": s["v"]}
    if c["kind"] == "copy":
        cache.copy(s["src"], s["dst"])
        return {"k": s["k"], "v": s["v"]}
    if c["kind"] == "compact":
        s["table"].copy_(s["found"][0])
        s["refs"].copy_(s["found"][1])
        cache.compact()
        return {"table": s["table"], "refs": s["refs"], "k": s["k"], "v": s["v"]}
    out, lse = cache.attention(0, s["q"], s["seqs"], s["q_start"], s["max_q"], shared=c["shared"], causal=c["causal"],
                               window=c["window"], scale=s["scale"], lse=True)
    return {"out": out, "lse": lse}


# ------------------------------------------------------------------------------------- the plain forms, in 32 bits
def _rotated(x, cos, sin, pos, interleaved, sign=1.0):
    """x [tokens][heads][dim] in the arithmetic of cos and sin's type."""
    rot = 2 * cos.shape[1]
    x = x.to(cos.dtype)
    cs, sn = cos[pos.long()][:, None], sin[pos.long()][:, None] * sign
    head = x[..., :rot]
    a, b = (head[..., 0::2], head[..., 1::2]) if interleaved else (head[..., :rot // 2], head[..., rot // 2:])
    u, w = a * cs - b * sn, b * cs + a * sn
    turned = torch.stack([u, w], -1).flatten(-2) if interleaved else torch.cat([u, w], -1)
    return torch.cat([turned, x[..., rot:]], -1)


def _token_places(s):
    """Batch index and position of every query token."""
    qs = s["q_start"].long()
    t = torch.arange(s["tokens"], device=qs.device)
    i = torch.searchsorted(qs[1:], t, right=True)
    seq = s["seqs"].long()[i]
    return seq, s["len"].long()[seq] - (qs[i + 1] - t)


def _fork(s):
    p, ch = s["parents"].long(), s["children"].long()
    s["table"][ch] = s["table"][p]
    s["len"][ch] = s["len"][p]
    held = _ceil(s["len"][p].long(), s["case"]["page"])
    mapped = torch.arange(s["table"].shape[1], device=ch.device) < held[:, None]
    s["refs"].index_add_(0, s["table"][ch].long().reshape(-1), mapped.int().reshape(-1))


def _append(s):
    ps, seqs, table, refs = s["case"]["page"], s["children"].long(), s["table"], s["refs"]
    old, new = s["len"].long()[seqs], s["len"].long()[seqs] + s["grow"].long()
    rows, b0, b1 = table[seqs].long(), -(-old // ps), -(-new // ps)
    last = rows.gather(1, (old // ps)[:, None])[:, 0]
    # a partly filled page that others map too is copied to a page of the sequence's own
    cow = (old % ps != 0) & (refs[last] > 1)
    first = torch.where(cow, b0 - 1, b0)
    block = torch.arange(rows.shape[1], device=seqs.device)
    wants = (block >= first[:, None]) & (block < b1[:, None])
    rank = wants.reshape(-1).cumsum(0).view_as(wants) - 1
    free = torch.sort((refs != 0).int(), stable=True).indices  # the lowest free pages first
    got = free[rank.clamp(min=0)]
    table[seqs] = torch.where(wants, got, rows).int()
    refs.index_add_(0, got.reshape(-1), wants.int().reshape(-1))
    refs.index_add_(0, last, -cow.int())
    s["len"][seqs] = new.int()
    # sequences with nothing to copy rewrite their own page with itself
    to = torch.where(cow, got.gather(1, (old // ps)[:, None])[:, 0], last)
    s["k"][:, to] = s["k"][:, last]
    s["v"][:, to] = s["v"][:, last]


def _free(s):
    seqs = s["children"].long()
    held = _ceil(s["len"].long()[seqs], s["case"]["page"])
    mapped = torch.arange(s["table"].shape[1], device=seqs.device) < held[:, None]
    s["refs"].index_add_(0, s["table"][seqs].long().reshape(-1), -mapped.int().reshape(-1))
    s["len"][seqs] = 0


def _compact(s):
    refs = s["refs"]
    pages = torch.arange(refs.numel(), device=refs.device)
    live = refs > 0
    used = live.sum()
    high, hole = live & (pages >= used), ~live & (pages < used)
    # the k-th live page past the used count goes to the k-th hole below it
    src, dst = high.nonzero()[:, 0], hole.nonzero()[:, 0]
    s["k"][:, dst] = s["k"][:, src]
    s["v"][:, dst] = s["v"][:, src]
    to = pages.clone()
    to[src] = dst
    s["table"].copy_(to[s["table"].long()])
    refs[dst] = refs[src]
    refs[src] = 0


def _attend(s):
    c, ps = s["case"], s["case"]["page"]
    dev, n, kv, d = s["q"].device, c["n"], c["kv_heads"], c["dim"]
    group = c["heads"] // kv
    seqs, qs = s["seqs"].long(), s["q_start"].long()
    length = s["len"].long()[seqs]
    span = s["table"].shape[1] * ps
    pages = s["table"].long()[seqs]
    blocks = torch.arange(s["table"].shape[1], device=dev) < (-(-length // ps))[:, None]
    pages = torch.where(blocks, pages, 0)
    keys = s["k"][0][pages].float().view(n, span, kv, d)
    values = s["v"][0][pages].float().view(n, span, kv, d)
    count = qs[1:] - qs[:-1]
    i = torch.arange(s["max_q"], device=dev)
    rows = (qs[:-1, None] + i).clamp(max=s["tokens"] - 1)
    q = s["q"].float()[rows].view(n, s["max_q"], kv, group, d)
    logits = torch.einsum("nikgd,njkd->nkgij", q, keys) * s["scale"]
    pos = (length - count)[:, None] + i
    j = torch.arange(span, device=dev)
    sees = (j < length[:, None, None]).expand(n, s["max_q"], span)
    if c["causal"]:
        sees = sees & (j <= pos[..., None])
    if c["window"] >= 0:
        sees = sees & ((j - pos[..., None]).abs() <= c["window"])
    logits = logits.masked_fill_(~sees[:, None, None], -math.inf)
    top = logits.amax(-1, keepdim=True)
    p = logits.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    out = torch.einsum("nkgij,njkd->nikgd", p, values) / total[..., 0].permute(0, 3, 1, 2)[..., None]
    lse = (top + total.log())[..., 0].permute(0, 3, 1, 2)
    keep = i < count[:, None]
    return {"out": out[keep].view(s["tokens"], c["heads"], d).to(s["q"].dtype), "lse": lse[keep].reshape(s["tokens"], c["heads"])}


def run(state):
    s = state
    if own:
        return _run_own(s)
    c = s["case"]
    if c["kind"] == "rotate":
        return _rotated(s["x"], s["cos"], s["sin"], s["pos"], c["interleaved"], -1.0 if c["backward"] else 1.0).to(s["x"].dtype)
    if c["kind"] == "store":
        seq, pos = _token_places(s)
        page, slot = s["table"][seq, pos // c["page"]].long(), pos % c["page"]
        q = _rotated(s["q_in"], s["cos"], s["sin"], pos, c["interleaved"]).to(s["k"].dtype)
        s["k"][0][page, slot] = _rotated(s["k_in"], s["cos"], s["sin"], pos, c["interleaved"]).to(s["k"].dtype)
        s["v"][0][page, slot] = s["v_in"].to(s["k"].dtype)
        return {"q": q, "k": s["k"], "v": s["v"]}
    if c["kind"] == "branch":
        _fork(s)
        _append(s)
        grown = s["table"].clone(), s["len"].clone(), s["refs"].clone()
        _free(s)
        return {"table": grown[0], "len": grown[1], "grown": grown[2], "refs": s["refs"], "k": s["k"], "v": s["v"]}
    if c["kind"] == "copy":
        s["k"][:, s["dst"].long()] = s["k"][:, s["src"].long()]
        s["v"][:, s["dst"].long()] = s["v"][:, s["src"].long()]
        return {"k": s["k"], "v": s["v"]}
    if c["kind"] == "compact":
        s["table"].copy_(s["found"][0])
        s["refs"].copy_(s["found"][1])
        _compact(s)
        return {"table": s["table"], "refs": s["refs"], "k": s["k"], "v": s["v"]}
    return _attend(s)


# ------------------------------------------------------------------------------------- what a pass cannot do without
def work(case):
    c, es = case, SIZE[case["dtype"]]
    if c["kind"] == "rotate":
        n = c["tokens"] * c["heads"] * c["dim"]
        return {"bytes": 2 * n * es + min(c["tokens"], c["positions"]) * c["rot"] * 4 + 4 * c["tokens"],
                "flops": 3 * c["tokens"] * c["heads"] * c["rot"]}
    row = c["kv_heads"] * c["dim"]
    page = c.get("layers", 1) * c["page"] * row * es * 2  # a page's keys and values in every layer
    if c["kind"] == "store":
        tokens = sum(_lengths(c)[1])
        n = tokens * (c["heads"] * c["dim"] + 2 * row)
        spots = min(tokens, c["held"] + c["queries"])
        return {"bytes": n * (SIZE[c["source"]] + es) + spots * c["rot"] * 4,
                "flops": 3 * tokens * (c["heads"] + c["kv_heads"]) * c["rot"]}
    if c["kind"] == "branch":
        held, grown = _ceil(c["held"], c["page"]), _ceil(c["held"] + c["grow"], c["page"])
        copies = c["n"] if c["held"] % c["page"] else 0
        index = 4 * c["n"] * (2 * held + 2 * grown + 8) + 4 * c["pool"]
        return {"bytes": 2 * copies * page + index, "flops": 0}
    if c["kind"] == "copy":
        return {"bytes": 2 * c["count"] * page + 8 * c["count"], "flops": 0}
    if c["kind"] == "compact":
        b = _ceil(c["held"], c["page"])
        live = (c["n"] - len(range(2, c["n"], 3))) * b
        moved = live * (c["pool"] - live) // c["pool"]  # of pages spread evenly over the pool
        return {"bytes": 2 * moved * page + 8 * c["n"] * b + 8 * c["pool"], "flops": 0}
    own_len, q = _lengths(c)
    pairs = 0
    for o, m in zip(own_len, q):
        length = c["shared"] + o
        # keys in sight of the m last positions: all, those up to the position, and those within the window
        w = c["window"] if c["window"] >= 0 else length
        for p in range(length - m, length):
            pairs += min(length, p + 1 if c["causal"] else p + w + 1) - max(0, p - w)
    lo = c["shared"] + min(o - m for o, m in zip(own_len, q))
    seen = c["shared"] - (max(0, min(c["shared"], lo - c["window"])) if c["window"] >= 0 else 0)
    tail = sum(min(o, m + c["window"]) if c["window"] >= 0 else o for o, m in zip(own_len, q))
    tokens = sum(q)
    return {"bytes": 2 * (seen + tail) * row * es + tokens * c["heads"] * (2 * c["dim"] * es + 4),
            "flops": 4 * pairs * c["heads"] * c["dim"]}


# ------------------------------------------------------------------------------------- the definitions, in 64 bits
def _turn(x, cos, sin, pos, interleaved, transpose):
    """Each pair (x, y) of a head as the complex number x + iy, times cos + i sin (conjugated for the transpose)."""
    half = cos.shape[1]
    x = x.double()
    z = torch.complex(cos[pos.long()].double(), sin[pos.long()].double())[:, None]
    z = z.conj() if transpose else z
    out = x.clone()
    at = torch.arange(half, device=x.device)
    first, second = (2 * at, 2 * at + 1) if interleaved else (at, at + half)
    w = torch.complex(x[..., first], x[..., second]) * z
    out[..., first], out[..., second] = w.real, w.imag
    return out


def exact(case, seed):
    c = case
    if c["kind"] in ("branch", "copy", "compact"):
        return None  # nothing is computed: pages and whole numbers move
    s = prepare(case, seed)
    if c["kind"] == "rotate":
        return _turn(s["x"], s["cos"], s["sin"], s["pos"], c["interleaved"], c["backward"])
    seqs, qs, table, length = s["seqs"].tolist(), s["q_start"].tolist(), s["table"].cpu(), s["len"].tolist()
    if c["kind"] == "store":
        pos = torch.cat([torch.arange(length[q] - (qs[i + 1] - qs[i]), length[q]) for i, q in enumerate(seqs)]).to(s["k"].device)
        result = {"q": _turn(s["q_in"], s["cos"], s["sin"], pos, c["interleaved"], False), "k": None, "v": None}
        if s["k"].numel() <= 1 << 28:
            turned = _turn(s["k_in"], s["cos"], s["sin"], pos, c["interleaved"], False)
            k, v = s["k"].double(), s["v"].double()
            for i, q in enumerate(seqs):
                p = pos[qs[i]:qs[i + 1]].cpu()
                page = table[q][p // c["page"]].long().to(k.device)
                slot = (p % c["page"]).to(k.device)
                k[0, page, slot] = turned[qs[i]:qs[i + 1]]
                v[0, page, slot] = s["v_in"][qs[i]:qs[i + 1]].double()
            result["k"], result["v"] = k, v
        return result
    if work(case)["flops"] > 2e12:
        return None
    group = c["heads"] // c["kv_heads"]
    out = torch.zeros(s["tokens"], c["heads"], c["dim"], dtype=torch.float64, device=s["q"].device)
    lse = torch.full((s["tokens"], c["heads"]), -math.inf, dtype=torch.float64, device=s["q"].device)
    for i, q in enumerate(seqs):
        pages = table[q][:_ceil(length[q], c["page"])].long().to(s["k"].device)
        k = s["k"][0][pages].flatten(0, 1)[:length[q]].double()
        v = s["v"][0][pages].flatten(0, 1)[:length[q]].double()
        x = s["q"][qs[i]:qs[i + 1]].double()
        p = torch.arange(length[q] - x.shape[0], length[q], device=x.device)[:, None]
        j = torch.arange(length[q], device=x.device)[None]
        hidden = (j > p) if c["causal"] else torch.zeros_like(j > p)
        if c["window"] >= 0:
            hidden = hidden | (j < p - c["window"]) | (j > p + c["window"])
        for h in range(c["heads"]):
            a = (x[:, h] @ k[:, h // group].T) * s["scale"]
            a[hidden] = -math.inf
            r = torch.logsumexp(a, 1)
            out[qs[i]:qs[i + 1], h] = torch.exp(a - r[:, None]) @ v[:, h // group]
            lse[qs[i]:qs[i + 1], h] = r
    return {"out": out, "lse": lse}
