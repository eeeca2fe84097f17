"""More operators of the prompt cache (a sliding window whose first tokens stay visible, trees of drafted tokens, a
cache held in 8 bits): the cases they are measured on, their plain forms and their definitions in 64 bits.

A case is a dict of plain values. ``prepare`` makes what a serving program has in hand, ``run`` makes one pass:
the operators' plain form in 32-bit torch where ``own`` is false, this repository's entry points where it
is true. ``exact`` evaluates the definition in 64 bits.

Kinds:
    attend  queries against the cached keys of their sequences. ``held``: what a value is held in (i8: 8 bits and a
            scale for each token and key head). ``window`` and ``sinks``: a row at position p sees the tokens j with
            |p - j| <= window and the first ``sinks``. ``tree``: an entry's rows are drafted tokens, each with a parent among
            them or none; a row sees the text before them, its ancestors and itself
    keep    the drafted tokens of one path through each tree become the end of their sequence's text
    store   rotary positions on q and k, k and v quantised into the pages of their sequences, and read back
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
        # one token for each of 3 long chats in a window, this framework's head shape: latency counts
        dict(name="sinks few", kind="attend", dtype="bf16", held="16", n=3, queries=1, shared=0, text=1500, heads=4, kv_heads=2,
             dim=256, page=16, causal=True, window=511, sinks=4, tree=False),
        # one token for each of 128 long chats
        dict(name="sinks decode", kind="attend", dtype="bf16", held="16", n=128, queries=1, shared=0, text=5900, heads=32,
             kv_heads=8, dim=128, page=32, causal=True, window=2047, sinks=16, tree=False),
        # prompts of ragged lengths, some of their tokens cached before
        dict(name="sinks prompts", kind="attend", dtype="f16", held="16", n=4, queries=2900, shared=0, text=3300, heads=16,
             kv_heads=4, dim=128, page=64, causal=True, window=1023, sinks=4, tree=False),
        # 11 drafted tokens for each of 4 short texts: latency counts
        dict(name="tree few", kind="attend", dtype="f16", held="16", n=4, queries=11, shared=0, text=300, heads=16, kv_heads=4,
             dim=128, page=16, causal=True, window=-1, sinks=0, tree=True),
        # 31 drafted tokens for each of 64 texts
        dict(name="tree verify", kind="attend", dtype="bf16", held="16", n=64, queries=31, shared=0, text=4000, heads=32, kv_heads=8,
             dim=128, page=32, causal=True, window=-1, sinks=0, tree=True),
        # 96 continuations behind one document, each with a tree of up to 24
        dict(name="tree behind a document", kind="attend", dtype="f16", held="16", n=96, queries=24, shared=4096, text=200, heads=4,
             kv_heads=2, dim=256, page=64, causal=True, window=-1, sinks=0, tree=True),
        # what verification accepts of those trees stays, in every layer
        dict(name="keep", kind="keep", dtype="bf16", held="16", n=64, queries=31, text=300, layers=12, kv_heads=4, dim=128, page=32),
        # one decode step of 64 sequences into 16-token pages
        dict(name="store decode", kind="store", dtype="bf16", source="bf16", n=64, queries=1, text=900, heads=32, kv_heads=8,
             dim=128, rot=128, page=16, interleaved=False),
        # prompts of this framework's own head shape from a 32-bit projection
        dict(name="store prompts", kind="store", dtype="f16", source="f32", n=24, queries=1000, text=0, heads=4, kv_heads=2, dim=256,
             rot=256, page=64, interleaved=False),
        # one token for each of 4 short sequences: latency counts
        dict(name="8 bits few", kind="attend", dtype="bf16", held="i8", n=4, queries=1, shared=0, text=700, heads=16, kv_heads=4,
             dim=128, page=16, causal=True, window=-1, sinks=0, tree=False),
        # one token for each of 64 long sequences
        dict(name="8 bits decode", kind="attend", dtype="bf16", held="i8", n=64, queries=1, shared=0, text=8192, heads=32, kv_heads=8,
             dim=128, page=32, causal=True, window=-1, sinks=0, tree=False),
        # prompts of ragged lengths, small heads
        dict(name="8 bits prompts", kind="attend", dtype="f16", held="i8", n=6, queries=2000, shared=0, text=2500, heads=12,
             kv_heads=12, dim=64, page=128, causal=True, window=-1, sinks=0, tree=False),
    ]


def _log(rng, lo, hi):
    """A whole number of [lo, hi], spread over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["attend", "attend", "attend", "attend", "store", "keep"])
    while True:
        dim = rng.choice([64, 128, 256])
        kv = rng.choice([1, 2, 4, 8])
        heads = kv * rng.choice([1, 2, 4, 5, 7, 8])
        c = dict(kind=kind, dtype=rng.choice(["bf16", "f16"]), n=_log(rng, 1, 256), kv_heads=kv, dim=dim,
                 page=rng.choice([8, 16, 32, 64, 128]))
        if kind == "store":
            c.update(source=rng.choice([c["dtype"], "f32"]), queries=_log(rng, 1, 2048), text=_log(rng, 1, 4096), heads=heads,
                     rot=rng.choice([dim, dim // 2]), interleaved=rng.random() < 0.5)
        elif kind == "keep":
            c.update(held=rng.choice(["16", "i8"]), queries=_log(rng, 1, 64), text=_log(rng, 1, 2048), layers=_log(rng, 1, 24))
        else:
            form = rng.choice(["sinks", "tree", "8 bits"])
            held = "i8" if form == "8 bits" or rng.random() < 0.3 else "16"
            tree = form == "tree" or (form == "8 bits" and rng.random() < 0.2)
            window = _log(rng, 16, 4096) if form == "sinks" or rng.random() < 0.2 else -1
            queries = _log(rng, 2, 96) if tree else 1 if rng.random() < 0.5 else _log(rng, 2, 2048)
            shared = rng.choice([0, 0, 1]) * _log(rng, 1, 16384) // c["page"] * c["page"]
            c.update(held=held, queries=queries, shared=shared, text=queries + _log(rng, 1, 8192), heads=heads,
                     causal=tree or rng.random() < 0.8, window=window, sinks=_log(rng, 1, 256) if window >= 0 else 0, tree=tree)
        if _fits(c):
            return c


def _ceil(a, b):
    return -(-a // b)


def _pool(c):
    """Pages of the case's pool."""
    grown = c["text"] + (c["queries"] if c["kind"] != "attend" else 0)
    return c.get("shared", 0) // c["page"] + c["n"] * _ceil(grown, c["page"]) + 7


def _fits(c):
    """Whether a drawn case costs no more than the largest listed ones."""
    if 2 * c.get("layers", 1) * _pool(c) * c["page"] * c["kv_heads"] * c["dim"] * 2 > (6e8 if c["kind"] == "keep" else 3.5e9):
        return False
    if c["kind"] == "attend":
        span = c["shared"] + c["text"]
        # the plain form holds every score and every gathered key in 32 bits
        if c["n"] * c["queries"] * c["heads"] * span > 6.5e8 or c["n"] * span * c["kv_heads"] * c["dim"] > 1e9:
            return False
    w = work(c)
    return w["bytes"] < 1.5e9 and w["flops"] < 3e11


def _lengths(c):
    """Tokens of each sequence past the shared ones, and its queries: ragged, as a batch's are."""
    n = c["n"]
    q = [max(1, c["queries"] - (i * 31 % max(1, c["queries"] // 4 + 1)) * (i > 0)) for i in range(n)]
    if c["kind"] != "attend":
        return [c["text"] + x for x in q], q
    text = [max(1, c["text"] - (i * 7919 % max(1, c["text"] // 3 + 1)) * (i > 0)) for i in range(n)]
    return text, [min(t, x) for t, x in zip(text, q)]


def _parents(c):
    """Each drafted token's parent in its entry (-1: none): one chain, which side branches leave, after the entry's number."""
    out = []
    for i, m in enumerate(_lengths(c)[1]):
        out.append([-1 if r < 2 and i % 3 == 0 else r - 1 if r % 3 else (r * (7 + i)) % (r + 1) - 1 for r in range(m)])
    return out


def _tables(positions, rot, dev):
    """cos and sin of every position's rot / 2 angles (theta 1e4), in 32 bits from 64."""
    f = 1e4 ** (-torch.arange(0, rot, 2, dtype=torch.float64, device=dev) / rot)
    a = torch.arange(positions, dtype=torch.float64, device=dev)[:, None] * f
    return a.cos().float(), a.sin().float()


def prepare(case, seed):
    c, dev = case, torch.device("cuda")
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    dt, pool, ps, kv, d, n = DTYPES[c["dtype"]], _pool(c), c["page"], c["kv_heads"], c["dim"], c["n"]
    s = {"case": c}

    def ints(v):
        return torch.tensor(v, dtype=torch.int32, device=dev)

    def cached():
        """A cache that has been in use: what a token's heads hold differs in size from token to token."""
        shape = (c.get("layers", 1), pool, ps, kv, d)
        if c.get("held", "i8") == "16":
            t = torch.empty(shape, device=dev, dtype=dt)
            for part in t.view(-1, kv, d).split(1 << 17):
                part.copy_(torch.randn(part.shape, generator=g, device=dev))
            return t, None
        t = torch.empty(shape, device=dev, dtype=torch.int8)
        sizes = (torch.randn(shape[:2] + (kv, ps), generator=g, device=dev) * 0.3).exp() * (3.0 / 127)
        for part in t.view(-1, kv, d).split(1 << 17):
            x = torch.randn(part.shape, generator=g, device=dev)
            part.copy_((x * (127 / x.abs().amax(-1, keepdim=True))).round())
        return t, sizes

    (s["k"], s["k_scale"]), (s["v"], s["v_scale"]) = cached(), cached()
    order = torch.randperm(pool, generator=g, device=dev).cpu()  # pages are handed out in no order
    shared = c.get("shared", 0)
    tail, q = _lengths(c)
    blocks = [_ceil(t, ps) for t in tail]
    table, used = torch.zeros(n, shared // ps + max(blocks), dtype=torch.int32), torch.zeros(pool, dtype=torch.int32)
    at = shared // ps
    table[:, :at] = order[:at]
    used[order[:at]] = n
    for i, b in enumerate(blocks):
        table[i, shared // ps:shared // ps + b] = order[at:at + b]
        used[order[at:at + b]] = 1
        at += b
    s["table"], s["refs"] = table.to(dev), used.to(dev)
    s["len"] = ints([shared + t for t in tail])
    s["seqs"] = torch.randperm(n, generator=g, device=dev).int()  # the batch's order is not the cache's
    batch = s["seqs"].tolist()
    s["q_start"] = torch.tensor([0] + [q[b] for b in batch]).cumsum(0).int().to(dev)
    s["tokens"], s["max_q"] = sum(q), max(q)

    if c["kind"] == "attend":
        s["q"] = (torch.randn(s["tokens"], c["heads"], d, generator=g, device=dev) * 2).to(dt)
        s["scale"] = 1.0 / math.sqrt(d)
        if c["tree"]:
            s["parents"] = ints(sum([_parents(c)[b] for b in batch], []))
        return s
    if c["kind"] == "keep":
        parents, kept, counts = _parents(c), [], []
        for b in batch:  # a path from some node of the tree up to the text
            path, r = [], (seed + 5 * b) % q[b]
            while r >= 0:
                path.append(r)
                r = parents[b][r]
            counts.append(len(path))
            kept += path[::-1] + [0] * (q[b] - len(path))
        s["kept"], s["counts"] = ints(kept), ints(counts)
        s["found"] = [s["len"].clone(), s["refs"].clone()]  # the cache as a pass finds it
        return s
    # q, k and v side by side in the rows of one projection that go on past them
    rows = torch.randn(s["tokens"], (c["heads"] + 2 * kv) * d + 64, generator=g, device=dev).to(DTYPES[c["source"]])[:, :-64]
    s["q_in"], s["k_in"], s["v_in"] = rows.unflatten(1, (c["heads"] + 2 * kv, d)).split([c["heads"], kv, kv], 1)
    s["cos"], s["sin"] = _tables(c["text"] + c["queries"], c["rot"], dev)
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
    c = s["case"]
    if "cache" not in s:  # the handle that a program keeps: pointers and sizes, no data
        s["cache"] = _package().PageCache(s["k"], s["v"], s["table"], s["len"], s["refs"], s["k_scale"], s["v_scale"])
    cache = s["cache"]
    if c["kind"] == "attend":
        sees, places = cache.tree(s["parents"], s["seqs"], s["q_start"], s["max_q"]) if c["tree"] else (None, None)
        out, lse = cache.attention(0, s["q"], s["seqs"], s["q_start"], s["max_q"], shared=c["shared"], causal=c["causal"],
                                   window=c["window"], scale=s["scale"], lse=True, sinks=c["sinks"], tree=sees)
        return {"out": out, "lse": lse, "places": places} if c["tree"] else {"out": out, "lse": lse}
    if c["kind"] == "keep":
        s["len"].copy_(s["found"][0])
        s["refs"].copy_(s["found"][1])
        cache.keep(s["seqs"], s["q_start"], s["kept"], s["counts"])
        return _cache_state(s)
    q = cache.store(0, s["q_in"], s["k_in"], s["v_in"], s["cos"], s["sin"], s["seqs"], s["q_start"], interleaved=c["interleaved"],
                    dtype=DTYPES[c["dtype"]])
    k, v = cache.load(0, s["seqs"], s["q_start"], s["tokens"], dtype=DTYPES[c["dtype"]])
    return {"q": q, "k": k, "v": v}


def _cache_state(s):
    if s["k_scale"] is None:
        return {"len": s["len"], "refs": s["refs"], "k": s["k"], "v": s["v"]}
    return {"len": s["len"], "refs": s["refs"], "k": s["k"], "v": s["v"], "k_scale": s["k_scale"], "v_scale": s["v_scale"]}


# ------------------------------------------------------------------------------------- the plain forms, in 32 bits
def _rotated(x, cos, sin, pos, interleaved):
    """x [tokens][heads][dim] in 32 bits."""
    rot = 2 * cos.shape[1]
    x = x.float()
    cs, sn = cos[pos][:, None], sin[pos][:, None]
    head = x[..., :rot]
    a, b = (head[..., 0::2], head[..., 1::2]) if interleaved else (head[..., :rot // 2], head[..., rot // 2:])
    u, w = a * cs - b * sn, b * cs + a * sn
    turned = torch.stack([u, w], -1).flatten(-2) if interleaved else torch.cat([u, w], -1)
    return torch.cat([turned, x[..., rot:]], -1)


def _quantised(x):
    """Codes of [-127, 127] and the scale of each head of x [tokens][heads][dim]."""
    top = x.abs().amax(-1, keepdim=True)
    some = top > 0
    codes = (x * torch.where(some, 127.0 / top, 1.0)).round().clamp(-127, 127).to(torch.int8)
    return codes, torch.where(some, top * (1.0 / 127), 1.0)[..., 0]


def _token_places(s):
    """Sequence and place in it of every row."""
    qs = s["q_start"].long()
    t = torch.arange(s["tokens"], device=qs.device)
    i = torch.searchsorted(qs[1:], t, right=True)
    seq = s["seqs"].long()[i]
    return seq, s["len"].long()[seq] - (qs[i + 1] - t)


def _store(s):
    c = s["case"]
    seq, pos = _token_places(s)
    page, slot, dt = s["table"][seq, pos // c["page"]].long(), pos % c["page"], DTYPES[c["dtype"]]
    q = _rotated(s["q_in"], s["cos"], s["sin"], pos, c["interleaved"]).to(dt)
    out = {"q": q}
    for name, x in (("k", _rotated(s["k_in"], s["cos"], s["sin"], pos, c["interleaved"])), ("v", s["v_in"].float())):
        codes, scale = _quantised(x)
        s[name][0][page, slot] = codes
        s[name + "_scale"][0][page, :, slot] = scale
        out[name] = (s[name][0][page, slot].float() * s[name + "_scale"][0][page, :, slot][..., None]).to(dt)
    return out


def _keep(s):
    ps, seqs, qs = s["case"]["page"], s["seqs"].long(), s["q_start"].long()
    s["len"].copy_(s["found"][0])
    s["refs"].copy_(s["found"][1])
    old, count = s["len"].long()[seqs], qs[1:] - qs[:-1]
    text = old - count
    t = torch.arange(s["tokens"], device=qs.device)
    i = torch.searchsorted(qs[1:], t, right=True)
    at = t - qs[i]
    some = at < s["counts"].long()[i]
    i, at, src = i[some], at[some], s["kept"].long()[some]
    a, b = text[i] + src, text[i] + at
    pa, pb = s["table"][seqs[i], a // ps].long(), s["table"][seqs[i], b // ps].long()
    s["k"][:, pb, b % ps] = s["k"][:, pa, a % ps]
    s["v"][:, pb, b % ps] = s["v"][:, pa, a % ps]
    if s["k_scale"] is not None:
        s["k_scale"][:, pb, :, b % ps] = s["k_scale"][:, pa, :, a % ps]
        s["v_scale"][:, pb, :, b % ps] = s["v_scale"][:, pa, :, a % ps]
    new = text + s["counts"].long()
    block = torch.arange(s["table"].shape[1], device=qs.device)
    gone = (block >= (-(-new // ps))[:, None]) & (block < (-(-old // ps))[:, None])
    s["refs"].index_add_(0, s["table"][seqs].long().reshape(-1), -gone.int().reshape(-1))
    s["len"][seqs] = new.int()
    return _cache_state(s)


def _ancestors(s, count, i):
    """[n][max_q][max_q]: whether a row's drafted token is, or descends from, that of the column; pointers double each step."""
    qs = s["q_start"].long()
    m = s["max_q"]
    rows = (qs[:-1, None] + i).clamp(max=s["tokens"] - 1)
    up = torch.where(i < count[:, None], s["parents"].long()[rows], -1)
    up = torch.cat([torch.where(up < 0, m, up), torch.full_like(up[:, :1], m)], 1)  # the last column: the text
    sees = torch.eye(m + 1, device=qs.device).expand(len(count), -1, -1)
    for _ in range(max(1, (m - 1).bit_length())):
        sees = torch.maximum(sees, sees.gather(1, up[..., None].expand(-1, -1, m + 1)))
        up = up.gather(1, up)
    return sees[:, :m, :m] > 0


def _attend(s):
    c, ps = s["case"], s["case"]["page"]
    dev, n, kv, d = s["q"].device, c["n"], c["kv_heads"], c["dim"]
    group = c["heads"] // kv
    seqs, qs = s["seqs"].long(), s["q_start"].long()
    length = s["len"].long()[seqs]
    span = s["table"].shape[1] * ps
    blocks = torch.arange(s["table"].shape[1], device=dev) < (-(-length // ps))[:, None]
    pages = torch.where(blocks, s["table"].long()[seqs], 0)
    keys, values = s["k"][0][pages].float(), s["v"][0][pages].float()
    if s["k_scale"] is not None:
        keys *= s["k_scale"][0][pages].transpose(-1, -2)[..., None]
        values *= s["v_scale"][0][pages].transpose(-1, -2)[..., None]
    keys, values = keys.view(n, span, kv, d), values.view(n, span, kv, d)
    count = qs[1:] - qs[:-1]
    i = torch.arange(s["max_q"], device=dev)
    rows = (qs[:-1, None] + i).clamp(max=s["tokens"] - 1)
    q = s["q"].float()[rows].view(n, s["max_q"], kv, group, d)
    logits = torch.einsum("nikgd,njkd->nkgij", q, keys) * s["scale"]
    text, j = length - count, torch.arange(span, device=dev)
    drafted = _ancestors(s, count, i) if c["tree"] else None
    pos = text[:, None] + (drafted.sum(-1) - 1 if c["tree"] else i)
    sees = (j < length[:, None, None]).expand(n, s["max_q"], span)
    if c["causal"] and not c["tree"]:
        sees = sees & (j <= pos[..., None])
    if c["window"] >= 0:
        sees = sees & (((j - pos[..., None]).abs() <= c["window"]) | (j < c["sinks"]))
    if c["tree"]:  # among the drafted tokens the tree alone decides
        of = j - text[:, None]
        sees = sees & (of < 0)[:, None]
        one = drafted.gather(2, of.clamp(0, s["max_q"] - 1)[:, None].expand(-1, s["max_q"], -1))
        sees = sees | (one & ((of >= 0) & (of < count[:, None]))[:, None])
    logits = logits.masked_fill_(~sees[:, None, None], -math.inf)
    top = logits.amax(-1, keepdim=True)
    p = logits.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    out = torch.einsum("nkgij,njkd->nikgd", p, values) / total[..., 0].permute(0, 3, 1, 2)[..., None]
    lse = (top + total.log())[..., 0].permute(0, 3, 1, 2)
    keep = i < count[:, None]
    result = {"out": out[keep].view(s["tokens"], c["heads"], d).to(s["q"].dtype), "lse": lse[keep].reshape(s["tokens"], c["heads"])}
    return {**result, "places": pos[keep].int()} if c["tree"] else result


def run(state):
    if own:
        return _run_own(state)
    return {"attend": _attend, "keep": _keep, "store": _store}[state["case"]["kind"]](state)


# ------------------------------------------------------------------------------------- what a pass cannot do without
def work(case):
    c, es = case, SIZE[case["dtype"]]
    row = c["kv_heads"] * c["dim"]
    held = row * 2 if c.get("held", "i8") == "16" else row + 4 * c["kv_heads"]  # bytes of a token's keys
    text, q = _lengths(c)
    tokens = sum(q)
    if c["kind"] == "store":
        spots = min(tokens, c["text"] + c["queries"])
        return {"bytes": tokens * (c["heads"] * c["dim"] * (SIZE[c["source"]] + es) + 2 * (row * (SIZE[c["source"]] + es) + 2 * held))
                + spots * c["rot"] * 4, "flops": tokens * (3 * (c["heads"] + c["kv_heads"]) * c["rot"] + 6 * row)}
    if c["kind"] == "keep":
        kept = sum(max(1, m // 3) for m in q)  # a path is about a third of its tree
        return {"bytes": 4 * c["layers"] * kept * held + 4 * (2 * tokens + 4 * c["n"]), "flops": 0}
    w, pairs, seen, parents = c["window"], 0, 0, _parents(c) if c["tree"] else None
    for i, (t, m) in enumerate(zip(text, q)):
        length = c["shared"] + t
        depth = []
        for r in range(m):
            if c["tree"]:
                depth.append(depth[parents[i][r]] + 1 if parents[i][r] >= 0 else 0)
                p, last = length - m + depth[r], length - m
            else:
                p, last = length - m + r, length
            hi = min(last, p + 1 if c["causal"] else last, p + w + 1 if w >= 0 else last)
            lo = max(0, p - w) if w >= 0 else 0
            pairs += max(0, hi - lo) + min(c["sinks"], lo, last) + (depth[r] + 1 if c["tree"] else 0)
        lo = max(0, length - m - w - c["tree"]) if w >= 0 else 0
        # the shared tokens are read once, for the first sequence
        seen += length - lo + min(c["sinks"], lo) if i == 0 else max(0, t - max(0, lo - c["shared"]))
        if i and c["sinks"] > c["shared"]:
            seen += max(0, min(c["sinks"], lo) - c["shared"])
    return {"bytes": 2 * seen * held + tokens * c["heads"] * (2 * c["dim"] * es + 4), "flops": 4 * pairs * c["heads"] * c["dim"]}


# ------------------------------------------------------------------------------------- the definitions, in 64 bits
def _turned(x, cos, sin, pos, interleaved):
    """Each pair (x, y) of a head as the complex number x + iy, times cos + i sin."""
    at = torch.arange(cos.shape[1], device=x.device)
    first, second = (2 * at, 2 * at + 1) if interleaved else (at, at + cos.shape[1])
    out = x.double()
    z = torch.complex(out[..., first], out[..., second]) * torch.complex(cos[pos].double(), sin[pos].double())[:, None]
    out[..., first], out[..., second] = z.real, z.imag
    return out


def _nearest(x):
    """What a head's 8 bits stand for: the nearest of 255 even steps between the ends of its largest magnitude."""
    step = x.abs().amax(-1, keepdim=True) / 127
    step[step == 0] = 1.0
    return torch.round(x / step) * step


def exact(case, seed):
    c = case
    if c["kind"] == "keep":
        return None  # nothing is computed: rows and whole numbers move
    if work(case)["flops"] > 1e12:
        return None
    s = prepare(case, seed)
    seqs, qs, table, length = s["seqs"].tolist(), s["q_start"].tolist(), s["table"].cpu(), s["len"].tolist()
    dev = s["k"].device
    if c["kind"] == "store":
        pos = torch.cat([torch.arange(length[q] - (qs[i + 1] - qs[i]), length[q]) for i, q in enumerate(seqs)]).to(dev)
        return {"q": _turned(s["q_in"], s["cos"], s["sin"], pos, c["interleaved"]),
                "k": _nearest(_turned(s["k_in"], s["cos"], s["sin"], pos, c["interleaved"])), "v": _nearest(s["v_in"].double())}
    group, parents = c["heads"] // c["kv_heads"], s["parents"].tolist() if c["tree"] else None
    out = torch.zeros(s["tokens"], c["heads"], c["dim"], dtype=torch.float64, device=dev)
    lse = torch.full((s["tokens"], c["heads"]), -math.inf, dtype=torch.float64, device=dev)

    def held(name, pages, count):
        x = s[name][0][pages].double()
        if s[name + "_scale"] is not None:
            x = x * s[name + "_scale"][0][pages].double().permute(0, 2, 1).unsqueeze(-1)
        return x.flatten(0, 1)[:count]

    for i, q in enumerate(seqs):
        count, rows = length[q], qs[i + 1] - qs[i]
        pages = table[q][:_ceil(count, c["page"])].long().to(dev)
        k, v = held("k", pages, count), held("v", pages, count)
        j = torch.arange(count, device=dev)[None]
        if c["tree"]:
            line = torch.zeros(rows, rows, dtype=torch.bool)
            for r in range(rows):
                if parents[qs[i] + r] >= 0:
                    line[r] = line[parents[qs[i] + r]]
                line[r, r] = True
            p = (count - rows + line.sum(1) - 1).to(dev)[:, None]
            hidden = torch.zeros(rows, count, dtype=torch.bool, device=dev)
        else:
            p = torch.arange(count - rows, count, device=dev)[:, None]
            hidden = (j > p) if c["causal"] else torch.zeros(rows, count, dtype=torch.bool, device=dev)
        if c["window"] >= 0:
            hidden = hidden | (((j < p - c["window"]) | (j > p + c["window"])) & (j >= c["sinks"]))
        if c["tree"]:
            hidden[:, count - rows:] = ~line.to(dev)
        x = s["q"][qs[i]:qs[i + 1]].double()
        for h in range(c["heads"]):
            a = (x[:, h] @ k[:, h // group].T) * s["scale"]
            a[hidden] = -math.inf
            r = torch.logsumexp(a, 1)
            out[qs[i]:qs[i + 1], h] = torch.exp(a - r[:, None]) @ v[:, h // group]
            lse[qs[i]:qs[i + 1], h] = r
    return {"out": out, "lse": lse, "places": None} if c["tree"] else {"out": out, "lse": lse}
