"""Embed many texts behind one instruction with a causal tower: the instruction is run once.

A small causal decoder with random int8 weights (the library's W8A8 products) embeds each text as the
mean of its last layer's rows, as an instruction-tuned embedder does. The instruction's keys and values are
stored once in a paged cache, every text is a fork of it, and the texts' attention reads the
instruction's pages once for the batch (e2cuda_rope_table, e2cuda_pages_fork / _append / _store /
_attention / _free / _compact). For comparison the same texts are run with the instruction recomputed for
each of them; the embeddings agree.

    python examples/prompt_cache.py [--texts 64] [--instruction 2048] [--text 40] [--layers 4]
"""
from __future__ import annotations

import argparse
import importlib.util
import sys
from pathlib import Path

import numpy as np
import torch

ROOT = Path(__file__).resolve().parent.parent


def load_package():
    if "e2c_b200" not in sys.modules:
        pkg = ROOT / "e2.c_b200"
        spec = importlib.util.spec_from_file_location("e2c_b200", pkg / "__init__.py", submodule_search_locations=[str(pkg)])
        mod = importlib.util.module_from_spec(spec)
        sys.modules["e2c_b200"] = mod
        spec.loader.exec_module(mod)
    return sys.modules["e2c_b200"]


class Tower:
    """A causal decoder: RMSNorm, q|k|v, rotary attention over the cache, o, RMSNorm, gated MLP."""

    HIDDEN, HEADS, KV, DIM, FFN, PAGE = 512, 8, 2, 128, 1024, 32

    def __init__(self, e2c, layers: int, max_tokens: int, seed: int = 0):
        self.e2c, self.layers = e2c, layers
        rng = np.random.default_rng(seed)

        def weight(n, k):
            w = rng.integers(-127, 128, (n, k), dtype=np.int8)
            return e2c.Weight(w=w, scale=np.full(n, 1.0 / (73.0 * np.sqrt(k)), np.float32))

        width = (self.HEADS + 2 * self.KV) * self.DIM
        self.w = [dict(qkv=weight(width, self.HIDDEN), o=weight(self.HIDDEN, self.HEADS * self.DIM),
                       up=weight(2 * self.FFN, self.HIDDEN), down=weight(self.HIDDEN, self.FFN)) for _ in range(layers)]
        # trained on 4096 positions, used on four times as many
        self.cos, self.sin = e2c.rope_table(max(max_tokens, 16384), self.DIM,
                                            scaling=e2c.RopeScaling(e2c.ROPE_BY_ROTATIONS, 4096, 4.0, 0, 0, 0))

    def linear(self, x, w):
        q, s = self.e2c.quantize_rows(x.contiguous())
        return self.e2c.i8_gemm(w, q, s)

    @staticmethod
    def norm(x):
        return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6)

    def run(self, cache, x, seqs, q_start, max_q, shared):
        """The rows x (the last tokens of their sequences, which append has grown) through every layer."""
        for layer, w in enumerate(self.w):
            rows = self.linear(self.norm(x), w["qkv"]).unflatten(1, (self.HEADS + 2 * self.KV, self.DIM))
            q, k, v = rows.split([self.HEADS, self.KV, self.KV], 1)
            q = cache.store(layer, q, k, v, self.cos, self.sin, seqs, q_start)
            a = cache.attention(layer, q, seqs, q_start, max_q, shared=shared)
            x = x + self.linear(a.flatten(1).float(), w["o"])
            gate, up = self.linear(self.norm(x), w["up"]).chunk(2, -1)
            x = x + self.linear(torch.nn.functional.gelu(gate, approximate="tanh") * up, w["down"])
        return self.norm(x)


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def pooled(x, lengths):
    """Unit-length means of each text's rows."""
    parts = torch.stack([p.mean(0) for p in x.split(lengths)])
    return parts / parts.norm(dim=1, keepdim=True)


def embed(e2c, texts: int, instruction: int, text: int, layers: int, seed: int = 0):
    """(shared, recomputed, milliseconds of each): embeddings of the texts behind the instruction."""
    rng = np.random.default_rng(seed)
    lengths = [int(n) for n in rng.integers(max(1, text // 2), text + 1, texts)]
    tower = Tower(e2c, layers, instruction + text)
    page = tower.PAGE
    g = torch.Generator(device="cuda").manual_seed(seed)
    prompt = torch.randn(instruction, tower.HIDDEN, generator=g, device="cuda")
    rows = torch.randn(sum(lengths), tower.HIDDEN, generator=g, device="cuda")
    per_text = -(-(instruction + text) // page) + 1
    starts = np.concatenate([[0], np.cumsum(lengths)]).tolist()

    def new_cache(n_pages):
        return e2c.PageCache.new(layers, n_pages, page, tower.KV, tower.DIM, texts + 1, per_text, torch.bfloat16)

    cache = new_cache(-(-instruction // page) + texts * (-(-text // page) + 2))
    children = ints(range(1, texts + 1))

    def shared():
        cache.append(ints([0]), ints([instruction]))
        tower.run(cache, prompt, ints([0]), ints([0, instruction]), instruction, 0)
        cache.fork(ints([0] * texts), children)
        cache.append(children, ints(lengths))
        x = tower.run(cache, rows, children, ints(starts), max(lengths), instruction // page * page)
        cache.free(torch.cat([ints([0]), children]))
        cache.compact()
        return pooled(x, lengths)

    whole = new_cache(texts * per_text)
    full = [instruction + n for n in lengths]
    full_starts = ints(np.concatenate([[0], np.cumsum(full)]).tolist())
    full_rows = torch.cat([torch.cat([prompt, r]) for r in rows.split(lengths)])

    def recomputed():
        whole.append(children, ints(full))
        x = tower.run(whole, full_rows, children, full_starts, max(full), 0)
        whole.free(children)
        return pooled(torch.cat([p[instruction:] for p in x.split(full)]), lengths)

    out, ms = [], []
    for f in (shared, recomputed):
        f()
        torch.cuda.synchronize()
        a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        a.record()
        out.append(f())
        b.record()
        e2c.check()
        ms.append(a.elapsed_time(b))
    return out[0], out[1], ms


def main():
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    for name, value in (("texts", 64), ("instruction", 2048), ("text", 40), ("layers", 4)):
        ap.add_argument("--" + name, type=int, default=value)
    a = ap.parse_args()
    one, other, ms = embed(load_package(), a.texts, a.instruction, a.text, a.layers)
    print(f"{a.texts} texts behind {a.instruction} tokens: shared {ms[0]:.2f} ms, recomputed {ms[1]:.2f} ms, "
          f"least cosine {(one * other).sum(1).min().item():.6f}")


if __name__ == "__main__":
    main()
