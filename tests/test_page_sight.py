"""The entry points for sinks, trees of drafted tokens and pages of 8 bits without a GPU: every refusal comes before any device
work, and leaves a message. Pointers below are never dereferenced: each call is refused by its argument checks."""
from __future__ import annotations

import ctypes as C

import pytest

from test_prompt_cache import ATTENTION, PTR, STORE, pages


def codes(e2c, **over):
    return pages(e2c, **dict(dict(type=e2c.I8, k_scale=PTR, v_scale=PTR), **over))


@pytest.mark.parametrize("over", [dict(k_scale=None), dict(v_scale=None), dict(k_scale=PTR + 4), dict(v_scale=PTR + 8), dict(head_dim=32)],
                         ids=str)
def test_bad_cache_of_8_bits_is_refused(e2c, over):
    lib, p = e2c.lib(), codes(e2c, **over)
    a = C.addressof(p)
    assert lib.e2cuda_pages_compact(a, None, None) == -1 and e2c.last_error().startswith("pages_compact")
    assert lib.e2cuda_pages_load(a, 0, PTR, None, PTR, 1, 1, PTR, PTR, 1, None) == -1
    assert lib.e2cuda_pages_attention_ws_bytes(a, 1, 1, 1, 4, 0) == 0


def sight(e2c, **over):
    return e2c.Sight(**dict(dict(causal=1, window=-1, sinks=0, words=0, tree=None), **over))


def attend(e2c, p, s, q_type, **over):
    a = dict(ATTENTION, **over)
    return e2c.lib().e2cuda_pages_attention_sight(C.addressof(p), a["layer"], q_type, a["q"], a["ldq"], a["seqs"], a["q_start"], a["n"], a["T"],
                                                  a["max_q"], a["heads"], a["shared"], None if s is None else C.addressof(s), a["scale"],
                                                  a["out"], a["ldo"], a["lse"], a["ws"], a["ws_bytes"], None)


BAD_SIGHT = [dict(sinks=-1), dict(tree=PTR, words=0), dict(tree=PTR + 2, words=1), dict(tree=PTR, words=-1)]


@pytest.mark.parametrize("over", BAD_SIGHT, ids=str)
def test_bad_sight_is_refused(e2c, over):
    assert attend(e2c, pages(e2c), sight(e2c, **over), e2c.BF16) == -1
    assert e2c.last_error().startswith("pages_attention")


def test_tree_with_fewer_words_than_rows_is_refused(e2c):
    assert attend(e2c, pages(e2c), sight(e2c, tree=PTR, words=1), e2c.BF16, T=40, max_q=33) == -1
    assert "33" in e2c.last_error()


def test_no_sight_is_refused(e2c):
    assert attend(e2c, pages(e2c), None, e2c.BF16) == -1


@pytest.mark.parametrize("cache,q_type", [("16", 2), ("16", 0), ("16", 3), ("8", 0), ("8", 3), ("8", 7), ("8", -1)])
def test_q_of_another_type_is_refused(e2c, cache, q_type):
    p = pages(e2c) if cache == "16" else codes(e2c)
    assert attend(e2c, p, sight(e2c), q_type) == -1
    assert "type" in e2c.last_error()


def test_attention_without_q_type_is_refused_over_8_bits(e2c):
    """The older entry takes q in the cache's type, which 8 bits are not for q."""
    p = codes(e2c)
    assert e2c.lib().e2cuda_pages_attention(C.addressof(p), *ATTENTION.values(), None) == -1


AT = dict(layer=0, x_type=1, q=PTR, ldq=256, k=PTR, ldk=128, v=PTR, ldv=128, q_out=0x2000, q_type=1, ldo=256, cos=PTR, sin=PTR,
          positions=64, rot=64, flags=0, pos=PTR, seqs=PTR, q_start=PTR, n=2, T=4, heads=4)
BAD_AT = [dict(q_type=2), dict(q_type=0), dict(x_type=2), dict(q=None), dict(rot=65), dict(rot=66), dict(positions=0), dict(flags=2),
          dict(ldk=64), dict(heads=3), dict(layer=2)]


@pytest.mark.parametrize("over", BAD_AT, ids=str)
def test_bad_store_at_is_refused(e2c, over):
    p = pages(e2c)
    assert e2c.lib().e2cuda_pages_store_at(C.addressof(p), *dict(AT, **over).values(), None) == -1
    assert e2c.last_error().startswith("pages_store")


@pytest.mark.parametrize("over", [dict(q_type=0), dict(q_type=3), dict(x_type=3), dict(x_type=-1), dict(x_type=0, q_out=PTR)], ids=str)
def test_bad_store_into_8_bits_is_refused(e2c, over):
    p = codes(e2c)
    assert e2c.lib().e2cuda_pages_store_at(C.addressof(p), *dict(AT, **over).values(), None) == -1
    assert e2c.last_error().startswith("pages_store")


def test_store_of_fp32_needs_a_type_over_8_bits(e2c):
    p = codes(e2c)
    assert e2c.lib().e2cuda_pages_store(C.addressof(p), *dict(STORE, x_type=0).values(), None) == -1


LOAD = dict(layer=0, seqs=PTR, first=None, q_start=PTR, n=1, T=4, k=PTR, v=PTR, type=1)


@pytest.mark.parametrize("over", [dict(layer=2), dict(seqs=None), dict(q_start=None), dict(n=0), dict(T=-1), dict(k=None), dict(v=PTR + 8),
                                  dict(type=3), dict(type=-1)], ids=str)
def test_bad_load_is_refused(e2c, over):
    p = pages(e2c)
    assert e2c.lib().e2cuda_pages_load(C.addressof(p), *dict(LOAD, **over).values(), None) == -1
    assert e2c.last_error().startswith("pages_load")


TREE = dict(parents=PTR, seqs=PTR, q_start=PTR, n=1, T=4, tree=PTR, words=1, pos=None)


@pytest.mark.parametrize("over", [dict(parents=None), dict(seqs=None), dict(q_start=None), dict(n=0), dict(T=-1), dict(tree=None),
                                  dict(words=0), dict(T=1 << 20, words=1 << 12)], ids=str)
def test_bad_tree_is_refused(e2c, over):
    p = pages(e2c)
    assert e2c.lib().e2cuda_pages_tree(C.addressof(p), *dict(TREE, **over).values(), None) == -1
    assert e2c.last_error().startswith("pages_tree")


KEEP = dict(seqs=PTR, q_start=PTR, kept=PTR, counts=PTR, n=1, T=4)


@pytest.mark.parametrize("over", [dict(seqs=None), dict(q_start=None), dict(kept=None), dict(counts=None), dict(n=-1), dict(n=5), dict(T=-1)],
                         ids=str)
def test_bad_keep_is_refused(e2c, over):
    p = pages(e2c)
    assert e2c.lib().e2cuda_pages_keep(C.addressof(p), *dict(KEEP, **over).values(), None) == -1
    assert e2c.last_error().startswith("pages_keep")


def test_nothing_to_do(e2c):
    lib, p = e2c.lib(), codes(e2c)
    a = C.addressof(p)
    assert attend(e2c, p, sight(e2c), e2c.F16, T=0) == 0
    assert lib.e2cuda_pages_load(a, *dict(LOAD, T=0).values(), None) == 0
    assert lib.e2cuda_pages_tree(a, *dict(TREE, T=0).values(), None) == 0
    assert lib.e2cuda_pages_keep(a, *dict(KEEP, n=0).values(), None) == 0
    assert lib.e2cuda_pages_keep(a, *dict(KEEP, T=0).values(), None) == 0
