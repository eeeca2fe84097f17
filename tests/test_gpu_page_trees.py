"""Trees of few drafted rows behind long texts, whose items are divided among blocks and joined: on the GPU, against the
64-bit form of test_gpu_page_sight.py, with its tolerances."""
from __future__ import annotations

import numpy as np
import pytest

from test_gpu_page_sight import assert_codes, dev, largest, make_codes, random_parents, sight64, tree_mask, tree_words
from test_gpu_prompt_cache import assert_attention, make_batch

pytestmark = pytest.mark.gpu

SHAPES = {
    # texts, rows an entry at most, H, KV, D, page: entries by the lane of one warp (up to 32), or planned by the block
    "few long ones, 8 rows": ([9000, 8771, 5003], 2, 8, 2, 128, 16),
    "few long ones, 16 rows": ([9000, 8771, 5003], 4, 16, 4, 128, 32),
    "few long ones, heads of 64": ([9000, 8771, 5003], 4, 8, 4, 64, 8),
    "few long ones, heads of 256": ([4100, 3771, 9001], 5, 6, 2, 256, 64),
    "many, 8 rows": ([1500 + 7 * i for i in range(70)], 4, 4, 2, 128, 16),
    "many, 16 rows": ([1500 - 5 * i for i in range(70)], 8, 8, 4, 64, 128),
    "many, heads of 256": ([700 + 11 * i for i in range(70)], 4, 8, 2, 256, 32),
    # 16 blocks side by side for a share's key heads
    "many heads": ([3000 + 77 * i for i in range(40)], 2, 32, 16, 64, 16),
}


@pytest.mark.parametrize("held", ["f16", "bf16", "i8"])
@pytest.mark.parametrize("window,sinks", [(-1, 0), (600, 5), (2500, 130)])
@pytest.mark.parametrize("case", list(SHAPES))
def test_few_drafts_behind_long_texts(e2c, torch_cuda, case, window, sinks, held):
    torch = torch_cuda
    texts, most, H, KV, D, page = SHAPES[case]
    rng = np.random.default_rng(len(case))
    rows = [most - i % min(most, 3) for i in range(len(texts))]
    make, name = (make_codes, "bf16") if held == "i8" else (make_batch, held)
    cache, q, seqs, q_start, max_q = make(e2c, torch, 16, [t + r for t, r in zip(texts, rows)], rows, 0, H, KV, D, page, name)
    parents = [random_parents(rng, rows[s]) for s in seqs.tolist()]
    tree, _ = cache.tree(dev(torch, sum(parents, [])), seqs, q_start, max_q)
    out, lse = cache.attention(0, q, seqs, q_start, max_q, window=window, sinks=sinks, tree=tree, lse=True)
    again = cache.attention(0, q, seqs, q_start, max_q, window=window, sinks=sinks, tree=tree)
    e2c.check()
    want = sight64(torch, cache, 0, q, seqs, q_start, True, window, D ** -0.5, sinks, [tree_mask(p) for p in parents])
    if held == "i8":
        assert_codes(torch, out, lse, want, name, max(texts) + most, largest(cache))
    else:
        assert_attention(torch, out, lse, want, name, max(texts) + most)
    assert torch.equal(again, out), "two calls differ"


@pytest.mark.parametrize("held", ["f16", "i8"])
@pytest.mark.parametrize("n", [3, 70])
def test_rows_without_bits(e2c, torch_cuda, n, held):
    """Such a row sees the text; where every logit is -infinity it is NaN, and where there is no text it is zeros, in items that
    blocks share too."""
    torch = torch_cuda
    lens, rows, H, KV, D = [6000 if i % 2 == 0 else 2 for i in range(n)], [2] * n, 8, 2, 128
    make = make_codes if held == "i8" else make_batch
    cache, q, seqs, q_start, max_q = make(e2c, torch, 17, lens, rows, 0, H, KV, D, 32, "f16")
    masks = [np.array([[False, False], [True, False]]) for _ in lens]
    tree = torch.tensor(tree_words(masks, 1), device="cuda")
    out, lse = cache.attention(0, q, seqs, q_start, max_q, tree=tree, lse=True)
    e2c.check()
    want = sight64(torch, cache, 0, q, seqs, q_start, True, -1, D ** -0.5, 0, masks)
    if held == "i8":
        assert_codes(torch, out, lse, want, "f16", 6000, largest(cache))
    else:
        assert_attention(torch, out, lse, want, "f16", 6000)
    short = (cache.length[seqs.long()] == 2).repeat_interleave(2)
    none = short & (torch.arange(2 * n, device="cuda") % 2 == 0)
    assert torch.isinf(lse[none]).all() and (out[none] == 0).all() and not torch.isinf(lse[~none]).any()
    if held == "f16":  # -infinity for every key of the text
        cache.k[0].nan_to_num_(0.0)
        cache.k[0, ..., 0] = -float("inf")
        q[..., 0] = 1.0
        out, lse = cache.attention(0, q, seqs, q_start, max_q, tree=tree, lse=True)
        e2c.check()
        assert torch.isnan(out[~none]).all() and (out[none] == 0).all() and (lse == -float("inf")).all()


def test_bounds_of_any_size(e2c, torch_cuda):
    """A bound on an entry's rows may be one kept for all batches; a number of sinks below zero is refused, however far."""
    torch = torch_cuda
    cache, q, seqs, q_start, max_q = make_batch(e2c, torch, 18, [50, 40], [3, 2], 0, 4, 2, 64, 16, "f16")
    parents = dev(torch, [-1, 0, 0, -1, -1])
    want, pos = cache.tree(parents, seqs, q_start, max_q)
    tree, at = cache.tree(parents, seqs, q_start, 2 ** 31 - 1)
    assert torch.equal(tree, want) and torch.equal(at, pos)
    out = cache.attention(0, q, seqs, q_start, 2 ** 31 - 1, tree=tree)
    assert torch.equal(out, cache.attention(0, q, seqs, q_start, max_q, tree=want))
    e2c.check()
    for sinks in (-1, -2 ** 31 - 5, -2 ** 32):
        with pytest.raises(e2c.E2CudaError, match="sinks"):
            cache.attention(0, q, seqs, q_start, max_q, window=3, sinks=sinks)


def test_a_tree_without_words_is_refused(e2c, torch_cuda):
    """An empty tensor has no address, and is not taken for no tree."""
    torch = torch_cuda
    cache, q, seqs, q_start, max_q = make_batch(e2c, torch, 19, [50, 40], [3, 2], 0, 4, 2, 64, 16, "f16")
    with pytest.raises(e2c.E2CudaError, match="tree of 5 rows of words"):
        cache.attention(0, q, seqs, q_start, max_q, tree=torch.zeros(5, 0, dtype=torch.int32, device="cuda"))
