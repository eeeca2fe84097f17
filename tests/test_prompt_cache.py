"""The prompt-cache entry points without a GPU: every refusal comes before any device work, and leaves a
message. Pointers below are never dereferenced: each call is refused by its argument checks."""
from __future__ import annotations

import ctypes as C

import pytest

PTR = 0x1000  # 16-byte aligned, never read


def pages(e2c, **over):
    f = dict(k=PTR, v=PTR, table=PTR, len=PTR, refs=PTR, ws=PTR, type=e2c.BF16, layers=2, n_pages=16, page=16, kv_heads=2,
             head_dim=64, max_seqs=4, max_blocks=8)
    f.update(over)
    return e2c.Pages(**f)


BAD_CACHES = [dict(k=None), dict(v=None), dict(table=None), dict(len=None), dict(refs=None), dict(ws=None), dict(type=0), dict(type=3),
              dict(layers=0), dict(n_pages=0), dict(page=4), dict(page=24), dict(page=2048), dict(kv_heads=0), dict(head_dim=96),
              dict(max_seqs=0), dict(max_blocks=0), dict(max_blocks=1 << 21), dict(k=PTR + 8), dict(refs=PTR + 4),
              dict(n_pages=1 << 28), dict(page=1024, max_blocks=1 << 20 | 1)]


@pytest.mark.parametrize("over", BAD_CACHES, ids=[str(o) for o in BAD_CACHES])
def test_bad_cache_is_refused(e2c, over):
    lib, p = e2c.lib(), pages(e2c, **over)
    a = C.addressof(p)
    for rc in (lib.e2cuda_pages_fork(a, PTR, PTR, 1, None), lib.e2cuda_pages_append(a, PTR, PTR, 1, None),
               lib.e2cuda_pages_free(a, PTR, 1, None), lib.e2cuda_pages_compact(a, None, None),
               lib.e2cuda_pages_copy(a, PTR, PTR, 1, None),
               lib.e2cuda_pages_attention(a, 0, PTR, 256, PTR, PTR, 1, 1, 1, 4, 0, 1, -1, 1.0, PTR, 256, None, PTR, 1 << 30, None)):
        assert rc == -1 and e2c.last_error().startswith("pages_")
    assert lib.e2cuda_pages_attention_ws_bytes(a, 1, 1, 1, 4, 0) == 0


@pytest.mark.parametrize("n", [-1, 5])
def test_bad_lists_are_refused(e2c, n):
    """More entries than sequences cannot be distinct."""
    lib, p = e2c.lib(), pages(e2c)
    a = C.addressof(p)
    assert lib.e2cuda_pages_fork(a, PTR, PTR, n, None) == -1
    assert lib.e2cuda_pages_append(a, PTR, PTR, n, None) == -1
    assert lib.e2cuda_pages_free(a, PTR, n, None) == -1
    assert lib.e2cuda_pages_copy(a, PTR, PTR, n if n < 0 else 17, None) == -1
    assert "list" in e2c.last_error()
    assert lib.e2cuda_pages_append(a, None, PTR, 1, None) == -1
    assert lib.e2cuda_pages_append(a, PTR, None, 1, None) == -1


@pytest.mark.parametrize("n", [0])
def test_empty_lists_do_nothing(e2c, n):
    lib, p = e2c.lib(), pages(e2c)
    a = C.addressof(p)
    assert lib.e2cuda_pages_fork(a, None, None, n, None) == 0
    assert lib.e2cuda_pages_append(a, None, None, n, None) == 0
    assert lib.e2cuda_pages_free(a, None, n, None) == 0
    assert lib.e2cuda_pages_copy(a, None, None, n, None) == 0


ATTENTION = dict(layer=0, q=PTR, ldq=256, seqs=PTR, q_start=PTR, n=2, T=4, max_q=2, heads=4, shared=0, causal=1, window=-1,
                 scale=1.0, out=PTR, ldo=256, lse=None, ws=PTR, ws_bytes=1 << 40)
BAD_ATTENTION = [dict(layer=2), dict(layer=-1), dict(q=None), dict(q=PTR + 2), dict(out=PTR + 8), dict(ldq=255), dict(ldq=260),
                 dict(ldo=128), dict(seqs=None), dict(q_start=None), dict(n=0), dict(T=-1), dict(max_q=0), dict(max_q=5),
                 dict(heads=3), dict(heads=1), dict(heads=258, ldq=1 << 20, ldo=1 << 20), dict(shared=8), dict(shared=-16),
                 dict(shared=256), dict(scale=float("nan")), dict(scale=float("inf")), dict(out=None)]


@pytest.mark.parametrize("over", BAD_ATTENTION, ids=[str(o) for o in BAD_ATTENTION])
def test_bad_attention_is_refused(e2c, over):
    p = pages(e2c)
    assert e2c.lib().e2cuda_pages_attention(C.addressof(p), *dict(ATTENTION, **over).values(), None) == -1
    assert e2c.last_error().startswith("pages_attention")


BAD_SIZES = [dict(n=0), dict(T=0), dict(max_q=0), dict(heads=3), dict(heads=1), dict(heads=258), dict(heads=256 * 129), dict(shared=-16)]


@pytest.mark.parametrize("over", BAD_SIZES, ids=[str(o) for o in BAD_SIZES])
def test_bad_attention_workspace_is_refused(e2c, over):
    """The size is asked for before the call: what the call refuses has none, and says so."""
    lib, p = e2c.lib(), pages(e2c)
    lib.e2cuda_pages_copy(C.addressof(p), None, None, -1, None)  # leaves another message
    size = lib.e2cuda_pages_attention_ws_bytes(C.addressof(p), *dict(dict(n=2, T=4, max_q=2, heads=4, shared=0), **over).values())
    assert size == 0
    assert e2c.last_error().startswith("pages_attention")


def test_no_rows_do_nothing(e2c):
    p = pages(e2c)
    assert e2c.lib().e2cuda_pages_attention(C.addressof(p), *dict(ATTENTION, T=0).values(), None) == 0


STORE = dict(layer=0, x_type=1, q=PTR, ldq=256, k=PTR, ldk=128, v=PTR, ldv=128, q_out=0x2000, ldo=256, cos=PTR, sin=PTR,
             positions=64, rot=64, flags=0, seqs=PTR, q_start=PTR, n=2, T=4, heads=4)
BAD_STORE = [dict(layer=2), dict(x_type=2), dict(x_type=7), dict(q=None), dict(k=None), dict(v=None), dict(q_out=None), dict(cos=None),
             dict(ldq=255), dict(ldk=127), dict(ldv=127), dict(ldo=255), dict(positions=0), dict(rot=0), dict(rot=63), dict(rot=66),
             dict(flags=2), dict(n=0), dict(T=-1), dict(heads=3), dict(seqs=None), dict(x_type=0, q_out=PTR),
             dict(q_out=PTR, ldo=512)]


@pytest.mark.parametrize("over", BAD_STORE, ids=[str(o) for o in BAD_STORE])
def test_bad_store_is_refused(e2c, over):
    p = pages(e2c)
    assert e2c.lib().e2cuda_pages_store(C.addressof(p), *dict(STORE, **over).values(), None) == -1
    assert e2c.last_error().startswith("pages_store")


ROPE = dict(x=PTR, ldx=256, x_type=1, y=0x2000, ldy=256, y_type=1, cos=PTR, sin=PTR, positions=64, rot=64, pos=PTR, T=4, heads=4,
            head_dim=64, flags=0)
BAD_ROPE = [dict(x=None), dict(y=None), dict(cos=None), dict(sin=None), dict(ldx=255), dict(ldy=255), dict(x_type=1, y_type=2),
            dict(x_type=1, y_type=0), dict(x_type=3), dict(y_type=-1), dict(positions=0), dict(rot=0), dict(rot=7), dict(rot=66),
            dict(T=-1), dict(heads=0), dict(flags=4), dict(pos=None, T=65), dict(y=PTR, x_type=0), dict(y=PTR, ldy=512)]


@pytest.mark.parametrize("over", BAD_ROPE, ids=[str(o) for o in BAD_ROPE])
def test_bad_rope_is_refused(e2c, over):
    assert e2c.lib().e2cuda_rope(*dict(ROPE, **over).values(), None) == -1
    assert e2c.last_error().startswith("rope")


BAD_TABLE = [dict(cos=None), dict(sin=None), dict(positions=0), dict(rot=0), dict(rot=3), dict(rot=514), dict(theta=0.0),
             dict(theta=float("nan")), dict(s=dict(kind=5)), dict(s=dict(kind=-1)), dict(s=dict(kind=1, factor=0.5)),
             dict(s=dict(kind=2, factor=float("nan"))), dict(s=dict(kind=3, factor=2.0, original=0)),
             dict(s=dict(kind=3, factor=2.0, original=64, fast=1.0, slow=4.0)),
             dict(s=dict(kind=4, factor=2.0, original=64), theta=0.5)]


@pytest.mark.parametrize("over", BAD_TABLE, ids=[str(o) for o in BAD_TABLE])
def test_bad_rope_table_is_refused(e2c, over):
    a = dict(cos=PTR, sin=PTR, positions=8, rot=8, theta=1e4, s=None)
    a.update(over)
    if a["s"] is not None:
        a["s"] = C.byref(e2c.RopeScaling(**a["s"]))
    assert e2c.lib().e2cuda_rope_table(*a.values(), None) == -1
    assert e2c.last_error().startswith("rope_table")


def test_ws_bytes(e2c):
    lib = e2c.lib()
    assert lib.e2cuda_pages_ws_bytes(1000, 10) >= 4 * 3 * 1010
    assert lib.e2cuda_pages_ws_bytes(-1, 10) == 0


def test_host_tensors_are_refused(e2c):
    """Every tensor of a call passes one of these; a host address must not reach a kernel."""
    torch = pytest.importorskip("torch")
    rows, ints, table = torch.zeros(3, 2, 64), torch.zeros(3, dtype=torch.int32), torch.zeros(8, 32)
    for f, args in ((e2c._rows, (rows, "x", 0)), (e2c._ints, (ints, 3, "x", 0)), (e2c._table, (table, table, 0))):
        with pytest.raises(e2c.E2CudaError, match="cuda:0, got cpu"):
            f(*args)


@pytest.mark.parametrize("ld", [2 ** 31, 2 ** 32, 2 ** 32 + 128])
def test_rows_further_apart_than_an_int_are_refused(e2c, ld):
    """The library's row strides are ints; a view of a larger tensor must not be read at another one."""
    class View:
        shape = (3, 2, 64)
        device = "cuda:0"

        def stride(self):
            return (ld, 64, 1)

        def get_device(self):
            return 0

    with pytest.raises(e2c.E2CudaError, match="elements apart"):
        e2c._rows(View(), "q", 0)
