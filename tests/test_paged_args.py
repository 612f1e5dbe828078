"""Refusals of the paged cache's C entries and the oracle's own cases, on the
CPU: arguments are checked before a GPU is touched."""

import ctypes
import os

import numpy as np
import pytest

import mlxvs_b200 as mv
from mlxvs_b200 import paged
from oracle import paged as O


@pytest.fixture(scope="module")
def lib():
    if not os.path.exists(mv.library_path()):
        from mlxvs_b200 import build

        build.build()
    return mv._load()


AT = 4096  # an aligned address that nothing reads


def cache(**kw):
    c = dict(keys=AT, values=AT, kp=2048, kr=256, kh=128, vp=2048, vr=256, vh=128, pages=10,
             codes=AT, scales=AT, page=8, heads=2, dim=128, type=1, ks=1.0, vs=1.0)
    c.update(kw)
    return paged._CACHE.pack(*c.values())


def queries(**kw):
    q = dict(q=AT, tokens=3, ts=1024, hs=128, table=AT, rows=4, width=5, requests=AT, lengths=AT,
             heads=8, type=1)
    q.update(kw)
    return paged._QUERIES.pack(*q.values())


def refused(lib, rc, text):
    assert rc == 1, lib.mlxvs_last_error()
    assert text.encode() in lib.mlxvs_last_error(), lib.mlxvs_last_error()


@pytest.mark.parametrize("change,text", [
    (dict(page=0), "page_size must be in [1, 1024]"),
    (dict(page=1025), "page_size must be in [1, 1024]"),
    (dict(pages=-1), "number of pages"),
    (dict(heads=0), "key heads"),
    (dict(dim=0), "head dimension"),
    (dict(dim=132), "multiple of 8"),
    (dict(dim=264), "at most 256"),
    (dict(dim=24, type=2), "multiple of 16"),
    (dict(type=0), "the cache must have their type"),
    (dict(type=7), "the cache must have their type"),
    (dict(keys=0), "must not be NULL"),
    (dict(values=AT + 8), "16-byte aligned"),
    (dict(kr=257), "strides must be multiples of 16 bytes"),
    (dict(vp=-8), "strides must be multiples of 16 bytes"),
    (dict(ks=0.0), "positive and finite"),
    (dict(vs=float("nan")), "positive and finite"),
])
def test_cache_refusals(lib, change, text):
    c = cache(**change)
    refused(lib, lib.mlxvs_paged_attention_device(c, queries(), None, 0, 1.0, AT, None, None), text)
    refused(lib, lib.mlxvs_paged_store_device(c, AT, AT, 1, 3, 256, 128, 256, 128, AT, None), text)


@pytest.mark.parametrize("change,text", [
    (dict(type=2), "must be float16 or bfloat16"),
    (dict(tokens=-1), "tokens must be in"),
    (dict(heads=7), "times the key heads"),
    (dict(heads=0), "times the key heads"),
    (dict(heads=2 * 129), "times the key heads"),
    (dict(rows=-1), "table must be int32"),
    (dict(q=0), "q and lengths must not be NULL"),
    (dict(lengths=0), "q and lengths must not be NULL"),
    (dict(table=0), "table must not be NULL"),
    (dict(requests=0, rows=2), "needs a row of the table"),
    (dict(q=AT + 2), "16-byte aligned"),
    (dict(ts=1001), "multiples of 16 bytes"),
])
def test_query_refusals(lib, change, text):
    q = queries(**change)
    refused(lib, lib.mlxvs_paged_attention_device(cache(), q, None, 0, 1.0, AT, None, None), text)
    refused(lib, lib.mlxvs_paged_select_device(cache(), q, 4, 1, 1, AT, None), text)


def test_other_refusals(lib):
    attend = lib.mlxvs_paged_attention_device
    refused(lib, attend(None, queries(), None, 0, 1.0, AT, None, None), "must not be NULL")
    refused(lib, attend(cache(), None, None, 0, 1.0, AT, None, None), "must not be NULL")
    refused(lib, attend(cache(), queries(), AT, 0, 1.0, AT, None, None), "pages must be int32")
    refused(lib, attend(cache(), queries(), None, 0, float("inf"), AT, None, None), "scale")
    refused(lib, attend(cache(), queries(), None, 0, 1.0, None, None, None), "out must not be NULL")
    select = lib.mlxvs_paged_select_device
    for n, first, last in ((0, 0, 0), (257, 1, 1)):
        refused(lib, select(cache(), queries(), n, first, last, AT, None), "n must be in [1, 256]")
    for first, last in ((-1, 1), (3, 2), (1, -1)):
        refused(lib, select(cache(), queries(), 4, first, last, AT, None), "together at most n")
    refused(lib, select(cache(codes=0), queries(), 4, 1, 1, AT, None), "codes and scales")
    refused(lib, select(cache(codes=AT + 4), queries(), 4, 1, 1, AT, None), "16-byte aligned")
    refused(lib, select(cache(), queries(), 4, 1, 1, None, None), "pages must not be NULL")
    store = lib.mlxvs_paged_store_device
    args = [AT, AT, 1, 3, 256, 128, 256, 128, AT, None]
    for i, bad, text in ((0, None, "must not be NULL"), (1, AT + 4, "aligned"), (2, 2, "bfloat16"),
                         (3, -1, "tokens"), (4, 255, "strides"), (8, None, "must not be NULL")):
        refused(lib, store(cache(), *args[:i], bad, *args[i + 1:]), text)
    refused(lib, store(cache(scales=0), *args), "codes and scales")
    tables = lib.mlxvs_paged_tables_device
    args = [AT, AT, 2, 16, AT, 5, AT, 4, 3, AT, AT, AT, AT, AT, None]
    for i, bad, text in ((0, None, "past and fresh"), (2, -1, "requests"), (3, 0, "page_size"),
                         (4, None, "free_pages"), (6, None, "table"), (7, -1, "table"),
                         (8, -1, "num_tokens"), (9, None, "outputs"), (12, None, "outputs")):
        refused(lib, tables(*args[:i], bad, *args[i + 1:]), text)


def test_structs_match_the_header():
    """The packed structs have the C layout (no padding anywhere)."""

    class Cache(ctypes.Structure):
        _fields_ = [("p", ctypes.c_void_p * 2), ("s", ctypes.c_int64 * 7),
                    ("c", ctypes.c_void_p * 2), ("i", ctypes.c_int32 * 4),
                    ("f", ctypes.c_float * 2)]

    class Queries(ctypes.Structure):
        _fields_ = [("q", ctypes.c_void_p), ("s", ctypes.c_int64 * 3), ("t", ctypes.c_void_p),
                    ("r", ctypes.c_int64 * 2), ("m", ctypes.c_void_p * 2),
                    ("i", ctypes.c_int32 * 2)]

    assert ctypes.sizeof(Cache) == paged._CACHE.size
    assert ctypes.sizeof(Queries) == paged._QUERIES.size


def test_python_refusals():
    torch = pytest.importorskip("torch")
    x = torch.zeros(2, 4, 64, dtype=torch.float16)
    with pytest.raises(ValueError, match="CUDA tensor"):
        mv.paged_attention(x, x, x, x, x)
    with pytest.raises(ValueError, match="CUDA tensor"):
        mv.paged_select(x, x, x, x, x, 16, 4)
    with pytest.raises(ValueError, match="CUDA tensor"):
        mv.paged_store(x, x, x, x, x)
    with pytest.raises(ValueError, match="CUDA tensor"):
        mv.paged_tables(x, x, x, x, 16, 4)


def test_oracle_known_answers():
    """Cases small enough to do by hand."""
    table, starts, rows, lengths, slots, used = O.paged_tables(
        [3, 0], [2, 1], [[7, -1], [-1, -1]], [5, 6, 9], 4, 4)
    assert table.tolist() == [[7, 5], [6, -1]] and starts.tolist() == [0, 2, 3]
    assert rows.tolist() == [0, 0, 1, -1] and lengths.tolist() == [4, 5, 1, 0]
    assert slots.tolist() == [31, 20, 24, -1] and used.tolist() == [2, 0]
    codes, scale = O.page_bounds(np.array([[1.0, -0.75], [0.505, 0.25]]))
    assert codes.tolist() == [[32, -48], [64, 16]] and scale == 1 / 64
    assert O.query_codes(np.array([[1.0, -0.5], [0.25, 0.5]])).tolist() == [[0, -16], [40, 16]]
    keys = np.zeros((2, 2, 1, 2))
    values = np.arange(8.0).reshape(2, 2, 1, 2)
    out, lse, _ = O.paged_attention(np.ones((2, 1, 2)), keys, values, np.array([[1, 0], [0, 1]]), [3, 0],
                                    [0, 1], 1.0)
    assert np.allclose(out[0, 0], [10 / 3, 13 / 3]) and np.allclose(lse[0, 0], np.log(3))
    assert (out[1] == 0).all() and lse[1, 0] == -np.inf


def test_bounds_hold():
    """Codes bound the keys but for the last half step below 128."""
    rng = np.random.default_rng(0)
    for _ in range(50):
        rows = rng.standard_normal((9, 32)) * 2.0 ** rng.integers(-20, 20)
        codes, scale = O.page_bounds(rows)
        top = np.abs(rows).max()
        assert 63 <= np.abs(codes).max() <= 127
        assert (codes[0] * scale <= rows.min(0) + top / 127).all()
        assert (codes[1] * scale >= rows.max(0) - top / 127).all()
        inner = np.abs(codes[1]) < 127
        assert (codes[1] * scale >= rows.max(0))[inner].all()
