"""Refusals of the drafted-token and 8-bit cache entry points, all before any GPU work."""
import ctypes as C

import pytest
import torch

from pluto_b200 import PlutoStatusError
from pluto_b200.layers import KeyValueCache, gqa_decode, kv_layout

ONE = 16   # a non-null "device pointer" that a refused call never reads


def code(engine, fn, *args):
    try:
        engine.check(fn(*args))
    except PlutoStatusError as error:
        return error.code, error.message
    return "Ok", ""


def cache(engine, dtype=1, **other):
    s = engine.KvCacheStruct()
    s.k_base = s.v_base = ONE
    s.page_size, s.page_stride, s.token_stride, s.dtype, s.num_pages = 16, 16 * 2 * 64, 2 * 64, dtype, 4
    for name, value in other.items():
        setattr(s, name, value)
    return s


def scales(engine, **other):
    s = engine.KvScalesStruct()
    s.k = s.v = ONE
    s.page_stride, s.token_stride = 32, 2
    for name, value in other.items():
        setattr(s, name, value)
    return s


def tree(engine, c, s=None, **other):
    a = dict(stream=None, q=ONE, q_dtype=1, gate=None, gate_dtype=0, gt=0, gh=0, cache=C.cast(C.pointer(c), C.c_void_p) if c else None,
             scales=C.cast(C.pointer(s), C.c_void_p) if s else None, prefix=ONE, max_prefix=100, parents=None, counts=None, out=ONE,
             out_dtype=1, lse=None, ws=ONE, ws_bytes=1 << 40, batch=1, nodes=3, hq=4, hkv=2, dim=64, rnd=1)
    a.update(other)
    return code(engine, engine.lib().pluto_gqa_tree_decode, *a.values())


BAD_CACHES = [dict(k_base=None), dict(v_base=None), dict(dtype=3), dict(page_size=0), dict(token_stride=127), dict(page_stride=1),
              dict(block_table=ONE, max_blocks=0), dict(block_table=ONE, max_blocks=1, num_pages=0), dict(k_base=17)]


def test_tree_decode_refuses(engine):
    for bad in BAD_CACHES:
        assert tree(engine, cache(engine, **bad))[0] == "InvalidArgument", bad
    assert tree(engine, None)[0] == "InvalidArgument"
    assert tree(engine, cache(engine, k_bases=ONE, v_bases=ONE))[0] == "Unimplemented"
    for bad in (dict(batch=0), dict(batch=65536), dict(nodes=0), dict(nodes=129), dict(hq=0), dict(hkv=0), dict(hq=5), dict(dim=0),
                dict(dim=257), dict(max_prefix=-1), dict(max_prefix=2 ** 31 - 1), dict(q_dtype=2), dict(out_dtype=7),
                dict(gate=ONE, gate_dtype=5), dict(q=None), dict(prefix=None), dict(out=None), dict(ws=None), dict(ws_bytes=0), dict(ws=8)):
        assert tree(engine, cache(engine), **bad)[0] == "InvalidArgument", bad
    # an 8-bit cache and its scales belong together
    assert tree(engine, cache(engine, dtype=2))[0] == "InvalidArgument"
    assert tree(engine, cache(engine), scales(engine))[0] == "InvalidArgument"
    for bad in (dict(k=None), dict(v=None), dict(token_stride=1), dict(page_stride=1)):
        assert tree(engine, cache(engine, dtype=2), scales(engine, **bad))[0] == "InvalidArgument", bad


def test_workspace_query(engine):
    size = engine.lib().pluto_gqa_tree_decode_workspace_bytes
    assert size(1, 1, 24, 4, 256) > 0 and size(16, 128, 40, 8, 128) > 0
    for bad in ((0, 1, 4, 2, 64), (1, 0, 4, 2, 64), (1, 129, 4, 2, 64), (1, 1, 5, 2, 64), (1, 1, 4, 2, 257)):
        assert size(*bad) == 0


@pytest.mark.parametrize("name", ["pluto_kv8_append", "pluto_kv8_read"])
def test_kv8_refuses(engine, name):
    def call(c=None, s=None, **other):
        c, s = c or cache(engine, dtype=2), s or scales(engine)
        a = dict(stream=None, k=ONE, v=ONE, dtype=1, b=0, t=128, h=64, cache=C.cast(C.pointer(c), C.c_void_p),
                 scales=C.cast(C.pointer(s), C.c_void_p), positions=None, counts=None, batch=1, tokens=3, heads=2, dim=64)
        a.update(other)
        return code(engine, getattr(engine.lib(), name), *a.values())
    for bad in BAD_CACHES[:2] + BAD_CACHES[3:8]:
        assert call(cache(engine, **{**dict(dtype=2), **bad}))[0] == "InvalidArgument", bad
    assert call(cache(engine, dtype=1))[0] == "InvalidArgument"
    for bad in (dict(k=None), dict(v=None), dict(k=17), dict(dtype=2), dict(batch=0), dict(tokens=0), dict(heads=0), dict(dim=0), dict(dim=257),
                dict(h=63), dict(cache=None), dict(scales=None), dict(batch=1 << 20, tokens=1 << 20)):
        assert call(**bad)[0] == "InvalidArgument", bad


def test_keep_prepare_and_verify_refuse(engine):
    L = engine.lib()
    c = cache(engine)
    p = C.cast(C.pointer(c), C.c_void_p)
    good = [None, p, None, ONE, ONE, ONE, 1, 4, 2, 64]
    for at, value in ((1, None), (3, None), (4, None), (5, None), (6, 0), (7, 0), (7, 129), (8, 0), (9, 300)):
        bad = list(good)
        bad[at] = value
        assert code(engine, L.pluto_kv_keep, *bad)[0] == "InvalidArgument", at
    good = [None, ONE, ONE, ONE, 1, 256, 64, ONE, ONE, ONE, None, None, ONE, 1, p, None, 1, 4, 4, 2, 64, 32, 1e-6, 1e4, 1]
    for at, value in ((1, None), (2, None), (3, None), (4, 2), (7, None), (8, None), (12, None), (13, 3), (14, None), (16, 0), (17, 0),
                      (18, 5), (20, 300), (21, 0), (21, 33), (21, 66), (22, 0.0), (22, float("nan")), (23, -1.0)):
        bad = list(good)
        bad[at] = value
        assert code(engine, L.pluto_draft_prepare, *bad)[0] == "InvalidArgument", at
    bad = list(good)
    bad[10], bad[17] = ONE, 129   # a tree of more nodes than an ancestor set holds
    assert code(engine, L.pluto_draft_prepare, *bad)[0] == "InvalidArgument"
    good = [None, ONE, ONE, 0, ONE, ONE, ONE, None, None, ONE, ONE, ONE, 1, 4, 100]
    for at, value in ((1, None), (3, 2), (4, None), (5, None), (6, None), (9, None), (10, None), (11, None), (12, 0), (12, 65536), (13, 0),
                      (13, 129), (14, 0), (14, 1048577)):
        bad = list(good)
        bad[at] = value
        assert code(engine, L.pluto_verify_drafts, *bad)[0] == "InvalidArgument", at
    bad = list(good)
    bad[7] = ONE
    assert code(engine, L.pluto_verify_drafts, *bad)[0] == "Unimplemented"   # a tree with draft probabilities


def test_python_layer_refuses_on_the_cpu():
    """8-bit pools never reach the functions of the other storage types."""
    codes = torch.zeros(1, 8, 2, 64, dtype=torch.float8_e4m3fn)
    with pytest.raises(PlutoStatusError, match="8-bit"):
        kv_layout(codes, codes, None, 8, 1024, 128)
    q = torch.zeros(1, 4, 64, dtype=torch.bfloat16)
    with pytest.raises(PlutoStatusError, match="8-bit"):
        gqa_decode(q, codes, codes, torch.ones(1, dtype=torch.int32), 8)
    with pytest.raises(PlutoStatusError):
        KeyValueCache.Create(8, 2, 64, dtype=torch.float16, device="cpu")
