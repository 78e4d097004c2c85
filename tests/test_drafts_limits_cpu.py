"""Limits of the drafted-token entry points that are refused before any GPU work: addresses off their elements, lengths whose
slots would not fit 32 bits."""
import ctypes as C

import pytest

from pluto_b200 import PlutoStatusError

ONE, ODD = 16, 18   # "device pointers" that a refused call never reads


def refused(engine, fn, args, at, value):
    args = list(args)
    args[at] = value
    with pytest.raises(PlutoStatusError) as error:
        engine.check(fn(*args))
    return error.value.code == "InvalidArgument"


def cache_of(engine, dtype):
    s = engine.KvCacheStruct()
    s.k_base = s.v_base = ONE
    s.page_size, s.page_stride, s.token_stride, s.dtype, s.num_pages = 16, 16 * 2 * 64, 2 * 64, dtype, 4
    return s


def test_addresses_off_their_elements(engine):
    L, c = engine.lib(), cache_of(engine, 0)
    p = C.cast(C.pointer(c), C.c_void_p)
    keep = [None, p, None, ONE, ONE, ONE, 1, 4, 2, 64]
    assert all(refused(engine, L.pluto_kv_keep, keep, at, ODD) for at in (3, 4, 5))
    prepare = [None, ONE, ONE, ONE, 0, 256, 64, ONE, ONE, ONE, ONE, ONE, ONE, 0, p, None, 1, 4, 4, 2, 64, 32, 1e-6, 1e4, 1]
    assert all(refused(engine, L.pluto_draft_prepare, prepare, at, ODD) for at in (1, 2, 3, 7, 8, 9, 10, 11, 12))
    tree = [None, ONE, 0, ONE, 0, 256, 64, p, None, ONE, 100, ONE, ONE, ONE, 0, ONE, ONE, 1 << 40, 1, 3, 4, 2, 64, 1]
    assert all(refused(engine, L.pluto_gqa_tree_decode, tree, at, ODD) for at in (1, 3, 9, 11, 12, 13, 15, 16))
    verify = [None, ONE, ONE, 0, ONE, ONE, ONE, None, ONE, ONE, ONE, ONE, 1, 4, 100]
    assert all(refused(engine, L.pluto_verify_drafts, verify, at, ODD) for at in (1, 2, 4, 5, 6, 8, 9, 10, 11))
    c.block_table, c.max_blocks = ODD, 1
    assert refused(engine, L.pluto_kv_keep, keep, 1, p)


def test_positions_off_their_elements(engine):
    L, c, s = engine.lib(), cache_of(engine, 2), engine.KvScalesStruct()
    s.k = s.v = ONE
    s.page_stride, s.token_stride = 32, 2
    args = [None, ONE, ONE, 0, 0, 128, 64, C.cast(C.pointer(c), C.c_void_p), C.cast(C.pointer(s), C.c_void_p), ONE, ONE, 1, 3, 2, 64]
    for fn in (L.pluto_kv8_append, L.pluto_kv8_read):
        assert all(refused(engine, fn, args, at, ODD) for at in (1, 2, 9, 10))


def test_prefixes_whose_tiles_pass_32_bits(engine):
    L, c = engine.lib(), cache_of(engine, 0)
    tree = [None, ONE, 0, None, 0, 0, 0, C.cast(C.pointer(c), C.c_void_p), None, ONE, 100, None, None, ONE, 0, None, ONE, 1 << 40, 1, 3, 4, 2, 64, 1]
    assert all(refused(engine, L.pluto_gqa_tree_decode, tree, 10, n) for n in (2 ** 31 - 1, 2 ** 31 - 1024, -1))
