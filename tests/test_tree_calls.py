"""CPU: what the entry points of a step over drafted trees refuse, before anything is launched."""
import ctypes

import pytest
import torch

from omni_npu_amd import _lib
from omni_npu_amd import kernels as K


def _buffer(n=1 << 16):
    raw = ctypes.create_string_buffer(n + 16)
    return raw, ctypes.addressof(raw) // 16 * 16 + 16


def _caller(fn, base):
    def rc(**swap):
        args = list(base)
        for i, x in swap.items():
            args[int(i[1:])] = x
        return fn(*args)
    return rc


def test_tree_decode_codes():
    lib = _lib.load()
    raw, p = _buffer()
    #        q, strides, T, k cache, strides, v cache, strides, pages, page, table, stride, blocks, lens, qsl, bits, stride, words, B, s, Hq, ...
    rc = _caller(lib.mlahip_gqa_tree_decode, [p, 1024, 128, 10, p, 32768, 256, 128, p, 32768, 256, 128, 4, 128, p, 4, 4, p, None, p, 1, 1, 2, 5, 8, 2,
                                              128, 0, 0, None, None, 0.1, 0, p, 1024, 128, None, p, 1 << 20, 4, 2, 16, None])
    assert rc(_19=None) == -1 and rc(_0=None) == -1 and rc(_17=None) == -1
    assert rc(_21=0) == -2 and rc(_21=9) == -2 and rc(_20=0) == -2 and rc(_19=p + 4) == -2
    assert rc(_23=65) == -2 and rc(_23=0) == -2
    assert rc(_26=96) == -3 and rc(_27=1) == -3
    assert rc(_13=24) == -2 and rc(_25=3) == -2 and rc(_32=-1) == -2
    assert rc(_37=None) == -4 and rc(_38=100) == -4
    assert rc(_40=3) == -2 and rc(_41=48) == -2 and rc(_41=256) == -2
    assert rc(_41=128) == -2                                   # two key heads to a workgroup of 128 rows
    assert rc(_41=64, _40=1, _26=256) == -2                    # heads of 256
    assert rc(_22=0) == 0 and rc(_3=0) == 0                    # nothing to do
    assert "gqa_tree_decode" in (rc(_41=48), lib.mlahip_last_error_string().decode())[1]
    del raw


def test_tree_plan():
    """Both sides choose alike, what the entry point takes; gqa_decode's choices stay its own."""
    from omni_npu_amd import _host
    host, seen = _host.load(), set()
    for batch in (1, 3, 32, 500):
        for q_len in (1, 5, 26, 60, 512):
            for hq, hk in ((8, 8), (32, 8), (64, 4), (6, 3), (1, 1)):
                for d in (64, 128, 256):
                    for es in (1, 2):
                        for longest in (1, 64, 1280, 2049, 16384, 1 << 30):
                            chunks, heads, rows = K.gqa_tree_plan(batch, q_len, hq, hk, d, es, longest)
                            assert (chunks, heads, rows) == tuple(host.gqa_tree_plan(batch, q_len, hq, hk, d, es, longest))
                            seen.add(rows)
                            assert 0 <= chunks <= 1 << 16 and hk % heads == 0
                            if rows == 128:
                                assert heads == 1 and q_len * hq // hk > 32
                            else:
                                assert (chunks, heads, rows) == K.gqa_plan(batch, q_len, hq, hk, d, es, longest)
    assert seen == {16, 32, 64, 128}
    for plan in (K.gqa_tree_plan, host.gqa_tree_plan):
        with pytest.raises(ValueError, match="gqa_plan"):
            plan(0, 1, 8, 2, 128, 2, 100)


def test_step_tables_codes():
    lib = _lib.load()
    raw, p = _buffer()
    at = lambda i: p + 1024 * i
    #      context, qsl, B, s, table, stride, blocks, page, lens, positions, slots, T, parents, bits, stride, words, held, free, num, capacity, stream
    rc = _caller(lib.mlahip_step_tables, [at(0), None, 4, 3, at(1), 8, 8, 16, at(2), at(3), at(4), 12, at(5), at(6), 1, 1, at(7), at(8), at(9), 50, None])
    assert all(rc(**{f"_{i}": None}) == -1 for i in (0, 4, 8, 9, 10, 12, 13, 16, 17, 18))
    assert rc(_2=-1) == -2 and rc(_3=0) == -2 and rc(_7=0) == -2 and rc(_6=0) == -2 and rc(_5=7) == -2 and rc(_11=-1) == -2 and rc(_2=1 << 24) == -2
    assert rc(_11=11) == -2 and rc(_3=4) == -2                 # fewer places than tokens
    assert rc(_15=0) == -2 and rc(_14=0) == -2 and rc(_3=65, _2=1, _11=65) == -2 and rc(_19=-1) == -2
    assert rc(_6=1 << 30, _5=1 << 30) == -2
    assert rc(_8=at(0)) == -3 and rc(_9=at(4) + 88) == -3 and rc(_16=at(0) + 12) == -3 and rc(_17=at(1)) == -3 and rc(_13=at(5)) == -3 and rc(_18=at(7)) == -3
    assert rc(_0=at(0) + 2) == -2 and rc(_9=at(3) + 4) == -2
    assert rc(_2=0, _11=0) == 0                                # nothing to do
    del raw


def test_keep_rows_codes():
    lib = _lib.load()
    raw, p = _buffer()
    at = lambda i: p + 1024 * i

    def rc(cache=(None, 64, 16, 16), **swap):
        c = (ctypes.c_int64 * 4)(at(0) if cache[0] is None else cache[0], *cache[1:])
        #                                 caches, number, pages, page, table, stride, blocks, context, lens, B, accepted, stride, most, num, kept, stream
        return _caller(lib.mlahip_keep_rows, [c, 1, 8, 4, at(1), 6, 6, at(2), at(3), 3, at(4), 5, 5, at(5), at(6), None])(**swap)

    assert all(rc(**{f"_{i}": None}) == -1 for i in (0, 4, 7, 8, 10, 13, 14)) and rc(cache=(0, 64, 16, 16)) == -1
    assert rc(_1=0) == -2 and rc(_2=0) == -2 and rc(_3=0) == -2 and rc(_5=5) == -2 and rc(_6=0) == -2 and rc(_9=-1) == -2 and rc(_11=4) == -2 and rc(_12=-1) == -2
    assert rc(cache=(None, 64, 8, 16)) == -2 and rc(cache=(None, 64, 16, 0)) == -2 and rc(cache=(None, 8, 16, 16)) == -2 and rc(cache=(None, 48, 16, 16)) == -2
    assert rc(cache=(None, 1 << 24, 1 << 22, 1 << 22)) == -2   # rows of 4 MB
    assert rc(_14=at(2)) == -3 and rc(_14=at(3) + 8) == -3 and rc(_14=at(4) + 40) == -3 and rc(_14=at(5)) == -3 and rc(_14=at(1) + 64) == -3
    assert rc(_14=at(6) + 2) == -2
    two = (ctypes.c_int64 * 8)(at(0), 64, 16, 16, at(0), 64, 16, 8)
    assert rc(_0=two, _1=2) == -3                              # the same cache twice
    two[4] += 512
    assert rc(_0=two, _1=2, _9=0) == 0
    assert rc(_9=0) == 0
    del raw


def test_host_tensors_are_refused():
    z = lambda *s: torch.zeros(*s, dtype=torch.bfloat16)
    i32 = lambda *s: torch.zeros(*s, dtype=torch.int32)
    i64 = lambda *s: torch.zeros(*s, dtype=torch.int64)
    with pytest.raises(ValueError, match="no CPU path"):
        K.gqa_tree_decode(z(1, 4, 64), z(2, 16, 2, 64), z(2, 16, 2, 64), i32(1, 2), i32(1), i64(1, 1), 1.0, z(1, 4, 64))
    with pytest.raises(ValueError, match="no CPU path"):
        K.step_tables(i32(1), i32(1, 2), 16, i32(1), i64(1), i64(1))
    with pytest.raises(ValueError, match="no CPU path"):
        K.keep_rows([torch.zeros(4, 2, 8)], i32(1, 2), i32(1), i32(1), i32(1, 2), i32(1), i32(1))
    with pytest.raises(ValueError, match="no caches"):
        K.keep_rows([], i32(1, 2), i32(1), i32(1), i32(1, 2), i32(1), i32(1))
