"""CPU: what the entry points for layers with ordinary key and value heads refuse, before anything is launched, and the rule that cuts a
step into pieces."""
import ctypes

import pytest
import torch

from omni_npu_amd import _host, _lib
from omni_npu_amd import kernels as K


def _buffer(n=1 << 12):
    raw = ctypes.create_string_buffer(n + 16)
    return raw, ctypes.addressof(raw) // 16 * 16 + 16


def test_gqa_decode_codes():
    lib = _lib.load()
    raw, p = _buffer()
    #        q, strides, T, k cache, strides, v cache, strides, pages, page, table, stride, blocks, lens, qsl, B, s, Hq, Hk, D, types, scales
    base = [p, 1024, 128, 2, p, 32768, 256, 128, p, 32768, 256, 128, 4, 128, p, 4, 4, p, None, 2, 1, 8, 2, 128, 0, 0, None, None, 0.1, 0, p, 1024,
            128, None, p, 1 << 20, 4, 2, 16, None]

    def rc(**swap):
        args = list(base)
        for i, x in swap.items():
            args[int(i[1:])] = x
        return lib.mlahip_gqa_decode(*args), lib.mlahip_last_error_string().decode()

    assert rc(_0=None)[0] == -1 and rc(_30=None)[0] == -1
    assert rc(_23=96)[0] == -3 and rc(_24=1)[0] == -3 and rc(_25=2)[0] == -3
    assert rc(_13=24)[0] == -2 and rc(_13=8)[0] == -2 and rc(_16=0)[0] == -2 and rc(_15=3)[0] == -2
    assert rc(_21=7)[0] == -2 and rc(_20=0)[0] == -2 and rc(_29=-1)[0] == -2 and rc(_36=-1)[0] == -2
    assert rc(_16=1 << 24, _15=1 << 24)[0] == -2               # more than 2^31 tokens of room
    assert rc(_1=1028)[0] == -2 and rc(_6=257)[0] == -2 and rc(_0=p + 2)[0] == -2 and rc(_31=1022)[0] == -2
    code, said = rc(_35=lib.mlahip_gqa_decode_workspace_bytes(2, 1, 8, 128, 4) - 1)
    assert code == -4 and "workspace" in said
    assert rc(_34=None)[0] == -4
    assert all(rc(_37=n)[0] == -2 for n in (-1, 0, 3, 4, 16)) and all(rc(_38=n)[0] == -2 for n in (0, 8, 48, 128))
    assert rc(_19=0)[0] == 0 and rc(_3=0)[0] == 0             # nothing to do
    assert lib.mlahip_gqa_decode_workspace_bytes(2, 1, 8, 128, 0) == 0
    del raw


def test_prologue_codes():
    lib = _lib.load()
    raw, p = _buffer()
    #        q, k, v with strides, T, Hq, Hk, D, type, gammas, eps, cos, sin, stride, rows, type, R, pairs, positions, slots, caches, ...
    base = [p, 512, 128, p, 512, 128, p, 512, 128, 2, 2, 1, 128, 0, p, p, 1e-6, p, p, 64, 100, 1, 128, 0, p, p, p, 16384, 128, 128, p, 16384, 128,
            128, 128, 2, 0, None, None, p, 256, 128, None, 0, 0, None]

    def rc(**swap):
        args = list(base)
        for i, x in swap.items():
            args[int(i[1:])] = x
        return lib.mlahip_qk_norm_rope_cache(*args)

    for null in (0, 3, 6, 17, 18, 24, 25, 26, 30, 39):
        assert rc(**{f"_{null}": None}) == -1, null
    assert rc(_13=1) == -3 and rc(_21=2) == -3 and rc(_36=2) == -3
    assert rc(_12=120) == -2 and rc(_12=272) == -2 and rc(_22=136) == -2 and rc(_22=144) == -2 and rc(_22=0) == -2 and rc(_20=0) == -2
    assert rc(_35=0) == -2 and rc(_34=0) == -2 and rc(_9=-1) == -2
    assert rc(_1=513) == -2 and rc(_28=130) == -2 and rc(_19=66) == -2 and rc(_0=p + 2) == -2
    assert rc(_9=0) == 0
    del raw


def test_copy_pages_codes():
    lib = _lib.load()
    raw, p = _buffer()
    I = lambda *x: (ctypes.c_int32 * len(x))(*x)

    def rc(src, dst, rows=None, pages=8, page=4, cache=(None, 64, 16, 16), table=None, n_caches=1):
        c = (ctypes.c_int64 * 4)(p if cache[0] is None else cache[0], *cache[1:])
        return lib.mlahip_copy_pages(c, n_caches, I(*src), I(*dst), None if rows is None else I(*rows), len(src), pages, page, table, 4, 2, 4, None)

    assert rc([], []) == 0
    assert rc([0], [8]) == -2 and rc([-1], [1]) == -2 and rc([0], [1], [5]) == -2 and rc([0], [1], [-1]) == -2
    assert rc([0, 1], [2, 2]) == -3 and rc([0, 1], [1, 2]) == -3 and rc([3], [3]) == -3
    many = list(range(60))
    assert rc(many, [200 + i for i in many[:-1]] + [200], pages=400) == -3            # (the marks' path: 200 twice)
    assert rc(many, [200 + i for i in many[:-1]] + [59], pages=400) == -3
    assert rc([0], [1], cache=(0, 64, 16, 16)) == -1 and rc([0], [1], n_caches=0) == -2
    assert rc([0], [1], cache=(None, 64, 8, 16)) == -2 and rc([0], [1], cache=(None, 64, 16, 0)) == -2 and rc([0], [1], cache=(None, 8, 16, 16)) == -2
    assert rc([0], [1], [2], table=p) == -3
    del raw


def test_host_tensors_are_refused():
    z = lambda *s, **k: torch.zeros(*s, **k)
    bf = dict(dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="no CPU path"):
        K.gqa_decode(z(1, 4, 64, **bf), z(2, 16, 2, 64, **bf), z(2, 16, 2, 64, **bf), z(1, 2, dtype=torch.int32), z(1, dtype=torch.int32), 1.0,
                     z(1, 4, 64, **bf))
    with pytest.raises(ValueError, match="no CPU path"):
        K.qk_norm_rope_cache(z(1, 4, 64, **bf), z(1, 2, 64, **bf), z(1, 2, 64, **bf), z(8, 32), z(8, 32), z(1, dtype=torch.int64))
    with pytest.raises(ValueError, match="no CPU path"):
        K.copy_pages(z(4, 2, 8), [0], [1])


def test_the_native_host_side_cuts_steps_as_the_wrapper_does():
    host = _host.load()
    for batch in (1, 3, 64, 300):
        for q_len in (1, 2, 17):
            for hq, hk in ((4, 1), (32, 8), (20, 4), (15, 5), (64, 64)):
                for d in (64, 128, 256):
                    for es in (1, 2):
                        for longest in (1, 64, 300, 1280, 1281, 131072):
                            chunks, heads, rows = K.gqa_plan(batch, q_len, hq, hk, d, es, longest)
                            assert (chunks, heads, rows) == tuple(host.gqa_plan(batch, q_len, hq, hk, d, es, longest))
                            assert chunks >= 0 and hk % heads == 0 and heads <= (4 if d == 256 or rows == 64 or rows == 32 and d == 128 and es == 2 else 8)
                            assert rows in ((16, 32) if d == 256 else (16, 32, 64))


def test_copy_pages_takes_what_the_native_side_does_not():
    """Tuples, tensors of numbers, single tensors and mistakes: the general path takes or names them (no GPU here: it says so)."""
    z = torch.zeros(4, 2, 8)
    for caches, src, dst in ((z, [0], [1]), ((z, z), (0,), (1,)), ([z], torch.tensor([0]), torch.tensor([1])), (iter([z]), [0], [1])):
        with pytest.raises(ValueError, match="no CPU path"):
            K.copy_pages(caches, src, dst)
    with pytest.raises(TypeError, match="whole numbers"):
        K.copy_pages([z], [0.0], [1])
    with pytest.raises(TypeError, match="whole numbers"):
        K.copy_pages([z], [True], [1])
    with pytest.raises(ValueError, match="sources"):
        K.copy_pages([], [0], [1])
