"""Scratch memory of the attention over ordinary heads, which is kept until the process ends: refused calls take none."""
import pytest
import torch

from tests.test_gqa_decode_gpu import call, check, make

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def side(dev):
    """A stream without scratch memory; one for all, as torch hands out 32 in turn and other tests count on new ones too."""
    return torch.cuda.Stream(dev)


def _args(dev, b=2, hq=8, hk=2, d=128, page=32):
    z = lambda *s: torch.zeros(*s, dtype=torch.bfloat16, device=dev)
    i = lambda *s: torch.ones(*s, dtype=torch.int32, device=dev)
    return [z(b, hq, d), z(4, page, hk, d), z(4, page, hk, d), i(b, 100), i(b), 0.1, z(b, hq, d)]


@pytest.mark.parametrize("form", [dict(d=96), dict(d=16), dict(b=65536), dict(page=24), dict(page=8)], ids=str)
@pytest.mark.parametrize("chunks", [None, 8])
def test_what_the_shapes_refuse(dev, side, form, chunks):
    _refused(dev, side, _args(dev, **form), num_chunks=chunks)


@pytest.mark.parametrize("kw", [dict(num_chunks=1 << 24), dict(num_chunks=(1 << 24) - 1), dict(num_chunks=8, heads_per_group=3),
                                dict(num_chunks=8, heads_per_group=8), dict(num_chunks=8, rows_per_group=48), dict(num_chunks=8, rows_per_group=0)], ids=str)
def test_what_the_launch_refuses(dev, side, kw):
    _refused(dev, side, _args(dev), **kw)


def test_what_addresses_and_strides_refuse(dev, side):
    args = _args(dev)
    odd = torch.zeros(2 * 8 * 128 + 1, dtype=torch.bfloat16, device=dev)[1:].view(2, 8, 128)
    _refused(dev, side, [odd] + args[1:], num_chunks=8)
    _refused(dev, side, args[:3] + [args[3][:1].expand(2, 100)] + args[4:], num_chunks=8)       # (rows that share their memory)


def _refused(dev, side, args, **kw):
    from omni_npu_amd import kernels as K
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        before = K.retained_workspace_bytes()
        with pytest.raises(K._lib.MlaHipError):
            K.gqa_decode(*args, **kw)
        assert K.retained_workspace_bytes() == before
    torch.cuda.synchronize()


def test_scratch_is_taken_as_it_is_needed_and_kept(dev, side):
    """By the native side and by the general one (which another number of pieces than a 16-bit one goes to): what there is serves smaller calls."""
    from omni_npu_amd import kernels as K
    c = make(dev, [300, 700, 64], hq=8, hk=2, seed=1)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        held = [K.retained_workspace_bytes()]
        for chunks in (9, 5, (1 << 16) + 5, 40, 9):
            check(c, *call(dev, c, 1, num_chunks=chunks))
            held.append(K.retained_workspace_bytes())
    need = lambda n: K._lib.load().mlahip_gqa_decode_workspace_bytes(3, 1, 8, 128, n)
    assert [b - a for a, b in zip(held, held[1:])] == [need(9), 0, need((1 << 16) + 5), 0, 0]


@pytest.mark.parametrize("lens,counts", [([500], [200]), ([500, 301, 0, 77], [150, 301, 0, 1]), ([90] * 70, [3] * 70)], ids=["one", "some", "many"])
def test_one_piece_has_no_partial_results(dev, lens, counts):
    """However many tokens and heads: its scratch memory goes by the requests, and nothing behind it is touched."""
    from omni_npu_amd import kernels as K
    need = K._lib.load().mlahip_gqa_decode_workspace_bytes
    assert need(len(lens), 1 << 14, 64, 128, 1) == need(len(lens), 1, 1, 64, 1) <= 8 * len(lens) + 256
    c = make(dev, lens, q_lens=counts, hq=6, hk=2, d=64, page=16, seed=4)
    n = need(len(lens), max(counts), 6, 64, 1)
    memory = torch.full((n + (1 << 20),), 77, dtype=torch.uint8, device=dev)
    for window in (None, 60):
        check(c, *call(dev, c, max(counts), varlen=True, num_chunks=1, window=window, workspace=memory[:n]), window=window)
    assert (memory[n:] == 77).all()
