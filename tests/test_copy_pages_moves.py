"""Pages that move with a block table: a page moves to one place, so a source named twice is refused, however many pairs there are."""
import ctypes

import pytest
import torch

from omni_npu_amd import _lib


@pytest.mark.parametrize("pairs", [2, 48, 49, 60, 201])
def test_a_source_named_twice_is_refused_with_a_table(pairs):
    lib = _lib.load()
    raw = ctypes.create_string_buffer(1 << 12)
    p = ctypes.addressof(raw) // 16 * 16 + 16
    I = lambda x: (ctypes.c_int32 * len(x))(*x)

    def rc(src, table):
        c = (ctypes.c_int64 * 4)(p, 64, 16, 16)
        dst = [2000 + i for i in range(len(src))]
        return lib.mlahip_copy_pages(c, 1, I(src), I(dst), None, len(src), 4000, 4, table, 4, 2, 4, None), lib.mlahip_last_error_string().decode()

    src = list(range(pairs - 1)) + [0]                         # (at both ends)
    code, said = rc(src, p)
    assert code == -3 and "page 0" in said and "moves" in said
    src[-2:] = [pairs, pairs]                                  # (side by side)
    assert pairs == 2 or rc(src, p)[0] == -3
    del raw


@pytest.mark.gpu
@pytest.mark.parametrize("pairs", [2, 60, 201])
def test_copies_of_one_page_to_many_places(dev, pairs):
    """Right without a table; with one refused before anything is copied, by lists and by tensors."""
    from omni_npu_amd import kernels as K
    cache = torch.arange(1 + 2 * pairs, device=dev, dtype=torch.int32)[:, None, None].expand(-1, 4, 16).contiguous()
    src, dst = [0] * pairs, list(range(1, 1 + 2 * pairs, 2))
    table = torch.zeros(3, 5, dtype=torch.int32, device=dev)
    before = cache.clone()
    for s, d in ((src, dst), (torch.tensor(src), tuple(dst))):
        with pytest.raises(ValueError, match="two places"):
            K.copy_pages(cache, s, d, block_table=table)
    assert torch.equal(cache, before) and not table.any()
    K.copy_pages(cache, src, dst)
    before[1::2] = 0
    assert torch.equal(cache, before)
