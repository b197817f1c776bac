"""Caches whose pages lie in each other: a copy of one page would write rows of another, in no order."""
import ctypes

import pytest
import torch

from omni_npu_amd import _lib


@pytest.mark.parametrize("page_stride,row_stride,pages,page,fine", [
    (64, 16, 8, 4, True), (48, 16, 8, 4, False), (16, 16, 8, 4, False), (60, 16, 8, 4, False), (1 << 40, 16, 8, 4, True),
    (16, 128, 8, 4, True), (16, 112, 8, 4, False), (16, 1 << 31, 8, 4, True), (32, 256, 8, 4, True), (16, 16, 1, 4, True), (16, 16, 8, 1, True)])
def test_pages_that_share_rows_are_refused(page_stride, row_stride, pages, page, fine):
    lib = _lib.load()
    raw = ctypes.create_string_buffer(1 << 12)
    p = ctypes.addressof(raw) // 16 * 16 + 16
    I = lambda *x: (ctypes.c_int32 * len(x))(*x)
    rc = lib.mlahip_copy_pages((ctypes.c_int64 * 4)(p, page_stride, row_stride, 16), 1, I(), I(), None, 0, pages, page, None, 0, 0, 0, None)
    assert rc == (0 if fine else -2)                           # (no pairs: nothing is launched)
    assert fine or "share memory" in lib.mlahip_last_error_string().decode()
    del raw


@pytest.mark.gpu
def test_layouts_of_one_allocation(dev):
    """Pages inside rows, rows inside pages and keys beside values are caches; pages that overlap are none."""
    from omni_npu_amd import kernels as K
    base = torch.arange(7 * 5 * 2 * 16, device=dev, dtype=torch.int32).view(7, 5, 2, 16)
    for view in (lambda x: x[:, :, 0], lambda x: x[:, :, 0].transpose(0, 1), lambda x: x[:, 1:4, 1], lambda x: x[:, :, 0].transpose(0, 1)[:4]):
        got, want = base.clone(), base.clone()
        K.copy_pages(view(got), [0, 1], [3, 2], rows=[2, 3])
        view(want)[3, :2], view(want)[2, :3] = view(base)[0, :2], view(base)[1, :3]
        assert torch.equal(got, want)
    with pytest.raises(ValueError, match="share memory"):
        K.copy_pages(base.view(-1).as_strided((8, 4, 16), (32, 16, 1)), [0], [3])
