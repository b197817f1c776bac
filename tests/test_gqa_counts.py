"""CPU: rows of tokens that are counted in 32 bits."""
import ctypes

import pytest

from omni_npu_amd import _lib


@pytest.mark.parametrize("batch,q_len,fine", [(2047, 1 << 20, True), (2048, 1 << 20, False), (4096, 1 << 20, False), (65535, 1 << 15, True),
                                              (65535, (1 << 15) + 1, False)])
def test_tokens_of_all_requests_fit_32_bits(batch, q_len, fine):
    """Without query_start_loc a request's rows begin at its number times q_len: request 4096 of 2^20 tokens would begin at row 0 again.  (Every call
    here lacks scratch memory: what is fine is refused for that.)"""
    lib = _lib.load()
    raw = ctypes.create_string_buffer(1 << 12)
    p = ctypes.addressof(raw) // 16 * 16 + 16
    call = lambda qsl: lib.mlahip_gqa_decode(p, 128, 128, 100, p, 2048, 128, 128, p, 2048, 128, 128, 4, 16, p, 4, 4, p, qsl, batch, q_len, 1, 1,
                                             128, 0, 0, None, None, 0.1, 0, p, 128, 128, None, None, 0, 1, 1, 64, None)
    assert call(None) == (-4 if fine else -2) and call(p) == -4
    del raw
