"""Batches in which a few requests have most of the keys, and so most of the partial results."""
import pytest
import torch

from tests.test_gqa_decode_gpu import call as chain
from tests.test_gqa_decode_gpu import check as check_chain
from tests.test_gqa_decode_gpu import make
from tests.test_gqa_tree_gpu import call, check, tree

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("q_len,hq,hk", [(1, 8, 2), (3, 10, 5), (1, 1, 1)])
@pytest.mark.parametrize("lens,chunks", [([20] * 9 + [4000] + [33] * 10, 100), ([2500, 2500, 7, 0, 2600] + [40] * 20, 180), ([5] * 70 + [3000, 1, 0, 3000], 190),
                                         ([1100, 3, 3, 3, 3, 1100], 48)], ids=["one", "three", "behind64", "ends"])
def test_a_few_long_requests(dev, d, q_len, hq, hk, lens, chunks):
    """More partial results than are joined side by side, in one request and in several, behind the 64 that a wavefront looks at first, at the batch's ends."""
    c = make(dev, lens, q_len=q_len, hq=hq, hk=hk, d=d, page=16, seed=len(lens))
    assert chunks <= 8 * len(lens)
    check_chain(c, *chain(dev, c, q_len, num_chunks=chunks))
    tree(c, seed=2)
    check(c, *call(dev, c, q_len, num_chunks=chunks))
    check(c, *call(dev, c, q_len, num_chunks=chunks, rows_per_group=128, heads_per_group=1))


def test_ragged_token_counts(dev):
    """Requests without tokens, one of many tokens among the long ones; rows behind the last request stay."""
    counts = [1, 7, 0, 2, 1] + [1] * 16
    lens = [2600, 2600, 2600, 40, 0] + [20] * 16
    c = make(dev, lens, q_lens=counts, hq=8, hk=2, d=64, page=16, seed=6)
    out, lse = chain(dev, c, 7, varlen=True, num_chunks=160)
    check_chain(c, out, lse)


def test_a_long_request_takes_its_own_time(dev):
    """One of 131 072 keys among 63 of 100 takes little longer than by itself, where four wavefronts join each of its rows, and the others' begins: chunks are
    (4096 + 63 x 4) / 256 = 17 units of 32 keys, so a workgroup has up to five of them one after the other, 3.5 us each."""
    from omni_npu_amd import kernels as K
    n, page, hq, hk, d = 131072, 128, 32, 8, 64
    k = torch.zeros(n // page + 64, page, hk, d, dtype=torch.bfloat16, device=dev)
    v, q = torch.zeros_like(k), torch.zeros(64, hq, d, dtype=torch.bfloat16, device=dev)
    out = torch.empty_like(q)
    table = torch.zeros(64, n // page, dtype=torch.int32, device=dev)
    table[0] = torch.arange(n // page)
    table[1:, 0] = n // page + torch.arange(63)
    lens = torch.tensor([n] + [100] * 63, dtype=torch.int32, device=dev)

    def us(b):
        best = float("inf")
        for _ in range(8):
            start, end = torch.cuda.Event(True), torch.cuda.Event(True)
            start.record()
            for _ in range(20):
                K.gqa_decode(q[:b], k, v, table[:b], lens[:b], 0.125, out[:b], num_chunks=256, heads_per_group=8, rows_per_group=16)
            end.record()
            torch.cuda.synchronize()
            best = min(best, start.elapsed_time(end) * 50)
        return best

    us(1), us(64)
    alone, among = us(1), us(64)
    assert among < 1.25 * (alone + 5 * 3.5), (alone, among)
