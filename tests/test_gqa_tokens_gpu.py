"""Requests that have more tokens in the batch than a call does: the ones that are done see the keys of their own places, the others stay as they were."""
import pytest
import torch

from oracle import heads_oracle as H
from tests.test_gqa_decode_gpu import call, make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("q_len", [1, 2, 3, 5])
@pytest.mark.parametrize("window", [None, 1, 30, 90])
@pytest.mark.parametrize("chunks", [None, 0, 7])
@pytest.mark.parametrize("lens,counts", [([10], [4]), ([300, 40, 3, 129, 9, 0], [6, 1, 5, 17, 9, 2]), ([40] * 70, [1, 3, 7, 0, 2] * 14)],
                         ids=["one", "ragged", "many"])
def test_more_tokens_than_are_done(dev, q_len, window, chunks, lens, counts):
    c = make(dev, lens, q_lens=counts, hq=6, hk=2, d=64, page=16, seed=q_len)
    out, lse = call(dev, c, q_len, varlen=True, window=window, num_chunks=chunks)
    o, l, weight, reach = H.gqa(c["q"], c["k"], c["v"], c["table"], c["lens"], c["scale"], c["start"], window or 0)
    done = torch.cat([torch.arange(n) < q_len for n in counts])
    assert ((out.double() - o).abs() <= H.gqa_tolerance(o, weight, reach, c["dtype"], 64))[done].all()
    assert torch.equal(torch.isinf(lse[done]), torch.isinf(l[done])) and (out[done][torch.isinf(l[done])] == 0).all()
    assert torch.isnan(out[~done].float()).all() and torch.isnan(lse[~done]).all()


def test_token_counts_out_of_range(dev):
    """Starts that fall, and counts near 2^31: rows without a key, or none."""
    c = make(dev, [20, 20, 20], q_lens=[2, 2, 2], hq=6, hk=2, d=64, page=16)
    c["start"] = torch.tensor([0, 2 ** 31 - 1, 2, 6], dtype=torch.int32)
    out, lse = call(dev, c, 2, varlen=True, window=4)
    o, l, weight, reach = H.gqa(c["q"][2:], c["k"], c["v"], c["table"][2:], c["lens"][2:], c["scale"], torch.tensor([0, 4]), 4)
    assert (out[:2] == 0).all() and torch.isinf(lse[:2]).all()
    assert ((out[2:4].double() - o[:2]).abs() <= H.gqa_tolerance(o, weight, reach, c["dtype"], 64)[:2]).all()
    assert torch.isnan(out[4:].float()).all() and torch.isnan(lse[4:]).all()
