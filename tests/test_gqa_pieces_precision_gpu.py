"""Requests in pieces whose scores are large: a piece counts by how many keys it has, and by how far its largest score lies below another's, whatever the scores' size.
The ordinary attention and the drafted trees'."""
import math

import pytest
import torch

from tests.test_gqa_decode_gpu import call as chain
from tests.test_gqa_decode_gpu import make
from tests.test_gqa_precision_gpu import tolerance
from tests.test_gqa_tree_gpu import call, tree
from tests.test_gqa_tree_precision_gpu import exact, places

pytestmark = pytest.mark.gpu

BOTH = pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "fp16"])
FORMS = pytest.mark.parametrize("rows", [None, 16, 64, 128], ids=["chain", "tree16", "tree64", "tree128"])


def run(dev, c, rows, chunks):
    """As gqa_decode, or as trees that are chains."""
    if rows is None:
        return chain(dev, c, 1, num_chunks=chunks)
    return call(dev, c, 1, num_chunks=chunks, rows_per_group=rows, heads_per_group=1)


def close(c, out, lse, **more):
    o, l, weight, reach = exact(c)
    tol = tolerance(c, o, weight, torch.zeros_like(reach), l) + more.get("also", 0.0) * (weight + o.abs())
    err = (out.double() - o).abs()
    assert (err <= tol).all(), f"worst {(err / tol).max():.3g} of the tolerance"
    assert torch.allclose(lse.double(), l, rtol=2.0 ** -21)


@BOTH
@FORMS
@pytest.mark.parametrize("scale", [2.0 ** -11, 2.0 ** -6, 0.25, 8.0, 4096.0, 2.0 ** 14])
@pytest.mark.parametrize("sign", [1.0, -1.0])
@pytest.mark.parametrize("lens,chunks", [([300, 33, 70], 7), ([1100], 3), ([1100], 35), ([40, 900], 12)])
def test_equal_scores_in_pieces(dev, dtype, rows, scale, sign, lens, chunks):
    """Pieces of different lengths, all scores one number of up to 2^36 (exact in fp32): the mean of the values, to the probabilities' and sums' roundings and, by
    their logarithms' own, a few times 2^-20."""
    c = tree(make(dev, lens, hq=4, hk=2, d=64, dtype=dtype, page=16, seed=4), seed=4)
    c["scale"] = scale
    c["q"].zero_()
    c["q"][..., 0] = 32768.0 * sign
    c["k"][..., 0] = 100.0
    close(c, *run(dev, c, rows, chunks), also=2.0 ** -18)


@BOTH
@FORMS
@pytest.mark.parametrize("first", [0, 1, 2, 3])
@pytest.mark.parametrize("chunks", [8, 16])
@pytest.mark.parametrize("d", [64, 128])
def test_pieces_a_step_apart(dev, dtype, rows, first, chunks, d):
    """Scores of 2^27, where neighbours in fp32 lie 16 apart, in log2 units: pieces of the one weigh 2^-16 of pieces of the next, wherever in the request."""
    n = 512
    c = tree(make(dev, [n, n], hq=4, hk=2, d=d, dtype=dtype, page=16, seed=5), seed=5)
    c["scale"] = 16 * math.log(2.0)
    c["q"].zero_()
    c["q"][..., 0], c["q"][..., 1] = 4096.0, 1.0
    c["k"][..., 0] = 2048.0
    for b in range(2):                                        # (the larger ones last, or first)
        at = places(c, b, n)
        c["k"][at[0], at[1], :, 1] = (first + ((torch.arange(n) >= n // 2) == (b == 0)).to(dtype))[:, None]
    close(c, *run(dev, c, rows, chunks * 2), also=2.0 ** -18)
