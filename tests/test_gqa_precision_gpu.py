"""How near the attention over ordinary key and value heads comes to its 64-bit statement: results are off by their own rounding, and by
little else."""
import pytest
import torch

from oracle import heads_oracle as H
from tests.test_gqa_decode_gpu import call, make

pytestmark = pytest.mark.gpu

# Of a probability, what two operands leave of it: the first part, 1 - 2^-6 of it, is rounded by a relative u, so the rest is at most 2^-6 + u of it,
# and is rounded by u again.
LEFT = {t: H.U[t] * (2.0 ** -6 + H.U[t]) for t in (torch.bfloat16, torch.float16)}


def tolerance(c, o, weight, reach, lse):
    """The result's own rounding; probabilities off by LEFT (of which numerator and denominator take the same ones: weight + |o| in all); in fp16 a
    rest below 2^-14 is rounded by 2^-25, for every key, against a sum of at least one; a sum of n products in fp32, n 2^-24 of their sizes; scores' errors
    and the smaller roundings as H.gqa_tolerance has them."""
    n = int(c["lens"].max())
    v = c["v"].float().abs().amax() * (1.0 if c["v_scale"] is None else c["v_scale"].max())
    small = n * 2.0 ** -25 * (c["dtype"] == torch.float16)
    part = 1.01 * LEFT[c["dtype"]] + n * 2.0 ** -24 + 2 * (c["d"] + 4) * 2.0 ** -24 * reach[..., None] + 2.0 ** -19
    return H.U[c["dtype"]] * o.abs() + part * (weight + o.abs()) + small * (float(v) + o.abs()) + 1e-30


def close(c, out, lse):
    k, v = (c[n].float() for n in ("k", "v"))
    o, l, weight, reach = H.gqa(c["q"], k, v, c["table"], c["lens"], c["scale"], c["start"], 0, c["k_scale"], c["v_scale"])
    tol = tolerance(c, o, weight, reach, l)
    err = (out.double() - o).abs()
    assert (err <= tol).all(), f"worst {(err / tol).max():.3g} of the tolerance"
    n = int(c["lens"].max())
    off = 1.01 * LEFT[c["dtype"]] + n * (2.0 ** -24 + 2.0 ** -25 * (c["dtype"] == torch.float16)) + (c["d"] + 4) * 2.0 ** -24 * reach + 2.0 ** -18 * (1 + l.abs())
    assert ((lse.double() - l).abs() <= off).all()


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "fp16"])
@pytest.mark.parametrize("fp8", [False, True], ids=["same", "e4m3"])
@pytest.mark.parametrize("q_len,hq,hk", [(1, 8, 2), (3, 16, 2), (5, 26, 2)])
@pytest.mark.parametrize("chunks", [0, 7])
def test_results_are_off_by_their_own_rounding(dev, d, dtype, fp8, q_len, hq, hk, chunks):
    """Few keys and many, so that probabilities' roundings would not average out."""
    c = make(dev, [6, 11, 40, 700, 7], q_len=q_len, hq=hq, hk=hk, d=d, dtype=dtype, fp8=fp8, page=16, seed=d + q_len)
    close(c, *call(dev, c, q_len, num_chunks=chunks))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "fp16"])
@pytest.mark.parametrize("chunks", [0, 6])
def test_an_infinite_value_gives_an_infinity(dev, dtype, chunks):
    """In every key's place once, of its sign, whatever its probability: 64 requests of 64 keys, each with one; the other dims are as without it."""
    c = make(dev, [64] * 64, hq=8, hk=2, d=64, dtype=dtype, page=16, seed=3)
    ref, ref_lse = call(dev, c, 1, num_chunks=chunks)
    for b in range(64):
        c["v"][c["table"][b, b // 16], b % 16, :, b] = float("inf") if b % 2 else -float("inf")
    out, lse = call(dev, c, 1, num_chunks=chunks)
    at = torch.arange(64)
    there = out[at, :, at].float()
    assert torch.isinf(there).all() and ((there > 0) == (at % 2 == 1)[:, None]).all()
    out[at, :, at] = ref[at, :, at]
    assert torch.equal(out, ref) and torch.equal(lse, ref_lse)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "fp16"])
@pytest.mark.parametrize("gap", [4, 14, 22, 24, 26, 30])
@pytest.mark.parametrize("heads,chunks", [(8, 0), (1, 0), (8, 5)])
def test_many_keys_far_below_one(dev, dtype, gap, heads, chunks):
    """The first key takes nearly everything and has small values; 8191 others lie ``gap`` powers of two below it.  In fp16 a probability is off by
    2^-25 at most where the largest are 2^13 and more, and a result below 2^-14 by 2^-25."""
    n, g = 8192, torch.Generator().manual_seed(gap)
    c = make(dev, [n], hq=8, hk=8, d=64, dtype=dtype, page=128, seed=gap)
    c["scale"] = 1.0
    c["q"].zero_()
    c["q"][..., 0] = 8.0
    c["k"][..., 0] = (4.0 + (torch.rand(c["k"].shape[:3], generator=g) * 0.4 - gap * 0.6931) / 8).to(dtype)
    c["v"] += 1.0
    first = c["table"][0, 0]
    c["k"][first, 0, :, 0] = 4.0
    c["v"][first, 0] = c["v"][first, 0] * 2.0 ** -10
    out, lse = call(dev, c, 1, heads_per_group=heads, num_chunks=chunks)
    o, l, weight, reach = H.gqa(c["q"], c["k"], c["v"], c["table"], c["lens"], 1.0, c["start"])
    tol = H.gqa_tolerance(o, weight, reach, dtype, 64)
    if dtype == torch.float16:
        tol = tol + 1.02 * n * 2.0 ** -38 * (c["v"].abs().max().double() + o.abs()) + 2.0 ** -25
    err = (out.double() - o).abs()
    assert (err <= tol).all(), f"worst {(err / tol).max():.3g} of the tolerance"


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "fp16"])
@pytest.mark.parametrize("scale", [1.0, 8.0, 64.0, 4096.0])
@pytest.mark.parametrize("order", ["rising", "falling", "mixed"])
@pytest.mark.parametrize("sign", [1.0, -1.0])
def test_scores_whose_steps_are_large(dev, dtype, scale, order, sign):
    """Scores of up to 2^36, whose neighbours in fp32 lie further apart than a reference below them: one key takes everything."""
    n, g = 200, torch.Generator().manual_seed(1)
    c = make(dev, [n], hq=4, hk=2, d=64, dtype=dtype, page=16, seed=2)
    c["scale"] = scale
    c["q"].zero_()
    c["q"][..., 0] = 32768.0 * sign
    size = {"rising": torch.arange(n), "falling": torch.arange(n).flip(0), "mixed": torch.randperm(n, generator=g)}[order] + 1.0
    rows = c["table"][0].long()[torch.arange(n) // 16], torch.arange(n) % 16
    c["k"][rows[0], rows[1], :, 0] = size.to(dtype)[:, None]
    key = int((size * sign).argmax())
    for heads in (1, 2):
        out, lse = call(dev, c, 1, heads_per_group=heads, num_chunks=0)
        assert torch.equal(out[0], c["v"][rows[0][key], rows[1][key]].repeat_interleave(2, 0))
        assert torch.allclose(lse.double(), torch.tensor(32768.0 * sign * scale * float(size[key]), dtype=torch.float64), rtol=2.0 ** -21)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "fp16"])
@pytest.mark.parametrize("scale", [1.0, 64.0, 4096.0, 2.0 ** 20])
@pytest.mark.parametrize("requests,chunks", [(1, 3), (1, 20), (3, 5), (3, 40)])
def test_pieces_with_scores_whose_steps_are_large(dev, dtype, scale, requests, chunks):
    """The same with each request in pieces, the largest score in its first, last or a middle one."""
    n = 400
    c = make(dev, [n] * requests, hq=4, hk=2, d=64, dtype=dtype, page=16, seed=2)
    c["scale"] = scale
    c["q"].zero_()
    c["q"][..., 0] = 32768.0
    c["k"][..., 0] = -(torch.arange(c["k"].shape[0] * 16).view(-1, 16, 1) % 251 + 1.0).to(dtype)
    at = torch.tensor([(0, n - 1, 170)[b] for b in range(requests)])
    page, row = c["table"][torch.arange(requests), at // 16].long(), at % 16
    c["k"][page, row, :, 0] = 200.0
    out, lse = call(dev, c, 1, num_chunks=chunks)
    assert torch.equal(out, c["v"][page, row].repeat_interleave(2, 1))
    assert torch.allclose(lse.double(), torch.tensor(32768.0 * 200 * scale, dtype=torch.float64), rtol=2.0 ** -21)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "fp16"])
@pytest.mark.parametrize("lens,chunks", [([1, 2, 40, 700], 0), ([1, 2, 40, 700], 9), ([5000], 1), ([5000], 40), ([5000, 3000, 20], 30)])
@pytest.mark.parametrize("d", [64, 256])
def test_values_of_the_largest_size(dev, dtype, lens, chunks, d):
    """All values are the type's largest, of one sign for a dim: so are the results, however many are summed and joined."""
    c = make(dev, lens, hq=6, hk=2, d=d, dtype=dtype, page=16, seed=7)
    sign = 1.0 - 2.0 * (torch.arange(d) % 2)
    c["v"][...] = (sign * torch.finfo(dtype).max).to(dtype)
    out, lse = call(dev, c, 1, num_chunks=chunks)
    assert torch.equal(out, c["v"][0, 0, 0].expand_as(out))
    o, l, weight, reach = H.gqa(c["q"], c["k"], torch.zeros_like(c["v"]), c["table"], c["lens"], c["scale"], c["start"])
    assert ((lse.double() - l).abs() <= 1.01 * LEFT[dtype] + 5000 * 2.0 ** -24 + (d + 4) * 2.0 ** -24 * reach + 2.0 ** -18 * (1 + l.abs())).all()
