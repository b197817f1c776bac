"""How near the attention of drafted trees comes to its 64-bit statement, with 16 to 128 rows to a workgroup: results are off by their own rounding, and by
little else; scores and values of any size, and ones that are no numbers."""
import pytest
import torch

from oracle import tree_oracle as T
from tests.test_gqa_decode_gpu import make
from tests.test_gqa_precision_gpu import LEFT, tolerance
from tests.test_gqa_tree_gpu import call, tree

pytestmark = pytest.mark.gpu

BOTH = pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "fp16"])
ROWS = pytest.mark.parametrize("rows", [16, 64, 128])


def own_rows(rows, d=64):
    return dict(rows_per_group=32 if rows == 64 and d == 256 else rows, heads_per_group=1)


def exact(c):
    k, v = (c[n].float() for n in ("k", "v"))
    return T.gqa(c["q"], k, v, c["table"], c["lens"], c["visible"], c["scale"], c["start"], 0, c["k_scale"], c["v_scale"])


def places(c, b, n):
    """Pages and rows of a request's first n keys."""
    at, page = torch.arange(n), c["k"].shape[1]
    return c["table"][b].long()[at // page], at % page


def seen(c, b, q_len):
    return T.seen(c["visible"][b * q_len:(b + 1) * q_len], int(c["lens"][b]), q_len)


@pytest.mark.parametrize("d", [64, 128, 256])
@BOTH
@pytest.mark.parametrize("fp8", [False, True], ids=["same", "e4m3"])
@pytest.mark.parametrize("q_len,hq,hk", [(1, 8, 2), (6, 26, 2), (33, 16, 4)])
@pytest.mark.parametrize("chunks", [0, 7])
@ROWS
def test_results_are_off_by_their_own_rounding(dev, d, dtype, fp8, q_len, hq, hk, chunks, rows):
    c = tree(make(dev, [q_len, q_len + 4, 40, 400, 34], q_len=q_len, hq=hq, hk=hk, d=d, dtype=dtype, fp8=fp8, page=16, seed=d + q_len), seed=q_len)
    out, lse = call(dev, c, q_len, num_chunks=chunks, **own_rows(rows, d))
    o, l, weight, reach = exact(c)
    tol = tolerance(c, o, weight, reach, l)
    err = (out.double() - o).abs()
    assert (err <= tol).all(), f"worst {(err / tol).max():.3g} of the tolerance"
    off = 1.01 * LEFT[dtype] + 400 * (2.0 ** -24 + 2.0 ** -25 * (dtype == torch.float16)) + (d + 4) * 2.0 ** -24 * reach + 2.0 ** -18 * (1 + l.abs())
    assert ((lse.double() - l).abs() <= off).all()


@BOTH
@pytest.mark.parametrize("chunks", [0, 6])
@pytest.mark.parametrize("q_len", [1, 3])
@ROWS
def test_an_infinite_value_gives_an_infinity(dev, dtype, chunks, q_len, rows):
    """In a key's place that every token sees, of its sign, whatever its probability; the other dims are as without it."""
    c = tree(make(dev, [64] * 60, q_len=q_len, hq=8, hk=2, d=64, dtype=dtype, page=16, seed=3), seed=3)
    ref, ref_lse = call(dev, c, q_len, num_chunks=chunks, **own_rows(rows))
    for b in range(60):
        c["v"][c["table"][b, b // 16], b % 16, :, b] = float("inf") if b % 2 else -float("inf")
    out, lse = call(dev, c, q_len, num_chunks=chunks, **own_rows(rows))
    t, at = torch.arange(60 * q_len), torch.arange(60).repeat_interleave(q_len)
    there = out[t, :, at].float()
    assert torch.isinf(there).all() and ((there > 0) == (at % 2 == 1)[:, None]).all()
    out[t, :, at] = ref[t, :, at]
    assert torch.equal(out, ref) and torch.equal(lse, ref_lse)


@BOTH
@pytest.mark.parametrize("gap", [4, 14, 22, 24, 26, 30])
@pytest.mark.parametrize("chunks", [0, 5])
@ROWS
def test_many_keys_far_below_one(dev, dtype, gap, chunks, rows):
    """The first key takes nearly everything and has small values; 8191 others lie ``gap`` powers of two below it.  In fp16 a probability is off by
    2^-25 at most where the largest are 2^12 and more (a reference of 128 rows is a whole number, up to one above 2^13's), and a result below 2^-14 by 2^-25."""
    n, g = 8192, torch.Generator().manual_seed(gap)
    c = tree(make(dev, [n], q_len=3, hq=8, hk=8, d=64, dtype=dtype, page=128, seed=gap), parents=[-1, 0, 1])
    c["scale"] = 1.0
    c["q"].zero_()
    c["q"][..., 0] = 8.0
    c["k"][..., 0] = (4.0 + (torch.rand(c["k"].shape[:3], generator=g) * 0.4 - gap * 0.6931) / 8).to(dtype)
    c["v"] += 1.0
    first = c["table"][0, 0]
    c["k"][first, 0, :, 0] = 4.0
    c["v"][first, 0] = c["v"][first, 0] * 2.0 ** -10
    out, lse = call(dev, c, 3, num_chunks=chunks, **own_rows(rows))
    o, l, weight, reach = exact(c)
    tol = 2.0 ** -8 * o.abs() if dtype == torch.bfloat16 else 2.0 ** -11 * o.abs() + 1.02 * n * 2.0 ** -37 * (c["v"].abs().max().double() + o.abs()) + 2.0 ** -25
    tol = tol + (1.01 * LEFT[dtype] + n * 2.0 ** -24 + 2 * 68 * 2.0 ** -24 * reach[..., None] + 2.0 ** -19) * (weight + o.abs())
    err = (out.double() - o).abs()
    assert (err <= tol).all(), f"worst {(err / tol).max():.3g} of the tolerance"


@BOTH
@pytest.mark.parametrize("scale", [1.0, 8.0, 64.0, 4096.0])
@pytest.mark.parametrize("order", ["rising", "falling", "mixed"])
@pytest.mark.parametrize("sign", [1.0, -1.0])
@ROWS
def test_scores_whose_steps_are_large(dev, dtype, scale, order, sign, rows):
    """Scores of up to 2^36, whose neighbours in fp32 lie further apart than a reference below them: of what a token sees one key takes everything."""
    n, s, g = 200, 9, torch.Generator().manual_seed(1)
    c = tree(make(dev, [n], q_len=s, hq=4, hk=2, d=64, dtype=dtype, page=16, seed=2), seed=2)
    c["scale"] = scale
    c["q"].zero_()
    c["q"][..., 0] = 32768.0 * sign
    size = {"rising": torch.arange(n), "falling": torch.arange(n).flip(0), "mixed": torch.randperm(n, generator=g)}[order] + 1.0
    at = places(c, 0, n)
    c["k"][at[0], at[1], :, 0] = size.to(dtype)[:, None]
    key = torch.where(seen(c, 0, s), size * sign, -torch.inf).argmax(1)
    out, lse = call(dev, c, s, num_chunks=0, **own_rows(rows))
    assert torch.equal(out, c["v"][at[0][key], at[1][key]].repeat_interleave(2, 1))
    want = 32768.0 * sign * scale * size[key].double()
    assert torch.allclose(lse.double(), want[:, None].expand(-1, 4), rtol=2.0 ** -21)


@BOTH
@pytest.mark.parametrize("scale", [1.0, 64.0, 4096.0, 2.0 ** 20])
@pytest.mark.parametrize("requests,chunks", [(1, 3), (1, 20), (3, 5), (3, 40)])
@ROWS
def test_pieces_with_scores_whose_steps_are_large(dev, dtype, scale, requests, chunks, rows):
    """The same with each request in pieces, the largest score in its first, a middle or its newest key, which its root sees."""
    n = 400
    c = tree(make(dev, [n] * requests, hq=4, hk=2, d=64, dtype=dtype, page=16, seed=2), seed=2)
    c["scale"] = scale
    c["q"].zero_()
    c["q"][..., 0] = 32768.0
    c["k"][..., 0] = -(torch.arange(c["k"].shape[0] * 16).view(-1, 16, 1) % 251 + 1.0).to(dtype)
    at = torch.tensor([(0, n - 1, 170)[b] for b in range(requests)])
    page, row = c["table"][torch.arange(requests), at // 16].long(), at % 16
    c["k"][page, row, :, 0] = 200.0
    out, lse = call(dev, c, 1, num_chunks=chunks, **own_rows(rows))
    assert torch.equal(out, c["v"][page, row].repeat_interleave(2, 1))
    assert torch.allclose(lse.double(), torch.tensor(32768.0 * 200 * scale, dtype=torch.float64), rtol=2.0 ** -21)


@BOTH
@pytest.mark.parametrize("scale", [2.0 ** -13, 2.0 ** -11, 2.0 ** -6, 0.25, 1.0, 3.0, 8.0, 64.0, 4096.0, 2.0 ** 14])
@pytest.mark.parametrize("sign", [1.0, -1.0])
@pytest.mark.parametrize("behind", [0, 1, 70])
@ROWS
def test_equal_scores_of_any_size_weigh_the_same(dev, dtype, scale, sign, behind, rows):
    """All keys' scores are one number, up to 2^36, behind ``behind`` keys of much smaller ones: a result is the mean of the others' values.  (The scores are
    exact in fp32, so nothing is off but the probabilities' second operands, the sums and the result, and below 2^10 a first tile's by half a step, 2^-15.)"""
    s = 9
    c = tree(make(dev, [300, 33 + behind, s + behind, 256], q_len=s, hq=8, hk=2, d=64, dtype=dtype, page=16, seed=2), seed=2)
    c["scale"] = scale
    c["q"].zero_()
    c["q"][..., 0] = 32768.0 * sign
    c["k"][..., 0] = 100.0
    for b in range(4):
        at = places(c, b, behind)
        c["k"][at[0], at[1], :, 0] = 100.0 - 50.0 * sign
    out, lse = call(dev, c, s, num_chunks=0, **own_rows(rows))
    o, l, weight, reach = exact(c)
    tol = tolerance(c, o, weight, torch.zeros_like(reach), l) + 2.0 ** -15 * (scale < 2.0 ** -12) * (weight + o.abs())
    err = (out.double() - o).abs()
    assert (err <= tol).all(), f"worst {(err / tol).max():.3g} of the tolerance"
    assert torch.allclose(lse.double(), l, rtol=2.0 ** -21)


@pytest.mark.parametrize("d", [64, 128, 256])
@BOTH
@pytest.mark.parametrize("fp8", [False, True], ids=["same", "e4m3"])
@pytest.mark.parametrize("scale", [2.0 ** -11, 1.0, 64.0, 2.0 ** 14])
@pytest.mark.parametrize("chunks", [0, 9])
@ROWS
def test_equal_scores_of_any_head_and_cache(dev, d, dtype, fp8, scale, chunks, rows):
    """The same with scales of the cache's heads, in pieces (their log-sum-exps' sums off by a few times 2^-20), and a value that is no number where some tokens
    do not see it, so that those are done by themselves."""
    s = 9
    c = tree(make(dev, [300, 75], q_len=s, hq=8, hk=2, d=d, dtype=dtype, fp8=fp8, page=16, seed=2), seed=2)
    c["scale"] = scale
    c["q"].zero_()
    c["q"][..., 0] = 32768.0
    for name, at, x in (("k", (Ellipsis, 0), 96.0), ("v", (c["table"][0, (300 - s + 3) // 16].long(), (300 - s + 3) % 16), float("nan"))):
        y = c[name].float()
        y[at] = x
        c[name] = y.to(c[name].dtype)
    if fp8:
        c["k_scale"] = torch.tensor([0.5, 4.0])
    rows_of = ~torch.cat((seen(c, 0, s)[:, 300 - s + 3], torch.zeros(s, dtype=torch.bool)))
    assert 0 < rows_of.sum() < 2 * s
    out, lse = call(dev, c, s, num_chunks=chunks, **own_rows(rows, d))
    o, l, weight, reach = exact(c)
    clean = dict(c, v=c["v"].float().nan_to_num(0.0))
    tol = tolerance(clean, o, weight, torch.zeros_like(reach), l) + 2.0 ** -18 * (weight + o.abs())
    err = (out.double() - o).abs()
    assert (err[rows_of] <= tol[rows_of]).all(), f"worst {(err / tol)[rows_of].max():.3g} of the tolerance"
    assert torch.isnan(out[~rows_of].float()).all() and torch.allclose(lse.double(), l, rtol=2.0 ** -21)


@BOTH
@pytest.mark.parametrize("lens,chunks", [([6, 7, 40, 700], 0), ([6, 7, 40, 700], 9), ([5000], 1), ([5000], 40), ([5000, 3000, 20], 30)])
@pytest.mark.parametrize("d", [64, 256])
@ROWS
def test_values_of_the_largest_size(dev, dtype, lens, chunks, d, rows):
    """All values are the type's largest, of one sign for a dim: so are the results, however many are summed and joined."""
    c = tree(make(dev, lens, q_len=6, hq=6, hk=2, d=d, dtype=dtype, page=16, seed=7), seed=7)
    sign = 1.0 - 2.0 * (torch.arange(d) % 2)
    c["v"][...] = (sign * torch.finfo(dtype).max).to(dtype)
    out, lse = call(dev, c, 6, num_chunks=chunks, **own_rows(rows, d))
    assert torch.equal(out, c["v"][0, 0, 0].expand_as(out))
    o, l, weight, reach = exact(dict(c, v=torch.zeros_like(c["v"])))
    assert ((lse.double() - l).abs() <= 1.01 * LEFT[dtype] + 5000 * 2.0 ** -24 + (d + 4) * 2.0 ** -24 * reach + 2.0 ** -18 * (1 + l.abs())).all()


@pytest.mark.parametrize("chunks", [0, 6])
@ROWS
def test_infinite_and_undefined_scores(dev, chunks, rows):
    """Scores of -inf weigh nothing; one of +inf or NaN makes the rows that see its key undefined, and no others.  (A neighbour's score
    may move a row's reference: two results that are each off by their rounding, LEFT and 2^-17 of values below 8.)"""
    s = 5

    def same(x, y):
        assert ((x.double() - y.double()).abs() <= 2.02 * 2.0 ** -8 * y.double().abs() + 2 * 16 * (LEFT[torch.bfloat16] + 2.0 ** -17)).all()

    c = tree(make(dev, [400, 130], q_len=s, hq=16, hk=2, d=64, page=16, seed=31), seed=31)
    c["q"][...] = c["q"].abs() + 0.5
    place = lambda b, key: (c["table"][b, key // 16].long(), key % 16)
    kw = dict(num_chunks=chunks, **own_rows(rows))
    for key in (0, 1, *range(32, 64), 200):                   # (a whole step of keys among them)
        c["k"][place(0, key)][0] = -float("inf")
    ref, ref_lse = call(dev, c, s, **kw)
    assert torch.isfinite(ref.float()).all()
    for bad in (float("inf"), float("nan")):
        for key in (150, 400 - s + 1):                        # (one of the context's, one of the tree's)
            was = c["k"][place(0, key)][1, 3].clone()
            c["k"][place(0, key)][1, 3] = bad
            out, lse = call(dev, c, s, **kw)
            c["k"][place(0, key)][1, 3] = was
            at = seen(c, 0, s)[:, key].nonzero()[:, 0]
            assert 0 < len(at) and torch.isnan(out[at, 8:].float()).all() and torch.isnan(lse[at, 8:]).all()
            out[at, 8:], lse[at, 8:] = ref[at, 8:], ref_lse[at, 8:]
            same(out, ref)
            same(lse, ref_lse)
    for bad in (float("inf"), float("nan")):                  # a query's
        q = c["q"].clone()
        c["q"][s + 2, 3, 5] = bad
        out, lse = call(dev, c, s, **kw)
        c["q"] = q
        assert torch.isnan(out[s + 2, 3].float()).all() and torch.isnan(lse[s + 2, 3])
        out[s + 2, 3], lse[s + 2, 3] = ref[s + 2, 3], ref_lse[s + 2, 3]
        same(out, ref)
        same(lse, ref_lse)
    c["k"][c["table"][1].long()[:9], :, 0] = -float("inf")    # every score of a row
    out, lse = call(dev, c, s, **kw)
    assert (out[s:, :8] == 0).all() and (lse[s:, :8] == -float("inf")).all() and torch.equal(out[s:, 8:], ref[s:, 8:])


@pytest.mark.parametrize("scale", [-0.2, 0.0, 3.0])
@pytest.mark.parametrize("fp8", [False, True], ids=["same", "e4m3"])
@ROWS
def test_scales_of_any_sign(dev, scale, fp8, rows):
    c = tree(make(dev, [500, 33], q_len=7, hq=6, hk=2, d=128, fp8=fp8, seed=32), seed=32)
    c["scale"] = scale
    out, lse = call(dev, c, 7, **own_rows(rows))
    o, l, weight, reach = exact(c)
    err, tol = (out.double() - o).abs(), tolerance(c, o, weight, reach, l)
    assert (err <= tol).all(), f"worst {(err / tol).max():.3g} of the tolerance"
