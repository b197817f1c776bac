"""Attention of tokens drafted as trees over a paged cache against its plain statement in 64 bits: types, head layouts, trees of one token to
hundreds, windows, places that hold infinities and NaN, strides, ragged and padded batches, pieces, graphs."""
import pytest
import torch

from oracle import heads_oracle as H
from oracle import tree_oracle as T
from tests.test_gqa_decode_gpu import E4M3, make
from tests.test_gqa_decode_gpu import call as chain

pytestmark = pytest.mark.gpu


def tree(c, seed=0, words=1, parents=None):
    """Random trees for a case's tokens: parents [T] and their bits."""
    g = torch.Generator().manual_seed(seed)
    sets, ups = [], []
    for a, z in zip(c["start"].tolist(), c["start"].tolist()[1:]):
        up = [-1 if i == 0 else int(torch.randint(-1, i, (1,), generator=g)) for i in range(z - a)] if parents is None else parents[a:z]
        ups += up
        sets += T.ancestors(up)
    c["parents"], c["visible"] = ups, T.words(sets, words)
    return c


def call(dev, c, q_len, window=None, varlen=False, **kw):
    from omni_npu_amd import kernels as K
    on = lambda x: None if x is None else x.to(dev)
    out = torch.full(c["q"].shape, float("nan"), dtype=c["dtype"], device=dev)
    lse = torch.full(c["q"].shape[:2], float("nan"), dtype=torch.float32, device=dev)
    K.gqa_tree_decode(on(c["q"]), on(c["k"]), on(c["v"]), on(c["table"]), on(c["lens"]), on(c["visible"]), c["scale"], out, q_len=q_len,
                      query_start_loc=on(c["start"]) if varlen else None, window=window, k_scale=on(c["k_scale"]), v_scale=on(c["v_scale"]),
                      lse_out=lse, **kw)
    torch.cuda.synchronize()
    return out.cpu(), lse.cpu()


def check(c, out, lse, window=0, rows=None):
    """Tolerances as in the chains' tests, and closer: a result is off by its own rounding and by what two operands leave of a probability."""
    k, v = (c[n].float() if c[n].dtype == E4M3 else c[n] for n in ("k", "v"))
    o, l, weight, reach = T.gqa(c["q"], k, v, c["table"], c["lens"], c["visible"], c["scale"], c["start"], window or 0, c["k_scale"], c["v_scale"])
    u, n = H.U[c["dtype"]], max(1, int(c["lens"].max()))
    big = v.float().abs()[torch.isfinite(v.float())].amax() * (1.0 if c["v_scale"] is None else c["v_scale"].max())
    small = n * 2.0 ** -25 * (c["dtype"] == torch.float16)     # (a rest below 2^-14 is rounded by 2^-25, for every key, against a sum of at least one)
    part = 1.01 * u * (2.0 ** -6 + u) + n * 2.0 ** -24 + 2 * (c["d"] + 4) * 2.0 ** -24 * reach[..., None] + 2.0 ** -19
    tol = u * o.abs() + part * (weight + o.abs()) + small * (float(big) + o.abs()) + 1e-30
    err = (out.double() - o).abs()
    if rows is not None:
        o, l, err, tol, out, lse, reach = (x[rows] for x in (o, l, err, tol, out, lse, reach))
    assert (err <= tol).all(), f"worst {(err / tol).max():.3g} of the tolerance"
    assert torch.equal(torch.isinf(lse), torch.isinf(l))
    fine = torch.isfinite(l)
    off = u * 1.01 + (c["d"] + 4) * 2.0 ** -24 * reach + 2.0 ** -18 * (1 + l.abs())
    assert ((lse.double() - l).abs()[fine] <= off[fine]).all()
    assert (out[~fine] == 0).all()


@pytest.mark.parametrize("lens,q_len", [([1], 1), ([8], 8), ([1021], 8), ([13, 64, 65, 700], 13), ([0, 70, 0, 2500], 26), ([60, 61, 95, 96, 97], 60)], ids=str)
@pytest.mark.parametrize("chunks", [0, None, 3, 37])
def test_lengths_and_chunks(dev, lens, q_len, chunks):
    """Trees that are all there is, contexts of one key, requests without keys, trees across tiles of keys and pages."""
    c = tree(make(dev, lens, q_len=q_len, page=16, seed=q_len), seed=len(lens))
    check(c, *call(dev, c, q_len, num_chunks=chunks))


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "fp16"])
@pytest.mark.parametrize("fp8", [False, True], ids=["same", "e4m3"])
@pytest.mark.parametrize("q_len,hq,hk", [(3, 4, 1), (5, 8, 8), (7, 6, 3), (12, 32, 2), (30, 40, 4), (33, 5, 5)])
def test_types_and_head_layouts(dev, d, dtype, fp8, q_len, hq, hk):
    c = tree(make(dev, [77, 401, 130], q_len=q_len, hq=hq, hk=hk, d=d, dtype=dtype, fp8=fp8, page=64, seed=d + hq), seed=d)
    check(c, *call(dev, c, q_len))


@pytest.mark.parametrize("rows", [16, 32, 64, 128])
@pytest.mark.parametrize("q_len,hq,hk", [(1, 8, 2), (17, 2, 2), (40, 12, 3), (64, 16, 2)])
@pytest.mark.parametrize("chunks", [0, 5])
def test_rows_of_a_workgroup(dev, rows, q_len, hq, hk, chunks):
    c = tree(make(dev, [q_len, 300, 64 + q_len - 1, q_len + 1], q_len=q_len, hq=hq, hk=hk, page=48, seed=q_len), seed=rows)
    check(c, *call(dev, c, q_len, num_chunks=chunks, rows_per_group=rows, heads_per_group=1))


@pytest.mark.parametrize("q_len,words", [(64, 2), (65, 2), (100, 2), (129, 3), (300, 5), (512, 8)])
def test_large_trees(dev, q_len, words):
    c = tree(make(dev, [q_len, 700, q_len + 31], q_len=q_len, hq=4, hk=2, d=64, page=16, seed=q_len), seed=1, words=words)
    check(c, *call(dev, c, q_len))


@pytest.mark.parametrize("window", [1, 2, 5, 15, 64, 100, 1000])
@pytest.mark.parametrize("q_len,words", [(1, 1), (9, 1), (70, 2)])
@pytest.mark.parametrize("d,page", [(64, 16), (128, 128), (256, 48)])
def test_windows(dev, window, q_len, words, d, page):
    """Windows that end in the context, at its end, and within the tree: the newest of a token's bits then."""
    c = tree(make(dev, [900, q_len, 64 + q_len, 257, 0], q_len=q_len, hq=8, hk=4, d=d, page=page, seed=window), seed=window, words=words)
    check(c, *call(dev, c, q_len, window=window), window=window)
    check(c, *call(dev, c, q_len, window=window, num_chunks=0), window=window)


@pytest.mark.parametrize("window", [2 ** 31 - 1, 2 ** 31, 2 ** 40, 1024])
def test_a_window_wider_than_any_request(dev, window):
    c = tree(make(dev, [300, 2, 1, 64], q_len=5, hq=8, hk=4, seed=30), seed=3)
    ref, ref_lse = call(dev, c, 5)
    check(c, ref, ref_lse)
    got, lse = call(dev, c, 5, window=window)
    assert torch.equal(got, ref) and torch.equal(lse, ref_lse)


@pytest.mark.parametrize("fp8", [False, True], ids=["same", "e4m3"])
@pytest.mark.parametrize("window", [None, 3, 200])
@pytest.mark.parametrize("q_len,hq,hk", [(1, 4, 2), (6, 8, 2), (33, 12, 3)])
def test_a_chain_is_gqa_decode(dev, fp8, window, q_len, hq, hk):
    """Tokens each behind the other: the masks of gqa_decode, and the same sums in the same order where the launches are alike."""
    c = tree(make(dev, [q_len, 300, 64 + q_len, 700], q_len=q_len, hq=hq, hk=hk, fp8=fp8, page=16, seed=q_len), parents=[i - 1 for i in range(q_len)] * 4)
    for kw in (dict(), dict(num_chunks=0, rows_per_group=16, heads_per_group=1)):
        ref, ref_lse = chain(dev, c, q_len, window=window, **kw)
        got, lse = call(dev, c, q_len, window=window, **kw)
        assert torch.allclose(got.float(), ref.float(), rtol=4 * H.U[c["dtype"]], atol=1e-3) and torch.allclose(lse, ref_lse, atol=1e-4)
    check(c, got, lse, window=window)


@pytest.mark.parametrize("bits", [0, -1, 0x5555555555555555])
def test_bits_that_are_no_tree(dev, bits):
    """None (the context alone, or nothing), all (bits past the request's tokens are not looked at), tokens without their own."""
    c = make(dev, [7, 300, 64, 20], q_len=7, hq=8, hk=2, page=16, seed=5)
    c["visible"] = torch.full((28, 2), bits, dtype=torch.int64)
    for window in (None, 3, 40):
        check(c, *call(dev, c, 7, window=window), window=window)


@pytest.mark.parametrize("chunks", [0, None, 9])
@pytest.mark.parametrize("window", [None, 30])
def test_ragged_requests(dev, chunks, window):
    """One to sixty tokens, none, an idle place; rows behind the last request, and tokens past q_len, stay as they were."""
    counts = [60, 1, 0, 7, 33, 0, 12]
    c = tree(make(dev, [200, 40, 70, 7, 33, 0, 500], q_lens=counts, hq=6, hk=2, d=64, page=16, seed=9), seed=2)
    out, lse = call(dev, c, 60, varlen=True, window=window, num_chunks=chunks)
    check(c, out, lse, window=window)
    wide = dict(c, q=torch.cat((c["q"], torch.randn(5, 6, 64).to(c["dtype"]))), visible=torch.cat((c["visible"], torch.full((5, 1), -1))))
    got, got_lse = call(dev, wide, 60, varlen=True, window=window, num_chunks=chunks)
    assert torch.equal(got[:113], out) and torch.equal(got_lse[:113], lse) and torch.isnan(got[113:]).all() and torch.isnan(got_lse[113:]).all()
    few, few_lse = call(dev, c, 20, varlen=True, window=window, num_chunks=chunks)
    done = torch.cat([torch.arange(n) < 20 for n in counts])
    check(dict(c), few.nan_to_num(0.0), few_lse, window=window, rows=done)
    assert torch.isnan(few[~done]).all()


def test_more_tokens_than_keys(dev):
    """The first tokens' keys would lie in front of the first one: they see nothing, the others what there is."""
    c = tree(make(dev, [3, 1, 10], q_len=12, hq=8, hk=2, d=64, page=16, seed=8), seed=6)
    check(c, *call(dev, c, 12))


@pytest.mark.parametrize("what,fp8", [(float("nan"), False), (float("inf"), False), (-float("inf"), False), (float("nan"), True)], ids=str)
@pytest.mark.parametrize("chunks", [0, 6])
@pytest.mark.parametrize("q_len,hq,hk,rows", [(9, 8, 2, None), (9, 16, 1, 16), (5, 4, 2, 64), (33, 4, 4, 32)])
def test_what_a_token_does_not_see_does_not_reach_it(dev, what, fp8, chunks, q_len, hq, hk, rows):
    """Pages' free rows, and tokens that are not among a token's ancestors: their keys and values hold what is no number."""
    c = tree(make(dev, [q_len, 150, 64 + q_len], q_len=q_len, hq=hq, hk=hk, d=64, fp8=fp8, page=16, seed=q_len), seed=4)
    bad = 3 % q_len
    sees = torch.tensor([c["visible"][t, 0].item() >> bad & 1 for t in range(3 * q_len)], dtype=torch.bool)
    assert 0 < sees.sum() < 3 * q_len
    used = torch.zeros(c["k"].shape[:2], dtype=torch.bool)
    for b, n in enumerate(c["lens"].tolist()):
        pos = torch.arange(n)
        used[c["table"][b].long()[pos // 16], pos % 16] = True
    for name in ("k", "v"):
        x = c[name].float()
        x[~used] = what
        for b, n in enumerate(c["lens"].tolist()):
            at = n - q_len + bad
            x[c["table"][b, at // 16].long(), at % 16] = what
        c[name] = x.to(c[name].dtype)
    check(c, *call(dev, c, q_len, num_chunks=chunks, rows_per_group=rows), rows=~sees)


def test_views_of_wider_tensors(dev):
    from omni_npu_amd import kernels as K
    c = tree(make(dev, [300, 77, 640], q_len=6, hq=12, hk=4, d=128, page=64, seed=42), seed=7)
    ref, ref_lse = call(dev, c, 6)
    check(c, ref, ref_lse)
    on = {n: c[n].to(dev) for n in ("q", "k", "v", "table", "lens", "visible")}
    wide_q = torch.full((18, 12 + 8, 128), float("nan"), dtype=c["dtype"], device=dev)
    wide_q[:, :12] = on["q"]
    wide_out = torch.full((18, 2, 14, 128), 7.0, dtype=c["dtype"], device=dev)
    table = torch.full((5, on["table"].shape[1] + 9), -3, dtype=torch.int32, device=dev)
    table[:3, :on["table"].shape[1]] = on["table"]
    bits = torch.full((18, 5), -1, dtype=torch.int64, device=dev)
    bits[:, 2:3] = on["visible"]
    bits[:, 3] = 0
    for view in (bits[:, 2:3], bits[:, 2:4]):
        for chunks in (None, 0, 6):
            wide_out.fill_(7.0)
            K.gqa_tree_decode(wide_q[:, :12], on["k"], on["v"], table[:, :on["table"].shape[1]], on["lens"], view, c["scale"], wide_out[:, 1, 1:13], q_len=6,
                              num_chunks=chunks)
            got = wide_out.cpu()
            check(c, got[:, 1, 1:13], ref_lse)
            got[:, 1, 1:13] = 7.0
            assert (got == 7.0).all()


@pytest.mark.parametrize("batch", [65, 300])
@pytest.mark.parametrize("chunks", [0, 1, 50, 300])
def test_many_requests(dev, batch, chunks):
    g = torch.Generator().manual_seed(batch)
    lens = [int(n) for n in torch.randint(0, 90, (batch,), generator=g)]
    lens[0], lens[-1], lens[batch // 2] = 0, 0, 400
    c = tree(make(dev, lens, q_len=4, hq=4, hk=2, d=64, page=16, seed=batch), seed=batch)
    check(c, *call(dev, c, 4, num_chunks=chunks))


def test_the_general_path_and_a_workspace_of_the_callers(dev):
    """What the native side leaves to it, with the same results; a workspace that is too small is refused."""
    from omni_npu_amd import kernels as K
    c = tree(make(dev, [300, 700, 64], q_len=5, hq=8, hk=2, seed=1), seed=1)
    ref, ref_lse = call(dev, c, 5, num_chunks=9)
    need = K._lib.load().mlahip_gqa_decode_workspace_bytes(3, 5, 8, 128, 9)
    ws = torch.empty(need, dtype=torch.uint8, device=dev)
    got, lse = call(dev, c, 5, num_chunks=9, workspace=ws)
    assert torch.equal(got, ref) and torch.equal(lse, ref_lse)
    with pytest.raises(K._lib.MlaHipError):
        call(dev, c, 5, num_chunks=9, workspace=ws[:need - 16])


def test_refusals(dev):
    from omni_npu_amd import kernels as K
    c = tree(make(dev, [30, 70], q_len=5, hq=8, hk=2, seed=1), seed=1)
    v = c["visible"]
    for bad in (v[:-1], v.to(torch.int32), v[:, 0], v.expand(-1, 9), v.view(2, 5).t(), v.view(5, 2)):
        with pytest.raises(ValueError, match="visible"):
            call(dev, dict(c, visible=bad), 5)
    with pytest.raises(ValueError, match="hold no bits"):
        call(dev, dict(c, visible=torch.zeros(130, 1, dtype=torch.int64), q=torch.zeros(130, 8, 128, dtype=torch.bfloat16)), 65)
    q = torch.zeros(10, 8, 128, dtype=torch.bfloat16, device=dev, requires_grad=True)
    with pytest.raises(RuntimeError, match="no backward"):
        K.gqa_tree_decode(q, c["k"].to(dev), c["v"].to(dev), c["table"].to(dev), c["lens"].to(dev), v.to(dev), 0.1, torch.empty_like(q), q_len=5)
