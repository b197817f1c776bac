"""Attention over a paged cache of ordinary key and value heads against its plain statement in 64 bits: head layouts, types, lengths from
nothing to several chunks, windows, masked places that hold infinities and NaN, strides, graphs."""
import math

import pytest
import torch

from oracle import heads_oracle as H

pytestmark = pytest.mark.gpu

E4M3 = torch.float8_e4m3fn


def make(dev, lens, q_len=1, hq=8, hk=2, d=128, dtype=torch.bfloat16, fp8=False, page=128, seed=0, q_lens=None, blocks=None, gain=1.0):
    g = torch.Generator().manual_seed(seed)
    b = len(lens)
    per = [-(-max(n, 0) // page) for n in lens]
    pages = sum(per) + 2
    table = torch.zeros(b, blocks or max(max(per), 1) + 1, dtype=torch.int32)
    order, at = torch.randperm(pages, generator=g).to(torch.int32), 0
    for i, n in enumerate(per):
        n = min(n, table.shape[1])
        table[i, :n] = order[at:at + n]
        at += n
    counts = q_lens or [q_len] * b
    start = torch.tensor([0] + counts).cumsum(0).to(torch.int32)
    c = dict(q=(torch.randn(int(start[-1]), hq, d, generator=g) * gain).to(dtype), table=table,
             lens=torch.tensor(lens, dtype=torch.int32), start=start, k_scale=None, v_scale=None, scale=d ** -0.5, d=d, dtype=dtype)
    for name in ("k", "v"):
        x = torch.randn(pages, page, hk, d, generator=g)
        if fp8:
            c[name] = (x * 30).clamp(-448, 448).to(E4M3)
            c[name + "_scale"] = 0.02 + 0.02 * torch.rand(hk, generator=g)
        else:
            c[name] = x.to(dtype)
    return c


def call(dev, c, q_len, window=None, varlen=False, **kw):
    from omni_npu_amd import kernels as K
    on = lambda x: None if x is None else x.to(dev)
    out = torch.full(c["q"].shape, float("nan"), dtype=c["dtype"], device=dev)
    lse = torch.full(c["q"].shape[:2], float("nan"), dtype=torch.float32, device=dev)
    K.gqa_decode(on(c["q"]), on(c["k"]), on(c["v"]), on(c["table"]), on(c["lens"]), c["scale"], out, q_len=q_len,
                 query_start_loc=on(c["start"]) if varlen else None, window=window, k_scale=on(c["k_scale"]), v_scale=on(c["v_scale"]),
                 lse_out=lse, **kw)
    torch.cuda.synchronize()
    return out.cpu(), lse.cpu()


def check(c, out, lse, window=0, rows=None):
    k, v = (c[n].float() if c[n].dtype == E4M3 else c[n] for n in ("k", "v"))
    o, l, weight, reach = H.gqa(c["q"], k, v, c["table"], c["lens"], c["scale"], c["start"], window or 0, c["k_scale"], c["v_scale"])
    tol = H.gqa_tolerance(o, weight, reach, c["dtype"], c["d"])
    err = (out.double() - o).abs()
    assert (err <= tol).all(), f"worst {(err / tol).max():.3g} of the tolerance"
    assert torch.equal(torch.isinf(lse), torch.isinf(l))
    fine = torch.isfinite(l)
    # the rounded probabilities' sum is off by u at most, the scores as in the result; the sum's own roundings stay below 2^-18
    off = H.U[c["dtype"]] * 1.01 + (c["d"] + 4) * 2.0 ** -24 * reach + 2.0 ** -18 * (1 + l.abs())
    assert ((lse.double() - l).abs()[fine] <= off[fine]).all()
    assert (out[~fine] == 0).all()


LENS = [[1], [2, 17, 64], [1021], [63, 64, 65, 128, 129, 700], [2500, 1, 33], [0, 5, 0, 260]]


@pytest.mark.parametrize("lens", LENS, ids=str)
@pytest.mark.parametrize("chunks", [0, None, 3, 37])
def test_lengths_and_chunks(dev, lens, chunks):
    c = make(dev, lens, seed=len(lens))
    check(c, *call(dev, c, 1, num_chunks=chunks))


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "fp16"])
@pytest.mark.parametrize("fp8", [False, True], ids=["same", "e4m3"])
@pytest.mark.parametrize("hq,hk", [(4, 1), (8, 8), (6, 3), (32, 2), (40, 4), (5, 5)])
def test_types_and_head_layouts(dev, d, dtype, fp8, hq, hk):
    c = make(dev, [77, 401, 130], hq=hq, hk=hk, d=d, dtype=dtype, fp8=fp8, page=64, seed=d + hq)
    check(c, *call(dev, c, 1))


@pytest.mark.parametrize("q_len,hq,hk", [(2, 8, 2), (3, 8, 8), (4, 20, 4), (5, 32, 2), (17, 12, 3)])
@pytest.mark.parametrize("fp8", [False, True], ids=["same", "e4m3"])
@pytest.mark.parametrize("chunks", [0, None, 11])
def test_several_tokens(dev, q_len, hq, hk, fp8, chunks):
    c = make(dev, [q_len, 300, 64 + q_len - 1, 1], q_len=q_len, hq=hq, hk=hk, fp8=fp8, page=16, seed=q_len)
    check(c, *call(dev, c, q_len, num_chunks=chunks))


@pytest.mark.parametrize("window", [1, 15, 64, 100, 1000])
@pytest.mark.parametrize("q_len", [1, 3])
@pytest.mark.parametrize("d,page", [(64, 16), (128, 128), (256, 48)])
def test_windows(dev, window, q_len, d, page):
    c = make(dev, [900, 3, 64, 257, 0], q_len=q_len, hq=8, hk=4, d=d, page=page, seed=window)
    check(c, *call(dev, c, q_len, window=window), window=window)


@pytest.mark.parametrize("window", [2 ** 31 - 1, 2 ** 31, 2 ** 40, 1024])
def test_a_window_wider_than_any_request(dev, window):
    """No window then, with requests of fewer keys than tokens too."""
    c = make(dev, [300, 2, 1, 64], q_len=5, hq=8, hk=4, seed=30)
    ref, ref_lse = call(dev, c, 5)
    check(c, ref, ref_lse)
    got, lse = call(dev, c, 5, window=window)
    assert torch.equal(got, ref) and torch.equal(lse, ref_lse)


@pytest.mark.parametrize("chunks", [0, 6])
def test_infinite_and_undefined_scores(dev, chunks):
    """Scores of -inf weigh nothing wherever they come; one of +inf or NaN makes its row undefined, and no other row."""
    c = make(dev, [400, 130], hq=4, hk=2, d=64, page=16, seed=31)
    c["q"][...] = c["q"].abs() + 0.5
    page = lambda b, key: (c["table"][b, key // 16], key % 16)
    plain, plain_lse = call(dev, c, 1, num_chunks=chunks)
    check(c, plain, plain_lse)
    gone = [0, 1, *range(32, 64), 200, 399]                  # (a whole step of keys among them)
    kept = torch.tensor([i for i in range(400) if i not in gone])
    few = dict(c, table=torch.arange(26, dtype=torch.int32)[None], lens=torch.tensor([len(kept)], dtype=torch.int32), q=c["q"][:1],
               start=torch.tensor([0, 1]))
    for n in ("k", "v"):                                     # the request without them
        rows = c[n][c["table"][0].long()[kept // 16], kept % 16]
        few[n] = torch.cat([rows, torch.zeros(416 - len(kept), 2, 64, dtype=rows.dtype)]).view(26, 16, 2, 64)
    for key in gone:
        c["k"][page(0, key)][0] = -float("inf")
    ref, ref_lse = call(dev, c, 1, num_chunks=chunks)
    o, l, weight, reach = H.gqa(few["q"], few["k"], few["v"], few["table"], few["lens"], few["scale"], few["start"])
    assert ((ref[0, :2].double() - o[0, :2]).abs() <= H.gqa_tolerance(o, weight, reach, c["dtype"], 64)[0, :2]).all()
    assert torch.equal(ref[0, 2:], plain[0, 2:]) and torch.equal(ref[1], plain[1]) and torch.equal(ref_lse[1], plain_lse[1])
    for bad in (float("inf"), float("nan")):
        was = c["k"][page(0, 150)][1, 3].clone()
        c["k"][page(0, 150)][1, 3] = bad
        out, lse = call(dev, c, 1, num_chunks=chunks)
        c["k"][page(0, 150)][1, 3] = was
        assert torch.isnan(out[0, 2:].float()).all() and torch.isnan(lse[0, 2:]).all()
        out[0, 2:], lse[0, 2:] = ref[0, 2:], ref_lse[0, 2:]
        assert torch.equal(out, ref) and torch.equal(lse, ref_lse)
    q = c["q"].clone()
    c["q"][1, 0, 5] = float("nan")
    out, lse = call(dev, c, 1, num_chunks=chunks)
    assert torch.isnan(out[1, 0].float()).all() and torch.isnan(lse[1, 0])
    c["q"] = q
    out[1, 0], lse[1, 0] = ref[1, 0], ref_lse[1, 0]
    assert torch.equal(out, ref) and torch.equal(lse, ref_lse)
    c["k"][c["table"][1].long()[:9], :, 0] = -float("inf")    # every score of a row
    out, lse = call(dev, c, 1, num_chunks=chunks)
    assert (out[1, :2] == 0).all() and (lse[1, :2] == -float("inf")).all() and torch.equal(out[1, 2:], ref[1, 2:])


@pytest.mark.parametrize("scale", [-0.2, 0.0, 3.0])
@pytest.mark.parametrize("fp8", [False, True], ids=["same", "e4m3"])
def test_scales_of_any_sign(dev, scale, fp8):
    c = make(dev, [500, 33], q_len=2, hq=6, hk=2, d=128, fp8=fp8, seed=32)
    c["scale"] = scale
    check(c, *call(dev, c, 2))


def test_ragged_token_counts(dev):
    c = make(dev, [300, 40, 7, 0, 129], q_lens=[1, 4, 0, 2, 3], hq=12, hk=4, seed=3)
    for chunks in (None, 0, 9):
        check(c, *call(dev, c, 4, varlen=True, num_chunks=chunks))


def test_a_row_without_a_key_is_zero(dev):
    """More tokens than keys: the first ones see nothing."""
    c = make(dev, [2, 1, 0, 3], q_len=3, hq=4, hk=2, seed=4)
    out, lse = call(dev, c, 3)
    check(c, out, lse)
    assert (out[0] == 0).all() and torch.isinf(lse[0]).all() and (out[6:9] == 0).all()


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("q_len,window", [(1, None), (2, None), (1, 40), (3, 40)])
@pytest.mark.parametrize("fp8", [False, True], ids=["same", "e4m3"])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_what_lies_in_masked_places_does_not_matter(dev, bad, q_len, window, fp8, d):
    """Behind a request's last key, in front of its window and in pages of nobody there may be anything; a later token's key may be
    infinite without a trace in an earlier token's row."""
    c = make(dev, [200, 33, 130], q_len=q_len, hq=6, hk=2, d=d, fp8=fp8, page=32, seed=q_len)
    fill = torch.tensor(bad).to(E4M3) if fp8 else bad
    ref, ref_lse = call(dev, c, q_len, window=window)
    used = torch.zeros(c["k"].shape[:2], dtype=torch.bool)
    for b, n in enumerate(c["lens"].tolist()):
        first = max(0, n - q_len + 1 - window) if window else 0
        for j in range(first, n):
            used[c["table"][b, j // 32], j % 32] = True
    for name in ("k", "v"):
        x = c[name].view(torch.uint8) if fp8 else c[name]
        x[~used] = fill.view(torch.uint8) if fp8 else fill
    got, got_lse = call(dev, c, q_len, window=window)
    assert torch.equal(got, ref) and torch.equal(got_lse, ref_lse)
    if q_len > 1:                                             # the newest token's key and value: seen by the last row of a request only
        for b, n in enumerate(c["lens"].tolist()):
            for name in ("k", "v"):
                x = c[name].view(torch.uint8) if fp8 else c[name]
                x[c["table"][b, (n - 1) // 32], (n - 1) % 32] = fill.view(torch.uint8) if fp8 else fill
        got, got_lse = call(dev, c, q_len, window=window)
        old = torch.arange(got.shape[0]) % q_len != q_len - 1
        assert torch.equal(got[old], ref[old]) and torch.equal(got_lse[old], ref_lse[old])
        if not fp8 or bad != bad:
            assert not torch.isfinite(got[~old].float()).all()


@pytest.mark.parametrize("chunks,heads", [(0, 1), (0, 2), (3, 2)])
def test_a_long_piece_is_begun_again_from_its_first_page(dev, chunks, heads):
    """More pages than a wavefront holds numbers of, and an infinity that the newest token alone sees."""
    c = make(dev, [9000, 4000], q_len=2, hq=6, hk=2, page=16, seed=13)
    kw = dict(num_chunks=chunks, heads_per_group=heads)
    ref, ref_lse = call(dev, c, 2, **kw)
    check(c, ref, ref_lse)
    for b, n in enumerate(c["lens"].tolist()):
        c["v"][c["table"][b, (n - 1) // 16], (n - 1) % 16] = float("inf")
    got, lse = call(dev, c, 2, **kw)
    assert torch.equal(got[0::2], ref[0::2]) and torch.equal(lse, ref_lse) and torch.isinf(got[1::2].float()).all()


def test_first_call_of_a_kernel_under_capture(dev):
    """A graph may be captured from a shape that has not run before."""
    from omni_npu_amd import kernels as K
    c = make(dev, [500, 90], q_len=5, hq=26, hk=2, d=64, dtype=torch.float16, fp8=True, seed=14)
    on = {n: c[n].to(dev) for n in ("q", "k", "v", "table", "lens", "k_scale", "v_scale")}
    out = torch.zeros_like(on["q"])
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        K._workspace(dev, 1 << 26, "gqa")
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            K.gqa_decode(on["q"], on["k"], on["v"], on["table"], on["lens"], c["scale"], out, q_len=5, k_scale=on["k_scale"],
                         v_scale=on["v_scale"], rows_per_group=64)
        for _ in range(2):
            out.fill_(float("nan"))
            graph.replay()
            torch.cuda.synchronize()
            ref, _ = call(dev, c, 5, rows_per_group=64, num_chunks=0)
            o, _, weight, reach = H.gqa(c["q"], c["k"].float(), c["v"].float(), c["table"], c["lens"], c["scale"], c["start"], 0, c["k_scale"],
                                        c["v_scale"])
            tol = H.gqa_tolerance(o, weight, reach, c["dtype"], 64)
            assert ((out.cpu().double() - o).abs() <= tol).all() and ((ref.double() - o).abs() <= tol).all()
    torch.cuda.current_stream().wait_stream(side)


@pytest.mark.parametrize("rows", [16, 32, 64])
@pytest.mark.parametrize("heads", [1, 2, 4, 8])
@pytest.mark.parametrize("d,fp8", [(64, False), (64, True), (128, False), (128, True), (256, False), (256, True)])
def test_every_form_of_a_workgroup(dev, rows, heads, d, fp8):
    """Heads and rows of a workgroup as a caller asks for them: the same attention; what does not fit is refused."""
    from omni_npu_amd import _lib
    c = make(dev, [300, 47, 900], q_len=3, hq=88, hk=8, d=d, fp8=fp8, page=32, seed=rows + heads)
    waves = 4 if d == 256 or rows == 64 or rows == 32 and d == 128 and not fp8 else 8
    kw = dict(num_chunks=5, heads_per_group=heads, rows_per_group=rows)
    if heads > waves or rows == 64 and d == 256:
        with pytest.raises(_lib.MlaHipError, match="to a workgroup"):
            call(dev, c, 3, **kw)
        return
    check(c, *call(dev, c, 3, **kw))
    check(c, *call(dev, c, 3, **dict(kw, num_chunks=0)))


def test_scores_that_outgrow_each_other(dev):
    """Keys of growing length: a row's reference is replaced again and again; and queries so large that one key takes everything."""
    c = make(dev, [1500, 700], hq=4, hk=2, seed=9)
    c["k"] = (c["k"].float() * torch.linspace(0.1, 3, c["k"].shape[1])[None, :, None, None]).to(c["dtype"])
    check(c, *call(dev, c, 1, num_chunks=5))
    c = make(dev, [1500, 700], hq=4, hk=2, seed=10, gain=30.0)
    check(c, *call(dev, c, 1, num_chunks=5))


def test_strides_of_interleaved_and_head_major_caches(dev):
    """Keys and values side by side in one allocation, head-major pages, q and out as views: the same bits as dense tensors."""
    from omni_npu_amd import kernels as K
    c = make(dev, [300, 90], hq=8, hk=2, page=32, seed=5)
    ref, _ = call(dev, c, 1)
    pages = c["k"].shape[0]
    both = torch.stack((c["k"], c["v"]), dim=3).to(dev)                       # [pages, page, hk, 2, d]
    major = torch.stack((c["k"], c["v"])).permute(1, 0, 3, 2, 4).contiguous().to(dev)   # [pages, 2, hk, page, d]
    for k, v in ((both[:, :, :, 0], both[:, :, :, 1]), (major[:, 0].transpose(1, 2), major[:, 1].transpose(1, 2))):
        assert k.shape == (pages, 32, 2, 128)
        wide = torch.zeros(2, 20, 128, dtype=c["dtype"], device=dev)
        wide[:, 4:12] = c["q"].to(dev)
        out = torch.full((8, 2, 136), float("nan"), dtype=c["dtype"], device=dev)
        view = out.transpose(0, 1)[..., :128]
        K.gqa_decode(wide[:, 4:12], k, v, c["table"].to(dev), c["lens"].to(dev), c["scale"], view)
        assert torch.equal(view.cpu(), ref)
        assert torch.isnan(out[..., 128:].float()).all()


def test_page_numbers_outside_the_cache_and_lengths_beyond_the_table(dev):
    """Read as the cache's first or last page; a length beyond the table's room counts as the room."""
    c = make(dev, [300, 256], page=64, seed=6, blocks=5)
    c["lens"][1] = 5000
    c["table"][1] = torch.tensor([1, 2, 3, 1, 2])
    ref = dict(c, table=c["table"].clone())
    ref["table"][0, 1], ref["table"][0, 2] = 0, c["k"].shape[0] - 1
    c["table"][0, 1], c["table"][0, 2] = -7, 1 << 30
    out, lse = call(dev, c, 1)
    check(ref, out, lse)


def test_rows_behind_the_batch_stay(dev):
    """query_start_loc that covers fewer tokens than q has: the others' results are left as they were."""
    from omni_npu_amd import kernels as K
    c = make(dev, [100, 50], q_lens=[2, 1], seed=7)
    q = torch.cat((c["q"], torch.full((3, 8, 128), float("nan"), dtype=c["dtype"]))).to(dev)
    out = torch.full(q.shape, 7.0, dtype=c["dtype"], device=dev)
    K.gqa_decode(q, c["k"].to(dev), c["v"].to(dev), c["table"].to(dev), c["lens"].to(dev), c["scale"], out, q_len=2,
                 query_start_loc=c["start"].to(dev))
    ref, lse = call(dev, c, 2, varlen=True)
    check(c, ref, lse)
    assert torch.equal(out[:3].cpu(), ref) and (out[3:] == 7).all()


def test_replays_follow_lengths_and_tables(dev):
    """A captured call replayed over other lengths, with eager work between; a larger eager call on the same stream does not take its
    scratch away."""
    from omni_npu_amd import kernels as K
    c = make(dev, [700, 64, 1300, 5], seed=8, hq=16, hk=4)
    q, k, v, table, lens = (c[n].to(dev) for n in ("q", "k", "v", "table", "lens"))
    out = torch.zeros_like(q)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        K.gqa_decode(q, k, v, table, lens, c["scale"], out)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            K.gqa_decode(q, k, v, table, lens, c["scale"], out)
        big = make(dev, [900] * 40, seed=2)
        for now in ([700, 64, 1300, 5], [1, 0, 1250, 384], [1408, 128, 3, 0], [700, 64, 1300, 5]):
            now = [min(n, 128 * int(table.shape[1])) for n in now]
            c["lens"] = torch.tensor(now, dtype=torch.int32)
            lens.copy_(c["lens"])
            out.fill_(float("nan"))
            graph.replay()
            torch.cuda.synchronize()
            got = out.cpu()
            o, l, weight, reach = H.gqa(c["q"], c["k"], c["v"], c["table"], c["lens"], c["scale"], c["start"])
            assert ((got.double() - o).abs() <= H.gqa_tolerance(o, weight, reach, c["dtype"], 128)).all()
            call(dev, big, 1)
            eager = torch.full_like(q, float("nan"))
            K.gqa_decode(q, k, v, table, lens, c["scale"], eager)
            torch.cuda.synchronize()
            assert torch.equal(eager, out)
    torch.cuda.current_stream().wait_stream(side)


def test_same_bits_every_time(dev):
    c = make(dev, [3000, 100, 1700], hq=32, hk=8, seed=11)
    first = call(dev, c, 1)
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(first, call(dev, c, 1)))


def test_a_caller_s_workspace(dev):
    from omni_npu_amd import _lib
    c = make(dev, [1000, 600], seed=12)
    ref = call(dev, c, 1, num_chunks=6)
    need = _lib.load().mlahip_gqa_decode_workspace_bytes(2, 1, 8, 128, 6)
    got = call(dev, c, 1, num_chunks=6, workspace=torch.empty(need, dtype=torch.uint8, device=dev))
    assert all(torch.equal(a, b) for a, b in zip(ref, got))
    with pytest.raises(_lib.MlaHipError, match="workspace"):
        call(dev, c, 1, num_chunks=6, workspace=torch.empty(need - 1, dtype=torch.uint8, device=dev))


def test_refusals(dev):
    from omni_npu_amd import kernels as K
    c = make(dev, [100, 50])
    on = {n: c[n].to(dev) for n in ("q", "k", "v", "table", "lens")}
    good = (on["q"], on["k"], on["v"], on["table"], on["lens"], c["scale"], torch.empty_like(on["q"]))

    def refused(err, match, swap, **kw):
        args = list(good)
        for i, x in swap.items():
            args[i] = x
        with pytest.raises(err, match=match):
            K.gqa_decode(*args, **kw)

    refused(ValueError, "bf16 or fp16", {0: on["q"].float()})
    refused(ValueError, "q and out", {6: torch.empty(2, 8, 64, dtype=torch.bfloat16, device=dev)})
    refused(TypeError, "like the queries", {1: on["k"].half()})
    refused(ValueError, "agree", {2: on["v"][:-1]})
    refused(ValueError, "query heads", {0: on["q"][:, :7], 6: torch.empty_like(on["q"][:, :7])})
    refused(ValueError, "window", {}, window=0)
    refused(ValueError, "q_len", {}, q_len=0)
    refused(ValueError, "q_len", {}, q_len=(1 << 32) + 1, query_start_loc=torch.zeros(3, dtype=torch.int32, device=dev))
    for name in ("num_chunks", "heads_per_group", "rows_per_group", "max_seq_len"):
        refused(ValueError, name, {}, **{name: -1})
        if name != "max_seq_len":
            refused(ValueError, name, {}, **{name: 1 << 32})
    refused(ValueError, "query tokens", {}, q_len=2)
    refused(ValueError, "seq_lens", {4: on["lens"].long()})
    refused(ValueError, "block_table", {3: on["table"][:1]})
    refused(ValueError, "query_start_loc", {}, query_start_loc=torch.zeros(2, dtype=torch.int32, device=dev))
    refused(ValueError, "lse_out", {}, lse_out=torch.empty(2, 8, dtype=torch.float16, device=dev))
    refused(ValueError, "goes with a float8", {}, k_scale=torch.ones(2, device=dev))
    refused(ValueError, "no CPU path", {3: c["table"]})
    refused(RuntimeError, "no backward", {0: on["q"].clone().requires_grad_()})
    refused(K._lib.MlaHipError, "64, 128 or 256", {i: good[i][..., :96] for i in (0, 1, 2, 6)})
    refused(K._lib.MlaHipError, "multiple of 16", {1: on["k"][:, :24], 2: on["v"][:, :24]})
    q = torch.zeros(2 * 8 * 128 + 1, dtype=torch.bfloat16, device=dev)[1:].view(2, 8, 128)
    refused(K._lib.MlaHipError, "16-byte aligned", {0: q})


def test_no_tokens(dev):
    from omni_npu_amd import kernels as K
    c = make(dev, [5])
    none = torch.empty(0, 8, 128, dtype=torch.bfloat16, device=dev)
    K.gqa_decode(none, c["k"].to(dev), c["v"].to(dev), c["table"].to(dev), c["lens"].to(dev)[:0], 1.0, none)
    K.gqa_decode(none, c["k"].to(dev), c["v"].to(dev), c["table"].to(dev), c["lens"].to(dev), 1.0, none,
                 query_start_loc=torch.zeros(2, dtype=torch.int32, device=dev))
