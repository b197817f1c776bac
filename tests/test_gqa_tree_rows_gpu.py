"""Attention of drafted trees with 128 rows to a workgroup, whatever the rule would choose, and with what it chooses: against the plain statement in 64 bits."""
import pytest
import torch

from oracle import tree_oracle as T
from tests.test_gqa_decode_gpu import make
from tests.test_gqa_tree_gpu import call, check, tree

pytestmark = pytest.mark.gpu

WIDE = dict(rows_per_group=128, heads_per_group=1)


@pytest.mark.parametrize("lens,q_len", [([1], 1), ([8], 8), ([31], 8), ([1021], 8), ([13, 64, 65, 700], 13), ([0, 70, 0, 2500], 26),
                                        ([60, 61, 95, 96, 97], 60)], ids=str)
@pytest.mark.parametrize("chunks", [0, 3, 37])
def test_lengths_and_chunks(dev, lens, q_len, chunks):
    """Fewer tiles than the pipeline is deep, pieces of one tile, requests without keys."""
    c = tree(make(dev, lens, q_len=q_len, page=16, seed=q_len), seed=len(lens))
    check(c, *call(dev, c, q_len, num_chunks=chunks, **WIDE))


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "fp16"])
@pytest.mark.parametrize("fp8", [False, True], ids=["same", "e4m3"])
@pytest.mark.parametrize("q_len,hq,hk,page", [(3, 4, 1, 16), (5, 8, 8, 64), (7, 6, 3, 48), (12, 32, 2, 128), (30, 40, 4, 80), (33, 5, 5, 32), (64, 28, 4, 16)])
def test_types_and_head_layouts(dev, d, dtype, fp8, q_len, hq, hk, page):
    c = tree(make(dev, [77, 401, 130], q_len=q_len, hq=hq, hk=hk, d=d, dtype=dtype, fp8=fp8, page=page, seed=d + hq), seed=d)
    for chunks in (0, 11):
        check(c, *call(dev, c, q_len, num_chunks=chunks, **WIDE))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "fp16"])
@pytest.mark.parametrize("gain", [0.0, 12.0, -12.0])
def test_scores_that_grow(dev, dtype, gain):
    """Scores that outgrow their rows' references again and again, at places that differ from row to row, and equal ones."""
    c = tree(make(dev, [600, 333], q_len=20, hq=8, hk=1, d=64, dtype=dtype, page=16, seed=3, gain=abs(gain)), seed=3)
    for b, n in enumerate(c["lens"].tolist()):                 # (the largest last, or first)
        size = torch.linspace(0.05, 1.0, n) if gain > 0 else torch.linspace(1.0, 0.05, n)
        at = torch.arange(n)
        rows = c["table"][b].long()[at // 16], at % 16
        c["k"][rows] = (c["k"][rows].float() * size[:, None, None]).to(dtype)
    for chunks in (0, 5):
        check(c, *call(dev, c, 20, num_chunks=chunks, **WIDE))


@pytest.mark.parametrize("q_len,words", [(64, 2), (65, 2), (129, 3), (300, 5), (512, 8)])
@pytest.mark.parametrize("d,hq", [(64, 4), (128, 6), (256, 2)])
def test_large_trees(dev, q_len, words, d, hq):
    """Several groups of rows, tokens that are shared by two, trees over many tiles."""
    c = tree(make(dev, [q_len, 700, q_len + 31], q_len=q_len, hq=hq, hk=2, d=d, page=16, seed=q_len), seed=1, words=words)
    check(c, *call(dev, c, q_len, num_chunks=0, **WIDE))
    check(c, *call(dev, c, q_len, num_chunks=13, **WIDE))


@pytest.mark.parametrize("window", [1, 2, 5, 15, 64, 100, 1000, 2 ** 31])
@pytest.mark.parametrize("q_len,words", [(1, 1), (9, 1), (70, 2)])
@pytest.mark.parametrize("d,page,fp8", [(64, 16, False), (128, 128, True), (128, 48, False), (256, 16, False), (256, 64, True)])
def test_windows(dev, window, q_len, words, d, page, fp8):
    c = tree(make(dev, [900, q_len, 64 + q_len, 257, 0], q_len=q_len, hq=8, hk=4, d=d, page=page, fp8=fp8, seed=window % 1001), seed=window % 1001, words=words)
    for chunks in (0, 7):
        check(c, *call(dev, c, q_len, window=window, num_chunks=chunks, **WIDE), window=window if window < 2 ** 30 else 0)


@pytest.mark.parametrize("bits", [0, -1, 0x5555555555555555])
def test_bits_that_are_no_tree(dev, bits):
    c = make(dev, [7, 300, 64, 20], q_len=7, hq=8, hk=2, page=16, seed=5)
    c["visible"] = torch.full((28, 2), bits, dtype=torch.int64)
    for window in (None, 3, 40):
        check(c, *call(dev, c, 7, window=window, **WIDE), window=window)


@pytest.mark.parametrize("chunks", [0, 9])
@pytest.mark.parametrize("window", [None, 30])
def test_ragged_requests(dev, chunks, window):
    """One to sixty tokens, none, an idle place; rows behind the last request, and tokens past q_len, stay as they were."""
    counts = [60, 1, 0, 7, 33, 0, 12]
    c = tree(make(dev, [200, 40, 70, 7, 33, 0, 500], q_lens=counts, hq=6, hk=2, d=64, page=16, seed=9), seed=2)
    out, lse = call(dev, c, 60, varlen=True, window=window, num_chunks=chunks, **WIDE)
    check(c, out, lse, window=window)
    more = dict(c, q=torch.cat((c["q"], torch.randn(5, 6, 64).to(c["dtype"]))), visible=torch.cat((c["visible"], torch.full((5, 1), -1))))
    got, got_lse = call(dev, more, 60, varlen=True, window=window, num_chunks=chunks, **WIDE)
    assert torch.equal(got[:113], out) and torch.equal(got_lse[:113], lse) and torch.isnan(got[113:]).all() and torch.isnan(got_lse[113:]).all()
    few, few_lse = call(dev, c, 20, varlen=True, window=window, num_chunks=chunks, **WIDE)
    done = torch.cat([torch.arange(n) < 20 for n in counts])
    check(dict(c), few.nan_to_num(0.0), few_lse, window=window, rows=done)
    assert torch.isnan(few[~done]).all()


def test_more_tokens_than_keys(dev):
    c = tree(make(dev, [3, 1, 10], q_len=12, hq=8, hk=2, d=64, page=16, seed=8), seed=6)
    check(c, *call(dev, c, 12, **WIDE))


@pytest.mark.parametrize("what,fp8", [(float("nan"), False), (float("inf"), False), (-float("inf"), False), (float("nan"), True)], ids=str)
@pytest.mark.parametrize("chunks", [0, 6])
@pytest.mark.parametrize("q_len,hq,hk,d", [(9, 8, 2, 64), (33, 16, 4, 128), (50, 32, 2, 64), (20, 16, 2, 256)])
def test_what_a_token_does_not_see_does_not_reach_it(dev, what, fp8, chunks, q_len, hq, hk, d):
    """Pages' free rows, and tokens that are not among a token's ancestors: their keys and values hold what is no number."""
    c = tree(make(dev, [q_len, 150, 64 + q_len], q_len=q_len, hq=hq, hk=hk, d=d, fp8=fp8, page=16, seed=q_len), seed=4)
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
    check(c, *call(dev, c, q_len, num_chunks=chunks, **WIDE), rows=~sees)


@pytest.mark.parametrize("rows", [16, 32, 64, 128])
@pytest.mark.parametrize("where", ["context", "behind"])
@pytest.mark.parametrize("which", ["k", "v"])
def test_a_window_that_ends_at_different_keys(dev, rows, where, which):
    """Tokens deeper in a tree see fewer keys of the context: one at the window's end, no number, reaches those that see it and no others."""
    q_len, window = 10, 40
    c = tree(make(dev, [97, 150, 46], q_len=q_len, hq=8, hk=2, d=64, page=16, seed=11), parents=[i - 1 for i in range(q_len)] * 3)
    sees = torch.zeros(3 * q_len, dtype=torch.bool)
    for b, n in enumerate(c["lens"].tolist()):
        at = n - q_len - window + (4 if where == "context" else 0)     # (a first token of a tree sees from one further on)
        if at >= 0:
            c[which][c["table"][b, at // 16].long(), at % 16] = float("nan")
            sees[b * q_len:(b + 1) * q_len] = T.seen(c["visible"][b * q_len:(b + 1) * q_len], n, q_len, window)[:, at]
    assert bool(sees.any()) == (where == "context")
    for chunks in (0, 4):
        out, lse = call(dev, c, q_len, window=window, num_chunks=chunks, rows_per_group=rows, heads_per_group=1)
        check(c, out, lse, window=window, rows=~sees)
        assert torch.isnan(out[sees]).any(-1).all()


@pytest.mark.parametrize("rows", [64, 128])
def test_a_score_without_end(dev, rows):
    """Keys whose scores are minus infinity weigh nothing, as if their bits were not set; a row whose scores all are gives zeros and minus infinity."""
    c = tree(make(dev, [70, 9, 200], q_len=9, hq=16, hk=1, d=64, page=16, seed=2), seed=5)
    c["q"] = c["q"].abs() + 0.5
    without, bad = dict(c, visible=c["visible"].clone()), dict(c, k=c["k"].clone())
    for b, n in enumerate(c["lens"].tolist()):
        for i in range(9) if b == 1 else (0, 4):
            bad["k"][c["table"][b, (n - 9 + i) // 16].long(), (n - 9 + i) % 16] = -float("inf")
            without["visible"][b * 9:(b + 1) * 9] &= ~(1 << i)
    for chunks in (0, 5):
        check(without, *call(dev, bad, 9, num_chunks=chunks, rows_per_group=rows, heads_per_group=1))


@pytest.mark.parametrize("fp8", [False, True], ids=["same", "e4m3"])
@pytest.mark.parametrize("rows", [None, 16, 128])
def test_views_of_wider_tensors(dev, fp8, rows):
    """Heads, rows and pages of wider tensors, keys and values of one, tables and bits with strides of their own."""
    from omni_npu_amd import kernels as K
    c = tree(make(dev, [300, 77, 640], q_len=6, hq=12, hk=4, d=128, page=64, fp8=fp8, seed=42), seed=7)
    pages = c["k"].shape[0]
    both = torch.zeros(pages + 1, 64 + 3, 2, 5, 128, dtype=torch.float32)
    both[:pages, :64, 0, :4], both[:pages, :64, 1, :4] = c["k"].float(), c["v"].float()
    both = both.to(c["k"].dtype).to(dev)
    k, v = both[:pages, :64, 0, :4], both[:pages, :64, 1, :4]
    on = {n: None if c[n] is None else c[n].to(dev) for n in ("q", "table", "lens", "visible", "k_scale", "v_scale")}
    q = torch.full((18, 20, 128), float("nan"), dtype=c["dtype"], device=dev)
    q[:, :12] = on["q"]
    bits = torch.full((18, 5), -1, dtype=torch.int64, device=dev)
    bits[:, 2:3] = on["visible"]
    for chunks in (None, 0, 6):
        out = torch.full((18, 2, 14, 128), 7.0, dtype=c["dtype"], device=dev)
        lse = torch.empty(18, 12, device=dev)
        K.gqa_tree_decode(q[:, :12], k, v, on["table"], on["lens"], bits[:, 2:3], c["scale"], out[:, 1, 1:13], q_len=6, k_scale=on["k_scale"],
                          v_scale=on["v_scale"], lse_out=lse, num_chunks=chunks, rows_per_group=rows, heads_per_group=rows and 1)
        got = out.cpu()
        check(c, got[:, 1, 1:13], lse.cpu())
        got[:, 1, 1:13] = 7.0
        assert (got == 7.0).all()


@pytest.mark.parametrize("rows", [16, 64, 128])
def test_pages_further_apart_than_32_bits_reach(dev, rows):
    """Pages of one cache lie 3 GB apart."""
    from omni_npu_amd import kernels as K
    c = tree(make(dev, [40, 25], q_len=6, hq=8, hk=2, d=64, page=16, seed=12), seed=12)
    pages, apart = c["k"].shape[0], 3 * 2 ** 29
    base = torch.empty(2, (pages - 1) * apart + 16 * 128, dtype=c["dtype"], device=dev)
    k, v = (base[i].as_strided((pages, 16, 2, 64), (apart, 128, 64, 1), base[i].storage_offset()) for i in (0, 1))
    k.copy_(c["k"])
    v.copy_(c["v"])
    for chunks in (0, 3):
        out, lse = torch.empty(12, 8, 64, dtype=c["dtype"], device=dev), torch.empty(12, 8, device=dev)
        K.gqa_tree_decode(c["q"].to(dev), k, v, c["table"].to(dev), c["lens"].to(dev), c["visible"].to(dev), c["scale"], out, q_len=6, lse_out=lse,
                          num_chunks=chunks, rows_per_group=rows, heads_per_group=1)
        check(c, out.cpu(), lse.cpu())


@pytest.mark.parametrize("batch", [65, 300])
@pytest.mark.parametrize("chunks", [0, 1, 50, 300])
def test_many_requests(dev, batch, chunks):
    g = torch.Generator().manual_seed(batch)
    lens = [int(n) for n in torch.randint(0, 90, (batch,), generator=g)]
    lens[0], lens[-1], lens[batch // 2] = 0, 0, 400
    c = tree(make(dev, lens, q_len=4, hq=4, hk=2, d=64, page=16, seed=batch), seed=batch)
    check(c, *call(dev, c, 4, num_chunks=chunks, **WIDE))


@pytest.mark.parametrize("lens,q_len,hq,hk,d", [([3000] * 6, 40, 32, 8, 128), ([9000, 20], 64, 32, 4, 64), ([1500] * 40, 20, 32, 4, 128), ([2500] * 16, 26, 16, 4, 256)])
def test_what_the_rule_chooses(dev, lens, q_len, hq, hk, d):
    """Work that it gives 128 rows to a workgroup."""
    from omni_npu_amd import kernels as K
    c = tree(make(dev, lens, q_len=q_len, hq=hq, hk=hk, d=d, page=64, seed=1), seed=1)
    room = c["table"].shape[1] * 64
    chunks, heads, rows = K.gqa_tree_plan(len(lens), q_len, hq, hk, d, 2, room)
    assert (heads, rows) == (1, 128)
    out, lse = call(dev, c, q_len)
    check(c, out, lse)
    again, again_lse = call(dev, c, q_len, num_chunks=chunks, **WIDE)
    assert torch.equal(out, again) and torch.equal(lse, again_lse)


def test_a_graph_over_other_requests(dev):
    """Captured once, replayed over other lengths, tables and trees, with eager work in between: each as the call by itself."""
    from omni_npu_amd import kernels as K
    q_len, hq, hk, d = 33, 16, 2, 128
    cases = [tree(make(dev, lens, q_len=q_len, hq=hq, hk=hk, d=d, page=16, blocks=80, seed=i), seed=i)
             for i, lens in enumerate(([1200, 33, 700], [40, 0, 1279], [33, 34, 35]))]
    most = max(c["k"].shape[0] for c in cases)
    pad = lambda x: torch.cat((x, torch.zeros(most - x.shape[0], *x.shape[1:], dtype=x.dtype)))
    names = ("q", "k", "v", "table", "lens", "visible")
    now = {n: (pad(cases[0][n]) if n in "kv" else cases[0][n]).to(dev) for n in names}
    out, lse = torch.empty_like(now["q"]), torch.empty(3 * q_len, hq, device=dev)

    def run(**kw):
        K.gqa_tree_decode(now["q"], now["k"], now["v"], now["table"], now["lens"], now["visible"], cases[0]["scale"], out, q_len=q_len, lse_out=lse, **kw)

    for kw in (dict(num_chunks=20, **WIDE), dict(num_chunks=0, **WIDE), dict()):
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            run(**kw)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            run(**kw)
        for c in cases + cases[:1]:
            for n in names:
                now[n].copy_(pad(c[n]) if n in "kv" else c[n])
            out.fill_(float("nan"))
            graph.replay()
            torch.cuda.synchronize()
            check(c, out.cpu(), lse.cpu())
            got = out.clone()
            run(**(kw or dict(max_seq_len=1280)))
            torch.cuda.synchronize()
            assert torch.allclose(got.float(), out.float(), rtol=2 ** -7, atol=1e-3)


@pytest.mark.parametrize("kw", [dict(heads_per_group=2), dict(heads_per_group=4), dict(rows_per_group=16), dict(rows_per_group=128), dict(num_chunks=3),
                                dict(heads_per_group=1)], ids=str)
@pytest.mark.parametrize("path", ["native", "general"])
def test_a_choice_of_the_callers_and_the_rules(dev, kw, path):
    """Where the rule would choose 128 rows, which go with one key head alone: what the caller names holds, and the rest follows it."""
    from omni_npu_amd import kernels as K
    c = tree(make(dev, [3000] * 6, q_len=40, hq=32, hk=8, page=64, seed=1), seed=1)
    assert K.gqa_tree_plan(6, 40, 32, 8, 128, 2, c["table"].shape[1] * 64)[2] == 128
    if path == "general":
        kw = dict(kw, workspace=torch.empty(1 << 28, dtype=torch.uint8, device=dev))
    check(c, *call(dev, c, 40, **kw))
