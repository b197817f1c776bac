"""The operators of layers with ordinary key and value heads together, as a serving step runs them: norms, positions and cache write, attention
over the pages, pages forked and moved between the steps.  Eager, captured and replayed, on two streams at once, over caches whose offsets
pass 32 bits."""
import pytest
import torch

from oracle import heads_oracle as H
from tests.test_gqa_decode_gpu import call, check, make

pytestmark = pytest.mark.gpu

E4M3 = torch.float8_e4m3fn


class Layer:
    """One layer's weights and caches, and its steps over a batch of requests."""

    def __init__(self, dev, hq=8, hk=2, d=64, r=64, pages=24, page=16, dtype=torch.bfloat16, fp8=False, seed=0):
        g = torch.Generator().manual_seed(seed)
        angle = torch.outer(torch.arange(512, dtype=torch.float64), 10000.0 ** (-torch.arange(0, r, 2, dtype=torch.float64) / r))
        self.hq, self.hk, self.d, self.dtype, self.page = hq, hk, d, dtype, page
        self.cos, self.sin = angle.cos().float().to(dev), angle.sin().float().to(dev)
        self.qg, self.kg = ((1 + 0.2 * torch.randn(d, generator=g)).to(dtype).to(dev) for _ in range(2))
        self.k, self.v = (torch.zeros(pages, page, hk, d, device=dev).to(E4M3 if fp8 else dtype) for _ in range(2))
        self.ks, self.vs = ((0.01 + 0.01 * torch.rand(hk, generator=g)).to(dev) if fp8 else None for _ in range(2))

    def step(self, qkv, positions, slots, table, lens, q_len, out, lse=None, q=None, window=None):
        from omni_npu_amd import kernels as K
        xq, xk, xv = (x.unflatten(1, (-1, self.d)) for x in qkv.split([n * self.d for n in (self.hq, self.hk, self.hk)], dim=1))
        q = torch.empty(xq.shape, dtype=self.dtype, device=qkv.device) if q is None else q
        K.qk_norm_rope_cache(xq, xk, xv, self.cos, self.sin, positions, slots, self.k, self.v, q_gamma=self.qg, k_gamma=self.kg, eps=1e-6,
                             q_out=q, k_scale=self.ks, v_scale=self.vs)
        K.gqa_decode(q, self.k, self.v, table, lens, self.d ** -0.5, out, q_len=q_len, window=window, k_scale=self.ks, v_scale=self.vs,
                     lse_out=lse)
        return q

    def check(self, q, table, lens, q_len, out, lse, window=None):
        """Against 64 bits, from the queries and the caches that the first operator has left."""
        cpu = lambda x: None if x is None else x.cpu()
        plain = lambda x: cpu(x).float() if x.dtype == E4M3 else cpu(x)
        start = torch.arange(0, len(lens) * q_len + 1, q_len)
        o, l, weight, reach = H.gqa(cpu(q), plain(self.k), plain(self.v), cpu(table), cpu(lens), self.d ** -0.5, start, window or 0, cpu(self.ks),
                                    cpu(self.vs))
        assert ((cpu(out).double() - o).abs() <= H.gqa_tolerance(o, weight, reach, self.dtype, self.d)).all()
        return cpu(lse)

    def tokens(self, dev, n, g):
        return torch.randn(n, (self.hq + 2 * self.hk) * self.d, generator=g).to(self.dtype).to(dev)


def places(table, lens, q_len, page):
    """Positions and slots of the newest ``q_len`` tokens of each request."""
    pos = (lens[:, None] - q_len + torch.arange(q_len, device=lens.device)).long()
    slots = table.gather(1, pos // page).long() * page + pos % page
    return pos.flatten(), slots.flatten()


@pytest.mark.parametrize("fp8", [False, True], ids=["same", "e4m3"])
@pytest.mark.parametrize("d,window", [(64, None), (128, 20), (256, None)])
def test_prompt_fork_decode_and_move(dev, fp8, d, window):
    """A prompt's tokens, written and attended; two requests that go on from it, the second in a copy of the last, half-filled page; their
    pages moved together; and the step after that.  Every step against the formulas, keys and values against one run of all tokens."""
    from omni_npu_amd import kernels as K
    L = Layer(dev, d=d, r=d, fp8=fp8)
    g = torch.Generator().manual_seed(5)
    table = torch.tensor([[20, 7, 13, 0], [20, 7, 9, 0]], dtype=torch.int32, device=dev)
    prompt = L.tokens(dev, 40, g)

    def step(x, tab, lens, q_len):
        pos, slots = places(tab, lens, q_len, 16)
        out = torch.full((x.shape[0], L.hq, d), float("nan"), dtype=L.dtype, device=dev)
        lse = torch.empty(x.shape[0], L.hq, dtype=torch.float32, device=dev)
        q = L.step(x, pos, slots, tab, lens, q_len, out, lse, window=window)
        torch.cuda.synchronize()
        L.check(q, tab, lens, q_len, out, lse, window)
        return out

    lens = lambda *n: torch.tensor(n, dtype=torch.int32, device=dev)
    step(prompt, table[:1], lens(40), 40)
    K.copy_pages([L.k, L.v], [13], [9], rows=[8])                                       # the second request's own last page
    new = L.tokens(dev, 6, g)
    step(new, table, lens(43, 43), 3)
    bits = lambda x: x.view(torch.uint8) if fp8 else x
    for c in (L.k, L.v):
        assert torch.equal(bits(c)[13, :8], bits(c)[9, :8]) and not torch.equal(bits(c)[13, 8:11], bits(c)[9, 8:11])
    last = L.tokens(dev, 2, g)
    before = [c.clone() for c in (L.k, L.v)]
    there = step(last, table, lens(44, 44), 1)
    for c, old in zip((L.k, L.v), before):
        c.copy_(old)
    K.copy_pages([L.k, L.v], [20, 7, 13, 9], [1, 2, 3, 4], block_table=table)            # moved to the front
    assert table.tolist() == [[1, 2, 3, 0], [1, 2, 4, 0]]
    for i in (20, 7, 13, 9):
        L.k[i].view(torch.uint8).fill_(0xff)                                            # (not a number, in every type)
        L.v[i].view(torch.uint8).fill_(0xff)
    assert torch.equal(step(last, table, lens(44, 44), 1), there)


@pytest.mark.parametrize("fp8", [False, True], ids=["same", "e4m3"])
def test_a_captured_step(dev, fp8):
    """One graph for every step of a padded batch: positions, slots, lengths and tables live on the device; pages are forked and moved by
    eager calls between the replays; requests end and their rows stay padding."""
    from omni_npu_amd import kernels as K
    L, ref = (Layer(dev, fp8=fp8, pages=40, hq=12, hk=4, seed=1) for _ in range(2))
    g = torch.Generator().manual_seed(6)
    b = 6
    table = torch.arange(b * 6, dtype=torch.int32, device=dev).view(b, 6).contiguous()
    lens = torch.zeros(b, dtype=torch.int32, device=dev)
    pos, slots = torch.zeros(b, dtype=torch.int64, device=dev), torch.full((b,), -1, dtype=torch.int64, device=dev)
    x = L.tokens(dev, b, g)
    q, out = (torch.empty(b, L.hq, L.d, dtype=L.dtype, device=dev) for _ in range(2))
    lse = torch.empty(b, L.hq, dtype=torch.float32, device=dev)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        L.step(x, pos, slots, table, lens, 1, out, lse, q)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            L.step(x, pos, slots, table, lens, 1, out, lse, q)
    torch.cuda.synchronize()
    n = [1, 33, 17, 0, 16, 70]
    for i, length in enumerate(n):                                                        # what the requests hold already
        if length > 1:
            rows = torch.arange(length - 1)
            for lay in (L, ref):
                lay.k[table[i].long()[rows // 16], rows % 16] = torch.randn(length - 1, L.hk, L.d, generator=torch.Generator().manual_seed(i)).to(L.k.dtype).to(dev)
                lay.v[table[i].long()[rows // 16], rows % 16] = torch.randn(length - 1, L.hk, L.d, generator=torch.Generator().manual_seed(9 + i)).to(L.k.dtype).to(dev)
    for t in range(5):
        now = torch.tensor([k + t if k else 0 for k in n], dtype=torch.int32, device=dev)
        if t == 3:
            now[2] = 0                                                                    # a request that has ended
            for lay in (L, ref):
                K.copy_pages([lay.k, lay.v], [int(table[5, 0]), int(table[5, 4])], [37, 36])
            table[5, 0], table[5, 4] = 37, 36
        p, s = places(table, now.clamp(min=1), 1, 16)
        live = now > 0
        lens.copy_(now), pos.copy_(p), slots.copy_(torch.where(live, s, -1)), x.copy_(L.tokens(dev, b, g))
        out.fill_(float("nan"))
        graph.replay()
        want = torch.full_like(out, float("nan"))
        want_lse = torch.empty_like(lse)
        qq = ref.step(x, pos, slots, table, lens, 1, want, want_lse)
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(lse, want_lse) and torch.equal(q, qq)
        assert torch.equal(L.k.view(torch.uint8), ref.k.view(torch.uint8)) and torch.equal(L.v.view(torch.uint8), ref.v.view(torch.uint8))
        assert (out[~live] == 0).all() and torch.isinf(lse[~live]).all()
        L.check(q, table, lens, 1, out, lse)


def test_two_streams_at_once(dev):
    """Two layers' steps on a stream each, interleaved from the host, without a wait between them: neither sees the other's scratch memory."""
    L = [Layer(dev, hq=16, hk=2, pages=600, seed=i) for i in range(2)]
    g = torch.Generator().manual_seed(8)
    table = torch.randperm(600, generator=g)[:8 * 32].to(torch.int32).view(8, 32).contiguous().to(dev)
    lens = torch.tensor([500, 3, 260, 17, 512, 100, 401, 64], dtype=torch.int32, device=dev)
    for lay in L:
        lay.k.copy_(torch.randn(lay.k.shape, generator=g).to(lay.dtype)), lay.v.copy_(torch.randn(lay.k.shape, generator=g).to(lay.dtype))
    pos, slots = places(table, lens, 1, 16)
    x = [lay.tokens(dev, 8, g) for lay in L]
    new = lambda: torch.full((8, 16, 64), float("nan"), dtype=torch.bfloat16, device=dev)
    ref = [new() for _ in L]
    for i, lay in enumerate(L):
        lay.step(x[i], pos, slots, table, lens, 1, ref[i])
    streams = [torch.cuda.Stream() for _ in L]
    outs = [[new() for _ in range(20)] for _ in L]
    torch.cuda.synchronize()
    for n in range(20):
        for i, lay in enumerate(L):
            with torch.cuda.stream(streams[i]):
                lay.step(x[i], pos, slots, table, lens, 1, outs[i][n])
    torch.cuda.synchronize()
    for i in range(2):
        assert torch.isfinite(ref[i]).all() and all(torch.equal(o, ref[i]) for o in outs[i])


def test_two_graphs_of_one_stream_and_a_larger_call_between(dev):
    """Graphs captured on one stream share its scratch memory, replayed one after the other; a call that needs more of it than there is
    leaves what a graph holds where it is."""
    from omni_npu_amd import kernels as K
    cases = [make(dev, [700, 333], hq=8, hk=2, seed=51), make(dev, [1500, 20, 900], hq=16, hk=4, d=64, page=16, seed=52)]
    refs = [call(dev, c, 1, num_chunks=12) for c in cases]
    on = [{n: c[n].to(dev) for n in ("q", "k", "v", "table", "lens")} for c in cases]
    outs = [torch.empty_like(o["q"]) for o in on]
    side, graphs = torch.cuda.Stream(), []
    for c, o, out in zip(cases, on, outs):
        with torch.cuda.stream(side):
            run = lambda: K.gqa_decode(o["q"], o["k"], o["v"], o["table"], o["lens"], c["scale"], out, num_chunks=12)
            run()
            torch.cuda.synchronize()
            graphs.append(torch.cuda.CUDAGraph())
            with torch.cuda.graph(graphs[-1], stream=side):
                run()
            torch.cuda.synchronize()
            big = make(dev, [900] * 40, hq=64, hk=2, d=64, page=64, seed=53)
            check(big, *call(dev, big, 1, num_chunks=300 * len(graphs)))
    for i in (0, 1, 1, 0, 1, 0):
        outs[i].fill_(float("nan"))
        torch.cuda.synchronize()
        graphs[i].replay()
        torch.cuda.synchronize()
        assert torch.equal(outs[i].cpu(), refs[i][0])


def test_on_a_stream_that_is_not_the_current_one_of_the_tensors(dev):
    """Tensors made on one stream, used on another that waits for it."""
    c = make(dev, [300, 77], seed=21)
    ref, ref_lse = call(dev, c, 1)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got, lse = call(dev, c, 1)
    assert torch.equal(got, ref) and torch.equal(lse, ref_lse)


@pytest.mark.parametrize("batch", [64, 65, 131, 700])
@pytest.mark.parametrize("chunks", [0, 1, 50, 300])
def test_many_requests(dev, batch, chunks):
    """More requests than a wavefront has lanes, empty ones among them, shared by few and by many chunks."""
    g = torch.Generator().manual_seed(batch)
    lens = [int(n) for n in torch.randint(0, 90, (batch,), generator=g)]
    lens[0], lens[-1], lens[batch // 2] = 0, 0, 400
    c = make(dev, lens, hq=4, hk=2, d=64, page=16, seed=batch)
    check(c, *call(dev, c, 1, num_chunks=chunks))


@pytest.mark.parametrize("chunks", [0, 7])
@pytest.mark.parametrize("d,page", [(64, 16), (64, 32), (128, 16), (256, 16), (256, 48)])
def test_more_pages_than_a_wavefront_holds_numbers_of(dev, chunks, d, page):
    c = make(dev, [64 * page + 1100, 1, 64 * page + 1, 64 * page], q_len=2, hq=6, hk=2, d=d, page=page, seed=page)
    check(c, *call(dev, c, 2, num_chunks=chunks))


@pytest.mark.parametrize("chunks", [None, 1, 2, 9, 200])
@pytest.mark.parametrize("n,q_len,window", [(1, 1, None), (33, 2, None), (2100, 1, None), (2100, 3, None), (5000, 1, 40), (5000, 2, 1500), (0, 1, None)])
def test_one_request_in_pieces(dev, chunks, n, q_len, window):
    c = make(dev, [n], q_len=q_len, hq=6, hk=2, d=64, page=16, seed=n)
    check(c, *call(dev, c, q_len, window=window, num_chunks=chunks), window=window)


@pytest.mark.parametrize("chunks", [None, 0, 5])
def test_many_tokens(dev, chunks):
    """A prompt's tokens behind a context, and a request that is only a prompt: many groups of rows."""
    c = make(dev, [500, 301, 77], q_lens=[150, 301, 1], hq=6, hk=2, d=64, page=16, seed=41)
    check(c, *call(dev, c, 301, varlen=True, num_chunks=chunks))
    check(c, *call(dev, c, 301, varlen=True, num_chunks=chunks, window=130), window=130)


@pytest.mark.parametrize("fp8", [False, True], ids=["same", "e4m3"])
def test_views_of_wider_tensors(dev, fp8):
    """Queries as a view of the projection's result, results into a wider tensor, rows of a wider block table: nothing beside them is touched."""
    from omni_npu_amd import kernels as K
    c = make(dev, [300, 77, 640], q_len=2, hq=12, hk=4, d=128, fp8=fp8, page=64, seed=42)
    ref, ref_lse = call(dev, c, 2)
    check(c, ref, ref_lse)
    on = {n: None if c[n] is None else c[n].to(dev) for n in ("q", "k", "v", "table", "lens", "k_scale", "v_scale")}
    wide_q = torch.full((6, 12 + 8, 128), float("nan"), dtype=c["dtype"], device=dev)
    wide_q[:, :12] = on["q"]
    wide_out = torch.full((6, 2, 14, 128), 7.0, dtype=c["dtype"], device=dev)
    table = torch.full((5, on["table"].shape[1] + 9), -3, dtype=torch.int32, device=dev)
    table[:3, :on["table"].shape[1]] = on["table"]
    for chunks in (None, 0, 6):
        wide_out.fill_(7.0)
        K.gqa_decode(wide_q[:, :12], on["k"], on["v"], table[:, :on["table"].shape[1]], on["lens"], c["scale"], wide_out[:, 1, 1:13], q_len=2,
                     k_scale=on["k_scale"], v_scale=on["v_scale"], num_chunks=chunks)
        got = wide_out.cpu()
        check(c, got[:, 1, 1:13], ref_lse)
        got[:, 1, 1:13] = 7.0
        assert (got == 7.0).all()


@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
def test_offsets_beyond_32_bits(dev, kind):
    """Caches of more than 2^32 elements: the pages in use lie at both ends."""
    from omni_npu_amd import kernels as K
    if torch.cuda.mem_get_info()[0] < 60 << 30:
        pytest.skip("not enough memory free")
    fp8 = kind == "e4m3"
    d, page, hk = 128, 128, 8
    pages = 2 ** 32 // (page * hk * d) + 40
    L = Layer(dev, hq=16, hk=hk, d=d, r=d, pages=2, page=page, fp8=fp8, seed=2)
    L.k, L.v = (torch.empty(pages, page, hk, d, device=dev, dtype=E4M3 if fp8 else torch.bfloat16) for _ in range(2))
    near = Layer(dev, hq=16, hk=hk, d=d, r=d, pages=8, page=page, fp8=fp8, seed=2)
    far_pages = [pages - 1, 3, pages - 7, pages // 2 + 5, pages - 2]
    table = torch.tensor([far_pages[:2], far_pages[2:4]], dtype=torch.int32, device=dev)
    small = torch.tensor([[0, 1], [2, 3]], dtype=torch.int32, device=dev)
    g = torch.Generator().manual_seed(3)
    out, want = (torch.full((400, 16, d), float("nan"), dtype=torch.bfloat16, device=dev) for _ in range(2))
    x = L.tokens(dev, 400, g)
    lens = torch.tensor([200, 200], dtype=torch.int32, device=dev)
    for lay, tab, o in ((L, table, out), (near, small, want)):
        pos, slots = places(tab, lens, 200, page)
        lay.step(x, pos, slots, tab, lens, 200, o)
    assert torch.isfinite(want).all() and torch.equal(out, want)
    K.copy_pages([L.k, L.v], [far_pages[0], far_pages[3]], [far_pages[4], 11])
    raw = lambda c: c.view(torch.uint8)
    for lay_c, near_c in ((L.k, near.k), (L.v, near.v)):
        for i, f in enumerate(far_pages[:4]):
            n = 128 if i % 2 == 0 else 72
            assert torch.equal(raw(lay_c)[f, :n], raw(near_c)[i, :n])
        assert torch.equal(raw(lay_c)[far_pages[4]], raw(near_c)[0]) and torch.equal(raw(lay_c)[11, :72], raw(near_c)[3, :72])
