"""The operators of a step over drafted trees together, as serving runs them: tables from lengths, norms, rotary positions and cache write, attention of
the trees, the accepted path's rows.  Against the same tokens one after the other, eager, captured and replayed."""
import pytest
import torch

from oracle import heads_oracle as H
from tests.test_heads_run_gpu import E4M3, Layer

pytestmark = pytest.mark.gpu


class Serving:
    """Requests whose tokens are drafted as trees, over two layers' caches, with all of their state on the device."""

    def __init__(self, dev, b, s, fp8=False, d=64, pages=120, page=16, room=12, seed=0, context=(40, 0, 17, 33, 5, 64)):
        self.dev, self.b, self.s, self.page = dev, b, s, page
        self.layers = [Layer(dev, hq=8, hk=2, d=d, r=d, pages=pages, page=page, fp8=fp8, seed=seed + i) for i in range(2)]
        i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)
        g = torch.Generator().manual_seed(seed)
        self.context = i32([context[i % len(context)] for i in range(b)])
        self.table, self.held = torch.full((b, room), -1, dtype=torch.int32, device=dev), i32([0] * b)
        self.free, self.num_free = i32(torch.randperm(pages, generator=g).tolist()), i32([pages])
        self.lens, self.kept = i32([0] * b), i32([0] * b)
        self.positions, self.slots = (torch.zeros(b * s, dtype=torch.int64, device=dev) for _ in range(2))
        self.parents, self.visible = i32([0] * (b * s)), torch.zeros(b * s, 1, dtype=torch.int64, device=dev)
        self.accepted, self.num = i32([[0] * s] * b), i32([0] * b)
        lay = self.layers[0]
        self.x = torch.zeros(2, b * s, (lay.hq + 2 * lay.hk) * d, dtype=lay.dtype, device=dev)
        self.q, self.out = (torch.zeros(2, b * s, lay.hq, d, dtype=lay.dtype, device=dev) for _ in range(2))

    def step(self):
        from omni_npu_amd import kernels as K
        K.step_tables(self.context, self.table, self.page, self.lens, self.positions, self.slots, q_len=self.s, parents=self.parents, visible=self.visible,
                      num_blocks=self.held, free_pages=self.free, num_free=self.num_free)
        for i, lay in enumerate(self.layers):
            q, k, v = (x.unflatten(1, (-1, lay.d)) for x in self.x[i].split([n * lay.d for n in (lay.hq, lay.hk, lay.hk)], dim=1))
            K.qk_norm_rope_cache(q, k, v, lay.cos, lay.sin, self.positions, self.slots, lay.k, lay.v, q_gamma=lay.qg, k_gamma=lay.kg, q_out=self.q[i],
                                 k_scale=lay.ks, v_scale=lay.vs)
            K.gqa_tree_decode(self.q[i], lay.k, lay.v, self.table, self.lens, self.visible, lay.d ** -0.5, self.out[i], q_len=self.s, k_scale=lay.ks,
                              v_scale=lay.vs)

    def keep(self):
        from omni_npu_amd import kernels as K
        K.keep_rows([c for lay in self.layers for c in (lay.k, lay.v)], self.table, self.context, self.lens, self.accepted, self.num, self.kept)
        self.context.copy_(self.kept)


def drafts(g, b, s):
    """Parents of b trees of s tokens and a path down each of them, of any length."""
    parents, paths = [], []
    for _ in range(b):
        up = [-1] + [int(torch.randint(0, i, (1,), generator=g)) for i in range(1, s)]
        path, at = [], int(torch.randint(0, s, (1,), generator=g))
        while at >= 0:
            path, at = [at] + path, up[at]
        parents.append(up)
        paths.append(path)
    return parents, paths


def run(dev, fp8, captured, d=64, steps=5):
    """Trees along one long text for each request: the path's tokens are the text's next ones, the others anything."""
    b, s = 6, 9
    sv = Serving(dev, b, s, fp8=fp8, d=d)
    g = torch.Generator().manual_seed(3)
    lay = sv.layers[0]
    width = (lay.hq + 2 * lay.hk) * d
    text = torch.randn(2, b, 160, width, generator=g).to(lay.dtype).to(dev)
    first = sv.context.tolist()
    done = [0] * b
    # the contexts: the text's first tokens, one chain after the other through the same step
    sv.context.zero_()
    for at in range(0, max(first), s):
        n = [min(s, max(0, c - at)) for c in first]
        sv.parents.copy_(torch.tensor([i - 1 for i in range(s)] * b, dtype=torch.int32))
        for i in range(b):
            sv.x[:, i * s:(i + 1) * s] = text[:, i, at:at + s]
        sv.accepted.copy_(torch.arange(s, dtype=torch.int32).expand(b, s))
        sv.num.copy_(torch.tensor(n, dtype=torch.int32))
        sv.step()
        sv.keep()
        assert sv.context.tolist() == [min(c, at + s) for c in first]
    graph = None
    if captured:
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        state = [x.clone() for x in (sv.context, sv.table, sv.held, sv.free, sv.num_free, *(c for lay in sv.layers for c in (lay.k, lay.v)))]
        sv.num.zero_()
        with torch.cuda.stream(side):
            sv.step()
            sv.keep()
            torch.cuda.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=side):
                sv.step()
                sv.keep()
        torch.cuda.synchronize()
        for x, old in zip((sv.context, sv.table, sv.held, sv.free, sv.num_free, *(c for lay in sv.layers for c in (lay.k, lay.v))), state):
            x.copy_(old)
    for step in range(steps):
        parents, paths = drafts(g, b, s)
        if step == 2:                                                # a request that ends: its pages go back with the next step
            sv.context[4] = -1
        sv.parents.copy_(torch.tensor([p for up in parents for p in up], dtype=torch.int32))
        sv.x.copy_(torch.randn(2, b * s, width, generator=g).to(lay.dtype))
        ctx = sv.context.tolist()
        for i, path in enumerate(paths):
            for k, at in enumerate(path):
                if ctx[i] >= 0:
                    sv.x[:, i * s + at] = text[:, i, ctx[i] + k]
            sv.accepted[i, :len(path)] = torch.tensor(path, dtype=torch.int32)
            sv.num[i] = len(path)
        if graph is not None:
            torch.randn(1000, device=dev).sum().item()
            graph.replay()
        else:
            sv.step()
            sv.keep()
        torch.cuda.synchronize()
        now = [c + len(p) if c >= 0 else -1 for c, p in zip(ctx, paths)]
        assert sv.context.tolist() == now
        used = [-(-(c + s) // sv.page) if c >= 0 else 0 for c in ctx]
        assert sv.held.tolist() == used and sv.num_free.item() == 120 - sum(used)
        assert len({*sv.free[:sv.num_free.item()].tolist(), *(p for i, n in enumerate(used) for p in sv.table[i, :n].tolist())}) == 120
        yield sv, text, ctx, paths, now


@pytest.mark.parametrize("fp8", [False, True], ids=["same", "e4m3"])
@pytest.mark.parametrize("captured", [False, True], ids=["eager", "graph"])
@pytest.mark.parametrize("d", [64, 128])
def test_steps_along_a_text(dev, fp8, captured, d):
    """After every step the caches hold the text so far, bit for bit as written one token after the other, and the path's results are those of attention
    over it."""
    from omni_npu_amd import kernels as K
    refs = [Layer(dev, hq=8, hk=2, d=d, r=d, pages=6 * 12, page=16, fp8=fp8, seed=i) for i in range(2)]
    steps = 0
    for sv, text, ctx, paths, now in run(dev, fp8, captured, d=d):
        steps += 1
        for i in range(sv.b):
            if now[i] < 0:
                continue
            n = now[i]
            pos = torch.arange(n, device=dev)
            rows = sv.table[i].long()[pos // 16] * 16 + pos % 16
            for j, (lay, ref) in enumerate(zip(sv.layers, refs)):
                slots = i * 192 + pos
                q, k, v = (x.unflatten(1, (-1, d)) for x in text[j, i, :n].split([m * d for m in (8, 2, 2)], dim=1))
                turned = torch.empty(n, 8, d, dtype=lay.dtype, device=dev)
                K.qk_norm_rope_cache(q, k, v, ref.cos, ref.sin, pos, slots, ref.k, ref.v, q_gamma=ref.qg, k_gamma=ref.kg, q_out=turned, k_scale=ref.ks,
                                     v_scale=ref.vs)
                bits = lambda c: c.view(torch.uint8).flatten(0, 1)
                for c, r in ((lay.k, ref.k), (lay.v, ref.v)):
                    assert torch.equal(bits(c)[rows], bits(r)[slots])
                at = torch.tensor(paths[i], device=dev) + i * sv.s
                m = len(paths[i])
                assert torch.equal(sv.q[j, at], turned[ctx[i]:])
                plain = lambda c: c.cpu().float() if c.dtype == E4M3 else c.cpu()
                o, _, weight, reach = H.gqa(turned[ctx[i]:].cpu(), plain(ref.k), plain(ref.v), torch.arange(12)[None] + 12 * i, torch.tensor([n]), d ** -0.5,
                                            torch.tensor([0, m]), 0, *(None if x is None else x.cpu() for x in (ref.ks, ref.vs)))
                assert ((sv.out[j, at].cpu().double() - o).abs() <= H.gqa_tolerance(o, weight, reach, lay.dtype, d)).all()
    assert steps == 5
