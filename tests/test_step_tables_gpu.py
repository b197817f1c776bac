"""A step's tables against their plain statement: pages taken and given back, lengths, positions, slots and what each token sees, whole numbers all."""
import pytest
import torch

from oracle import tree_oracle as T

pytestmark = pytest.mark.gpu


class Case:
    def __init__(self, seed, batch, page=16, room=12, counts=None, q_len=3, hi=100, tree=False, words=1, pages=True, padded=0, spare=40, idle=0.1, capacity=None):
        g = torch.Generator().manual_seed(seed)
        rnd = lambda lo, hi, n: [int(x) for x in torch.randint(lo, hi + 1, (n,), generator=g)]
        self.page, self.q_len, self.ragged = page, q_len, counts is not None
        self.counts = counts or [q_len] * batch
        self.ctx = [-1 - c if torch.rand(1, generator=g) < idle else c for c in rnd(0, hi, batch)]
        self.total = sum(self.counts) + padded
        self.parents = None
        if tree:
            self.parents = [p for n in self.counts for p in [int(torch.randint(-2, i + 2, (1,), generator=g)) for i in range(n)]] + rnd(-1, 5, padded)
        self.words = words
        self.held = None
        if pages:
            self.held = [min(room, max(0, h)) for h in [(-(-max(c, 0) // page)) + e for c, e in zip(self.ctx, rnd(-1, 2, batch))]]
        used = sum(self.held) if pages else batch * room
        order = torch.randperm(used + spare, generator=g).tolist()
        self.table = [[-7] * room for _ in range(batch)]
        at = 0
        for b in range(batch):
            for k in range(self.held[b] if pages else room):
                self.table[b][k] = order[at]
                at += 1
        capacity = used + spare if capacity is None else capacity
        self.free, self.num_free = (order[at:] + [-9] * capacity)[:capacity], min(spare, capacity)

    def expected(self):
        return T.step_tables(self.ctx, self.counts, self.table, self.page, self.total, self.parents, self.words, self.held, self.free, self.num_free)

    def on(self, dev):
        i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)
        b = len(self.ctx)
        start = [0]
        for n in self.counts:
            start.append(start[-1] + n)
        args = [i32(self.ctx), i32(self.table).view(b, -1), self.page, i32([77] * b),
                *(torch.full((self.total,), 55, dtype=torch.int64, device=dev) for _ in range(2))]
        kw = dict(q_len=self.q_len, query_start_loc=i32(start) if self.ragged else None)
        if self.parents is not None:
            kw.update(parents=i32(self.parents), visible=torch.full((self.total, self.words), 55, dtype=torch.int64, device=dev))
        if self.held is not None:
            kw.update(num_blocks=i32(self.held), free_pages=i32(self.free), num_free=i32([self.num_free]))
        return args, kw

    def check(self, args, kw):
        want = self.expected()
        assert args[3].tolist() == want["seq_lens"]
        assert args[4].tolist() == want["positions"]
        assert args[5].tolist() == want["slots"]
        assert args[1].tolist() == want["table"]
        if self.parents is not None:
            assert torch.equal(kw["visible"].cpu(), want["words"])
        if self.held is not None:
            assert kw["num_blocks"].tolist() == want["held"] and kw["num_free"].tolist() == [want["num_free"]]
            assert kw["free_pages"].tolist() == want["free"]


def run(dev, case):
    from omni_npu_amd import kernels as K
    args, kw = case.on(dev)
    K.step_tables(*args, **kw)
    torch.cuda.synchronize()
    case.check(args, kw)
    return args, kw


@pytest.mark.parametrize("batch", [1, 2, 63, 64, 200])
@pytest.mark.parametrize("page", [1, 7, 16, 128])
@pytest.mark.parametrize("q_len", [1, 5, 40])
@pytest.mark.parametrize("tree", [False, True])
@pytest.mark.parametrize("pages", [False, True])
def test_uniform_steps(dev, batch, page, q_len, tree, pages):
    run(dev, Case(batch + page, batch, page=page, room=150 // page + 2, q_len=q_len, tree=tree, pages=pages, spare=60 * batch))


@pytest.mark.parametrize("seed", range(12))
@pytest.mark.parametrize("tree", [False, True])
def test_ragged_steps(dev, seed, tree):
    """Requests without tokens, at the front and the end too; padding; tokens that outgrow the table."""
    g = torch.Generator().manual_seed(seed)
    batch = int(torch.randint(1, 80, (1,), generator=g))
    counts = [int(x) * (torch.rand(1, generator=g) > 0.3).item() for x in torch.randint(0, 70, (batch,), generator=g)]
    run(dev, Case(seed, batch, counts=counts, tree=tree, words=2, pages=seed % 3 > 0, padded=seed % 4 * 3, spare=[500, 20, 3, 0][seed % 4]))


@pytest.mark.parametrize("spare", [0, 1, 2, 5, 11, 30])
def test_too_few_pages(dev, spare):
    """From the first request that the list is too short for on none gets any, those that need none go on; tables without room."""
    case = Case(spare, 40, q_len=30, room=7, hi=110, spare=spare)
    args, kw = run(dev, case)
    assert spare > 5 or any(n == c for n, c in zip(case.expected()["seq_lens"], case.ctx) if c >= 0)


@pytest.mark.parametrize("capacity", [0, 3, 8, 20])
def test_a_list_without_room_takes_nothing_back(dev, capacity):
    case = Case(3, 30, q_len=1, spare=3, capacity=capacity, idle=0.7)
    run(dev, case)


def test_pages_given_back_come_out_in_their_order(dev):
    """A step, its end, the step again: the tables and the list as they were."""
    from omni_npu_amd import kernels as K
    case = Case(1, 20, q_len=50, spare=400, idle=0.0)
    case.held = [-(-c // 16) for c in case.ctx]
    args, kw = case.on(dev)
    before = [x.clone() for x in (kw["num_blocks"], kw["free_pages"], kw["num_free"])]
    K.step_tables(*args, **kw)
    table = args[1].clone()
    assert not torch.equal(kw["num_free"], before[2])
    kw["query_start_loc"] = torch.zeros(21, dtype=torch.int32, device=dev)
    K.step_tables(*args, **kw)
    for x, y in zip(before, (kw["num_blocks"], kw["free_pages"], kw["num_free"])):
        assert torch.equal(x, y)
    kw["query_start_loc"] = None
    K.step_tables(*args, **kw)
    assert torch.equal(table, args[1])


@pytest.mark.parametrize("batch", [1023, 1024, 1025, 3000, 9000])
@pytest.mark.parametrize("tree", [False, True])
def test_many_requests(dev, batch, tree):
    """More than a workgroup's threads, and more than its samples of the starts."""
    g = torch.Generator().manual_seed(batch)
    counts = [int(x) for x in torch.randint(0, 4, (batch,), generator=g)]
    run(dev, Case(batch, batch, counts=counts, tree=tree, hi=60, spare=batch, padded=5))
    run(dev, Case(batch, batch, q_len=2, tree=tree, hi=60, spare=batch // 4))


@pytest.mark.parametrize("total", [2047, 2048, 2049, 20000])
@pytest.mark.parametrize("pages", [False, True])
def test_prompts(dev, total, pages):
    """One launch and two; many pages for one request."""
    run(dev, Case(total, 3, counts=[5, total - 6, 1], page=16, room=1300, hi=30, pages=pages, spare=1400, idle=0.0))
    run(dev, Case(total, 1, q_len=total, page=16, room=1300, hi=30, pages=pages, spare=1400, idle=0.0))


@pytest.mark.parametrize("n,words", [(64, 1), (65, 2), (200, 4), (200, 2), (512, 8), (700, 11)])
def test_large_trees(dev, n, words):
    """A chain as deep as it is long, a bush, bits that the words do not hold (their depth counts all the same)."""
    for seed, up in enumerate(([i - 1 for i in range(n)], [-1] + [0] * (n - 1), [i - 2 for i in range(n)])):
        case = Case(seed, 2, counts=[n, n], tree=True, words=words, room=60, spare=100, idle=0.0)
        case.parents = up + case.parents[n:]
        run(dev, case)


def test_wild_values(dev):
    """Counts and starts that are none: nothing is read or written out of place."""
    from omni_npu_amd import kernels as K
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device=dev)
    i64 = lambda n: torch.full((n,), 55, dtype=torch.int64, device=dev)
    big = 2 ** 31 - 1
    lens, pos, slots = i32(0, 0, 0, 0), i64(12), i64(12)
    table = torch.arange(20, dtype=torch.int32, device=dev).view(4, 5).contiguous()
    K.step_tables(i32(big, 5, -big, big - 1), table, 4, lens, pos, slots, q_len=3)
    assert lens.tolist() == [big, 8, 0, big] and slots.tolist() == [-1] * 3 + [25, 26, 27] + [-1] * 6
    assert pos.tolist() == [big, big + 1, big + 2, 5, 6, 7, 0, 0, 0, big - 1, big, big + 1]
    held, free, num = i32(-5, 100, 2, 3), i32(40, 41, 42), i32(99)
    K.step_tables(i32(4, 5, 6, 7), table, 4, lens, pos, slots, query_start_loc=i32(-7, 2, 0, 9, 8), num_blocks=held, free_pages=free, num_free=num)
    torch.cuda.synchronize()
    assert all(-1 <= s < 43 * 4 for s in slots.tolist())


@pytest.mark.parametrize("total", [60, 3000])
def test_in_a_graph(dev, total):
    """One capture, steps of other lengths: state on the device, checked after every replay, with eager work between."""
    from omni_npu_amd import kernels as K
    b, n = 20, total // 20
    case = Case(1, b, q_len=n, tree=True, words=-(-n // 64), page=16, room=60, spare=900, hi=40)
    args, kw = case.on(dev)
    state = [x.clone() for x in (args[0], args[1], kw["num_blocks"], kw["free_pages"], kw["num_free"])]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        K.step_tables(*args, **kw)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            K.step_tables(*args, **kw)
    torch.cuda.synchronize()
    for x, old in zip((args[0], args[1], kw["num_blocks"], kw["free_pages"], kw["num_free"]), state):
        x.copy_(old)
    for step in range(5):
        ctx = [-1 if (i + step) % 7 == 0 else (37 * i + 61 * step) % 300 for i in range(b)]
        args[0].copy_(torch.tensor(ctx, dtype=torch.int32))
        case.ctx, case.table, case.held = ctx, args[1].tolist(), kw["num_blocks"].tolist()
        case.free, case.num_free = kw["free_pages"].tolist(), kw["num_free"].item()
        torch.randn(1000, device=dev).sum().item()
        graph.replay()
        torch.cuda.synchronize()
        case.check(args, kw)


def test_views(dev):
    """Rows of a wider table and of wider bit rows: nothing beside them is touched."""
    from omni_npu_amd import kernels as K
    case = Case(5, 12, q_len=6, tree=True, spare=60)
    args, kw = case.on(dev)
    wide = torch.full((14, 40), -3, dtype=torch.int32, device=dev)
    wide[:12, 5:17] = args[1]
    bits = torch.full((72, 4), 9, dtype=torch.int64, device=dev)
    args[1], kw["visible"] = wide[:12, 5:17], bits[:, 2:3]
    K.step_tables(*args, **kw)
    torch.cuda.synchronize()
    case.check(args, kw)
    wide[:12, 5:17], bits[:, 2] = -3, 9
    assert (wide == -3).all() and (bits == 9).all()


def test_refusals(dev):
    from omni_npu_amd import kernels as K
    base = Case(2, 4, tree=True)

    def refused(error, match, **swap):
        args, kw = base.on(dev)
        for name, x in swap.items():
            if name[0] == "_":
                args[int(name[1:])] = x(args, kw) if callable(x) else x
            else:
                kw[name] = x(args, kw) if callable(x) else x
        with pytest.raises(error, match=match):
            K.step_tables(*args, **kw)

    refused(ValueError, "pages of", _2=0)
    refused(ValueError, "tokens a request", q_len=0)
    refused(ValueError, "context_lens", _0=lambda a, k: a[0].long())
    refused(ValueError, "seq_lens", _3=lambda a, k: a[3][:3])
    refused(ValueError, "positions", _4=lambda a, k: a[4][:-1])
    refused(ValueError, "block_table", _1=lambda a, k: a[1][:3])
    refused(ValueError, "block_table", _1=lambda a, k: a[1].t().contiguous().t())
    refused(ValueError, "go together", visible=None)
    refused(ValueError, "go together", num_free=None)
    refused(ValueError, "visible", visible=lambda a, k: k["visible"][:-1])
    refused(ValueError, "parents", parents=lambda a, k: k["parents"].long())
    refused(ValueError, "places", q_len=4)
    refused(ValueError, "query_start_loc", query_start_loc=lambda a, k: a[0])
    refused(ValueError, "no CPU path", num_free=lambda a, k: k["num_free"].cpu())
    refused(K._lib.MlaHipError, "shares memory", _3=lambda a, k: a[0])
    refused(K._lib.MlaHipError, "shares memory", _4=lambda a, k: a[5])
    refused(K._lib.MlaHipError, "shares memory", num_blocks=lambda a, k: a[0])
    many = Case(2, 2, q_len=65, tree=True)
    args, kw = many.on(dev)
    with pytest.raises(ValueError, match="hold no bits"):
        K.step_tables(*args, **kw)
