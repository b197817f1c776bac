"""An accepted path's rows moved up behind the context: the bytes of the plain assignment, everything else left as it was."""
import pytest
import torch

from oracle import tree_oracle as T

pytestmark = pytest.mark.gpu


def _bytes(g, *shape):
    return torch.randint(0, 256, shape, generator=g, dtype=torch.uint8)


def path(g, s, n):
    """An increasing list of n numbers below s."""
    return torch.sort(torch.randperm(s, generator=g)[:n]).values.tolist()


def make(g, batch, page, s, most, hi=70, room=8, idle=0.1):
    ctx = [int(c) if torch.rand(1, generator=g) > idle else -1 for c in torch.randint(0, hi, (batch,), generator=g)]
    pages = batch * room + 3
    table = torch.randperm(pages, generator=g)[:batch * room].view(batch, room).tolist()
    num = [int(x) for x in torch.randint(0, most + 1, (batch,), generator=g)]
    entries = [path(g, s, n) + [-5] * (most - n) for n in num]
    return dict(ctx=ctx, lens=[c + s if c >= 0 else 0 for c in ctx], table=table, num=num, entries=entries, pages=pages, page=page)


def check(dev, c, caches, views=None):
    """views: what the call is given of the tensors (all of them otherwise)."""
    from omni_npu_amd import kernels as K
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)
    on = [x.to(dev) for x in caches]
    b = len(c["ctx"])
    out = i32([99] * b)
    K.keep_rows(views(on) if views else on, i32(c["table"]), i32(c["ctx"]), i32(c["lens"]), i32(c["entries"]).view(b, -1), i32(c["num"]), out)
    torch.cuda.synchronize()
    want, lens = [x.clone() for x in caches], []
    old, new = (views(x) if views else x for x in (caches, want))
    for b in range(len(c["ctx"])):
        moves, n = T.kept(c["ctx"][b], c["lens"][b], c["entries"][b], c["num"][b], c["table"][b], c["page"], c["pages"])
        lens.append(c["ctx"][b] + n if c["ctx"][b] >= 0 else c["ctx"][b])
        for (p0, r0), (p1, r1) in moves:
            for x, y in zip(old, new):
                y[p1, r1] = x[p0, r0]
    assert out.tolist() == lens
    for x, y in zip(on, want):
        assert torch.equal(x.cpu(), y)


@pytest.mark.parametrize("page,widths", [(128, [1024, 128]), (16, [256]), (128, [656]), (64, [4, 12, 128]), (7, [1, 3, 2, 16]), (1, [16]), (16, [2064, 48])])
@pytest.mark.parametrize("batch", [1, 5, 70])
@pytest.mark.parametrize("s,most", [(1, 1), (8, 4), (26, 6), (60, 23)])
def test_paths(dev, page, widths, batch, s, most):
    """Rows of any width; paths of one token to more than a lane reads at once, onto one another's places."""
    g = torch.Generator().manual_seed(page + batch + s)
    c = make(g, batch, page, s, most, hi=min(70, 8 * page), room=140 // page + 3)
    check(dev, c, [_bytes(g, c["pages"], page, w) for w in widths])


def test_a_path_that_moves_by_one(dev):
    """Every row is the next one's source."""
    g = torch.Generator().manual_seed(1)
    c = make(g, 3, 16, 40, 39, idle=0.0)
    c["num"], c["entries"] = [39, 20, 8], [list(range(1, 40))] * 3
    check(dev, c, [_bytes(g, c["pages"], 16, 64)])


@pytest.mark.parametrize("entries,kept", [([0, 1, 2, 3], 4), ([0, 2, 2, 5], 2), ([0, 3, 1, 5], 2), ([-1, 2, 3, 4], 0), ([0, 4, 7, 8], 3), ([5, 6, 7, 9], 3),
                                          ([0, 2 ** 31 - 1, 5, 6], 1), ([1, 2, -2 ** 31, 3], 2)], ids=str)
def test_where_a_path_ends(dev, entries, kept):
    """At its first entry that is no larger than the one before, or no token of its request."""
    g = torch.Generator().manual_seed(2)
    c = make(g, 2, 16, 8, 4, idle=0.0)
    c["num"], c["entries"] = [4, 4], [entries, entries]
    check(dev, c, [_bytes(g, c["pages"], 16, 64), _bytes(g, c["pages"], 16, 16)])
    assert T.kept(c["ctx"][0], c["lens"][0], entries, 4, c["table"][0], 16, c["pages"])[1] == kept


def test_pages_that_are_none(dev):
    """Entries of the table below zero and past the caches, places past the table: the path ends there."""
    g = torch.Generator().manual_seed(3)
    for bad in (-1, -2 ** 31, 10 ** 6):
        c = make(g, 6, 4, 12, 6, hi=16, idle=0.0, room=6)
        for b in range(6):
            c["table"][b][b] = bad
        check(dev, c, [_bytes(g, c["pages"], 4, 64)])
    c = make(g, 4, 4, 12, 6, hi=24, idle=0.0, room=5)
    c["num"] = [6, 6, 100, -3]
    c["entries"] = [[0, 1, 2, 3, 4, 11]] * 4
    check(dev, c, [_bytes(g, c["pages"], 4, 64)])
    c["ctx"], c["lens"] = [2 ** 31 - 1, 2 ** 31 - 3, 0, -2 ** 31], [2 ** 31 - 1, 2 ** 31 - 1, 3, 5]
    check(dev, c, [_bytes(g, c["pages"], 4, 64)])


def test_many_caches_take_several_launches(dev):
    g = torch.Generator().manual_seed(4)
    c = make(g, 5, 4, 9, 4, hi=20, room=9)
    check(dev, c, [_bytes(g, c["pages"], 4, 16 + 12 * (i % 3)) for i in range(400)])


def test_strided_caches_of_any_type(dev):
    """Rows of one interleaved allocation, views of a per-layer storage, pages inside rows: nothing beside the rows is touched."""
    g = torch.Generator().manual_seed(5)
    c = make(g, 6, 16, 12, 5, room=7)
    both = torch.randn(c["pages"], 16, 576, generator=g).bfloat16()
    layers = torch.randn(3, c["pages"], 16, 2, 64, generator=g)
    inside = torch.randn(16, c["pages"], 8, generator=g).half()
    check(dev, c, [both, layers, inside], lambda x: [x[0][..., :512], *x[1], x[2].transpose(0, 1)])


def test_a_tuple_and_a_single_cache(dev):
    from omni_npu_amd import kernels as K
    z = torch.arange(64, device=dev).view(4, 4, 4).clone()
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device=dev)
    out = i32(0)
    for caches in ((z,), z, iter([z])):
        ref = z.clone()
        ref[1, 1] = z[1, 2]
        K.keep_rows(caches, i32(1).view(1, 1), i32(0), i32(4), i32(0, 2).view(1, 2), i32(2), out)
        assert torch.equal(z, ref) and out.item() == 2


def test_no_entries_and_no_requests(dev):
    from omni_npu_amd import kernels as K
    z = torch.zeros(4, 4, 4, device=dev)
    i32 = lambda *s: torch.zeros(*s, dtype=torch.int32, device=dev)
    out = i32(2)
    K.keep_rows([z], i32(2, 3), i32(2) + 5, i32(2) + 9, i32(2, 0), i32(2) + 3, out)
    assert out.tolist() == [5, 5]
    K.keep_rows([z], i32(0, 3), i32(0), i32(0), i32(0, 2), i32(0), i32(0))


def test_offsets_beyond_32_bits(dev):
    from omni_npu_amd import kernels as K
    if torch.cuda.mem_get_info()[0] < 30 << 30:
        pytest.skip("not enough memory free")
    pages = 2 ** 33 // (128 * 1024) + 9
    cache = torch.empty(pages, 128, 1024, dtype=torch.uint8, device=dev)
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device=dev)
    far = [pages - 1, pages - 5, 3]
    for p in far:
        cache[p] = torch.randint(0, 256, (128, 1024), dtype=torch.uint8, device=dev)
    before = {p: cache[p].clone() for p in far}
    K.keep_rows([cache], i32(*far).view(1, 3), i32(126), i32(126 + 140), i32(0, 1, 5, 135).view(1, 4), i32(4), out := i32(0))
    torch.cuda.synchronize()
    assert out.item() == 130
    want = {p: x.clone() for p, x in before.items()}
    want[far[1]][0], want[far[1]][1] = before[far[1]][3], before[far[2]][5]                # places 128 and 129 from 131 and 261
    assert all(torch.equal(cache[p], want[p]) for p in far)


def test_refusals(dev):
    from omni_npu_amd import kernels as K
    z = torch.zeros(4, 4, 4, device=dev)
    i32 = lambda *s: torch.zeros(*s, dtype=torch.int32, device=dev)
    base = [[z], i32(2, 3), i32(2), i32(2), i32(2, 2), i32(2), i32(2)]

    def refused(error, match, **swap):
        args = list(base)
        for i, x in swap.items():
            args[int(i[1:])] = x
        with pytest.raises(error, match=match):
            K.keep_rows(*args)

    refused(ValueError, "no caches", _0=[])
    refused(ValueError, "same pages", _0=[z, z[:3]])
    refused(ValueError, "no CPU path", _0=[z.cpu()])
    refused(ValueError, "share memory", _0=[z[:1].expand(4, 4, 4)])
    refused(ValueError, "block_table", _1=i32(1, 3))
    refused(ValueError, "context_lens", _2=i32(2).long())
    refused(ValueError, "seq_lens", _3=i32(3))
    refused(ValueError, "accepted", _4=i32(2))
    refused(ValueError, "num_accepted", _5=i32(2, 1))
    refused(ValueError, "kept_lens", _6=i32(1))
    refused(K._lib.MlaHipError, "shares memory", _6=base[2])
    refused(K._lib.MlaHipError, "shares memory", _6=base[4].view(-1)[1:3])
    refused(RuntimeError, "no backward", _0=[z.clone().requires_grad_()])
