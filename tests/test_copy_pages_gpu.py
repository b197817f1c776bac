"""Pages copied, forked and moved in many caches at once: the bytes of the plain assignment, everything else left as it was."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def _bytes(g, *shape):
    return torch.randint(0, 256, shape, generator=g, dtype=torch.uint8)


def _plain(caches, src, dst, rows):
    out = [c.clone() for c in caches]
    for c, old in zip(out, caches):
        for i, (a, b) in enumerate(zip(src, dst)):
            n = c.shape[1] if rows is None else rows[i]
            c[b, :n] = old[a, :n]
    return out


@pytest.mark.parametrize("page,widths", [(128, [1024, 128]), (16, [256]), (128, [656]), (64, [4, 12, 128]), (7, [1, 3, 2, 16]), (1, [16])])
@pytest.mark.parametrize("pairs", [1, 5, 200])
@pytest.mark.parametrize("part", [False, True])
def test_copies(dev, page, widths, pairs, part):
    from omni_npu_amd import kernels as K
    g = torch.Generator().manual_seed(page + pairs)
    pages = 2 * pairs + 3
    caches = [_bytes(g, pages, page, w) for w in widths]
    order = torch.randperm(pages, generator=g).tolist()
    src, dst = [order[i % (pairs // 2 + 1)] for i in range(pairs)], order[-pairs:]     # (sources may repeat)
    rows = [int(i) for i in torch.randint(0, page + 1, (pairs,), generator=g)] if part else None
    on = [c.to(dev) for c in caches]
    K.copy_pages(on, src, dst, rows)
    for got, ref in zip(on, _plain(caches, src, dst, rows)):
        assert torch.equal(got.cpu(), ref)


def test_many_caches_take_several_launches(dev):
    from omni_npu_amd import kernels as K
    g = torch.Generator().manual_seed(1)
    caches = [_bytes(g, 40, 4, 16 + 16 * (i % 3)) for i in range(400)]
    on = [c.to(dev) for c in caches]
    src, dst = list(range(15)), list(range(20, 35))
    K.copy_pages(on, torch.tensor(src), torch.tensor(dst), torch.tensor([i % 5 for i in range(15)]))
    for got, ref in zip(on, _plain(caches, src, dst, [i % 5 for i in range(15)])):
        assert torch.equal(got.cpu(), ref)


def test_strided_caches_of_any_type(dev):
    """Rows of one interleaved allocation, views of a per-layer storage, a cache of one page size 1: nothing beside the rows is touched."""
    from omni_npu_amd import kernels as K
    g = torch.Generator().manual_seed(2)
    both = torch.randn(10, 32, 576, generator=g).bfloat16()
    layers = torch.randn(3, 10, 32, 2, 64, generator=g)
    on, lay = both.to(dev), layers.to(dev)
    K.copy_pages([on[..., :512], *lay], [1, 2], [5, 9], rows=[32, 7])
    both[5, :, :512] = both[1, :, :512]
    both[9, :7, :512] = both[2, :7, :512]
    layers[:, 5] = layers[:, 1]
    layers[:, 9, :7] = layers[:, 2, :7]
    assert torch.equal(on.cpu(), both) and torch.equal(lay.cpu(), layers)


@pytest.mark.parametrize("pairs", [1, 30, 300])
def test_moves_rewrite_the_table(dev, pairs):
    from omni_npu_amd import kernels as K
    g = torch.Generator().manual_seed(pairs)
    pages = 2 * pairs + 5
    caches = [_bytes(g, pages, 16, 64) for _ in range(3)]
    order = torch.randperm(pages, generator=g)
    src, dst = order[:pairs].tolist(), order[pairs:2 * pairs].tolist()
    wide = torch.randint(-1, pages + 2, (9, 21), generator=g, dtype=torch.int32)
    on, table = [c.to(dev) for c in caches], wide.to(dev)
    K.copy_pages(on, src, dst, block_table=table[:7, 2:19])
    ref = wide.clone()
    to = {a: b for a, b in zip(src, dst)}
    for i in range(7):
        for j in range(2, 19):
            ref[i, j] = to.get(int(wide[i, j]), int(wide[i, j]))
    assert torch.equal(table.cpu(), ref)
    for got, want in zip(on, _plain(caches, src, dst, None)):
        assert torch.equal(got.cpu(), want)


def test_far_pages(dev):
    """Offsets beyond 2^32 bytes."""
    from omni_npu_amd import kernels as K
    cache = torch.zeros(5000, 128, 8192, dtype=torch.uint8, device=dev)      # 5.2 GB
    cache[4999].fill_(9)
    cache[4100].fill_(5)
    K.copy_pages(cache, [4999, 4100], [1, 4998])
    assert (cache[1] == 9).all() and (cache[4998] == 5).all() and (cache[2] == 0).all() and (cache[4997] == 0).all()


def test_nothing_to_copy_and_replays(dev):
    from omni_npu_amd import kernels as K
    c = torch.arange(6 * 4 * 16, device=dev, dtype=torch.int32).view(6, 4, 16)
    ref = c.clone()
    K.copy_pages(c, [], [])
    assert torch.equal(c, ref)
    K.copy_pages(c, [0], [1], [0])
    assert torch.equal(c, ref)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        K.copy_pages(c, [2, 3], [4, 5])
    for i in range(3):
        c.add_(i + 1)
        ref = c.clone()
        graph.replay()
        torch.cuda.synchronize()
        ref[4], ref[5] = ref[2].clone(), ref[3].clone()
        assert torch.equal(c, ref)


def test_refusals(dev):
    from omni_npu_amd import kernels as K
    c = torch.zeros(6, 4, 16, device=dev)

    def refused(err, match, *args, **kw):
        with pytest.raises(err, match=match):
            K.copy_pages(*args, **kw)

    refused(ValueError, "pair 1", c, [0, 6], [1, 2])
    refused(ValueError, "pair 0", c, [0], [-1])
    refused(ValueError, "destination", c, [0, 1], [2, 2])
    refused(ValueError, "destination", c, [0, 1], [1, 2])
    refused(ValueError, "destination", c, [3], [3])
    refused(ValueError, "1 destinations", c, [0, 1], [2])
    refused(ValueError, "rows of", c, [0], [1], [5])
    refused(ValueError, "on the host", c, torch.tensor([0], device=dev), [1])
    refused(ValueError, "same pages", [c, c[:5]], [0], [1])
    refused(ValueError, "contiguous rows", c[..., ::2], [0], [1])
    refused(ValueError, "share memory", c[:1].expand(6, 4, 16), [0], [1])
    refused(ValueError, "moved whole", c, [0], [1], [2], torch.zeros(2, 2, dtype=torch.int32, device=dev))
    refused(ValueError, "int32", c, [0], [1], block_table=torch.zeros(2, 2, device=dev))
    refused(TypeError, "whole numbers", c, [0.0], [1])
    refused(ValueError, "no CPU path", c.cpu(), [0], [1])


@pytest.mark.parametrize("part", [False, True])
@pytest.mark.parametrize("widths", [[1024, 1024], [1024, 128], [656, 656]])
def test_copies_that_go_past_the_caches(dev, part, widths):
    """32 MB and more: whole pages and filled rows, caches of one size and of two, a table that follows."""
    from omni_npu_amd import kernels as K
    g = torch.Generator(device=dev).manual_seed(7)
    pairs, page = 400, 128
    pages = 2 * pairs + 5
    caches = [torch.randint(0, 256, (pages, page, w), generator=g, device=dev, dtype=torch.uint8) for w in widths]
    order = torch.randperm(pages, generator=g, device=dev)
    src, dst = order[:pairs], order[pairs:2 * pairs]
    rows = torch.randint(0, page + 1, (pairs,), generator=g, device=dev) if part else None
    table = None if part else torch.randint(0, pages, (37, 65), generator=g, device=dev, dtype=torch.int32)
    want = [c.clone() for c in caches]
    for c, old in zip(want, caches):
        keep = torch.arange(page, device=dev)[None, :, None] >= (rows[:, None, None] if part else page)
        c[dst] = torch.where(keep, old[dst], old[src])
    if table is not None:
        follow = torch.arange(pages, device=dev, dtype=torch.int32)
        follow[src] = dst.int()
        want_table = follow[table.long()]
    K.copy_pages(caches, src.tolist(), dst.tolist(), rows.tolist() if part else None, table)
    for got, ref in zip(caches, want):
        assert torch.equal(got, ref)
    assert table is None or torch.equal(table, want_table)
