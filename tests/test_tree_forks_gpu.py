"""A fork beside a list of free pages, as the documents have it: pages of its own by a step without tokens, copied into; either request may end first."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("first", [0, 1])
@pytest.mark.parametrize("context", [1, 16, 37, 48])
def test_a_fork_keeps_its_pages_when_the_other_ends(dev, first, context):
    from omni_npu_amd import kernels as K
    page, room, pages = 16, 6, 24
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device=dev)
    g = torch.Generator().manual_seed(context)
    caches = [torch.randint(0, 256, (pages, page, n), generator=g, dtype=torch.uint8).to(dev) for n in (32, 48)]
    free, count = torch.randperm(pages, generator=g).to(torch.int32).to(dev), i32(pages)
    table, held, lens = torch.full((3, room), -1, dtype=torch.int32, device=dev), i32(0, 0, 0), i32(0, 0, 0)
    none = torch.zeros(0, dtype=torch.int64, device=dev)

    def step(ctx, tokens=(0, 0, 0)):
        start = i32(0, *torch.tensor(tokens).cumsum(0).tolist())
        n = sum(tokens)
        K.step_tables(i32(*ctx), table, page, lens, none.new_zeros(n), none.new_zeros(n), query_start_loc=start, num_blocks=held, free_pages=free, num_free=count)

    step((context, -1, -1))
    step((context, context, -1))                              # the fork's place: a context, no tokens, no pages
    assert lens.tolist() == [context, context, 0] and held[0] == held[1] == -(-context // page)
    src, dst = (table[b, :held[b]].tolist() for b in (0, 1))
    assert len(set(src + dst)) == 2 * len(src)
    K.copy_pages(caches, src, dst, rows=[page] * (len(src) - 1) + [context - page * (len(src) - 1)])
    read = lambda b: [c[table[b, :held[b]].long()].flatten(0, 1)[:context].clone() for c in caches]
    want = read(0)
    assert all(torch.equal(x, y) for x, y in zip(read(1), want))
    stays = 1 - first
    step([context if b == stays else -1 for b in range(2)] + [-1])
    assert held[first] == 0 and count.item() == pages - len(src)
    step([context if b == stays else -1 for b in range(2)] + [0], (0, 0, page * room))       # a third one takes what has come back
    assert not set(table[2, :held[2]].tolist()) & set(table[stays, :held[stays]].tolist())
    for c in caches:
        c[table[2, :held[2]].long()] = 0
    assert all(torch.equal(x, y) for x, y in zip(read(stays), want))
