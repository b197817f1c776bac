"""Pages that go back to the list in numbers: requests that end with hundreds and thousands of them."""
import pytest
import torch

from tests.test_step_tables_gpu import Case, run

pytestmark = pytest.mark.gpu


class Ending(Case):
    """Requests that hold ``held`` pages each, in turn, of which some end."""

    def __init__(self, seed, batch, held, ends, page=16, spare=7, capacity=None, q_len=1, tree=False):
        room = max(held) + 2
        super().__init__(seed, batch, page=page, room=room, q_len=q_len, spare=spare, tree=tree, idle=0.0)
        g = torch.Generator().manual_seed(seed + 1)
        self.held = [held[b % len(held)] for b in range(batch)]
        self.ctx = [-1 if ends(b) else max(0, (h - 1) * page - q_len) for b, h in enumerate(self.held)]
        used = sum(self.held)
        order = torch.randperm(used + spare, generator=g).tolist()
        at, self.table = 0, []
        for h in self.held:
            self.table.append(order[at:at + h] + [-7] * (room - h))
            at += h
        capacity = used + spare if capacity is None else capacity
        self.free, self.num_free = (order[at:] + [-9] * capacity)[:capacity], min(spare, capacity)


@pytest.mark.parametrize("batch,held", [(1, [512]), (1, [8192]), (4, [8192, 1, 0, 3]), (64, [512, 2, 511, 1, 0]), (1024, [1, 2]), (1500, [3, 0, 40, 1, 2]), (3, [1025, 1, 1024])])
@pytest.mark.parametrize("which", ["all", "some", "first", "last"])
def test_requests_that_end(dev, batch, held, which):
    """All of a request's pages, of several with others between, next to requests that give one page back or two."""
    ends = {"all": lambda b: True, "some": lambda b: b % 3 != 1, "first": lambda b: b == 0, "last": lambda b: b == batch - 1}[which]
    run(dev, Ending(batch, batch, held, ends))
    run(dev, Ending(batch, batch, held, ends, q_len=3, tree=True, page=7))


@pytest.mark.parametrize("capacity", [0, 7, 500, 1030, 1500, 3000])
@pytest.mark.parametrize("batch", [20, 1100])
def test_a_list_without_room_for_all(dev, capacity, batch):
    """From the first request on that it has no room for, it takes none back."""
    run(dev, Ending(3, batch, [500, 2, 40, 1], lambda b: b % 5 != 2, capacity=capacity))


def test_pages_that_go_back_are_taken_by_others(dev):
    """A request ends with a thousand pages, which those behind it need in the same step."""
    case = Ending(5, 6, [1000, 0, 0, 0, 0, 0], lambda b: b == 0, spare=0)
    case.ctx = [-1] + [16 * 190] * 5
    run(dev, case)


def test_giving_back_takes_as_long_as_taking(dev):
    """8192 pages of one request, the list's in its table's place: a page to a thread either way."""
    from omni_npu_amd import kernels as K
    n, page = 8192, 16
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device=dev)
    pages = torch.randperm(n, generator=torch.Generator().manual_seed(1)).to(torch.int32).to(dev)
    table, free = pages[None].clone(), pages.clone()
    seq, positions, slots = i32(0), torch.zeros(1, dtype=torch.int64, device=dev), torch.zeros(1, dtype=torch.int64, device=dev)

    def us(ctx, held, count):
        best, context = float("inf"), i32(ctx)
        for _ in range(10):
            num_blocks, num_free = i32(held), i32(count)
            start, end = torch.cuda.Event(True), torch.cuda.Event(True)
            torch.cuda.synchronize()
            start.record()
            K.step_tables(context, table, page, seq, positions, slots, num_blocks=num_blocks, free_pages=free, num_free=num_free)
            end.record()
            torch.cuda.synchronize()
            best = min(best, start.elapsed_time(end) * 1e3)
        return best

    take, give = us(n * page - 1, 0, n), us(-1, n, 0)
    assert give < 2 * take + 20, (take, give)


@pytest.mark.parametrize("left", [0, 2, 9, 10, 4000])
def test_a_list_of_two_thousand_million_pages(dev, left):
    """Pages on the list and pages that go back are more than 2^31 together: from the first request that they do not fit for on, none go back."""
    from omni_npu_amd import kernels as K
    most = 2 ** 31 - 1
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device=dev)
    free = torch.empty(most, dtype=torch.int32, device=dev)
    free[-5000:] = 7
    held, table = [4, 6, 4001], torch.arange(3 * 4001, dtype=torch.int32, device=dev).view(3, 4001)
    num_blocks, num_free, seq = i32(*held), i32(most - left), i32(5, 5, 5)
    rows = lambda: torch.zeros(3, dtype=torch.int64, device=dev)
    K.step_tables(i32(-1, -1, -1), table, 16, seq, rows(), rows(), num_blocks=num_blocks, free_pages=free, num_free=num_free)
    back, given = [], 0
    for b, h in enumerate(held):
        given += h
        if given <= left:
            back += table[b, :h].tolist()
            held[b] = 0
    want = [7] * 5000
    want[5000 - left:5000 - left + len(back)] = back[::-1]
    assert num_blocks.tolist() == held and num_free.tolist() == [most - left + len(back)] and seq.tolist() == [0, 0, 0]
    assert free[-5000:].tolist() == want
