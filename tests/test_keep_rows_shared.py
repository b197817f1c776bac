"""CPU: caches of one call that share memory are refused, whatever their strides; those that only lie between each other are not."""
import ctypes
import random

import pytest

from omni_npu_amd import _lib

PAGES, PAGE = 6, 5


def call(caches, pages=PAGES, page=PAGE):
    """caches: (offset, page stride, row stride, bytes of a row); the entry's answer for a batch of none, which launches nothing."""
    lib = _lib.load()
    base = 1 << 40
    words = (ctypes.c_int64 * (4 * len(caches)))(*(x for at, *geometry in caches for x in (base + at, *geometry)))
    rc = lib.mlahip_keep_rows(words, len(caches), pages, page, None, 1, 1, None, None, 0, None, 0, 0, None, None, None)
    return rc, lib.mlahip_last_error_string().decode()


def taken(cache, pages=PAGES, page=PAGE):
    at, ps, rs, n = cache
    return {at + p * ps + r * rs + i for p in range(pages) for r in range(page) for i in range(n)}


def meet(caches, pages=PAGES, page=PAGE):
    sets = [taken(c, pages, page) for c in caches]
    return any(sets[i] & sets[k] for i in range(len(sets)) for k in range(i))


# of one storage: pages of rows of bytes
ROW, PAGE_B = 64, 64 * PAGE


@pytest.mark.parametrize("caches,fine", [
    ([(0, PAGE_B, ROW, 64), (0, PAGE_B, ROW, 64)], False),                            # the same twice
    ([(0, PAGE_B, ROW, 48), (48, PAGE_B, ROW, 16)], True),                            # parts of a row side by side
    ([(0, PAGE_B, ROW, 64), (48, PAGE_B, ROW, 16)], False),                           # a row and its last bytes
    ([(48, PAGE_B, ROW, 16), (0, PAGE_B, ROW, 49)], False),
    ([(0, PAGE_B, ROW, 64), (PAGE_B, PAGE_B, ROW, 64)], False),                       # pages 0 to 5 and 1 to 6 of one cache
    ([(0, PAGE_B, ROW, 64), (PAGES * PAGE_B, PAGE_B, ROW, 64)], True),                # one behind the other
    ([(0, 2 * PAGE_B, ROW, 64), (PAGE_B, 2 * PAGE_B, ROW, 64)], True),                # keys and values of one storage, page by page
    ([(0, 2 * PAGE_B, ROW, 64), (PAGE_B - 1, 2 * PAGE_B, ROW, 64)], False),
    ([(0, PAGE_B, ROW, 64), (3, PAGE_B, ROW, 1)], False),
    ([(0, 1000, 100, 10), (500, 1000, 20, 20)], True),                                # keys, then their scales, in a page of both
    ([(0, 1000, 100, 10), (409, 1000, 20, 20)], False),
    ([(0, 1000, 100, 10), (10, 1000, 20, 8)], True),                                  # rows of other strides between rows
    ([(0, 1000, 100, 10), (10, 1000, 24, 8)], False),                                 # (the last one reaches the second row)
    ([(0, 1000, 100, 10), (12, 1000, 50, 30)], True),
    ([(0, 16, 16 * PAGES, 16), (16 * PAGES * PAGE, 16, 16 * PAGES, 16)], True),       # pages inside rows
    ([(0, 16, 32 * PAGES, 16), (16 * PAGES, 16, 32 * PAGES, 16)], True),
    ([(0, 16, 32 * PAGES, 16), (16 * PAGES - 8, 16, 32 * PAGES, 16)], False),
], ids=str)
@pytest.mark.parametrize("turned", [False, True])
def test_two_caches(caches, fine, turned):
    assert meet(caches) != fine
    rc, said = call(caches[::-1] if turned else caches)
    assert (rc == 0) == fine and (fine or rc == -3 and "caches 0 and 1 share memory" in said)


@pytest.mark.parametrize("layers", [1, 40, 300])
def test_all_layers_of_one_storage(layers):
    """[pages, layers, 2, page, row], [pages, page, layers, row] and [layers, pages, page, row]; one that begins a byte early among them."""
    for caches in ([(i * PAGE_B, 2 * layers * PAGE_B, ROW, ROW) for i in range(2 * layers)],
                   [(i * ROW, layers * PAGE_B, layers * ROW, ROW) for i in range(layers)],
                   [(i * PAGES * PAGE_B, PAGE_B, ROW, ROW) for i in range(layers)]):
        random.Random(layers).shuffle(caches)
        assert call(caches)[0] == 0
        if layers > 1:
            at = next(i for i, c in enumerate(caches) if c[0] > 0)
            wrong = caches[:at] + [(caches[at][0] - 1, *caches[at][1:])] + caches[at + 1:]
            rc, said = call(wrong)
            assert rc == -3 and f" {at} " in said


@pytest.mark.parametrize("seed", range(40))
def test_any_layouts(seed):
    """As by their bytes; caches whose blocks lie differently far apart are refused where one begins in the other."""
    g = random.Random(seed)
    seen = set()
    for _ in range(60):
        pages, page = g.choice([(1, 4), (3, 1), (4, 3), (2, 5), (1, 1)])
        row_stride = g.randint(1, 12)
        inside = g.random() < 0.2 and pages > 1 and page > 1       # (pages inside rows)
        caches = []
        apart = g.randint(20, 90)
        for _ in range(g.randint(2, 4)):
            inner = row_stride if g.random() < 0.6 else g.randint(1, 12)
            n = g.randint(1, min(inner, 5))
            outer = max(apart, ((pages if inside else page) - 1) * inner + n) + (0 if g.random() < 0.8 else g.randint(1, 9))
            caches.append((g.randint(0, 160), *((inner, outer) if inside else (outer, inner)), n))
        rc, said = call(caches, pages, page)
        outers = {c[2] if inside or pages == 1 else c[1] for c in caches}
        ends = [max(taken(c, pages, page)) for c in caches]
        near = any(a[0] <= z and b[0] <= y for i, (a, y) in enumerate(zip(caches, ends)) for b, z in list(zip(caches, ends))[:i])
        really = meet(caches, pages, page)
        if len(outers) == 1:
            assert (rc != 0) == really, (caches, pages, page)
        else:
            assert rc != 0 if really else rc == 0 or near, (caches, pages, page)
        assert rc in (0, -3) and (rc == 0 or "share memory" in said)
        seen.add(rc)
    assert seen == {0, -3}


def test_what_ends_past_all_addresses():
    rc, said = call([(0, 1 << 62, 16, 16)])
    assert rc == -2 and "past all addresses" in said
