"""Plain statements of what a step over drafted trees runs: tables from lengths, attention where each token sees the context and its ancestors, the
accepted path's rows.  Test infrastructure only."""
import torch


def ancestors(parents):
    """Sets of token numbers: each token and what its parents lead to (a parent that is not in front of its token is none)."""
    out = []
    for i, up in enumerate(parents):
        out.append((out[up] if 0 <= up < i else set()) | {i})
    return out


def words(sets, n):
    """Bit rows int64 [len(sets), n]."""
    rows = []
    for s in sets:
        row = [0] * n
        for k in s:
            if k < 64 * n:
                row[k // 64] |= 1 << k % 64
        rows.append([w - (1 << 64) if w >> 63 else w for w in row])
    return torch.tensor(rows, dtype=torch.int64).view(len(sets), n)


def seen(visible, n, s, window=0):
    """[s, n] truth values: which of a request's n keys its s tokens see.  visible [s, W]."""
    out = torch.zeros(s, max(n, 0), dtype=torch.bool)
    for i in range(s):
        row = [w & (1 << 64) - 1 for w in visible[i].tolist()]
        keys = list(range(max(0, n - s))) + [n - s + k for k in range(min(s, 64 * len(row))) if row[k // 64] >> k % 64 & 1 and n - s + k >= 0]
        out[i, keys[-window:] if window else keys] = True
    return out


def gqa(q, k_cache, v_cache, block_table, seq_lens, visible, scale, q_start, window=0, k_scale=None, v_scale=None):
    """As heads_oracle.gqa, with a tree's masks: (o, lse, weight, reach) in fp64."""
    t, hq, d = q.shape
    page, hk = k_cache.shape[1], k_cache.shape[2]
    grp = hq // hk
    o, lse = torch.zeros(t, hq, d, dtype=torch.float64), torch.full((t, hq), -torch.inf, dtype=torch.float64)
    weight, reach = torch.zeros(t, hq, d, dtype=torch.float64), torch.zeros(t, hq, dtype=torch.float64)
    for b, n in enumerate(seq_lens.tolist()):
        n = max(0, min(n, block_table.shape[1] * page))
        t0, t1 = int(q_start[b]), int(q_start[b + 1])
        pos = torch.arange(n)
        rows = block_table[b].long()[pos // page] * page + pos % page
        k, v = (c.flatten(0, 1)[rows].double() for c in (k_cache, v_cache))
        if k_scale is not None:
            k = k * k_scale.double()[:, None]
        if v_scale is not None:
            v = v * v_scale.double()[:, None]
        sees = seen(visible[t0:t1], n, t1 - t0, window)
        for i in range(t1 - t0):
            at = sees[i].nonzero()[:, 0]
            if at.numel() == 0:
                continue
            for h in range(hk):
                heads = slice(h * grp, (h + 1) * grp)
                qq, kk, vv = q[t0 + i, heads].double(), k[at, h], v[at, h]
                s = qq @ kk.t() * scale
                top = s.amax(1, keepdim=True)
                p = torch.exp(s - top)
                tot = p.sum(1, keepdim=True)
                o[t0 + i, heads] = p @ vv / tot
                lse[t0 + i, heads] = (top + tot.log())[:, 0]
                weight[t0 + i, heads] = p @ vv.abs() / tot
                reach[t0 + i, heads] = (qq.abs() @ kk.abs().t()).amax(1) * abs(scale)
    return o, lse, weight, reach


def step_tables(ctx, counts, table, page, total, parents=None, n_words=0, held=None, free=None, num_free=0):
    """Lists of whole numbers: dict(seq_lens, positions, slots, words, table, held, free, num_free)."""
    table, room = [list(r) for r in table], len(table[0]) if table else 0
    lens = [0 if c < 0 else c + n for c, n in zip(ctx, counts)]
    fits = [True] * len(ctx)
    if held is not None:
        held, free = [min(max(h, 0), room) for h in held], list(free)
        num_free = min(max(num_free, 0), len(free))
        need = [-(-n // page) for n in lens]
        back, given = [], 0
        for b, n in enumerate(need):
            if n < held[b]:
                given += held[b] - n
                if num_free + given <= len(free):
                    back += table[b][n:held[b]]
                    held[b] = n
        free[num_free:num_free + len(back)] = back[::-1]
        num_free += len(back)
        top, taken = num_free, 0
        for b, n in enumerate(need):
            if n > room:
                fits[b] = False
            elif n > held[b]:
                taken += n - held[b]
                if taken > top:
                    fits[b] = False
                    continue
                while held[b] < n:
                    num_free -= 1
                    table[b][held[b]] = free[num_free]
                    held[b] += 1
    positions, slots, sees, t = [0] * total, [-1] * total, [set() for _ in range(total)], 0
    for b, n in enumerate(counts):
        up = parents[t:t + n] if parents is not None else [i - 1 for i in range(n)]
        line = ancestors(up)
        for i in range(n):
            if t + i < total and ctx[b] >= 0:
                positions[t + i] = ctx[b] + len(line[i]) - 1
                at = ctx[b] + i
                if fits[b] and at // page < room and table[b][at // page] >= 0:
                    slots[t + i] = table[b][at // page] * page + at % page
                sees[t + i] = line[i]
        t += n
    return dict(seq_lens=[n if ok else c for n, c, ok in zip(lens, ctx, fits)], positions=positions, slots=slots,
                words=words(sees, n_words) if parents is not None else None, table=table, held=held, free=free, num_free=num_free)


def kept(ctx, n, entries, num, table, page, num_pages):
    """The rows (from, to) of one request's path as (page, row) pairs, and how many of its entries count."""
    if ctx < 0:
        return [], 0
    place = lambda x: (table[x // page], x % page) if 0 <= x // page < len(table) and 0 <= table[x // page] < num_pages else None
    moves, last = [], -1
    for d, a in enumerate(entries[:max(0, num)]):
        if a <= last or ctx + a >= n or place(ctx + a) is None or place(ctx + d) is None:
            break
        moves.append((place(ctx + a), place(ctx + d)))
        last = a
    return moves, len(moves)
