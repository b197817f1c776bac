"""The operators of a speculative step, as cases that can be timed and compared: several tokens of each request are drafted as a tree,
attended at once, and the rows of the path that is kept move up behind the context.

``tables``: what a step reads besides its queries, made on the GPU from the requests' lengths.  Pages out of a list of free ones into the
block tables (and back, where a request got shorter), sequence lengths, positions, slots, and for drafted trees which tokens each token sees.
``attend``: attention of the drafted tokens over the paged cache of ordinary key and value heads, each seeing the whole context and its own
ancestors, whole contexts or a sliding window.
``keep``: the rows of the accepted path moved to the places behind the context, in all layers' caches at once.

Where ``own`` is true the calls are this package's; where it is false the same is computed by elementary torch operations, sums in 32
bits, rounded once.
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
GOLDEN = 0.6180339887498949


def _tables(name=None, batch=1, q_len=1, ragged=False, lo=1, hi=1, page=128, tree=False, pages=True, idle=0, room=0, padded=0, ended=0):
    case = dict(op="tables", batch=batch, q_len=q_len, ragged=ragged, lo=lo, hi=hi, page=page, tree=tree, pages=pages, idle=idle, room=room,
                padded=padded, ended=ended)
    return case if name is None else dict(name=name, **case)


def _attend(name=None, batch=1, q_len=8, ragged=False, lo=1, hi=1, q_heads=32, kv_heads=8, dim=128, dtype="bf16", cache="same", page=128,
            window=0, idle=0, room=0):
    case = dict(op="attend", batch=batch, q_len=q_len, ragged=ragged, lo=lo, hi=hi, q_heads=q_heads, kv_heads=kv_heads, dim=dim, dtype=dtype,
                cache=cache, page=page, window=window, idle=idle, room=room)
    return case if name is None else dict(name=name, **case)


def _keep(name=None, batch=1, q_len=8, kept=4, layers=1, page=128, heads=1, wide=512, narrow=64, context=1000):
    case = dict(op="keep", batch=batch, q_len=q_len, kept=kept, layers=layers, page=page, heads=heads, wide=wide, narrow=narrow,
                context=context)
    return case if name is None else dict(name=name, **case)


def listed():
    return [
        # one user's next token, nothing drafted: the smallest call there is, latency alone
        _tables("tables_one_token", batch=1, lo=1020, hi=1020, room=8192),
        # a decode batch with a drafted tree for each request, places of a captured graph left idle, a few requests just ended
        _tables("tables_tree_batch", batch=64, q_len=26, lo=4096, hi=8192, page=16, tree=True, idle=3, room=16384, ended=2),
        # trees of any size up to 64 tokens, many requests, in rows padded to a captured graph's size
        _tables("tables_tree_ragged", batch=500, q_len=64, ragged=True, lo=1, hi=6000, page=64, tree=True, room=8192, padded=77),
        # a prefill step: prompts of any length, most of their pages still to be taken
        _tables("tables_prompts", batch=9, q_len=16384, ragged=True, lo=0, hi=2000, room=32768),
        # one user in a chat, a small tree, on a rank of eight: latency alone
        _attend("tree_one_user", batch=1, q_len=8, lo=1021, hi=1021, q_heads=4, kv_heads=1, room=8192),
        # the benchmark's decode batch, 64 requests of 4k-8k tokens, eight drafted tokens each
        _attend("tree_batch", batch=64, q_len=8, lo=4096, hi=8192, room=8192),
        # few users and wide trees: 60 tokens a step
        _attend("tree_wide", batch=8, q_len=60, lo=2048, hi=16384, q_heads=64, kv_heads=8, room=16384),
        # throughput serving over the 8-bit cache, trees of 26 tokens, a graph's idle places
        _attend("tree_fp8", batch=32, q_len=26, lo=1024, hi=8192, q_heads=32, kv_heads=4, cache="fp8", idle=2, room=16384),
        # sliding-window layers with wide heads and small pages, fp16, trees of one to seven tokens
        _attend("tree_window", batch=33, q_len=7, ragged=True, lo=300, hi=9000, q_heads=16, kv_heads=4, dim=256, dtype="fp16", page=16,
                window=1024, room=16384),
        # one user's accepted tokens, a small model's layers: latency alone
        _keep("keep_one_user", batch=1, q_len=8, kept=3, layers=16, heads=2, wide=256, narrow=256),
        # a decode batch over a latent cache
        _keep("keep_latent_batch", batch=64, q_len=26, kept=5, layers=27),
        # throughput serving, wide rows, small pages
        _keep("keep_wide_batch", batch=256, q_len=60, kept=9, layers=32, page=16, heads=8, wide=1024, narrow=1024),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    """One more call of the same kinds, at sizes all over what the list spans."""
    op = rng.choice(["tables", "attend", "attend", "keep"])
    most = max(_cost(c) for c in listed() if c["op"] == op)
    while True:
        if op == "tables":
            tree = rng.random() < 0.6
            batch, hi = _log(rng, 1, 500), _log(rng, 20, 131072)
            c = _tables(batch=batch, q_len=_log(rng, 1, 128 if tree else 16384), ragged=rng.random() < 0.5, lo=rng.randint(0, hi), hi=hi,
                        page=rng.choice([16, 64, 128]), tree=tree, pages=rng.random() < 0.7, idle=rng.choice([0, 0, 3]), room=0,
                        padded=rng.choice([0, 0, 5]), ended=rng.choice([0, 0, 1]))
            c["room"] = -(-(hi + c["q_len"]) // 1024) * 1024
        elif op == "attend":
            kv = rng.choice([1, 2, 3, 4, 8])
            hi = _log(rng, 40, 65536)
            c = _attend(batch=_log(rng, 1, 64), q_len=_log(rng, 1, 128), ragged=rng.random() < 0.3, lo=rng.randint(max(hi // 8, 1), hi), hi=hi,
                        q_heads=kv * rng.choice([1, 2, 4, 5, 8, 16]), kv_heads=kv, dim=rng.choice([64, 128, 128, 256]),
                        dtype=rng.choice(["bf16", "bf16", "fp16"]), cache=rng.choice(["same", "same", "fp8"]),
                        page=rng.choice([16, 64, 128]), window=rng.choice([0, 0, 0, _log(rng, 20, 4096)]), idle=rng.choice([0, 0, 2]),
                        room=max(1024, 1 << (hi - 1).bit_length()))
        else:
            wide, narrow, heads = rng.choice([(512, 64, 1), (1024, 1024, 8), (128, 128, 2), (656, 0, 1)])
            q_len = _log(rng, 2, 64)
            c = _keep(batch=_log(rng, 1, 256), q_len=q_len, kept=rng.randint(1, min(12, (q_len + 1) // 2)), layers=rng.randint(1, 61),
                      page=rng.choice([16, 64, 128]), heads=heads, wide=wide, narrow=narrow, context=_log(rng, 1, 8192))
        if _cost(c) <= most and _room(c) <= 8e9:
            return c


def _spread(n, lo, hi, first):
    """n whole numbers all over lo .. hi, the first one given."""
    return [first] + [lo + round((hi - lo) * ((i * GOLDEN) % 1.0)) for i in range(1, n)]


def _tokens(case):
    """How many tokens each request has in the step (idle places of a ragged step have none)."""
    n = case["batch"]
    lens = _spread(n, 1, case["q_len"], case["q_len"]) if case["ragged"] else [case["q_len"]] * n
    if case["ragged"] and case["op"] == "tables" and not case["tree"]:  # (prompts: all of them together are one step's tokens)
        lens = [max(1, x * case["q_len"] // sum(lens)) for x in lens]
    return lens + [0 if case["ragged"] else case["q_len"]] * case["idle"]


def _contexts(case):
    """Cached tokens of each request in front of the step; -1: an idle place."""
    return _spread(case["batch"], case["lo"], case["hi"], case["hi"]) + [-1] * case["idle"]


def _lengths(case):
    """Lengths with the step's tokens, of which lo .. hi are the range."""
    n = [max(x, t) for x, t in zip(_spread(case["batch"], case["lo"], case["hi"], case["hi"]), _tokens(case))]
    return n + [0] * case["idle"]


def _kept(case):
    return _spread(case["batch"], 1, case["kept"], case["kept"])


def work(case):
    if case["op"] == "tables":
        tokens, ctx = _tokens(case), _contexts(case)
        places, b = sum(tokens) + case["padded"], len(tokens)
        taken = sum(-(-n // case["page"]) for n, c in zip(tokens, ctx) if c >= 0)
        nbytes = places * (16 + (12 if case["tree"] else 0)) + b * (12 if case["ragged"] else 8) + taken * 4
        if case["pages"]:
            nbytes += b * 4
        return {"bytes": nbytes, "flops": 0}
    if case["op"] == "attend":
        es = 1 if case["cache"] == "fp8" else 2
        d, hq, hk, w = case["dim"], case["q_heads"], case["kv_heads"], case["window"]
        tokens, lens = _tokens(case), _lengths(case)
        seen = [min(n, w + t - 1) if w else n for n, t in zip(lens, tokens)]
        nbytes = sum(seen) * 2 * hk * d * es + sum(tokens) * (hq * d * 4 + 8) + sum(-(-n // case["page"]) for n in seen) * 4
        pairs = sum(t * (min(n - t + 1, w) if w else n - t + 1) for n, t in zip(lens, tokens) if n)
        return {"bytes": nbytes, "flops": 4 * pairs * hq * d}
    row = case["layers"] * (case["wide"] + case["narrow"]) * (1 if case["wide"] == 656 else 2)
    return {"bytes": 2 * sum(n - 1 for n in _kept(case)) * row + case["batch"] * 20, "flops": 0}


def _cost(case):
    w = work(case)
    return max(w["bytes"] / 5e12, w["flops"] / 5e14)


def _room(case):
    if case["op"] == "attend":  # the keys, values and scores that the plain form lays out in 32 bits
        return (case["batch"] + case["idle"]) * case["hi"] * max(case["kv_heads"] * case["dim"] * 2, case["q_len"] * case["q_heads"] * 2) * 4
    if case["op"] == "keep":
        return case["layers"] * _keep_pages(case) * case["page"] * (case["wide"] + case["narrow"]) * 2
    return 0


def _keep_pages(case):
    return case["batch"] * (-(-case["q_len"] // case["page"]) + 1) + 1


def _to_e4m3(x):
    return x.clamp(-448.0, 448.0).to(torch.float8_e4m3fn)


def _draw_parents(tokens, g, dev):
    """A tree for each request: its first token is the root, every other one hangs under any of those before it."""
    index = torch.tensor([i for n in tokens for i in range(n)], dtype=torch.int64, device=dev)
    pick = torch.rand(index.numel(), generator=g, device=dev, dtype=torch.float64)
    return torch.where(index == 0, -1, torch.minimum((pick * index).long(), index - 1)).to(torch.int32)


def _ancestors(parents, begin, count, s):
    """[B, s, s] truth values: which of a request's tokens are a token's ancestors or itself.  parents [T], a request's from begin [B] on."""
    at = torch.arange(s, device=parents.device)
    there = at < count[:, None]
    p = parents.long()[(begin[:, None] + at).clamp(0, parents.numel() - 1)]
    p = torch.where(there & (p >= 0) & (p < at), p, s)  # (s: none)
    sees = torch.cat((torch.eye(s, device=p.device, dtype=torch.bool) & there[..., None], torch.zeros(s, dtype=torch.bool, device=p.device)
                      .expand(p.shape[0], 1, s)), dim=1)
    p = torch.cat((p, torch.full_like(p[:, :1], s)), dim=1)
    for _ in range(max(1, (s - 1).bit_length())):  # as far again with every step
        sees = sees | torch.gather(sees, 1, p[..., None].expand(-1, -1, s))
        p = torch.gather(p, 1, p)
    return sees[:, :s]


def _pack(sees):
    """Truth values [..., n] as words of 64 bits [..., ceil(n / 64)]."""
    n = sees.shape[-1]
    sees = torch.nn.functional.pad(sees, (0, -n % 64)).unflatten(-1, (-1, 64))
    return (sees.long() << torch.arange(64, device=sees.device)).sum(-1)


def prepare(case, seed):
    dev = torch.device("cuda", torch.cuda.current_device())
    g = torch.Generator(device=dev).manual_seed(seed)
    perm = lambda n: torch.randperm(n, generator=g, device=dev)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)
    s = {"case": case}
    page = case["page"]
    if case["op"] == "tables":
        tokens, ctx = _tokens(case), _contexts(case)
        b, total = len(tokens), sum(tokens) + case["padded"]
        starts = [0]
        for n in tokens:
            starts.append(starts[-1] + n)
        s["context_lens"], s["starts"] = i32(ctx), i32(starts)
        held = [-(-c // page) if c > 0 else 0 for c in ctx]
        for i in range(case["ended"]):  # an idle place, or the request in it, still holds pages
            held[-1 - i % b] += 3
        wide = -(-case["room"] // page)
        held = [min(n, wide) for n in held]
        pages = sum(held) + sum(-(-n // page) + 1 for n in tokens) + 16
        order = perm(pages).to(torch.int32)
        table, at = torch.zeros(b, wide, dtype=torch.int32, device=dev), 0
        for i, (c, n, h) in enumerate(zip(ctx, tokens, held)):
            h = h if case["pages"] else min(wide, -(-(max(c, 0) + n) // page))
            table[i, :h] = order[at:at + h]
            at += h
        s["block_table"] = table
        s["num_blocks"] = s["free_pages"] = s["num_free"] = None
        if case["pages"]:
            free = torch.zeros(pages, dtype=torch.int32, device=dev)
            free[:pages - at] = order[at:]
            s["num_blocks"], s["free_pages"], s["num_free"] = i32(held), free, i32([pages - at])
        s["parents"] = _draw_parents(tokens + [1] * case["padded"], g, dev) if case["tree"] else None
        s["visible"] = torch.empty(total, -(-case["q_len"] // 64), dtype=torch.int64, device=dev) if case["tree"] else None
        s["seq_lens"] = torch.empty(b, dtype=torch.int32, device=dev)
        s["positions"], s["slots"] = (torch.empty(total, dtype=torch.int64, device=dev) for _ in range(2))
    elif case["op"] == "attend":
        d, hq, hk, dt = case["dim"], case["q_heads"], case["kv_heads"], DTYPES[case["dtype"]]
        tokens, lens = _tokens(case), _lengths(case)
        b, total = len(lens), sum(tokens)
        per = [-(-n // page) for n in lens]
        pages = sum(per) + 2
        kind = torch.float8_e4m3fn if case["cache"] == "fp8" else dt
        s["k_cache"], s["v_cache"] = (torch.empty(pages, page, hk, d, dtype=kind, device=dev) for _ in range(2))
        for c in (s["k_cache"], s["v_cache"]):
            step = max(1, (1 << 28) // (page * hk * d))  # (no more than 1 GB of random numbers at a time)
            for at in range(0, pages, step):
                part = c[at:at + step]
                x = torch.randn(part.shape, generator=g, device=dev, dtype=torch.float32 if case["cache"] == "fp8" else dt)
                part.copy_(_to_e4m3(x * 20) if case["cache"] == "fp8" else x)
        order, table = perm(pages).to(torch.int32), torch.zeros(b, -(-max(case["room"], max(lens)) // page), dtype=torch.int32, device=dev)
        at = 0
        for i, n in enumerate(per):
            table[i, :n] = order[at:at + n]
            at += n
        s["block_table"], s["seq_lens"] = table, i32(lens)
        starts = [0]
        for n in tokens:
            starts.append(starts[-1] + n)
        s["begin"], s["count"] = i32(starts[:-1]), i32(tokens)
        s["starts"] = i32(starts) if case["ragged"] else None
        parents = _draw_parents(tokens, g, dev)
        sees = _ancestors(parents, s["begin"].long(), torch.tensor([n if x else 0 for n, x in zip(tokens, lens)], device=dev), case["q_len"])
        who, at = _of_tokens(s["begin"], s["count"], total)
        s["visible"] = _pack(sees)[who, at].contiguous()
        s["q"] = torch.randn(total, hq, d, generator=g, device=dev, dtype=dt)
        s["k_scale"] = s["v_scale"] = None
        if case["cache"] == "fp8":
            s["k_scale"], s["v_scale"] = (0.04 + 0.02 * torch.rand(hk, generator=g, device=dev) for _ in range(2))
        s["out"] = torch.empty_like(s["q"])
        s["longest"] = max(lens)
    else:
        b, q_len = case["batch"], case["q_len"]
        ctx = [case["context"] + i % (page + 3) for i in range(b)]
        pages, layers, heads = _keep_pages(case), case["layers"], case["heads"]
        if case["wide"] == 656:  # rows of 656 bytes
            s["wide"] = torch.randint(0, 256, (layers, pages, page, 656), generator=g, device=dev, dtype=torch.uint8)
        else:
            s["wide"] = torch.randn(layers, pages, page, heads, case["wide"] // heads, generator=g, device=dev, dtype=torch.bfloat16)
        s["narrow"] = None
        if case["narrow"]:
            s["narrow"] = torch.randn(layers, pages, page, heads, case["narrow"] // heads, generator=g, device=dev, dtype=torch.bfloat16)
        s["caches"] = list(s["wide"]) + (list(s["narrow"]) if case["narrow"] else [])
        order = perm(pages).to(torch.int32)
        table, at = torch.zeros(b, max(c + q_len for c in ctx) // page + 2, dtype=torch.int32, device=dev), 0
        for i, c in enumerate(ctx):  # (only the pages that the step's tokens lie in are its own here)
            first, last = c // page, (c + q_len - 1) // page
            table[i, first:last + 1] = order[at:at + last - first + 1]
            at += last - first + 1
        kept, most = _kept(case), case["kept"]
        # The root, then a path among the tokens behind the kept places, so that a second pass over the same caches moves the same rows.
        path = torch.zeros(b, most, dtype=torch.int64, device=dev)
        for i, n in enumerate(kept):
            path[i, 1:n] = n + torch.sort(perm(q_len - n)[:n - 1]).values
        s["block_table"], s["context_lens"], s["seq_lens"] = table, i32(ctx), i32([c + q_len for c in ctx])
        s["accepted"], s["num_accepted"] = path.to(torch.int32), i32(kept)
        s["kept_lens"] = torch.empty(b, dtype=torch.int32, device=dev)
    return s


def run(s):
    case = s["case"]
    if own:
        from omni_npu_amd import kernels as K
        if case["op"] == "tables":
            K.step_tables(s["context_lens"], s["block_table"], case["page"], s["seq_lens"], s["positions"], s["slots"], q_len=case["q_len"],
                          query_start_loc=s["starts"] if case["ragged"] or case["padded"] else None, parents=s["parents"], visible=s["visible"],
                          num_blocks=s["num_blocks"], free_pages=s["free_pages"], num_free=s["num_free"])
            return _tables_out(s)
        if case["op"] == "attend":
            K.gqa_tree_decode(s["q"], s["k_cache"], s["v_cache"], s["block_table"], s["seq_lens"], s["visible"], case["dim"] ** -0.5, s["out"],
                              q_len=case["q_len"], query_start_loc=s["starts"], window=case["window"] or None, k_scale=s["k_scale"],
                              v_scale=s["v_scale"], max_seq_len=s["longest"])
            return s["out"]
        K.keep_rows(s["caches"], s["block_table"], s["context_lens"], s["seq_lens"], s["accepted"], s["num_accepted"], s["kept_lens"])
        return s["wide"], s["narrow"], s["kept_lens"]
    if case["op"] == "tables":
        return _plain_tables(s)
    if case["op"] == "attend":
        return _plain_attend(s)
    return _plain_keep(s)


def _tables_out(s):
    return {n: s[n] for n in ("seq_lens", "positions", "slots", "visible", "block_table", "num_blocks", "free_pages", "num_free") if s[n] is not None}


def _of_tokens(begin, count, total):
    """The request of each token and its place in it."""
    t = torch.arange(total, device=begin.device)
    who = torch.searchsorted((begin + count).long(), t, right=True).clamp(max=begin.numel() - 1)
    return who, t - begin.long()[who]


def _plain_tables(s):
    case, dev = s["case"], s["block_table"].device
    page, ctx, starts, table = case["page"], s["context_lens"].long(), s["starts"].long(), s["block_table"]
    live = ctx >= 0
    count = starts[1:] - starts[:-1]
    length = torch.where(live, ctx.clamp(min=0) + count, 0)
    ok = torch.ones_like(live)
    if case["pages"]:
        held, n_free, free = s["num_blocks"].long(), s["num_free"].long(), s["free_pages"]
        target = -(-length // page)
        ok = target <= table.shape[1]
        give = torch.where(ok, (held - target).clamp(min=0), 0)
        given = give.cumsum(0)
        back = given + n_free <= free.numel()
        give = torch.where(back, give, 0)
        n_back = give.sum()
        # (the pages that each request gives, the first of them last, and those it takes, from the list's end)
        col = torch.arange(table.shape[1], device=dev)
        rank = col - target[:, None]
        at = n_free + n_back - 1 - (given - give)[:, None] - rank
        mine = (rank >= 0) & (rank < give[:, None])
        free = torch.cat((free, free[:1]))  # (one place more for what is not written)
        free[torch.where(mine, at, free.numel() - 1).flatten()] = table.flatten()
        free = free[:-1]
        n_free = n_free + n_back
        take = torch.where(ok, (target - held).clamp(min=0), 0)
        taken = take.cumsum(0)
        got = (take == 0) | (taken <= n_free)
        take = torch.where(got, take, 0)
        rank = col - held[:, None]
        at = n_free - 1 - (taken - take)[:, None] - rank
        mine = (rank >= 0) & (rank < take[:, None])
        table.copy_(torch.where(mine, free[at.clamp(0, free.numel() - 1)], table))
        s["free_pages"].copy_(free)
        s["num_blocks"].copy_(held - give + take)
        s["num_free"].copy_(n_free - take.sum())
        ok = ok & got
    s["seq_lens"].copy_(torch.where(ok, length, ctx))
    total = s["slots"].numel()
    who, i = _of_tokens(starts[:-1], count, total)
    used = (torch.arange(total, device=dev) < starts[-1]) & live[who]
    depth = i
    if case["tree"]:
        sees = _ancestors(s["parents"], starts[:-1], torch.where(live, count, 0), case["q_len"])
        place = (who, i.clamp(max=case["q_len"] - 1))
        depth = sees.sum(-1)[place] - 1
        s["visible"].copy_(torch.where(used[:, None], _pack(sees)[place], 0))
    s["positions"].copy_(torch.where(used, ctx[who] + depth, 0))
    at = ctx[who].clamp(min=0) + i
    inside = at < table.shape[1] * page
    slot = table[who, (at // page).clamp(max=table.shape[1] - 1)].long() * page + at % page
    s["slots"].copy_(torch.where(used & ok[who] & inside, slot, -1))
    return _tables_out(s)


def _plain_attend(s):
    case = s["case"]
    q, lens, page, n = s["q"], s["seq_lens"].long(), case["page"], case["q_len"]
    b, hk, d = lens.numel(), case["kv_heads"], case["dim"]
    at = torch.arange(s["longest"], device=q.device)
    rows = s["block_table"].long()[:, at // page] * page + at % page

    def keys(cache, scale):  # [B, Hk, keys, D]
        flat = cache.flatten(0, 1)
        x = flat.view(torch.uint8)[rows].view(torch.float8_e4m3fn).float() * scale[:, None] if scale is not None else flat[rows].float()
        return x.transpose(1, 2).contiguous()

    begin, count = s["begin"].long(), s["count"].long()
    i = torch.arange(n, device=q.device)
    token = (begin[:, None] + i).clamp(max=q.shape[0] - 1)  # [B, s]
    qr = q.float()[token].view(b, n, hk, -1, d).permute(0, 2, 1, 3, 4).reshape(b, hk, -1, d)
    scores = torch.matmul(qr, keys(s["k_cache"], s["k_scale"]).transpose(2, 3)) * d ** -0.5
    bits = (s["visible"][token][..., None] >> torch.arange(64, device=q.device) & 1).bool().flatten(2)[..., :n]  # [B, s, s]
    ctx = lens - count
    place = at - ctx[:, None]  # [B, keys]: a key's place among the step's tokens
    own_key = torch.gather(bits, 2, place.clamp(0, n - 1)[:, None].expand(-1, n, -1)) & (place < count[:, None])[:, None]
    seen = torch.where((place < 0)[:, None], True, own_key) & (at < lens[:, None])[:, None]
    if case["window"]:  # the newest ones of what a token sees
        seen &= seen.flip(2).cumsum(2, dtype=torch.int32).flip(2) <= case["window"]
    seen = seen[:, None, :, None].expand(b, hk, n, scores.shape[2] // n, -1).reshape(scores.shape)
    scores = scores.masked_fill(~seen, -math.inf)
    most = scores.amax(-1, keepdim=True)
    p = torch.exp(scores - torch.where(most == -math.inf, 0.0, most))
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p, keys(s["v_cache"], s["v_scale"])) / torch.where(total == 0, 1.0, total)
    o = o.view(b, hk, n, -1, d).permute(0, 2, 1, 3, 4).reshape(b, n, -1, d)
    who, i = _of_tokens(s["begin"], s["count"], q.shape[0])
    return o[who, i].to(q.dtype)


def _plain_keep(s):
    case, page = s["case"], s["case"]["page"]
    ctx, depth = s["context_lens"].long(), torch.arange(case["kept"], device=s["accepted"].device)
    kept = depth < s["num_accepted"][:, None]
    slot = lambda at: torch.gather(s["block_table"].long(), 1, at // page) * page + at % page
    src, dst = slot(ctx[:, None] + s["accepted"].long()), slot(ctx[:, None] + depth)
    src, dst = torch.where(kept, src, dst).flatten(), dst.flatten()
    for c in (s["wide"], s["narrow"]):
        if c is not None:
            flat = c.flatten(1, 2)
            flat[:, dst] = flat[:, src]
    s["kept_lens"].copy_(ctx + s["num_accepted"])
    return s["wide"], s["narrow"], s["kept_lens"]


def exact(case, seed):
    """The operators by their definitions, one request at a time."""
    s = prepare(case, seed)
    page = case["page"]
    if case["op"] == "tables":
        return _exact_tables(s)
    if case["op"] == "attend":
        out = torch.zeros(s["q"].shape, dtype=torch.float64, device=s["q"].device)
        group, begin = case["q_heads"] // case["kv_heads"], s["begin"].tolist()
        words = [[w & (1 << 64) - 1 for w in row] for row in s["visible"].tolist()]
        for b, (n, count) in enumerate(zip(_lengths(case), _tokens(case))):
            if n == 0:
                continue
            used = s["block_table"][b, :-(-n // page)].long()
            seen = torch.zeros(count, n, dtype=torch.bool)
            for i in range(count):
                line = [n - count + j for j in range(count) if words[begin[b] + i][j // 64] >> j % 64 & 1]
                most = case["window"] or n
                seen[i, line[-most:]] = True
                seen[i, max(0, n - count - max(0, most - len(line))):n - count] = True
            hidden = ~seen.to(out.device).repeat_interleave(group, 0)
            for h in range(case["kv_heads"]):
                k, v = (c[used, :, h].reshape(-1, case["dim"])[:n].double() for c in (s["k_cache"], s["v_cache"]))
                if s["k_scale"] is not None:
                    k, v = k * s["k_scale"][h].double(), v * s["v_scale"][h].double()
                rows, heads = slice(begin[b], begin[b] + count), slice(h * group, (h + 1) * group)
                x = s["q"][rows, heads].double().reshape(-1, case["dim"]) @ k.t() / math.sqrt(case["dim"])
                x[hidden] = -math.inf
                out[rows, heads] = (torch.softmax(x, dim=1) @ v).view(count, group, -1)
        return out
    wide, narrow = (None if c is None else c.clone() for c in (s["wide"], s["narrow"]))
    table, path = s["block_table"].tolist(), s["accepted"].tolist()
    where = lambda b, at: (table[b][at // page], at % page)
    ctx = s["context_lens"].tolist()
    moves = [(*where(b, ctx[b] + path[b][k]), *where(b, ctx[b] + k)) for b, n in enumerate(_kept(case)) for k in range(n) if path[b][k] != k]
    if moves:
        p0, r0, p1, r1 = (torch.tensor(x, device=wide.device) for x in zip(*moves))
        for c, old in ((wide, s["wide"]), (narrow, s["narrow"])):
            if c is not None:
                c[:, p1, r1] = old[:, p0, r0]
    return wide, narrow, torch.tensor([c + n for c, n in zip(ctx, _kept(case))], dtype=torch.int32, device=wide.device)


def _exact_tables(s):
    case, page, dev = s["case"], s["case"]["page"], s["slots"].device
    out = {n: x.clone() for n, x in _tables_out(s).items()}
    ctx, tokens, table = s["context_lens"].tolist(), _tokens(case), s["block_table"].tolist()
    room, total = len(table[0]), s["slots"].numel()
    fits = [True] * len(ctx)
    lens = [0 if c < 0 else c + n for c, n in zip(ctx, tokens)]
    if case["pages"]:
        held, capacity = s["num_blocks"].tolist(), s["free_pages"].numel()
        free = s["free_pages"].tolist()
        stack, behind = free[:s["num_free"].item()], free[s["num_free"].item():]
        need = [-(-n // page) for n in lens]
        back, given = [], 0
        for b, n in enumerate(need):
            if n <= room and n < held[b]:
                given += held[b] - n
                if len(stack) + given <= capacity:
                    back += table[b][n:held[b]]
                    held[b] = n
        stack += back[::-1]
        shown, taken, top = stack + free[len(stack):], 0, len(stack)
        for b, n in enumerate(need):
            if n > room:
                fits[b] = False
            elif n > held[b]:
                more = n - held[b]
                taken += more
                if taken > top:
                    fits[b] = False
                    continue
                for i in range(more):
                    table[b][held[b] + i] = stack.pop()
                held[b] = n
        out["block_table"], out["num_blocks"] = torch.tensor(table, dtype=torch.int32, device=dev), torch.tensor(held, dtype=torch.int32, device=dev)
        out["free_pages"], out["num_free"] = torch.tensor(shown, dtype=torch.int32, device=dev), torch.tensor([len(stack)], dtype=torch.int32, device=dev)
    out["seq_lens"] = torch.tensor([n if ok else c for n, c, ok in zip(lens, ctx, fits)], dtype=torch.int32, device=dev)
    positions, slots, t = [0] * total, [-1] * total, 0
    words = [[0] * out["visible"].shape[1] for _ in range(total)] if case["tree"] else None
    parents = s["parents"].tolist() if case["tree"] else None
    for b, n in enumerate(tokens):
        line = []
        for i in range(n):
            if case["tree"]:
                up = parents[t]
                line.append((line[up] if 0 <= up < i else set()) | {i})
            if ctx[b] >= 0:
                depth = len(line[i]) - 1 if case["tree"] else i
                positions[t] = ctx[b] + depth
                at = ctx[b] + i
                if fits[b] and at // page < room:
                    slots[t] = table[b][at // page] * page + at % page
                if case["tree"]:
                    for j in line[i]:
                        words[t][j // 64] |= 1 << j % 64
            t += 1
    out["positions"], out["slots"] = torch.tensor(positions, device=dev), torch.tensor(slots, device=dev)
    if case["tree"]:
        out["visible"] = torch.tensor([[w - (1 << 64) if w >> 63 else w for w in row] for row in words], device=dev)
    return out
