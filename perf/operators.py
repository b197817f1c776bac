"""The operators of a layer with ordinary key and value heads over a paged cache, as cases that can be timed and compared.

``rope_cache``: the step in front of the attention.  Per-head RMSNorm of queries and keys, rotary positions (half or interleaved
pairs, all of a head or its first part), keys and values into the paged cache of 16- or 8-bit values: one call per layer and step.
``attend``: attention of each request's newest tokens over that cache, ragged lengths, whole contexts or a sliding window.
``pages``: pages of all layers' caches copied, forked (their filled rows only) or moved with the block table rewritten.

Where ``own`` is true the calls are this package's; where it is false the same is computed by elementary torch operations in 32
bits, rounded once.
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
E4M3_MAX = 448.0
EPS = 1e-6


def _rope(name=None, tokens=1, start=0, q_heads=32, kv_heads=8, dim=128, rotary=128, interleaved=False, norm=True, dtype="bf16",
          cache="same", page=128, padded=0, base=1e6):
    case = dict(op="rope_cache", tokens=tokens, start=start, q_heads=q_heads, kv_heads=kv_heads, dim=dim, rotary=rotary,
                interleaved=interleaved, norm=norm, dtype=dtype, cache=cache, page=page, padded=padded, base=base)
    return case if name is None else dict(name=name, **case)


def _attend(name=None, batch=1, q_len=1, lo=1, hi=1, q_heads=32, kv_heads=8, dim=128, dtype="bf16", cache="same", page=128,
            window=0, idle=0, room=0):
    case = dict(op="attend", batch=batch, q_len=q_len, lo=lo, hi=hi, q_heads=q_heads, kv_heads=kv_heads, dim=dim, dtype=dtype,
                cache=cache, page=page, window=window, idle=idle, room=room)
    return case if name is None else dict(name=name, **case)


def _pages(name=None, layers=1, pages=64, page=128, heads=1, wide=512, narrow=64, pairs=1, part=False, move=False, requests=8,
           kept=8):
    case = dict(op="pages", layers=layers, pages=pages, page=page, heads=heads, wide=wide, narrow=narrow, pairs=pairs, part=part,
                move=move, requests=requests, kept=kept)
    return case if name is None else dict(name=name, **case)


def listed():
    return [
        # one user's next token on a rank of eight: the smallest call there is, latency alone
        _rope("rope_one_token", tokens=1, start=1020, q_heads=4, kv_heads=1),
        # a decode batch padded to a captured graph's size, far positions, part of the head rotated, interleaved pairs
        _rope("rope_decode_batch", tokens=64, start=100000, q_heads=32, kv_heads=8, rotary=64, interleaved=True, padded=5),
        # a prompt of odd length, small heads, without norms, fp16
        _rope("rope_prompt_fp16", tokens=2999, q_heads=16, kv_heads=4, dim=64, rotary=64, norm=False, dtype="fp16", page=16),
        # a large prefill step into the 8-bit cache
        _rope("rope_prefill_fp8", tokens=16384, q_heads=64, kv_heads=8, cache="fp8"),
        # one user in a chat, on a rank of eight: latency alone
        _attend("attend_one_user", batch=1, lo=1021, hi=1021, q_heads=4, kv_heads=1, room=8192),
        # the benchmark's decode batch: 64 requests of 4k-8k tokens
        _attend("attend_batch", batch=64, lo=4096, hi=8192, room=8192),
        # one document of 128k tokens being asked about
        _attend("attend_long", batch=1, lo=131072, hi=131072, q_heads=64, kv_heads=8, room=131072),
        # throughput serving over the 8-bit cache with one speculative token, lengths all over the range, a graph's idle places
        _attend("attend_fp8_mtp", batch=128, q_len=2, lo=2048, hi=16384, q_heads=64, kv_heads=8, cache="fp8", idle=3, room=16384),
        # sliding-window layers with wide heads and small pages, fp16
        _attend("attend_window", batch=33, lo=300, hi=9000, q_heads=16, kv_heads=4, dim=256, dtype="fp16", page=16, window=1024,
                room=16384),
        # a few requests forked: the filled rows of their last pages, in every layer of a latent cache
        _pages("pages_fork", layers=27, pages=96, pairs=6, part=True),
        # shared prefixes becoming private: whole pages of one small model's layers
        _pages("pages_copy", layers=16, pages=256, page=16, heads=8, wide=1024, narrow=1024, pairs=100),
        # a cache compacted: its last pages into the holes, the block tables after them
        _pages("pages_compact", layers=24, pages=512, pairs=200, move=True, requests=64, kept=48, heads=8, wide=1024, narrow=1024),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    """One more call of the same kinds, at sizes all over what the list spans."""
    op = rng.choice(["rope_cache", "attend", "attend", "pages"])
    most = max(_cost(c) for c in listed() if c["op"] == op)
    while True:
        kv = rng.choice([1, 2, 3, 4, 8])
        if op == "rope_cache":
            dim = rng.choice([64, 128, 256])
            tokens = _log(rng, 1, 16384)
            c = _rope(tokens=tokens, start=rng.choice([0, _log(rng, 1, 200000)]), q_heads=kv * rng.choice([1, 2, 4, 5, 8]), kv_heads=kv,
                      dim=dim, rotary=rng.choice([dim, dim // 2, dim // 4]), interleaved=rng.random() < 0.4,
                      norm=rng.random() < 0.6, dtype=rng.choice(["bf16", "bf16", "fp16"]), cache=rng.choice(["same", "same", "fp8"]),
                      page=rng.choice([16, 64, 128]), padded=min(tokens - 1, rng.choice([0, 0, 3])), base=rng.choice([1e4, 1e6]))
        elif op == "attend":
            hi = _log(rng, 20, 131072)
            window = rng.choice([0, 0, 0, _log(rng, 100, 4096)])
            c = _attend(batch=_log(rng, 1, 128), q_len=rng.choice([1, 1, 1, 2, 3, 4]), lo=rng.randint(max(hi // 8, 8), hi), hi=hi,
                        q_heads=kv * rng.choice([1, 2, 4, 5, 8, 16]), kv_heads=kv, dim=rng.choice([64, 128, 128, 256]),
                        dtype=rng.choice(["bf16", "bf16", "fp16"]), cache=rng.choice(["same", "same", "fp8"]),
                        page=rng.choice([16, 64, 128]), window=window, idle=rng.choice([0, 0, 2]),
                        room=max(1024, 1 << (hi - 1).bit_length()))
        else:
            wide, narrow, heads = rng.choice([(512, 64, 1), (1024, 1024, 8), (128, 128, 2), (656, 0, 1)])
            pages = _log(rng, 16, 512)
            c = _pages(layers=rng.randint(1, 32), pages=pages, page=rng.choice([16, 64, 128]), heads=heads, wide=wide, narrow=narrow,
                       pairs=_log(rng, 1, pages // 3), part=rng.random() < 0.3, requests=_log(rng, 1, 64), kept=rng.randint(1, 64))
            c["move"] = not c["part"] and rng.random() < 0.5
        if _cost(c) <= most and _room(c) <= 6e9:
            return c


def _lengths(case):
    """The requests' lengths: ragged over lo .. hi, then the idle places."""
    n, lo, hi = case["batch"], case["lo"], case["hi"]
    return [hi] + [lo + round((hi - lo) * ((i * 0.6180339887498949) % 1.0)) for i in range(1, n)] + [0] * case["idle"]


def _seen(case):
    """How many keys of each request are read: those that one of its tokens sees."""
    w, s = case["window"], case["q_len"]
    return [min(n, w + s - 1) if w else n for n in _lengths(case)]


def _rows(case):
    """How many rows of each pair's page are filled."""
    page, n = case["page"], case["pairs"]
    return [1 + round((page - 1) * ((i * 0.6180339887498949) % 1.0)) if case["part"] else page for i in range(1, n + 1)]


def work(case):
    es = 1 if case.get("cache") == "fp8" else 2
    if case["op"] == "rope_cache":
        t, d, hq, hk = case["tokens"], case["dim"], case["q_heads"], case["kv_heads"]
        kept = t - case["padded"]
        nbytes = t * hq * d * 4 + kept * 2 * hk * d * (2 + es) + t * case["rotary"] * 4 + t * 16
        flops = t * hq * (4 * case["norm"] * d + 3 * case["rotary"]) + kept * hk * (4 * case["norm"] * d + 3 * case["rotary"])
    elif case["op"] == "attend":
        d, hq, hk = case["dim"], case["q_heads"], case["kv_heads"]
        keys, tokens = sum(_seen(case)), (case["batch"] + case["idle"]) * case["q_len"]
        nbytes = keys * 2 * hk * d * es + tokens * hq * d * 4 + sum(-(-n // case["page"]) for n in _seen(case)) * 4
        flops = 4 * keys * case["q_len"] * hq * d
    else:
        row = case["layers"] * (case["wide"] + case["narrow"]) * (1 if case["wide"] == 656 else 2)
        nbytes, flops = 2 * sum(_rows(case)) * row + case["move"] * case["requests"] * case["kept"] * 8, 0
    return {"bytes": nbytes, "flops": flops}


def _cost(case):
    w = work(case)
    return max(w["bytes"] / 6e12, w["flops"] / 1e14)


def _room(case):
    if case["op"] == "attend":  # the keys and values that the plain form lays out in 32 bits
        return (case["batch"] + case["idle"]) * case["hi"] * max(case["kv_heads"] * case["dim"], case["q_len"] * case["q_heads"]) * 4
    if case["op"] == "pages":
        return case["layers"] * case["pages"] * case["page"] * (case["wide"] + case["narrow"]) * 2
    return 0


def _tables(case, dev):
    """cos / sin of position x frequency in 64 bits, rounded to 32: what a model makes once."""
    n = case["start"] + case["tokens"]
    inv = case["base"] ** (-torch.arange(0, case["rotary"], 2, dtype=torch.float64, device=dev) / case["rotary"])
    angle = torch.arange(n, dtype=torch.float64, device=dev)[:, None] * inv
    return angle.cos().float(), angle.sin().float()


def _to_e4m3(x):
    return x.clamp(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn)


def prepare(case, seed):
    dev = torch.device("cuda", torch.cuda.current_device())
    g = torch.Generator(device=dev).manual_seed(seed)
    dt = DTYPES.get(case.get("dtype"), torch.bfloat16)
    randn = lambda *shape, dtype=dt: torch.randn(*shape, generator=g, device=dev, dtype=torch.float32 if dtype == torch.float8_e4m3fn else dtype)
    perm = lambda n: torch.randperm(n, generator=g, device=dev)
    s = {"case": case}
    if case["op"] == "rope_cache":
        t, d, hq, hk, page = case["tokens"], case["dim"], case["q_heads"], case["kv_heads"], case["page"]
        pages = -(-t // page) + 3
        qkv = randn(t, (hq + 2 * hk) * d)  # one projection's result: the three are views of it
        s["q"], s["k"], s["v"] = (x.unflatten(1, (-1, d)) for x in qkv.split([hq * d, hk * d, hk * d], dim=1))
        s["positions"] = case["start"] + perm(t)
        slots = perm(pages * page)[:t]
        slots[t - case["padded"]:] = -1
        s["slots"] = slots
        s["cos"], s["sin"] = _tables(case, dev)
        s["q_gamma"] = (1 + 0.1 * randn(d)).to(dt) if case["norm"] else None
        s["k_gamma"] = (1 + 0.1 * randn(d)).to(dt) if case["norm"] else None
        s["k_scale"] = s["v_scale"] = None
        s["k_cache"], s["v_cache"] = randn(pages, page, hk, d), randn(pages, page, hk, d)
        if case["cache"] == "fp8":
            s["k_scale"], s["v_scale"] = (0.01 + 0.01 * torch.rand(hk, generator=g, device=dev) for _ in range(2))
            s["k_cache"], s["v_cache"] = _to_e4m3(s["k_cache"]), _to_e4m3(s["v_cache"])
        s["q_out"] = torch.empty(t, hq, d, dtype=dt, device=dev)
    elif case["op"] == "attend":
        d, hq, hk, page = case["dim"], case["q_heads"], case["kv_heads"], case["page"]
        lens = torch.tensor(_lengths(case), dtype=torch.int32)
        b = lens.numel()
        per = [-(-n // page) for n in lens.tolist()]
        pages = sum(per) + 2
        kind = torch.float8_e4m3fn if case["cache"] == "fp8" else dt
        s["k_cache"], s["v_cache"] = (torch.empty(pages, page, hk, d, dtype=kind, device=dev) for _ in range(2))
        for c in (s["k_cache"], s["v_cache"]):
            for at in range(0, pages, max(1, (1 << 28) // (page * hk * d))):  # (no more than 1 GB of random numbers at a time)
                part = c[at:at + max(1, (1 << 28) // (page * hk * d))]
                x = torch.randn(part.shape, generator=g, device=dev, dtype=torch.float32 if case["cache"] == "fp8" else dt)
                part.copy_(_to_e4m3(x * 20) if case["cache"] == "fp8" else x)
        order, table = perm(pages).to(torch.int32), torch.zeros(b, -(-max(case["room"], case["hi"]) // page), dtype=torch.int32, device=dev)
        at = 0
        for i, n in enumerate(per):
            table[i, :n] = order[at:at + n]
            at += n
        s["block_table"], s["seq_lens"] = table, lens.to(dev)
        s["q"] = randn(b * case["q_len"], hq, d)
        s["k_scale"] = s["v_scale"] = None
        if case["cache"] == "fp8":
            s["k_scale"], s["v_scale"] = (0.04 + 0.02 * torch.rand(hk, generator=g, device=dev) for _ in range(2))
        s["out"] = torch.empty_like(s["q"])
        s["longest"] = case["hi"]
    else:
        n, page, pages = case["pairs"], case["page"], case["pages"]
        tail = (case["heads"], case["wide"] // case["heads"])
        if case["wide"] == 656:  # rows of 656 bytes
            s["wide"] = torch.randint(0, 256, (case["layers"], pages, page, 656), generator=g, device=dev, dtype=torch.uint8)
        else:
            s["wide"] = randn(case["layers"], pages, page, *tail)
        s["narrow"] = randn(case["layers"], pages, page, case["heads"], case["narrow"] // case["heads"]) if case["narrow"] else None
        order = perm(pages)
        s["src"], s["dst"] = order[:n].clone(), order[n:2 * n].clone()
        rows = _rows(case)
        s["rows"] = torch.tensor(rows, device=dev)
        s["caches"] = list(s["wide"]) + (list(s["narrow"]) if case["narrow"] else [])
        s["src_host"], s["dst_host"], s["rows_host"] = s["src"].tolist(), s["dst"].tolist(), rows if case["part"] else None
        s["block_table"] = None
        if case["move"]:  # the tables name any page but the holes
            live = torch.cat((order[:n], order[2 * n:])).to(torch.int32)
            s["block_table"] = live[torch.randint(0, live.numel(), (case["requests"], case["kept"]), generator=g, device=dev)]
    return s


def run(s):
    op = s["case"]["op"]
    if own:
        from omni_npu_amd import kernels as K
        if op == "rope_cache":
            K.qk_norm_rope_cache(s["q"], s["k"], s["v"], s["cos"], s["sin"], s["positions"], s["slots"], s["k_cache"], s["v_cache"],
                                 q_gamma=s["q_gamma"], k_gamma=s["k_gamma"], eps=EPS, interleaved=s["case"]["interleaved"],
                                 q_out=s["q_out"], k_scale=s["k_scale"], v_scale=s["v_scale"])
            return s["q_out"], s["k_cache"], s["v_cache"]
        if op == "attend":
            K.gqa_decode(s["q"], s["k_cache"], s["v_cache"], s["block_table"], s["seq_lens"], s["case"]["dim"] ** -0.5, s["out"],
                         q_len=s["case"]["q_len"], window=s["case"]["window"] or None, k_scale=s["k_scale"], v_scale=s["v_scale"],
                         max_seq_len=s["longest"])
            return s["out"]
        K.copy_pages(s["caches"], s["src_host"], s["dst_host"], rows=s["rows_host"], block_table=s["block_table"])
        return s["wide"], s["narrow"], s["block_table"]
    if op == "rope_cache":
        return _plain_rope_cache(s)
    if op == "attend":
        return _plain_attend(s)
    return _plain_pages(s)


def _plain_norm_rope(x, gamma, cos, sin, interleaved):
    x = x.float()
    if gamma is not None:
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * gamma.float()
    r = cos.shape[-1]
    turned, rest = x[..., :2 * r], x[..., 2 * r:]
    a, b = (turned[..., 0::2], turned[..., 1::2]) if interleaved else (turned[..., :r], turned[..., r:])
    a, b = a * cos - b * sin, b * cos + a * sin
    turned = torch.stack((a, b), dim=-1).flatten(-2) if interleaved else torch.cat((a, b), dim=-1)
    return torch.cat((turned, rest), dim=-1)


def _plain_rope_cache(s):
    case, dt = s["case"], s["q"].dtype
    cos, sin = s["cos"][s["positions"]][:, None], s["sin"][s["positions"]][:, None]
    q = _plain_norm_rope(s["q"], s["q_gamma"], cos, sin, case["interleaved"])
    k, v = _plain_norm_rope(s["k"], s["k_gamma"], cos, sin, case["interleaved"]), s["v"].float()
    if s["k_scale"] is not None:
        k, v = _to_e4m3(k / s["k_scale"][:, None]), _to_e4m3(v / s["v_scale"][:, None])
    else:
        k, v = k.to(dt), v.to(dt)
    kept = case["tokens"] - case["padded"]  # (the padding is behind the tokens)
    slots = s["slots"][:kept]
    as_rows = lambda c: c.view(torch.uint8).flatten(0, 1) if c.dtype == torch.float8_e4m3fn else c.flatten(0, 1)
    as_new = lambda x: (x.view(torch.uint8) if x.dtype == torch.float8_e4m3fn else x)[:kept]
    as_rows(s["k_cache"])[slots] = as_new(k)
    as_rows(s["v_cache"])[slots] = as_new(v)
    s["q_out"].copy_(q)
    return s["q_out"], s["k_cache"], s["v_cache"]


def _plain_attend(s):
    case = s["case"]
    q, lens, page, n = s["q"], s["seq_lens"].long(), case["page"], case["q_len"]
    b, hk, d = lens.numel(), case["kv_heads"], case["dim"]
    at = torch.arange(case["hi"], device=q.device)
    rows = s["block_table"].long()[:, at // page] * page + at % page

    def keys(cache, scale):  # [B, Hk, keys, D]
        flat = cache.flatten(0, 1)
        x = flat.view(torch.uint8)[rows].view(torch.float8_e4m3fn).float() * scale[:, None] if scale is not None else flat[rows].float()
        return x.transpose(1, 2).contiguous()

    qr = q.float().view(b, n, hk, -1, d).permute(0, 2, 1, 3, 4).reshape(b, hk, -1, d)
    scores = torch.matmul(qr, keys(s["k_cache"], s["k_scale"]).transpose(2, 3)) * d ** -0.5
    last = lens[:, None] - n + torch.arange(n, device=q.device)  # a token's own key
    seen = at <= last[..., None]
    if case["window"]:
        seen &= at > last[..., None] - case["window"]
    seen = seen[:, None, :, None].expand(b, hk, n, scores.shape[2] // n, -1).reshape(scores.shape)
    scores = scores.masked_fill(~seen, -math.inf)
    most = scores.amax(-1, keepdim=True)
    p = torch.exp(scores - torch.where(most == -math.inf, 0.0, most))
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p, keys(s["v_cache"], s["v_scale"])) / torch.where(total == 0, 1.0, total)
    return o.view(b, hk, n, -1, d).permute(0, 2, 1, 3, 4).reshape(q.shape).to(q.dtype)


def _plain_pages(s):
    case = s["case"]
    if case["part"]:
        filled = (torch.arange(case["page"], device=s["src"].device) < s["rows"][:, None])[None, :, :, None]
        for c in (s["wide"], s["narrow"]):
            if c is not None:
                flat = c.flatten(3)
                flat[:, s["dst"]] = torch.where(filled, flat[:, s["src"]], flat[:, s["dst"]])
    else:
        s["wide"][:, s["dst"]] = s["wide"][:, s["src"]]
        if s["narrow"] is not None:
            s["narrow"][:, s["dst"]] = s["narrow"][:, s["src"]]
    if s["block_table"] is not None:
        to = torch.arange(case["pages"], dtype=torch.int32, device=s["src"].device)
        to[s["src"]] = s["dst"].to(torch.int32)
        s["block_table"].copy_(to[s["block_table"].long()])
    return s["wide"], s["narrow"], s["block_table"]


def exact(case, seed):
    """The operators by their definitions, in 64 bits, one request or one head at a time."""
    s = prepare(case, seed)
    if case["op"] == "rope_cache":
        def turned(x, gamma):
            y = torch.empty(x.shape, dtype=torch.float64, device=x.device)
            r = case["rotary"] // 2
            c, sn = s["cos"].double()[s["positions"]], s["sin"].double()[s["positions"]]
            for h in range(x.shape[1]):
                z = x[:, h].double()
                if gamma is not None:
                    z = z / torch.sqrt(z.pow(2).sum(1, keepdim=True) / case["dim"] + EPS) * gamma.double()
                y[:, h] = z
                for i in range(r):
                    a, b = (2 * i, 2 * i + 1) if case["interleaved"] else (i, i + r)
                    y[:, h, a] = z[:, a] * c[:, i] - z[:, b] * sn[:, i]
                    y[:, h, b] = z[:, a] * sn[:, i] + z[:, b] * c[:, i]
            return y

        q, k, v = turned(s["q"], s["q_gamma"]), turned(s["k"], s["k_gamma"]), s["v"].double()
        if s["k_scale"] is not None:
            k = (k / s["k_scale"].double().view(1, -1, 1)).clamp(-E4M3_MAX, E4M3_MAX)
            v = (v / s["v_scale"].double().view(1, -1, 1)).clamp(-E4M3_MAX, E4M3_MAX)
        caches = []
        for cache, new in ((s["k_cache"], k), (s["v_cache"], v)):
            rows = cache.double().flatten(0, 1)
            there = s["slots"] >= 0
            rows[s["slots"][there]] = new[there]
            caches.append(rows.view(cache.shape))
        return q, caches[0], caches[1]
    if case["op"] == "attend":
        out = torch.zeros(s["q"].shape, dtype=torch.float64, device=s["q"].device)
        group = case["q_heads"] // case["kv_heads"]
        for b, n in enumerate(_lengths(case)):
            used = s["block_table"][b, :-(-n // case["page"])].long()
            for h in range(case["kv_heads"]):
                k, v = (c[used, :, h].reshape(-1, case["dim"])[:n].double() for c in (s["k_cache"], s["v_cache"]))
                if s["k_scale"] is not None:
                    k, v = k * s["k_scale"][h].double(), v * s["v_scale"][h].double()
                for i in range(case["q_len"]):
                    end = n - case["q_len"] + i + 1
                    begin = max(0, end - case["window"]) if case["window"] else 0
                    if end <= begin:
                        continue
                    q = s["q"][b * case["q_len"] + i, h * group:(h + 1) * group].double()
                    p = torch.softmax(q @ k[begin:end].t() / math.sqrt(case["dim"]), dim=1)
                    out[b * case["q_len"] + i, h * group:(h + 1) * group] = p @ v[begin:end]
        return out
    wide, narrow = (None if c is None else c.clone() for c in (s["wide"], s["narrow"]))
    for i, (a, b) in enumerate(zip(s["src_host"], s["dst_host"])):
        n = _rows(case)[i]
        for c in (wide, narrow):
            if c is not None:
                c[:, b, :n] = c[:, a, :n]
    table = None
    if s["block_table"] is not None:
        table = s["block_table"].clone()
        for a, b in zip(s["src_host"], s["dst_host"]):
            table[s["block_table"] == a] = b
    return wide, narrow, table
