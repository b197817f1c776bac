"""Plain statements, in 64 bits, of what layers with ordinary key and value heads run around a paged cache: per-head RMSNorm, rotary
positions, cache write, attention over the pages.  Test infrastructure only."""
import torch

U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}     # half a step, relative


def norm_rope(x, gamma, cos, sin, positions, eps, interleaved):
    """x [T,H,D] -> (result, size) in fp64: size bounds what a result is the sum of, for tolerances."""
    y = x.double()
    if gamma is not None:
        y = y / torch.sqrt((y * y).mean(-1, keepdim=True) + eps) * gamma.double()
    c, s = (t.double()[positions][:, None] for t in (cos, sin))
    r = c.shape[-1]
    out, size = y.clone(), y.abs()
    a, b = (slice(0, 2 * r, 2), slice(1, 2 * r, 2)) if interleaved else (slice(0, r), slice(r, 2 * r))
    out[..., a] = y[..., a] * c - y[..., b] * s
    out[..., b] = y[..., b] * c + y[..., a] * s
    for i in (a, b):
        size[..., i] = y[..., a].abs() * torch.maximum(c.abs(), s.abs()) + y[..., b].abs() * torch.maximum(c.abs(), s.abs())
    return out, size


def gqa(q, k_cache, v_cache, block_table, seq_lens, scale, q_start, window=0, k_scale=None, v_scale=None):
    """q [T,Hq,D], caches [pages,page,Hk,D] -> (o [T,Hq,D], lse [T,Hq], tol [T,Hq,D]) in fp64.  ``tol`` without the result's own
    rounding, for probabilities rounded by a relative u: multiply by what of_tol says."""
    t, hq, d = q.shape
    page, hk = k_cache.shape[1], k_cache.shape[2]
    grp = hq // hk
    o, lse = torch.zeros(t, hq, d, dtype=torch.float64), torch.full((t, hq), -torch.inf, dtype=torch.float64)
    weight, reach = torch.zeros(t, hq, d, dtype=torch.float64), torch.zeros(t, hq, dtype=torch.float64)
    for b, n in enumerate(seq_lens.tolist()):
        n = min(n, block_table.shape[1] * page)
        t0, t1 = int(q_start[b]), int(q_start[b + 1])
        pos = torch.arange(max(n, 0))
        rows = block_table[b].long()[pos // page] * page + pos % page
        k, v = (c.flatten(0, 1)[rows].double() for c in (k_cache, v_cache))
        if k_scale is not None:
            k = k * k_scale.double()[:, None]
        if v_scale is not None:
            v = v * v_scale.double()[:, None]
        for i in range(t1 - t0):
            end = n - (t1 - t0) + i + 1
            begin = max(0, end - window) if window else 0
            if end <= begin:
                continue
            for h in range(hk):
                heads = slice(h * grp, (h + 1) * grp)
                qq, kk, vv = q[t0 + i, heads].double(), k[begin:end, h], v[begin:end, h]
                s = qq @ kk.t() * scale
                top = s.amax(1, keepdim=True)
                p = torch.exp(s - top)
                tot = p.sum(1, keepdim=True)
                o[t0 + i, heads] = p @ vv / tot
                lse[t0 + i, heads] = (top + tot.log())[:, 0]
                weight[t0 + i, heads] = p @ vv.abs() / tot
                reach[t0 + i, heads] = (qq.abs() @ kk.abs().t()).amax(1) * abs(scale)
    return o, lse, weight, reach


def gqa_tolerance(o, weight, reach, dtype, d):
    """How far a result may be from ``o``: its own rounding, u |o|; the probabilities' rounding, which moves o' = sum p' v / sum p' by at
    most u sum(w |v - o|) <= u (weight + |o|) to first order; and the scores' fp32 error, (d + 4) 2^-24 of the absolute products,
    which moves every probability by that much relatively (a factor of two for numerator and denominator)."""
    u = U[dtype]
    return u * o.abs() + (1.01 * u + 2 * (d + 4) * 2.0 ** -24 * reach[..., None] + 2.0 ** -19) * (weight + o.abs()) + 1e-30
