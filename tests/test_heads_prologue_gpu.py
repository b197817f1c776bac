"""Per-head RMSNorm, rotary positions and cache write of layers with ordinary key and value heads, against their plain statement in 64
bits: types, head widths, rotated parts, both pairings, strides, padding, positions outside the tables, refusals."""
import pytest
import torch

from oracle import heads_oracle as H

pytestmark = pytest.mark.gpu

E4M3, EPS = torch.float8_e4m3fn, 1e-6


def make(t, hq, hk, d, r, dtype=torch.bfloat16, seed=0, fp8=False, page=16, norm=True, table=torch.float32, far=0, pages=None):
    g = torch.Generator().manual_seed(seed)
    pages = pages or -(-t // page) + 2
    n = far + t + 5
    angle = torch.outer(torch.arange(n, dtype=torch.float64), 10000.0 ** (-torch.arange(0, r, 2, dtype=torch.float64) / r))
    qkv = torch.randn(t, (hq + 2 * hk) * d, generator=g).to(dtype)
    c = dict(qkv=qkv, cos=angle.cos().to(table), sin=angle.sin().to(table), positions=far + torch.randperm(t + 5, generator=g)[:t],
             slots=torch.randperm(pages * page, generator=g)[:t], d=d, hq=hq, hk=hk, dtype=dtype, fp8=fp8)
    c["qg"], c["kg"] = ((1 + 0.2 * torch.randn(d, generator=g)).to(dtype) if norm else None for _ in range(2))
    kind = E4M3 if fp8 else dtype
    c["kc"], c["vc"] = (torch.randn(pages, page, hk, d, generator=g).to(kind) for _ in range(2))
    c["ks"], c["vs"] = ((0.01 + 0.02 * torch.rand(hk, generator=g)) if fp8 else None for _ in range(2))
    return c


def views(qkv, c):
    return (x.unflatten(1, (-1, c["d"])) for x in qkv.split([c["hq"] * c["d"], c["hk"] * c["d"], c["hk"] * c["d"]], dim=1))


def expect(c, interleaved, positions=None, slots=None):
    """(q, k, v, tolerances of q and k) in 64 bits."""
    q, k, v = views(c["qkv"], c)
    pos = c["positions"] if positions is None else positions
    (q, qs), (k, ks) = (H.norm_rope(x, g, c["cos"], c["sin"], pos, EPS, interleaved) for x, g in ((q, c["qg"]), (k, c["kg"])))
    return q, k, v.double(), qs, ks


def close(got, ref, size, dtype, scale=None):
    """One rounding of the result, and fp32 errors: the norm's sum of up to 256 squares, root, quotient and three products in a row stay
    below 2^-19 of what a result is the sum of."""
    got, ref, size = got.double(), ref.double(), size.double()
    if scale is not None:                                     # e4m3: half a step is 2^-4 of the value, 2^-10 among the subnormal ones
        ref, size = (ref / scale.double()[:, None]).clamp(-448, 448), size / scale.double()[:, None]
        tol = torch.maximum(2.0 ** -4 * ref.abs(), torch.tensor(2.0 ** -10)) + 2.0 ** -18 * size
    else:
        tol = H.U[dtype] * ref.abs() + 2.0 ** -19 * size + 2.0 ** -24 * (dtype == torch.float16) + 1e-38
    assert ((got - ref).abs() <= tol).all(), f"worst {((got - ref).abs() / tol).max():.3g} of the tolerance"


def run(dev, c, interleaved=False, **kw):
    from omni_npu_amd import kernels as K
    on = lambda x: None if x is None else x.to(dev)
    q, k, v = views(c["qkv"].to(dev), c)
    kc, vc = on(c["kc"]).clone(), on(c["vc"]).clone()
    q_out = torch.full(q.shape, 7.0, dtype=c["dtype"], device=dev)
    K.qk_norm_rope_cache(q, k, v, on(c["cos"]), on(c["sin"]), on(c["positions"]), on(c["slots"]), kc, vc, q_gamma=on(c["qg"]), k_gamma=on(c["kg"]),
                         eps=EPS, interleaved=interleaved, q_out=q_out, k_scale=on(c["ks"]), v_scale=on(c["vs"]), **kw)
    torch.cuda.synchronize()
    return q_out.cpu(), kc.cpu(), vc.cpu()


def check_all(c, q_out, kc, vc, interleaved):
    q, k, v, qs, ks = expect(c, interleaved)
    close(q_out, q, qs, c["dtype"])
    there = (c["slots"] >= 0) & (c["slots"] < kc.shape[0] * kc.shape[1])
    rows = c["slots"][there]
    plain = lambda x: x.float() if c["fp8"] else x
    close(plain(kc).flatten(0, 1)[rows], k[there], ks[there], c["dtype"], c["ks"])
    if c["fp8"]:
        close(plain(vc).flatten(0, 1)[rows], v[there], v[there].abs(), c["dtype"], c["vs"])
    else:
        assert torch.equal(vc.flatten(0, 1)[rows], v[there].to(c["dtype"]))
    keep = torch.ones(kc.shape[0] * kc.shape[1], dtype=torch.bool)
    keep[rows] = False
    bits = lambda x: x.view(torch.uint8) if c["fp8"] else x
    for new, old in ((kc, c["kc"]), (vc, c["vc"])):
        assert torch.equal(bits(new).flatten(0, 1)[keep], bits(old).flatten(0, 1)[keep])


@pytest.mark.parametrize("d,r", [(16, 16), (64, 64), (64, 32), (80, 32), (96, 96), (128, 128), (128, 16), (192, 64), (256, 256), (256, 64)])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("fp8", [False, True], ids=["same", "e4m3"])
@pytest.mark.parametrize("norm", [False, True])
def test_widths_and_pairings(dev, d, r, interleaved, fp8, norm):
    c = make(37, 6, 2, d, r, fp8=fp8, norm=norm, seed=d + r)
    check_all(c, *run(dev, c, interleaved), interleaved)


@pytest.mark.parametrize("t", [1, 2, 63, 515, 4099])
@pytest.mark.parametrize("hq,hk", [(4, 1), (5, 5), (32, 8)])
def test_token_counts(dev, t, hq, hk):
    c = make(t, hq, hk, 128, 128, seed=t)
    check_all(c, *run(dev, c), False)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "fp16"])
@pytest.mark.parametrize("table", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
def test_types_and_far_positions(dev, dtype, table):
    c = make(50, 4, 4, 64, 64, dtype=dtype, table=table, far=200000, seed=1)
    check_all(c, *run(dev, c), False)


def test_padding_and_slots_past_the_cache_are_not_written(dev):
    c = make(20, 4, 2, 128, 128, seed=2)
    c["slots"][3], c["slots"][7], c["slots"][19] = -1, c["kc"].shape[0] * 16, 1 << 40
    check_all(c, *run(dev, c), False)


def test_positions_outside_the_tables_are_not_written(dev):
    c = make(12, 4, 2, 128, 128, seed=3)
    c["positions"][2], c["positions"][5] = -1, c["cos"].shape[0]
    q_out, kc, vc = run(dev, c)
    bad = torch.tensor([2, 5])
    assert (q_out[bad] == 7).all()
    for new, old in ((kc, c["kc"]), (vc, c["vc"])):
        assert torch.equal(new.flatten(0, 1)[c["slots"][bad]], old.flatten(0, 1)[c["slots"][bad]])
    good = torch.tensor([i for i in range(12) if i not in (2, 5)])
    q, _, _, qs, _ = expect(c, False, positions=c["positions"].clamp(0, c["cos"].shape[0] - 1))
    close(q_out[good], q[good], qs[good], c["dtype"])


def test_in_place_and_without_a_cache(dev):
    """Queries and keys rotated where they lie in the projection's result, the rest of it untouched; queries alone; keys to both."""
    from omni_npu_amd import kernels as K
    c = make(33, 6, 2, 128, 64, seed=4)
    on = lambda x: x.to(dev)
    q_ref, k_ref, _, qs, ks = expect(c, False)
    qkv = on(c["qkv"])
    q, k, v = views(qkv, c)
    args = (on(c["cos"]), on(c["sin"]), on(c["positions"]))
    K.qk_norm_rope_cache(q, k, None, *args, q_gamma=on(c["qg"]), k_gamma=on(c["kg"]), eps=EPS)
    close(q.cpu(), q_ref, qs, c["dtype"])
    close(k.cpu(), k_ref, ks, c["dtype"])
    assert torch.equal(v.cpu(), list(views(c["qkv"], c))[2])
    qkv = on(c["qkv"])
    q, k, v = views(qkv, c)
    K.qk_norm_rope_cache(q, None, None, *args, q_gamma=on(c["qg"]), eps=EPS)
    close(q.cpu(), q_ref, qs, c["dtype"])
    assert torch.equal(k.cpu(), list(views(c["qkv"], c))[1])
    kc, vc, k_out = on(c["kc"]), on(c["vc"]), torch.empty(33, 2, 128, dtype=c["dtype"], device=dev)
    slots = on(c["slots"])
    slots[4] = -1                                              # (a token that is not cached has its key all the same)
    K.qk_norm_rope_cache(q.clone(), k, v, *args, slots, kc, vc, k_gamma=on(c["kg"]), eps=EPS, k_out=k_out)
    close(k_out.cpu(), k_ref, ks, c["dtype"])
    keep = [i for i in range(33) if i != 4]
    assert torch.equal(kc.cpu().flatten(0, 1)[c["slots"][keep]], k_out.cpu()[keep])


@pytest.mark.parametrize("fp8", [False, True], ids=["same", "e4m3"])
def test_not_a_number_and_infinities(dev, fp8):
    """NaN stays NaN; an infinity saturates in the 8-bit cache and stays one in the others."""
    c = make(6, 2, 2, 64, 64, seed=5, fp8=fp8, norm=False)
    v0 = 4 * 64
    k0 = 2 * 64
    c["qkv"][1, v0 + 3], c["qkv"][1, v0 + 70], c["qkv"][2, k0 + 5] = float("nan"), float("inf"), float("nan")
    q_out, kc, vc = run(dev, c)
    v1, k2 = vc.float().flatten(0, 1)[c["slots"][1]], kc.float().flatten(0, 1)[c["slots"][2]]
    assert torch.isnan(v1[0, 3]) and (v1[1, 6] == (448 if fp8 else float("inf"))) and torch.isnan(v1).sum() == 1
    assert torch.isnan(k2[0]).nonzero().flatten().tolist() == [5, 37]   # the pair


@pytest.mark.parametrize("interleaved", [False, True])
def test_an_infinity_stays_where_it_is(dev, interleaved):
    """Behind the rotated part, and in a pair of its own: no other value of the head changes."""
    c = make(4, 2, 2, 128, 32, seed=8, norm=False)
    ref, _, _ = run(dev, c, interleaved)
    c["qkv"][1, 40], c["qkv"][2, 128 + 127], c["qkv"][3, 4] = float("inf"), float("nan"), float("inf")
    got, _, _ = run(dev, c, interleaved)
    changed = (got != ref).nonzero().tolist()
    pair = [4, 5] if interleaved else [4, 20]
    assert changed == [[1, 0, 40], [2, 1, 127], [3, 0, pair[0]], [3, 0, pair[1]]]


def test_head_major_and_side_by_side_caches(dev):
    from omni_npu_amd import kernels as K
    c = make(21, 4, 2, 128, 128, seed=6)
    _, kc, vc = run(dev, c)
    pages = kc.shape[0]
    q, k, v = views(c["qkv"].to(dev), c)
    args = [x.to(dev) for x in (c["cos"], c["sin"], c["positions"], c["slots"])]
    both = torch.stack((c["kc"], c["vc"]), dim=3).to(dev)
    major = torch.stack((c["kc"], c["vc"])).permute(1, 0, 3, 2, 4).contiguous().to(dev)
    for kk, vv in ((both[:, :, :, 0], both[:, :, :, 1]), (major[:, 0].transpose(1, 2), major[:, 1].transpose(1, 2))):
        K.qk_norm_rope_cache(q, k, v, *args, kk, vv, q_gamma=c["qg"].to(dev), k_gamma=c["kg"].to(dev), eps=EPS, q_out=torch.empty_like(q))
        assert torch.equal(kk.cpu(), kc) and torch.equal(vv.cpu(), vc) and kk.shape[0] == pages


def test_replays_follow_positions_and_slots(dev):
    from omni_npu_amd import kernels as K
    c = make(9, 4, 2, 128, 128, seed=7)
    q, k, v = views(c["qkv"].to(dev), c)
    cos, sin, pos, slots, kc, vc, qg, kg = (c[n].to(dev) for n in ("cos", "sin", "positions", "slots", "kc", "vc", "qg", "kg"))
    out = torch.zeros(q.shape, dtype=c["dtype"], device=dev)
    step = lambda: K.qk_norm_rope_cache(q, k, v, cos, sin, pos, slots, kc, vc, q_gamma=qg, k_gamma=kg, eps=EPS, q_out=out)
    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for i in range(3):
        c["positions"], c["slots"] = c["positions"].roll(1), c["slots"].roll(2)
        pos.copy_(c["positions"])
        slots.copy_(c["slots"])
        out.fill_(7)
        c["kc"], c["vc"] = kc.cpu(), vc.cpu()
        graph.replay()
        torch.cuda.synchronize()
        check_all(c, out.cpu(), kc.cpu(), vc.cpu(), False)
        eager = run(dev, c)
        assert all(torch.equal(a, b.cpu()) for a, b in zip(eager, (out, kc, vc)))


def test_refusals(dev):
    from omni_npu_amd import kernels as K
    c = make(5, 4, 2, 128, 128)
    q, k, v = (x.contiguous() for x in views(c["qkv"].to(dev), c))
    on = {n: c[n].to(dev) for n in ("cos", "sin", "positions", "slots", "kc", "vc", "qg", "kg")}
    good = [q, k, v, on["cos"], on["sin"], on["positions"], on["slots"], on["kc"], on["vc"]]

    def refused(err, match, swap, **kw):
        args = list(good)
        for i, x in swap.items():
            args[i] = x
        with pytest.raises(err, match=match):
            K.qk_norm_rope_cache(*args, **kw)

    refused(ValueError, "bf16 or fp16", {0: q.float()})
    refused(ValueError, "together", {2: None})
    refused(ValueError, "together", {7: None})
    refused(ValueError, "k must be", {1: k[:4]})
    refused(ValueError, "q_out must be", {}, q_out=torch.empty(5, 4, 64, dtype=torch.bfloat16, device=dev))
    refused(ValueError, "q_gamma must be", {}, q_gamma=on["qg"].float())
    refused(ValueError, "cos / sin", {3: on["cos"].half(), 4: on["sin"].half()})
    refused(ValueError, "cos / sin", {4: on["sin"][:-1]})
    refused(ValueError, "positions", {5: on["positions"].int()})
    refused(ValueError, "slot_mapping", {6: on["slots"][:4]})
    refused(TypeError, "like the queries", {7: on["kc"].half()})
    refused(ValueError, "agree", {8: on["vc"][:-1]})
    refused(ValueError, "goes with a float8", {}, k_scale=torch.ones(2, device=dev))
    refused(ValueError, "no CPU path", {5: c["positions"]})
    refused(RuntimeError, "no backward", {0: q.clone().requires_grad_()})
    refused(K._lib.MlaHipError, "multiples of 16", {3: on["cos"][:, :20], 4: on["sin"][:, :20]})
    odd = torch.zeros(q.numel() + 1, dtype=q.dtype, device=dev)[1:].view(q.shape)
    refused(K._lib.MlaHipError, "aligned", {0: odd}, q_out=q)
    with pytest.raises(ValueError, match="go with k"):
        K.qk_norm_rope_cache(q, None, None, on["cos"], on["sin"], on["positions"], k_gamma=on["kg"])


def test_no_tokens(dev):
    from omni_npu_amd import kernels as K
    c = make(1, 4, 2, 64, 64)
    z = lambda h: torch.empty(0, h, 64, dtype=torch.bfloat16, device=dev)
    i = torch.empty(0, dtype=torch.int64, device=dev)
    kc = c["kc"].to(dev)
    K.qk_norm_rope_cache(z(4), z(2), z(2), c["cos"].to(dev), c["sin"].to(dev), i, i, kc, kc.clone())
    K.qk_norm_rope_cache(z(4), None, None, c["cos"].to(dev), c["sin"].to(dev), i)
    assert torch.equal(kc.cpu(), c["kc"])


@pytest.mark.parametrize("d,interleaved", [(64, False), (128, True), (256, False)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "fp16"])
@pytest.mark.parametrize("fp8", [False, True], ids=["same", "e4m3"])
def test_large_batches_are_as_their_parts(dev, d, interleaved, dtype, fp8):
    """From 64 MB of input on values go past the caches: the same bits as in calls of a few hundred tokens."""
    from omni_npu_amd import kernels as K
    hq, hk = 30, 5
    t = (64 << 20) // (40 * d * 2) + 77
    g = torch.Generator(device=dev).manual_seed(d)
    qkv = torch.randn(t, 40 * d, generator=g, device=dev).to(dtype)
    angle = torch.outer(torch.arange(t, device=dev).float(), 10000.0 ** (-torch.arange(0, d, 2, device=dev).float() / d))
    gamma = (1 + 0.1 * torch.randn(d, generator=g, device=dev)).to(dtype)
    scale = torch.full((hk,), 0.02, device=dev) if fp8 else None
    positions, slots = torch.arange(t, device=dev), torch.randperm(t + 50, generator=g, device=dev)[:t]
    slots[5] = -1

    def outputs(step):
        q_out = torch.zeros(t, hq, d, dtype=dtype, device=dev)
        kc, vc = (torch.zeros(-(-(t + 50) // 16), 16, hk, d, device=dev).to(E4M3 if fp8 else dtype) for _ in range(2))
        for a in range(0, t, step):
            part = slice(a, min(a + step, t))
            q, k, v = (x.unflatten(1, (-1, d)) for x in qkv[part].split([hq * d, hk * d, hk * d], dim=1))
            K.qk_norm_rope_cache(q, k, v, angle.cos(), angle.sin(), positions[part], slots[part], kc, vc, q_gamma=gamma, k_gamma=gamma, eps=EPS,
                                 interleaved=interleaved, q_out=q_out[part], k_scale=scale, v_scale=scale)
        return q_out, kc.view(torch.uint8), vc.view(torch.uint8)

    for whole, parts in zip(outputs(t), outputs(3001)):
        assert torch.equal(whole, parts) and whole.any()
