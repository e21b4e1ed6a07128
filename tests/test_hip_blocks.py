"""GPU: the transformer-block operators (mggan/hip/blocks.py) against their definitions in 64 bits, element by element.

Tolerances: u = half a step of the type (2^-8 bf16, 2^-24 f32).  A sum of n products in f32 is off by at most n 2^-24 times the sum
of the products' absolute values (any order); exp and what is built on it by (8 + |z|) 2^-23 of its value (a rounded argument of
size |z| and a few steps of the instruction); every value that is rounded to the operands' type by u of itself.  The bounds below
carry these through the formulas with absolute values in the place of the terms."""
import pytest
import torch

pytestmark = pytest.mark.gpu

U = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}
F = 2.0 ** -24
TYPES = [torch.float32, torch.bfloat16]


def B():
    assert torch.cuda.is_available(), "GPU tests need a HIP device"
    from mggan.hip import blocks

    return blocks


def rnd(gen, *shape, dtype, std=1.0):
    return (torch.randn(*shape, generator=gen) * std).to(dtype).cuda()


def close(got, want, bound, what):
    assert got.shape == want.shape, what
    err = (got.double() - want).abs()
    bad = ~(err <= bound + 1e-37)
    assert not bad.any(), "{}: {} of {} beyond their bounds, worst {:.3g} times".format(
        what, int(bad.sum()), bad.numel(), float((err / (bound + 1e-37)).max()))


def act_of(z, act, slope):
    """(value, derivative, bound of the second derivative) in 64 bits."""
    if act == 0:
        return z, torch.ones_like(z), 0.0
    if act == 1:
        return torch.where(z > 0, z, z * slope), torch.where(z > 0, 1.0, slope).double(), 0.0
    s = torch.sigmoid(z)
    if act == 2:
        return s, s * (1 - s), 0.1
    if act == 4:
        return z * s, s * (1 + z * (1 - s)), 0.5
    phi, cdf = torch.exp(-0.5 * z * z) * 0.3989422804014327, 0.5 * torch.erfc(-z * 0.5 ** 0.5)
    return z * cdf, cdf + z * phi, 0.8


LAYERS = [  # rows, inputs, outputs: one row, odd sizes, tails of tiles and steps, several tiles, a long reduction with few outputs
    (1, 8, 8), (1, 1, 1), (3, 5, 7), (16, 64, 64), (17, 72, 40), (65, 136, 130), (130, 1000, 96), (300, 200, 520), (257, 513, 259),
    (2, 4096, 33), (5000, 24, 40), (1100, 264, 1032)]

# enough tiles of 128 x 128 and of 256 x 256 outputs for the kernels that take those, with ragged edges
BIG = [(1800, 200, 1736), (4000, 72, 3333), (4100, 328, 3400)]


def layer_bounds(x, w, b, dtype):
    K = w.shape[1]
    z = x.double() @ w.double().t() + (0 if b is None else b.double())
    size = x.double().abs() @ w.double().abs().t() + (0 if b is None else b.double().abs())
    return z, (K + 4) * F * size


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M,K,N,act", [s + (a,) for s in LAYERS for a in (0, 1, 2, 4, 5)] + [s + (5,) for s in BIG])
def test_linear_residual(M, K, N, act, dtype):
    blocks, gen, u = B(), torch.Generator().manual_seed(M + K + N), U[dtype]
    slope = 0.2
    x, w = rnd(gen, M, K, dtype=dtype), rnd(gen, N, K, dtype=dtype, std=K ** -0.5)
    b, r, dy = rnd(gen, N, dtype=dtype), rnd(gen, M, N, dtype=dtype), rnd(gen, M, N, dtype=dtype)
    if (M + act) % 3 == 0:
        b = None
    if (N + act) % 3 == 0:
        r = None
    leaves = [t.requires_grad_() for t in (x, w, b, r) if t is not None]
    y = blocks.linear_residual(x, w, b, r, act=act, slope=slope)
    grads = dict(zip([n for n, t in zip("xwbr", (x, w, b, r)) if t is not None], torch.autograd.grad(y, leaves, dy)))
    with torch.no_grad():
        y0 = blocks.linear_residual(x, w, b, r, act=act, slope=slope)
        assert torch.equal(y0, y)  # (keeping the activation's input changes nothing)
        z, ez = layer_bounds(x, w, b, dtype)
        a, d, d2 = act_of(z, act, slope)
        ref = a if r is None else a + r.double()
        ea = ez * (1.13 if act else 1.0) + (0 if act < 2 else (8 + z.abs()) * 2 * F * a.abs())
        close(y, ref, u * (1 + F) * (ref.abs() + ea) + ea + F * ref.abs() + F * a.abs(), "y")
        dyd = dy.double()
        dz = dyd * d
        # z kept in the operands' type: off by u |z|; its derivative moves by at most d2 times that
        edz = dyd.abs() * (d2 * (u * z.abs() + ez) + (0 if act < 2 else (8 + z.abs()) * 4 * F))
        if act == 1:  # on the step of the slope a value within the error of zero may fall on either side
            edz = edz + dyd.abs() * (z.abs() <= ez)
        es = edz + F * dz.abs()
        edz = es + u * (dz.abs() + es)
        xd, wd = x.double(), w.double()
        for name, got, want, err in (
                ("x", grads["x"], dz @ wd, edz @ wd.abs() + (N + 4) * F * ((dz.abs() + edz) @ wd.abs())),
                ("w", grads["w"], dz.t() @ xd, edz.t() @ xd.abs() + (M + 4) * F * ((dz.abs() + edz).t() @ xd.abs()))):
            close(got, want, err + u * (want.abs() + err), "d" + name)
        if b is not None:
            want, err = dz.sum(0), es.sum(0) + (M + 4) * F * (dz.abs() + es).sum(0)
            close(grads["b"], want, err + u * (want.abs() + err), "db")
        if r is not None:
            assert torch.equal(grads["r"], dy)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M,K,N,act,bias", [s + a for s in LAYERS for a in ((4, True), (5, False), (2, True), (1, False))] +
                         [s + (4, True) for s in BIG])
def test_gated_linear(M, K, N, act, bias, dtype):
    blocks, gen, u = B(), torch.Generator().manual_seed(M + K + N + 1), U[dtype]
    slope = 0.1
    x, w, v = rnd(gen, M, K, dtype=dtype), rnd(gen, N, K, dtype=dtype, std=K ** -0.5), rnd(gen, N, K, dtype=dtype, std=K ** -0.5)
    b, c = (rnd(gen, N, dtype=dtype), rnd(gen, N, dtype=dtype)) if bias else (None, None)
    dy = rnd(gen, M, N, dtype=dtype)
    leaves = [t.requires_grad_() for t in (x, w, v, b, c) if t is not None]
    y = blocks.gated_linear(x, w, v, b, c, act=act, slope=slope)
    grads = dict(zip([n for n, t in zip("xwvbc", (x, w, v, b, c)) if t is not None], torch.autograd.grad(y, leaves, dy)))
    with torch.no_grad():
        assert torch.equal(blocks.gated_linear(x, w, v, b, c, act=act, slope=slope), y)
        z, ez = layer_bounds(x, w, b, dtype)
        up, eu = layer_bounds(x, v, c, dtype)
        a, d, d2 = act_of(z, act, slope)
        ea = ez * 1.13 + (0 if act < 2 else (8 + z.abs()) * 2 * F * a.abs()) + F * a.abs()
        ref = a * up
        e = ea * (up.abs() + eu) + a.abs() * eu + F * ref.abs()
        close(y, ref, e + u * (ref.abs() + e), "y")
        dyd = dy.double()
        kz, ku = u * z.abs() + ez, u * up.abs() + eu  # what the kept inputs are off by
        ed = d2 * kz + (0 if act < 2 else (8 + z.abs()) * 4 * F)
        if act == 1:
            ed = ed + (z.abs() <= ez)
        dz, du = dyd * up * d, dyd * a
        es_z = dyd.abs() * (ed * (up.abs() + ku) + d.abs() * ku) + 3 * F * dz.abs()
        es_u = dyd.abs() * (1.13 * kz + (0 if act < 2 else (8 + z.abs()) * 2 * F * a.abs())) + 2 * F * du.abs()
        ez_, eu_ = es_z + u * (dz.abs() + es_z), es_u + u * (du.abs() + es_u)
        xd, wd, vd = x.double(), w.double(), v.double()
        err = ez_ @ wd.abs() + eu_ @ vd.abs() + (2 * N + 4) * F * ((dz.abs() + ez_) @ wd.abs() + (du.abs() + eu_) @ vd.abs())
        want = dz @ wd + du @ vd
        close(grads["x"], want, err + u * (want.abs() + err), "dx")
        for name, t, et in (("w", dz, ez_), ("v", du, eu_)):
            want = t.t() @ xd
            err = et.t() @ xd.abs() + (M + 4) * F * ((t.abs() + et).t() @ xd.abs())
            close(grads[name], want, err + u * (want.abs() + err), "d" + name)
        if bias:
            for name, t, et in (("b", dz, es_z), ("c", du, es_u)):
                want, err = t.sum(0), et.sum(0) + (M + 4) * F * (t.abs() + et).sum(0)
                close(grads[name], want, err + u * (want.abs() + err), "d" + name)


# ---- attention ---------------------------------------------------------------------------------------------------------------

def visible(N, M, scenes, kv_scenes, causal, prefix):
    """(N, M) truth values from the definition, scene by scene."""
    see = torch.zeros(N, M, dtype=torch.bool)
    for s, ((a, b), (c, d)) in enumerate(zip(scenes, kv_scenes)):
        see[a:b] = False
        i, j = torch.arange(b - a)[:, None], torch.arange(d - c)[None]
        ok = torch.ones(b - a, d - c, dtype=torch.bool)
        if causal:
            ok = (j <= i + (d - c) - (b - a)) | (j < (prefix[s] if prefix is not None else 0))
        see[a:b, c:d] = ok
    return see.cuda()


def reference(q, k, v, see, dout, scale, cap, xy, kv_xy, slopes):
    """{name: (value, bound)} in 64 bits; the bounds follow the kernels' roundings (module docstring)."""
    (N, H, D), (M, Hkv, _), dtype = q.shape, k.shape, q.dtype
    u, ub, G = U[dtype], 0.0 if dtype == torch.float32 else U[dtype], H // Hkv
    Q, K, V, dO = (t.detach().double().transpose(0, 1) for t in (q, k, v, dout))
    Kh, Vh = K.repeat_interleave(G, 0), V.repeat_interleave(G, 0)
    z = scale * (Q @ Kh.transpose(1, 2))
    es = (D + 8) * F * scale * (Q.abs() @ Kh.abs().transpose(1, 2))
    t = torch.tanh(z / cap) if cap else None
    s = cap * t if cap else z
    es = es + 8 * F * s.abs() + (0 if not cap else cap * (4 * F * t.abs() if dtype == torch.float32 else 8 * F))
    dist = None
    if xy is not None:
        dist = (xy.double()[:, None] - kv_xy.double()[None]).norm(dim=-1)
        bias = slopes.detach().double()[:, None, None] * dist
        s, es = s - bias, es + 8 * F * bias.abs()
    s = s.masked_fill(~see, -torch.inf)
    P = torch.softmax(s, -1).nan_to_num(0.0)
    n = see.sum(-1).double()[None, :, None]
    rel = 2 * (es * see).amax(-1, keepdim=True) + (n + 16) * F
    O = P @ Vh
    A = P @ Vh.abs()
    eO = (rel + ub) * A * (1 + ub) + (n + 4) * F * A
    eO = eO + u * (O.abs() + eO)
    dP = dO @ Vh.transpose(1, 2)
    edP = (D + 4) * F * (dO.abs() @ Vh.abs().transpose(1, 2))
    delta = (dO * O).sum(-1, keepdim=True)
    edelta = (dO.abs() * (eO + (D + 4) * F * O.abs())).sum(-1, keepdim=True)
    dL = P * (dP - delta)
    edL = (rel * dL.abs() + P * (edP + edelta) * (1 + rel) + 4 * F * P * (dP.abs() + delta.abs()))
    dS, eS = dL, edL
    if cap:
        fac = 1 - t * t
        efac = 2 * (es / cap + 8 * F) + 4 * F
        dS, eS = dL * fac, edL * fac + (dL.abs() + edL) * efac
    eS = eS + ub * (dS.abs() + eS)
    dQ, eQ = scale * (dS @ Kh), scale * ((eS + (n + 4) * F * (dS.abs() + eS)) @ Kh.abs())
    m = see.sum(0).double()[None, :, None] * G
    dK, eK = scale * (dS.transpose(1, 2) @ Q), scale * (eS.transpose(1, 2) @ Q.abs() + (m + 4) * F * ((dS.abs() + eS).transpose(1, 2) @ Q.abs()))
    dV, Pt = P.transpose(1, 2) @ dO, P.transpose(1, 2)
    eV = (rel * P).transpose(1, 2) @ dO.abs() + (ub * (1 + F) + (m + 4) * F) * (Pt @ dO.abs())
    fold = lambda x: x.view(Hkv, G, M, D).sum(1)
    out = {"out": (O, eO), "dq": (dQ, eQ + u * (dQ.abs() + eQ))}
    for nme, x, e in (("dk", fold(dK), fold(eK)), ("dv", fold(dV), fold(eV))):
        out[nme] = (x, e + u * (x.abs() + e))
    out = {nme: (x.transpose(0, 1), e.transpose(0, 1)) for nme, (x, e) in out.items()}
    if xy is not None:
        d = -(dL * dist).sum((1, 2))
        # sums of 32 terms, of a wave's tiles, of 64 lanes, in 64 bits from there: at most 2 Lk / 32 + 200 additions one after another
        out["dslopes"] = (d, ((edL + (8 + 200 + M / 16) * F * dL.abs()) * dist).sum((1, 2)))
    return out


def lengths_to_scenes(lengths, start=0):
    out = []
    for n in lengths:
        out.append((start, start + n))
        start += n
    return out


ATTENTION = {  # rows of each scene (keys, if other), heads, key heads, width, causal, prefix, cap, axes, rows behind the last scene
    "one_row": ([1], None, 1, 1, 8, False, None, 0.0, 0, 0),
    "one_row_causal_bias": ([1], None, 2, 1, 16, True, None, 5.0, 1, 3),
    "tiny_scenes": ([1, 2, 0, 3, 5, 1, 0, 7, 2, 4, 6, 1, 1], None, 4, 4, 32, False, None, 0.0, 2, 0),
    "tiny_scenes_cap": ([3, 1, 4, 1, 5, 9, 2, 6, 5, 3, 5, 8, 9, 7, 9], None, 4, 2, 32, False, None, 8.0, 2, 5),
    "scenes_64x20": ([20] * 64, None, 4, 4, 32, False, None, 0.0, 2, 0),
    "scenes_33": ([33, 31, 65, 64, 63, 1, 17], None, 3, 1, 24, False, None, 20.0, 2, 0),
    "causal": ([130, 257, 1, 64], None, 4, 2, 64, True, None, 0.0, 0, 1),
    "causal_prefix": ([100, 7, 300, 0, 45], None, 4, 1, 64, True, [30, 7, 0, 4, 200], 30.0, 0, 0),
    "causal_bias": ([513], None, 2, 2, 128, True, None, 0.0, 1, 0),
    "width_80": ([150, 90], None, 2, 2, 80, True, [0, 90], 0.0, 0, 0),
    "width_40_bias": ([77, 200], None, 4, 4, 40, False, None, 12.0, 1, 0),
    "more_keys": ([5, 1, 40], [100, 37, 41], 6, 2, 64, True, None, 0.0, 0, 0),
    "fewer_keys": ([50, 9, 30], [20, 0, 64], 2, 1, 32, True, [3, 0, 10], 0.0, 0, 2),
    "one_token_each": ([1] * 9, [1, 64, 65, 200, 0, 31, 129, 5, 700], 8, 2, 64, True, None, 15.0, 1, 0),
    "tokens_many_shares": ([1, 1], [3000, 2111], 4, 1, 32, True, None, 0.0, 0, 0),
    "tokens_20_heads_a_key_head": ([1] * 3, [700, 1, 90], 40, 2, 16, True, None, 0.0, 2, 1),
    "tokens_wide": ([1, 0, 1, 1], [400, 3, 77, 130], 4, 2, 128, False, None, 0.0, 0, 0),
    "tokens_wide_f": ([1, 1], [64, 129], 4, 4, 96, True, None, 9.0, 1, 0),
    "wide_launch": ([900, 1300, 2100], None, 8, 4, 64, True, None, 0.0, 0, 0),
    "wide_launch_bias": ([2000, 2300], None, 8, 8, 32, True, [100, 0], 25.0, 2, 0),
}


def make(case, dtype, seed=0):
    rows, keys, H, Hkv, D, causal, prefix, cap, axes, behind = ATTENTION[case]
    gen = torch.Generator().manual_seed(seed + len(case))
    scenes = lengths_to_scenes(rows)
    kv_scenes = scenes if keys is None else lengths_to_scenes(keys, 3)
    N = scenes[-1][1] + behind
    M = N if keys is None else kv_scenes[-1][1] + 4
    q, k, v, dout = (rnd(gen, n, h, D, dtype=dtype) for n, h in ((N, H), (M, Hkv), (M, Hkv), (N, H)))
    xy = kv_xy = slopes = None
    if axes:
        xy = (torch.rand(N, axes, generator=gen) * 12).cuda()
        kv_xy = xy if keys is None else (torch.rand(M, axes, generator=gen) * 12).cuda()
        slopes = (torch.rand(H, generator=gen) * 0.4).cuda()
    return q, k, v, dout, scenes, kv_scenes, dict(causal=causal, prefix=prefix, cap=cap, xy=xy, kv_xy=kv_xy, slopes=slopes)


def run_attention(q, k, v, dout, scenes, kv_scenes, opt):
    leaves = {"dq": q, "dk": k, "dv": v}
    if opt["slopes"] is not None:
        leaves["dslopes"] = opt["slopes"]
    for t in leaves.values():
        t.requires_grad_()
    out = B().attention(q, k, v, scenes, kv_scenes, **opt)
    return {"out": out.detach(), **dict(zip(leaves, torch.autograd.grad(out, list(leaves.values()), dout)))}


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("case", list(ATTENTION))
def test_attention(case, dtype):
    q, k, v, dout, scenes, kv_scenes, opt = make(case, dtype)
    got = run_attention(q, k, v, dout, scenes, kv_scenes, opt)
    with torch.no_grad():
        alone = B().attention(q, k, v, scenes, kv_scenes, **opt)  # (single rows over long caches take a kernel of their own here)
        see = visible(q.shape[0], k.shape[0], scenes, kv_scenes, opt["causal"], opt["prefix"])
        want = reference(q, k, v, see, dout, q.shape[2] ** -0.5, opt["cap"], opt["xy"], opt["kv_xy"], opt["slopes"])
        assert set(want) == set(got)
        for name, (x, e) in want.items():
            close(got[name], x, e, name)
        close(alone, *want["out"], "out without gradients")
        blind = ~see.any(1)
        assert not alone[blind].any() and not got["out"][blind].any() and not got["dq"][blind].any()
        unseen = ~see.any(0)
        assert not got["dk"][unseen].any() and not got["dv"][unseen].any()
