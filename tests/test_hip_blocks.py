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
    (2, 4096, 33), (5000, 24, 40), (1100, 264, 1032),
    (33, 40, 159), (70, 159, 127), (16, 333, 700), (15, 2005, 24), (40, 96, 320)]

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


BAD = [float("nan"), float("inf"), float("-inf")]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("width,cap,axes", [(32, 0.0, 2), (64, 20.0, 0), (128, 0.0, 1)])
def test_attention_values_that_are_not_finite_stay_in_their_scene(width, cap, axes, dtype):
    """Scene 1 of three holds NaN and infinities in every operand, and rows no scene names do: the others' results are what they were."""
    gen = torch.Generator().manual_seed(width)
    scenes, N = [(0, 21), (21, 60), (60, 147)], 150
    clean = {n: rnd(gen, N, h, width, dtype=dtype) for n, h in (("q", 4), ("k", 2), ("v", 2), ("dout", 4))}
    xy = (torch.rand(N, axes, generator=gen) * 9).cuda() if axes else None
    slopes = torch.rand(4, generator=gen).cuda() if axes else None
    ok = torch.ones(N, dtype=torch.bool)
    ok[21:60] = ok[147:] = False
    runs = []
    for poisoned in (False, True):
        t = {n: x.clone() for n, x in clean.items()}
        if poisoned:
            for i, x in enumerate(t.values()):
                x[147:] = BAD[0]
                x[40, :, i] = BAD[i % 3]
                x[25, 0, 5 + i:] = BAD[(i + 1) % 3]
        p = xy.clone() if axes else None
        if axes and poisoned:
            p[30] = BAD[1]
            p[148:] = BAD[0]
        opt = dict(causal=width == 64, prefix=[3, 9, 50] if width == 64 else None, cap=cap, xy=p, kv_xy=p, slopes=slopes.clone() if axes else None)
        r = run_attention(t["q"], t["k"], t["v"], t["dout"], scenes, scenes, opt)
        with torch.no_grad():
            r["alone"] = B().attention(t["q"], t["k"], t["v"], scenes, **opt)
        runs.append(r)
    for name in ("out", "alone", "dq", "dk", "dv"):
        got, want = runs[1][name][ok.cuda()], runs[0][name][ok.cuda()]
        assert torch.isfinite(got).all(), name
        # the sums are the same ones, through another product: off by their rounding at most
        torch.testing.assert_close(got.double(), want.double(), rtol=4 * U[dtype], atol=64 * F * float(want.abs().max()))
        assert not torch.isfinite(runs[1][name][21:60]).all(), name
    assert not torch.isfinite(runs[1]["out"][40]).all()


@pytest.mark.parametrize("dtype", TYPES)
def test_attention_values_that_are_not_finite_behind_the_causal_mask(dtype):
    """A key that a row does not see yet may be anything; rows that see it get what the definition gives, column by column."""
    gen = torch.Generator().manual_seed(5)
    N, at = 100, 70
    q, k, v = (rnd(gen, N, 2, 64, dtype=dtype) for _ in range(3))
    with torch.no_grad():
        want = B().attention(q, k, v, [(0, N)], causal=True)
        v[at, 0, 3], v[at, 0, 4], v[at + 5, 0, 4], v[at, 0, 5] = BAD[0], BAD[1], BAD[2], BAD[2]
        got = B().attention(q, k, v, [(0, N)], causal=True)
    seen = torch.zeros(N, 2, 64, dtype=torch.bool, device="cuda")
    seen[at:, 0, 3:6] = True
    torch.testing.assert_close(got[~seen].double(), want[~seen].double(), rtol=4 * U[dtype], atol=1e-5)
    assert got[at:, 0, 3].isnan().all()
    assert (got[at:at + 5, 0, 4] == float("inf")).all() and got[at + 5:, 0, 4].isnan().all()
    assert (got[at:, 0, 5] == float("-inf")).all()


@pytest.mark.parametrize("dtype", TYPES)
def test_attention_reads_views_of_packed_and_unaligned_operands(dtype):
    gen = torch.Generator().manual_seed(8)
    N, H, D, scenes = 90, 4, 40, [(0, 33), (33, 90)]
    packed = rnd(gen, N, 3, H, D, dtype=dtype)
    odd = rnd(gen, N * H * D + 1, dtype=dtype)[1:].view(N, H, D)
    dout = rnd(gen, N, D, H, dtype=dtype).transpose(1, 2)
    B_ = B()
    views = [(packed[:, 0], packed[:, 1], packed[:, 2]), (odd, packed[:, 1], packed[:, 2].transpose(0, 1).contiguous().transpose(0, 1)),
             (packed.transpose(2, 3).contiguous().transpose(2, 3)[:, 0], odd, odd)]
    for q, k, v in views:
        plain = [x.detach().clone(memory_format=torch.contiguous_format).requires_grad_() for x in (q, k, v)]
        leaves = [x.detach().requires_grad_() for x in (q, k, v)]
        a, b = B_.attention(*leaves, scenes), B_.attention(*plain, scenes)
        assert torch.equal(a, b)
        for x, y in zip(torch.autograd.grad(a, leaves, dout), torch.autograd.grad(b, plain, dout.contiguous())):
            assert torch.equal(x, y)


def test_attention_scene_tables():
    """Device tables in any order, with rows that several scenes name, padding entries and rows behind the operands."""
    gen = torch.Generator().manual_seed(9)
    N, B_ = 70, B()
    q, k, v = (rnd(gen, N, 2, 32, dtype=torch.float32) for _ in range(3))
    table = lambda rows: torch.tensor(rows, dtype=torch.int32, device="cuda")
    with torch.no_grad():
        want = B_.attention(q, k, v, [(0, 30), (30, 64)])
        assert torch.equal(B_.attention(q, k, v, table([[30, 64], [0, 30], [0, 0], [70, 70]])), want)
        assert torch.equal(B_.attention(q, k, v, table([[0, 64], [30, 64], [0, 30]])), want)  # the last one that names a row
        far = B_.attention(q, k, v, table([[0, 30], [30, 64], [64, 5000]]), table([[0, 30], [30, 64], [-7, 100000]]))
        assert torch.equal(far[:64], want[:64])
        assert torch.equal(far[64:], B_.attention(q, k, v, [(64, 70)], [(0, 70)])[64:])
        assert not B_.attention(q, k, v, table([[0, 0]])).any()
        assert not B_.attention(q, k, v, torch.zeros(0, 2, dtype=torch.int32, device="cuda")).any()
        assert B_.attention(q[:0], k, v, [(0, 0)]).shape == (0, 2, 32)
        assert not B_.attention(q, k[:0], v[:0], [(0, 70)], [(0, 0)]).any()
    # scenes that share keys: the gradients of the keys add up
    qq, kk, vv = (x[:40].clone().requires_grad_() for x in (q, k, v))
    shared = B_.attention(qq, kk, vv, [(0, 10), (10, 40)], [(0, 40), (0, 40)])
    one = B_.attention(qq, kk, vv, [(0, 40)])
    assert torch.equal(shared, one)
    for a, b in zip(torch.autograd.grad(shared, [qq, kk, vv], q[:40]), torch.autograd.grad(one, [qq, kk, vv], q[:40])):
        assert torch.equal(a, b)


def test_layers_read_views_and_empty_batches():
    gen = torch.Generator().manual_seed(10)
    B_ = B()
    for dtype in TYPES:
        wide = rnd(gen, 50, 100, dtype=dtype)
        w, up = rnd(gen, 24, 40, dtype=dtype), rnd(gen, 24, 40, dtype=dtype)
        bias = rnd(gen, 25, dtype=dtype)[1:]
        res = rnd(gen, 24, 50, dtype=dtype).t()
        for x in (wide[:, 8:48], wide[:, 3:43], wide[::2, 16:56], rnd(gen, 40, 50, dtype=dtype).t(), wide[:, :40].reshape(5, 10, 40)):
            plain, leaf = x.contiguous().clone().requires_grad_(), x.detach().requires_grad_()
            r = res[:x.shape[0]] if x.dim() == 2 else res.reshape(5, 10, 24)
            for f in (lambda t: B_.linear_residual(t, w, bias, r, act=B_.ACT_GELU), lambda t: B_.gated_linear(t, w, up, bias, None)):
                a, b = f(leaf), f(plain)
                assert torch.equal(a, b)
                assert torch.equal(torch.autograd.grad(a, leaf, torch.ones_like(a))[0], torch.autograd.grad(b, plain, torch.ones_like(b))[0])
        none = torch.zeros(0, 40, dtype=dtype, device="cuda", requires_grad=True)
        w_ = w.clone().requires_grad_()
        for y in (B_.linear_residual(none, w_, act=B_.ACT_SILU), B_.gated_linear(none, w_, up)):
            assert y.shape == (0, 24)
            dx, dw = torch.autograd.grad(y, [none, w_], y)
            assert dx.shape == (0, 40) and not dw.any()
        t = wide[:, :40].clone().requires_grad_()  # only some gradients wanted; a gradient that is broadcast
        y = B_.gated_linear(t, w, up)
        assert torch.equal(torch.autograd.grad(y.sum(), t)[0], torch.autograd.grad(B_.gated_linear(t, w, up), t, torch.ones_like(y))[0])


def block(x, p, table, heads, xy, slopes):
    """Attention and feed-forward of one block, as a user composes them."""
    B_ = B()
    N, C = x.shape
    qkv = B_.linear_residual(x, p["qkv"], p["qkv_b"]).view(N, 3, heads, C // heads)
    mixed = B_.attention(qkv[:, 0], qkv[:, 1], qkv[:, 2], table, causal=xy is None, cap=25.0, xy=xy, slopes=slopes)
    x = B_.linear_residual(mixed.reshape(N, C), p["out"], p["out_b"], x)
    return B_.linear_residual(B_.gated_linear(x, p["gate"], p["up"], act=B_.ACT_GELU), p["down"], None, x)


def block64(x, p, scenes, heads, xy, slopes):
    N, C = x.shape
    qkv = (x @ p["qkv"].t() + p["qkv_b"]).view(N, 3, heads, C // heads)
    see = visible(N, N, scenes, scenes, xy is None, None)
    q, k, v = (qkv[:, i].transpose(0, 1) for i in range(3))
    s = 25.0 * torch.tanh(q @ k.transpose(1, 2) * (C // heads) ** -0.5 / 25.0)
    if xy is not None:
        s = s - slopes[:, None, None] * (xy[:, None] - xy[None]).square().sum(-1).add(1e-300).sqrt()
    mixed = (torch.softmax(s.masked_fill(~see, -torch.inf), -1) @ v).transpose(0, 1).reshape(N, C)
    x = mixed @ p["out"].t() + p["out_b"] + x
    h = torch.nn.functional.gelu(x @ p["gate"].t()) * (x @ p["up"].t())
    return h @ p["down"].t() + x


def block_inputs(dtype, spatial, seed=3):
    gen = torch.Generator().manual_seed(seed)
    C, heads, hidden, lengths = 96, 3, 200, [20, 1, 33, 7, 64, 50]
    scenes, N = lengths_to_scenes(lengths), sum(lengths)
    sizes = {"qkv": (3 * C, C), "qkv_b": (3 * C,), "out": (C, C), "out_b": (C,), "gate": (hidden, C), "up": (hidden, C), "down": (C, hidden)}
    p = {n: rnd(gen, *s, dtype=dtype, std=s[-1] ** -0.5 if len(s) > 1 else 0.1) for n, s in sizes.items()}
    x, dy = rnd(gen, N, C, dtype=dtype), rnd(gen, N, C, dtype=dtype)
    xy = (torch.rand(N, 2, generator=gen) * 10).cuda() if spatial else None
    slopes = (torch.rand(heads, generator=gen) * 0.3).cuda() if spatial else None
    return x, dy, p, scenes, heads, xy, slopes


@pytest.mark.parametrize("spatial", [False, True])
@pytest.mark.parametrize("dtype", TYPES)
def test_block_of_all_three(dtype, spatial):
    """A block's output and every gradient against the same in 64 bits, by 2-norm.  Ten roundings to the operands' type lie in a row on the
    longest way (projections, scores' weights, outputs, their gradients), each at most u of its value; errors of products of independent
    terms add in squares, and a residual stream keeps what passes by them: 12 u; in f32 sums of up to 200 terms and 16-step functions
    count as 40 u."""
    x, dy, p, scenes, heads, xy, slopes = block_inputs(dtype, spatial)
    leaves = [x] + list(p.values()) + ([slopes] if spatial else [])
    for t in leaves:
        t.requires_grad_()
    y = block(x, p, scenes, heads, xy, slopes)
    got = torch.autograd.grad(y, leaves, dy)
    up = lambda t: t.detach().double().requires_grad_()
    x64, p64, s64 = up(x), {n: up(t) for n, t in p.items()}, up(slopes) if spatial else None
    y64 = block64(x64, p64, scenes, heads, None if xy is None else xy.double(), s64)
    want = torch.autograd.grad(y64, [x64] + list(p64.values()) + ([s64] if spatial else []), dy.double())
    for name, a, b in [("y", y, y64)] + list(zip(["x"] + list(p) + ["slopes"], got, want)):
        rel = float((a.detach().double() - b.detach()).norm() / b.detach().norm())
        assert rel <= (12 if dtype == torch.bfloat16 else 40) * U[dtype], (name, rel)


def test_gradients_against_differences():
    """Directional derivatives of the f32 block from values of the same kernels: central differences of step h have an error of h^2 times
    the third derivative and of 2^-24 |y| sqrt(terms) / h; h = 2^-6 leaves both below 2e-3 of the derivative here."""
    x, dy, p, scenes, heads, xy, slopes = block_inputs(torch.float32, True, seed=12)
    leaves = {"x": x, **p, "slopes": slopes}
    for t in leaves.values():
        t.requires_grad_()
    grads = dict(zip(leaves, torch.autograd.grad(block(x, p, scenes, heads, xy, slopes), list(leaves.values()), dy)))
    gen, h = torch.Generator().manual_seed(2), 2.0 ** -6
    for name, t in leaves.items():
        d = torch.randn(t.shape, generator=gen).cuda()
        d = (d / d.norm() * 0.5 + grads[name] / grads[name].norm() * 0.5).detach()
        value = []
        for sign in (1, -1):
            moved = {n: (u + sign * h * d if n == name else u).detach() for n, u in leaves.items()}
            with torch.no_grad():
                y = block(moved["x"], {n: moved[n] for n in p}, scenes, heads, xy, moved["slopes"])
            value.append(float((y.double() * dy.double()).sum()))
        numeric, formula = (value[0] - value[1]) / (2 * h), float((grads[name].double() * d.double()).sum())
        assert abs(numeric - formula) <= 5e-3 * abs(formula) + 5e-3, (name, numeric, formula)


@pytest.mark.parametrize("dtype", TYPES)
def test_runs_streams_and_graphs_give_the_same_bits(dtype):
    x, dy, p, scenes, heads, xy, slopes = block_inputs(dtype, True, seed=4)
    table = torch.tensor(scenes, dtype=torch.int32, device="cuda")
    leaves = [x] + list(p.values()) + [slopes]
    for t in leaves:
        t.requires_grad_()

    def step():
        y = block(x, p, table, heads, xy, slopes)
        return (y,) + torch.autograd.grad(y, leaves, dy)

    first = [t.detach().clone() for t in step()]
    for t, u in zip(first, step()):
        assert torch.equal(t, u)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        on_side = [step() for _ in range(2)]  # (two calls in flight on one stream, the first one's results alive)
    # two captured graphs of the same leaves, replayed in turn, with eager work between
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    for r in on_side:
        for t, u in zip(first, r):
            assert torch.equal(t, u)
    del on_side, r, u, t
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            outs = step()
        graphs.append((g, [t.detach() for t in outs]))
        del outs
    for i in range(4):
        for g, outs in graphs:
            for t in outs:
                t.zero_()
            g.replay()
            torch.cuda.synchronize()
            for t, u in zip(first, outs):
                assert torch.equal(t, u), i
        eager = step()
        assert torch.equal(eager[0], first[0])
        del eager
    # new values in place: a replay reads them, and the scene table in device memory too
    with torch.no_grad():
        x.mul_(0.5)
        table.copy_(torch.tensor([[0, 20], [20, 54], [54, 54], [54, 61], [61, 125], [125, 175]], dtype=torch.int32))
    want = [t.detach() for t in step()]
    for g, outs in graphs:
        g.replay()
        torch.cuda.synchronize()
        for t, u in zip(want, outs):
            assert torch.equal(t, u)


def test_serving_step_in_a_graph():
    """One new row per sequence over a growing cache: the graph reads the lengths when it runs."""
    gen = torch.Generator().manual_seed(6)
    S, room, H, Hkv, D = 5, 300, 8, 2, 64
    q = rnd(gen, S, H, D, dtype=torch.bfloat16)
    k, v = (rnd(gen, S * room, Hkv, D, dtype=torch.bfloat16) for _ in range(2))
    lens = [1, 17, 64, 200, 299]
    rows = torch.tensor([[s, s + 1] for s in range(S)], dtype=torch.int32, device="cuda")
    kv = torch.tensor([[s * room, s * room + n] for s, n in enumerate(lens)], dtype=torch.int32, device="cuda")
    B_ = B()
    with torch.no_grad():
        B_.attention(q, k, v, rows, kv)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = B_.attention(q, k, v, rows, kv)
        for step in range(3):
            g.replay()
            assert torch.equal(out, B_.attention(q, k, v, rows, kv))
            see = visible(S, S * room, [(s, s + 1) for s in range(S)], kv.tolist(), False, None)
            want = reference(q, k, v, see, q, D ** -0.5, 0.0, None, None, None)["out"]
            close(out, *want, "out")
            kv[:, 1] += torch.tensor([1, 1, 1, 1, 0 if step else 1], dtype=torch.int32, device="cuda")
            q.copy_(rnd(gen, S, H, D, dtype=torch.bfloat16))
            torch.cuda.synchronize()


def test_caches_beyond_32_bit_offsets():
    """Keys whose byte offsets pass 2^32 (2.2e9 elements of bf16): rows at both ends of the cache."""
    M, D = 17_200_000, 128
    k = torch.zeros(M, 1, D, dtype=torch.bfloat16, device="cuda")
    gen = torch.Generator().manual_seed(1)
    tail = rnd(gen, 700, 1, D, dtype=torch.bfloat16)
    k[-700:] = tail
    q = rnd(gen, 200, 2, D, dtype=torch.bfloat16)
    B_ = B()
    with torch.no_grad():
        a = B_.attention(q, k, k, [(0, 200)], [(M - 700, M)], causal=True)
        assert torch.equal(a, B_.attention(q, tail, tail, [(0, 200)], [(0, 700)], causal=True))
        a = B_.attention(q[:1], k, k, [(0, 1)], [(M - 700, M)])
        # the keys are split by the cache's size, and every share rounds its weights (u each) against a maximum of its own, so this one is not
        # the same bits as over the short cache: both are held to the definition, within (u + f32 sums) sum P |v| + u |out|
        see = torch.ones(1, 700, dtype=torch.bool, device="cuda")
        want = reference(q[:1], tail, tail, see, q[:1], D ** -0.5, 0.0, None, None, None)["out"]
        close(a, *want, "long cache")
        close(B_.attention(q[:1], tail, tail, [(0, 1)], [(0, 700)]), *want, "short cache")


def test_a_second_derivative_is_refused():
    gen = torch.Generator().manual_seed(1)
    x, w = rnd(gen, 4, 8, dtype=torch.float32).requires_grad_(), rnd(gen, 8, 8, dtype=torch.float32)
    for y in (B().linear_residual(x, w, act=B().ACT_SILU), B().attention(x.view(4, 1, 8), x.view(4, 1, 8), x.view(4, 1, 8), [(0, 4)])):
        g, = torch.autograd.grad(y.sum(), x, create_graph=True)
        with pytest.raises(RuntimeError):
            torch.autograd.grad(g.sum(), x)


def test_positions_written_before_the_backward_pass_are_noticed():
    """The distances are formed again in the backward pass: positions that changed in between raise, as every saved operand does."""
    gen = torch.Generator().manual_seed(2)
    q, xy = rnd(gen, 6, 2, 8, dtype=torch.float32).requires_grad_(), rnd(gen, 6, 2, dtype=torch.float32)
    slopes = torch.ones(2, device="cuda")
    out = B().attention(q, q, q, [(0, 6)], xy=xy, slopes=slopes)
    xy.add_(1.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        out.sum().backward()


def test_kept_values_go_through_saved_tensors():
    """Activation inputs and softmax statistics can be offloaded by hooks and are freed with the graph."""
    gen = torch.Generator().manual_seed(3)
    x, w = rnd(gen, 20, 32, dtype=torch.bfloat16).requires_grad_(), rnd(gen, 24, 32, dtype=torch.bfloat16)
    seen = []
    with torch.autograd.graph.saved_tensors_hooks(lambda t: (seen.append(tuple(t.shape)), t.cpu())[1], lambda t: t.cuda()):
        y = B().gated_linear(x, w, w)
        out = B().attention(y.view(20, 3, 8), y.view(20, 3, 8), y.view(20, 3, 8), [(0, 20)])
    offloaded, = torch.autograd.grad(out.float().square().sum(), x)
    assert (2, 20, 24) in seen and (20, 3, 8) in seen and any(len(s) == 1 and s[0] >= 3 * 3 * 20 for s in seen)
    y = B().gated_linear(x, w, w)
    out = B().attention(y.view(20, 3, 8), y.view(20, 3, 8), y.view(20, 3, 8), [(0, 20)])
    assert torch.equal(offloaded, torch.autograd.grad(out.float().square().sum(), x)[0])


def test_a_list_of_scenes_in_a_captured_graph():
    """The graph keeps the table that it reads, however many other lists come later; a list that is new in a capture is refused."""
    gen = torch.Generator().manual_seed(4)
    q = rnd(gen, 40, 2, 16, dtype=torch.float32)
    scenes = [(0, 7), (7, 40)]
    B_ = B()
    with torch.no_grad():
        want = B_.attention(q, q, q, scenes)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = B_.attention(q, q, q, scenes)
            with pytest.raises(ValueError, match="capture"):
                B_.attention(q, q, q, [(0, 9), (9, 40)])
        side = torch.cuda.Stream()
        for i in range(200):  # (the cache is emptied several times over, its memory used again)
            B_.attention(q, q, q, [(0, 1 + i % 39), (1 + i % 39, 40), (0, i // 39)])
            with torch.cuda.stream(side):
                B_.attention(q, q, q, [(0, 1 + i % 39), (1 + i % 39, 40), (0, i // 39)])
        for _ in range(3):
            out.zero_()
            g.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, want)
            assert torch.equal(B_.attention(q, q, q, scenes), want)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("Hkv,D,cap,axes,splits", [(2, 64, 0.0, 0, False), (8, 128, 5.0, 0, False), (1, 40, 0.0, 2, True), (4, 32, 3.0, 1, True)])
def test_a_few_rows_for_each_of_several_caches(dtype, Hkv, D, cap, axes, splits):
    """Chunks of 1 to 11 rows behind a mask, without a gradient: every row reads its own keys (split over shares where the caches are long),
    and the rows of a scene without keys and of no scene are zeros."""
    gen = torch.Generator().manual_seed(D)
    chunks, room, H = [1, 3, 11, 0, 8, 2], 2100 if splits else 150, 8
    lens = [room, 64, 77, 5, 0, room - 1]
    starts = [sum(chunks[:i]) for i in range(len(chunks))]
    scenes = [(a, a + n) for a, n in zip(starts, chunks)]
    kv = [(i * room, i * room + n) for i, n in enumerate(lens)]
    N, M = sum(chunks) + 1, room * len(chunks)
    prefix = [0, 70, 0, 0, 3, 4]
    q, k, v = rnd(gen, N, H, D, dtype=dtype), rnd(gen, M, Hkv, D, dtype=dtype), rnd(gen, M, Hkv, D, dtype=dtype)
    for a, b in zip([e for _, e in kv], [s for s, _ in kv[1:]] + [M]):
        k[a:b], v[a:b] = float("nan"), float("inf")  # (what no row sees)
    xy = kv_xy = slopes = None
    if axes:
        xy, kv_xy = rnd(gen, N, axes, dtype=torch.float32), rnd(gen, M, axes, dtype=torch.float32)
        slopes = torch.linspace(0.2, 1.0, H, device="cuda")
    see = visible(N, M, scenes, kv, True, prefix)
    clean = [t.where(torch.isfinite(t), torch.zeros_like(t)) for t in (k, v)]
    want = reference(q, *clean, see, q, D ** -0.5, cap, xy, kv_xy, slopes)["out"]
    with torch.no_grad():
        out = B().attention(q, k, v, scenes, kv, causal=True, prefix=prefix, cap=cap, xy=xy, kv_xy=kv_xy, slopes=slopes)
    close(out, *want, "out")
    assert not out[-1].any() and not out[starts[4]:starts[4] + 8].any()


def test_forward_mode_raises_instead_of_losing_the_tangent():
    B_, gen, fw = B(), torch.Generator().manual_seed(1), torch.autograd.forward_ad
    t, w = rnd(gen, 8, 16, dtype=torch.float32), rnd(gen, 16, 16, dtype=torch.float32)
    rows = lambda u: u.view(8, 2, 8)
    for call in (lambda u: B_.linear_residual(u, w), lambda u: B_.gated_linear(u, w, w), lambda u: B_.attention(rows(u), rows(u), rows(u), [(0, 8)])):
        want = call(t)
        with fw.dual_level():
            assert torch.equal(call(t), want)
            with pytest.raises(NotImplementedError):
                call(fw.make_dual(t, t))
