"""GPU: the transformer-block operators (mggan/hip/blocks.py) against their definitions in 64 bits with the roundings that the kernels
make on purpose carried out, so that the bounds hold what is f32 in between to f32.

u = half a step of the operands' type (2^-8 bf16, 2^-24 f32), F = 2^-24.  With bf16 operands the softmax's weights P, the scores' gradient dS
and a layer's dZ are rounded to bf16 where they enter a matrix instruction.  Where the value before that rounding is known to within e (P and
dS of the backward pass, dZ) the rounded value lies between the roundings of its two ends, and `entered` says how far that is from the
rounding of the exact value: zero but where a border between two steps lies in between.  Everything else is f32: a sum of n products is off by
n F of the sum of their absolute values, exp2 and rcp by a step (2 F) of their value.  Outputs are rounded once, by u."""
import pytest
import torch

from test_hip_blocks import B, F, TYPES, U, close, lengths_to_scenes, rnd, visible

pytestmark = pytest.mark.gpu

SERIES_FROM = 64.0  # caps above it, and all in f32: tanh by its series near zero


def entered(x, e, dtype):
    """x, known to within e, as it enters a product: (its rounding, how far that of the kernel's value can be from it).  Rounding never
    changes an order, so the kernel's value lies between the roundings of both ends."""
    if dtype == torch.float32:
        return x, e
    at = lambda t: t.to(torch.float32).to(dtype).double()
    c = at(x)
    return c, torch.maximum((at(x + e) - c).abs(), (at(x - e) - c).abs())


def attention64(q, k, v, see, dout, scale, cap=0.0, xy=None, kv_xy=None, slopes=None):
    """{name: (value, bound)}.  Scores: a product of D terms, its factor and a few roundings, (D + 8) F of the absolute terms.  The cap's
    tanh: its series is off by 8 F of itself, the quotient 1 - 2 / (e + 1) by at most 2 / (e + 1) times 5 F and a rounding, 12 F, whatever
    the value (it is taken where |x| >= 0.35, or everywhere in bf16 with a cap of at most 64: 64 x 12 F = 2^-14.4 against u = 2^-8 of the
    weights).  A weight is exp2 of a score less its row's maximum: 8 F of the largest score, and the sum's (n + 16) F; in bf16 the backward
    pass takes both statistics in one number of up to 32 + |score|, a rounding of F of it more."""
    (N, H, D), (M, Hkv, _), dtype = q.shape, k.shape, q.dtype
    u, half, G = U[dtype], dtype == torch.bfloat16, H // Hkv
    ub = u if half else 0.0
    Q, K, V, dO = (t.detach().double().transpose(0, 1) for t in (q, k, v, dout))
    Kh, Vh = K.repeat_interleave(G, 0), V.repeat_interleave(G, 0)
    z = scale * (Q @ Kh.transpose(1, 2))
    es = (D + 8) * F * scale * (Q.abs() @ Kh.abs().transpose(1, 2))
    s, fac, efac = z, 1.0, 0.0
    if cap:
        t = torch.tanh(z / cap)
        et = torch.full_like(t, 12 * F)
        if not half or cap > SERIES_FROM:
            et = torch.where((z / cap).abs() < 0.34, 8 * F * t.abs(), et)
        et = es / cap + 4 * F * (z / cap).abs() * (1 - t * t) + et
        s, es, fac = cap * t, cap * et + 2 * F * cap * t.abs(), 1 - t * t
        efac = 2 * t.abs() * et + 3 * F
    dist = None
    if xy is not None:
        dist = (xy.double()[:, None] - kv_xy.double()[None]).norm(dim=-1)
        bias = slopes.detach().double()[:, None, None] * dist
        s, es = s - bias, es + 8 * F * bias.abs()
    es = es + 8 * F * s.abs()
    s = s.masked_fill(~see, -torch.inf)
    P = torch.softmax(s, -1).nan_to_num(0.0)
    n = see.sum(-1).double()[None, :, None]
    rel = 2 * (es * see).amax(-1, keepdim=True) + (n + 16 + (32 if half else 0)) * F
    O, A = P @ Vh, P @ Vh.abs()
    eO = (rel + ub) * A + (n + 4) * F * A
    dP = dO @ Vh.transpose(1, 2)
    edP = (D + 4) * F * (dO.abs() @ Vh.abs().transpose(1, 2))
    delta = (dO * O).sum(-1, keepdim=True)
    edelta = (dO.abs() * (eO + (D + 4) * F * O.abs())).sum(-1, keepdim=True)  # (of the output before it is rounded)
    dL = P * (dP - delta)
    edL = rel * dL.abs() + P * (edP + edelta) * (1 + rel) + 4 * F * P * (dP.abs() + delta.abs())
    dS, eS = entered(dL * fac, edL * fac + (dL.abs() + edL) * efac, dtype)
    Pe, eP = entered(P, rel * P, dtype)
    m = see.sum(0).double()[None, :, None] * G
    dQ, eQ = scale * (dS @ Kh), scale * ((eS + (n + 4) * F * (dS.abs() + eS)) @ Kh.abs())
    dSt, eSt, Pt = dS.transpose(1, 2), eS.transpose(1, 2), Pe.transpose(1, 2)
    dK, eK = scale * (dSt @ Q), scale * (eSt @ Q.abs() + (m + 4) * F * ((dSt.abs() + eSt) @ Q.abs()))
    dV, eV = Pt @ dO, eP.transpose(1, 2) @ dO.abs() + (m + 4) * F * (Pt @ dO.abs())
    fold = lambda x: x.reshape(Hkv, G, M, D).sum(1)
    out = {"out": (O, eO), "dq": (dQ, eQ), "dk": (fold(dK), fold(eK)), "dv": (fold(dV), fold(eV))}
    out = {name: (x.transpose(0, 1), (e + u * (x.abs() + e)).transpose(0, 1)) for name, (x, e) in out.items()}
    if xy is not None:
        # row by row a - c b with a = sum P dP dist, b = sum P dist, c = sum P dP: nothing in it is rounded to bf16
        w, f = P * dP.abs(), (n + 8) * F
        a, b, c = (P * dP * dist).sum(-1, keepdim=True), (P * dist).sum(-1, keepdim=True), (P * dP).sum(-1, keepdim=True)
        ea = ((rel + f) * w * dist + P * edP * dist).sum(-1, keepdim=True)
        eb, ec = (rel + f) * b, ((rel + f) * w + P * edP).sum(-1, keepdim=True)
        row = a - c * b
        e = ea + c.abs() * eb + b * ec + eb * ec + 3 * F * (a.abs() + (c * b).abs())
        # (then sums of up to 12 in f32 -- two rows a lane, 64 lanes, four waves -- and the rest in 64 bits)
        out["dslopes"] = (-row.sum((1, 2)), (e + 14 * F * row.abs()).sum((1, 2)))
    return out


def run(q, k, v, dout, scenes, kv_scenes=None, **opt):
    """Output, output without a gradient kept, and all gradients."""
    leaves = {"dq": q, "dk": k, "dv": v}
    if opt.get("slopes") is not None:
        leaves["dslopes"] = opt["slopes"]
    leaves = {n: t.detach().requires_grad_() for n, t in leaves.items()}
    if "dslopes" in leaves:
        opt["slopes"] = leaves["dslopes"]
    out = B().attention(leaves["dq"], leaves["dk"], leaves["dv"], scenes, kv_scenes, **opt)
    got = {"out": out.detach(), **dict(zip(leaves, torch.autograd.grad(out, list(leaves.values()), dout)))}
    with torch.no_grad():
        return got, B().attention(q, k, v, scenes, kv_scenes, **opt)


def check(got, alone, want):
    assert set(got) == set(want)
    for name, (x, e) in want.items():
        close(got[name], x, e, name)
    close(alone, *want["out"], "out without gradients")


CAPS = [2.0, 50.0, 64.0, 100.0, 1e4, 1e6, 1e7, 2.0 ** 25, 2.0 ** 60]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("axes,D", [(0, 64), (1, 32), (2, 128)])
@pytest.mark.parametrize("cap", CAPS)
def test_caps_of_any_size(cap, axes, D, dtype):
    """A large cap leaves the scores as they are: the score's error is bounded by its own size, not by the cap's."""
    gen = torch.Generator().manual_seed(D)
    scenes, N, H, Hkv = [(0, 70), (70, 71), (71, 150)], 150, 4, 2
    q, k, v, dout = (rnd(gen, N, h, D, dtype=dtype, std=s) for h, s in ((H, 2.0), (Hkv, 1.0), (Hkv, 1.0), (H, 1.0)))
    xy = slopes = None
    if axes:
        xy, slopes = (torch.rand(N, axes, generator=gen) * 9).cuda(), (torch.rand(H, generator=gen) * 0.3).cuda()
    got, alone = run(q, k, v, dout, scenes, causal=True, cap=cap, xy=xy, slopes=slopes)
    see = visible(N, N, scenes, scenes, True, None)
    want = attention64(q, k, v, see, dout, D ** -0.5, cap, xy, xy, slopes)
    check(got, alone, want)
    if cap >= 2.0 ** 25:  # (tanh(x) = x - x^3 / 3 + ..: below 2^-40 of the scores here, so the same definition without a cap holds too)
        check(got, alone, attention64(q, k, v, see, dout, D ** -0.5, 0.0, xy, xy, slopes))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("cap", CAPS)
def test_caps_of_any_size_for_single_rows(cap, dtype):
    gen = torch.Generator().manual_seed(7)
    H, D, lens = 8, 64, [300, 1200, 1]
    kv, M = lengths_to_scenes(lens), sum(lens)
    q, k, v = rnd(gen, 3, H, D, dtype=dtype, std=2.0), rnd(gen, M, 2, D, dtype=dtype), rnd(gen, M, 2, D, dtype=dtype)
    scenes = [(i, i + 1) for i in range(3)]
    with torch.no_grad():
        out = B().attention(q, k, v, scenes, kv, cap=cap)
    close(out, *attention64(q, k, v, visible(3, M, scenes, kv, False, None), q, D ** -0.5, cap)["out"], "out")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("H,Hkv,per", [(40, 1, 2), (112, 2, 3)])
def test_several_heads_a_partial_result(H, Hkv, per, dtype):
    """Keys and heads of which a part each would pass 1 GiB: `per` heads of a key head are walked by one workgroup (the last part of 56
    fewer), and the parts are joined.  Scenes are independent, so three of them are held to the definition."""
    gen = torch.Generator().manual_seed(H)
    N, D, n = 40_000, 128, 40
    keys = N if Hkv == 1 else N // 2
    if Hkv == 2:
        N = keys
    parts = (1 << 30) // (8 * Hkv * keys * D)
    assert -(-(H // Hkv) // parts) == per
    scenes = [(i, i + n) for i in range(0, N, n)]
    q, dout = (torch.empty(N, H, D, dtype=dtype, device="cuda") for _ in range(2))
    k, v = (torch.empty(N, Hkv, D, dtype=dtype, device="cuda") for _ in range(2))
    cgen = torch.Generator(device="cuda").manual_seed(H)
    for t in (q, k, v, dout):
        t.normal_(generator=cgen)
    leaves = [t.requires_grad_() for t in (q, k, v)]
    out = B().attention(*leaves, scenes, causal=True)
    grads = torch.autograd.grad(out, leaves, dout)
    with torch.no_grad():
        for a, b in (scenes[0], scenes[len(scenes) // 2], scenes[-1]):
            see = visible(n, n, [(0, n)], [(0, n)], True, None)
            want = attention64(q[a:b], k[a:b], v[a:b], see, dout[a:b], D ** -0.5)
            for name, got in zip(("out", "dq", "dk", "dv"), (out,) + grads):
                close(got[a:b], *want[name], name)


def visible_only(q, k, v, dout, see, scale, cap):
    """The definition in 64 bits, each row over the keys that it sees and nothing else: what infinities and NaN become."""
    (N, H, D), G = q.shape, q.shape[1] // k.shape[1]
    q, k, v, dout = (t.detach().double().cpu() for t in (q, k, v, dout))
    out = {"out": torch.zeros_like(q), "dq": torch.zeros_like(q), "dk": torch.zeros_like(k), "dv": torch.zeros_like(v)}
    dot = lambda a, b: (a * b).sum(-1)
    for i in range(N):
        j = see[i].nonzero()[:, 0].cpu()
        for h in range(H):
            K, V, do = k[j, h // G], v[j, h // G], dout[i, h]
            z = scale * dot(K, q[i, h])
            t = torch.tanh(z / cap) if cap else None
            P = torch.softmax(cap * t if cap else z, 0)
            O = (P[:, None] * V).sum(0)
            dS = P * (dot(V, do) - dot(do, O)) * (1 - t * t if cap else 1.0)
            out["out"][i, h], out["dq"][i, h] = O, scale * (dS[:, None] * K).sum(0)
            out["dk"][j, h // G] += scale * dS[:, None] * q[i, h]
            out["dv"][j, h // G] += P[:, None] * do
    return out


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("cap", [0.0, 20.0])
@pytest.mark.parametrize("value", [float("nan"), float("inf"), float("-inf")])
@pytest.mark.parametrize("which", ["q", "k", "v", "dout"])
def test_what_a_value_that_is_not_finite_becomes(which, value, cap, dtype):
    """In every output and gradient the same places are +inf, -inf, NaN or finite as in the definition -- whether the tile that holds the
    value is partly masked (rows near it) or seen as a whole (rows far behind it).  Under a cap an infinite score is a finite one of slope zero,
    and zero times infinity is NaN."""
    gen = torch.Generator().manual_seed(11)
    N, H, D, at = 200, 2, 32, 10
    t = {n: rnd(gen, N, H, D, dtype=dtype) for n in ("q", "k", "v", "dout")}
    t["q"][:, 0, 3].abs_()  # (a key of -inf there leaves some rows finite scores and others none)
    t["q"][::3, 0, 3].neg_()
    t[which][at, 0, 3], t[which][at + 5, 1, 7] = value, value
    got, _ = run(t["q"], t["k"], t["v"], t["dout"], [(0, N)], causal=True, cap=cap)
    see = visible(N, N, [(0, N)], [(0, N)], True, None)
    want = visible_only(*t.values(), see, D ** -0.5, cap)
    kind = lambda x: torch.where(x.isnan(), 2, torch.where(x.isinf(), x.sign(), 0.0))
    for name, x in want.items():
        a, b = kind(got[name].double().cpu()), kind(x)
        assert torch.equal(a, b), (name, [(i, float(a[tuple(i)]), float(b[tuple(i)])) for i in (a != b).nonzero().tolist()[:6]], int((a != b).sum()))


# ---- every kernel that a call can reach ----------------------------------------------------------------------------------------

NAMES = {torch.float32: "f", torch.bfloat16: "DF16b"}


def launched(call):
    """(what call gives, the kernels that it and its backward pass launched, by their mangled names)"""
    from mggan.hip.lib import load

    load().launch_log(True)
    try:
        out = call()
        return out, [name for name, _ in load().read_launches()]
    finally:
        load().launch_log(False)


def ran(names, kernel, dtype, *args):
    """Whether the instantiation with these template arguments (numbers and truth values) is among the launches."""
    want = "{}I{}{}E".format(kernel, NAMES[dtype], "".join("L{}{}E".format("b" if isinstance(a, bool) else "i", int(a)) for a in args))
    return any(want in n for n in names)


def ways(dtype):
    """What is done to a score (the kernels' argument X), with a cap and axes that lead there."""
    small = [(0, 0.0, 0), (1, 9.0, 0), (2, 0.0, 1), (3, 30.0, 1), (4, 0.0, 2), (5, 64.0, 2)]
    return small if dtype == torch.float32 else small + [(9, 65.0, 0), (11, 500.0, 1), (13, 1e5, 2)]


WIDTHS = {32: 24, 64: 64, 96: 88, 128: 128}  # the kernels' widths, one of an operand's each


@pytest.mark.parametrize("dtype,X,cap,axes", [(t,) + w for t in TYPES for w in ways(t)])
@pytest.mark.parametrize("DP,QF", [(32, 1), (64, 1), (96, 1), (128, 1), (96, 2), (128, 2)])
def test_every_attention_kernel(DP, QF, dtype, X, cap, axes):
    """64 and 128 rows a workgroup, all widths, caps and distances: forward, dQ and dK / dV against the definition."""
    gen = torch.Generator().manual_seed(100 * DP + 10 * QF + X)
    D, (H, Hkv) = WIDTHS[DP], (86, 43) if QF == 2 else (4, 2)
    lengths, prefix = [150, 1, 40, 0, 107], [17, 0, 40, 2, 90]
    scenes, N = lengths_to_scenes(lengths), sum(lengths) + 2  # (three tiles of 128 rows: 258 workgroups with 86 heads; two rows of no scene)
    q, k, v, dout = (rnd(gen, N, h, D, dtype=dtype) for h in (H, Hkv, Hkv, H))
    xy = slopes = None
    if axes:
        xy, slopes = (torch.rand(N, axes, generator=gen) * 12).cuda(), (torch.rand(H, generator=gen) * 0.4).cuda()
    causal = X % 2 == 0
    opt = dict(causal=causal, prefix=prefix if causal else None, cap=cap, xy=xy, slopes=slopes)
    (got, alone), names = launched(lambda: run(q, k, v, dout, scenes, **opt))
    assert ran(names, "blk_attn_fwd_kernel", dtype, DP, QF, X) and ran(names, "blk_attn_dkv_kernel", dtype, DP, X)
    assert ran(names, "blk_attn_dq_kernel", dtype, DP, QF if dtype == torch.bfloat16 else 1, X)
    see = visible(N, N, scenes, scenes, causal, opt["prefix"])
    check(got, alone, attention64(q, k, v, see, dout, D ** -0.5, cap, xy, xy, slopes))


@pytest.mark.parametrize("dtype,X,cap,axes", [(t,) + w for t in TYPES for w in ways(t)])
@pytest.mark.parametrize("DP", list(WIDTHS))
def test_every_kernel_for_single_rows(DP, dtype, X, cap, axes):
    gen = torch.Generator().manual_seed(10 * DP + X)
    D, H, Hkv, lens = WIDTHS[DP], 6, 2, [1100, 1, 0, 133, 700]
    kv, M, S = lengths_to_scenes(lens, 2), sum(lens) + 5, len(lens)
    q, k, v = rnd(gen, S, H, D, dtype=dtype), rnd(gen, M, Hkv, D, dtype=dtype), rnd(gen, M, Hkv, D, dtype=dtype)
    xy = kv_xy = slopes = None
    if axes:
        xy, kv_xy = ((torch.rand(n, axes, generator=gen) * 12).cuda() for n in (S, M))
        slopes = (torch.rand(H, generator=gen) * 0.4).cuda()
    rows = [(i, i + 1) for i in range(S)]
    with torch.no_grad():
        out, names = launched(lambda: B().attention(q, k, v, rows, kv, causal=True, cap=cap, xy=xy, kv_xy=kv_xy, slopes=slopes))
    assert ran(names, "blk_attn_row_kernel", dtype, DP, X)
    close(out, *attention64(q, k, v, visible(S, M, rows, kv, True, None), q, D ** -0.5, cap, xy, kv_xy, slopes)["out"], "out")


@pytest.mark.parametrize("dtype", TYPES)
def test_values_that_are_not_finite_with_128_rows_a_workgroup(dtype):
    """The second run of such a workgroup goes over its rows 16 at a time: what no row sees changes nothing, what rows see is the definition's."""
    gen = torch.Generator().manual_seed(3)
    H, D, scenes, N = 86, 128, [(0, 100), (100, 290), (290, 300)], 300
    t = {n: rnd(gen, N, H, D, dtype=dtype) for n in ("q", "k", "v", "dout")}
    see = visible(N, N, scenes, scenes, True, None)
    want, _ = run(*t.values(), scenes, causal=True)
    for name, x in t.items():
        x[200 if name in "kv" else 150, 1, 5], x[130, 2, 9] = float("inf"), float("nan")
    (got, alone), names = launched(lambda: run(*t.values(), scenes, causal=True))
    assert ran(names, "blk_attn_fwd_kernel", dtype, 128, 2, 0) and ran(names, "blk_attn_dq_kernel", dtype, 128, 2 if dtype == torch.bfloat16 else 1, 0)
    kinds = visible_only(*(x[:, :3] for x in t.values()), see, D ** -0.5, 0.0)
    kind = lambda x: torch.where(x.isnan(), 2, torch.where(x.isinf(), x.sign(), 0.0))
    for name, x in kinds.items():
        assert torch.equal(kind(got[name][:, :3].double().cpu()), kind(x)), name
        assert torch.isfinite(got[name][:, 3:]).all(), name
        clean = torch.isfinite(x).all(-1)  # (rows without such a value: the sums are the same ones, through another product)
        clean[100:290, 1:] = False
        a, b = got[name][:, :3][clean.cuda()].double(), want[name][:, :3][clean.cuda()].double()
        torch.testing.assert_close(a, b, rtol=4 * U[dtype], atol=64 * F * float(b.abs().max()))
    assert torch.equal(kind(alone[:, :3].double().cpu()), kind(kinds["out"]))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("D", [32, 128])
def test_more_tiles_than_are_ranked_and_heads_walked_together(D, dtype):
    """131,100 rows: their tiles are taken from the last on, and with 2,048 workgroups of keys one walks both heads of a key head.  Output
    gradients are zero but in three scenes, which the slopes' gradient then is a sum over."""
    gen = torch.Generator(device="cuda").manual_seed(D)
    n, S, H = 60, 2185, 2
    N = n * S
    q, k, v, dout = (torch.randn(N, h, D, generator=gen, device="cuda").to(dtype) for h in (H, 1, 1, H))
    xy, slopes = torch.rand(N, 1, generator=gen, device="cuda") * 9, torch.tensor([0.05, 0.7], device="cuda")
    some = [0, 1100, S - 1]
    keep = torch.zeros(S, 1, dtype=torch.bool, device="cuda")
    keep[some] = True
    dout.mul_(keep.expand(S, n).reshape(N, 1, 1))
    scenes = [(i * n, i * n + n) for i in range(S)]
    (got, alone), names = launched(lambda: run(q, k, v, dout, scenes, causal=True, xy=xy, slopes=slopes))
    assert ran(names, "blk_attn_dkv_kernel", dtype, D, 2) and not any("blk_attn_sum_kernel" in name for name in names)
    see = visible(n, n, [(0, n)], [(0, n)], True, None)
    slope, err = 0.0, 0.0
    for s in some:
        at = slice(s * n, s * n + n)
        want = attention64(q[at], k[at], v[at], see, dout[at], D ** -0.5, 0.0, xy[at], xy[at], slopes)
        close(alone[at], *want["out"], "out without gradients")
        for name in ("out", "dq", "dk", "dv"):
            close(got[name][at], *want[name], name)
        slope, err = slope + want["dslopes"][0], err + want["dslopes"][1]
    close(got["dslopes"], slope, err, "dslopes")
    others = ~keep.expand(S, n).reshape(N)
    assert not any(got[name][others].any() for name in ("dq", "dk", "dv"))


def act64(z, ez, act, slope):
    """(value, derivative, what the value is off by, what the derivative is off by) of z known to within ez.  The slopes of value and
    derivative are at most 1.13 and 0.1 / 0.5 / 0.8; sigmoid and SiLU are evaluated to (8 + |z|) 2 F of themselves, their derivatives to twice
    that; GELU is z (0.5 + 0.5 erf): half a unit's few F times |z|, and of itself."""
    if act == 0:
        return z, torch.ones_like(z), ez, torch.zeros_like(z)
    if act == 1:
        a, d = torch.where(z > 0, z, z * slope), torch.where(z > 0, 1.0, slope).double()
        return a, d, ez * max(1.0, abs(slope)) + F * a.abs(), (z.abs() <= ez) * abs(1 - slope)
    grow = (8 + z.abs()) * 2 * F
    s = torch.sigmoid(z)
    if act == 2:
        return s, s * (1 - s), 0.25 * ez + grow * s, 0.1 * ez + 2 * grow
    if act == 4:
        a = z * s
        return a, s * (1 + z * (1 - s)), 1.13 * ez + grow * a.abs(), 0.5 * ez + 2 * grow
    cdf = 0.5 * torch.erfc(-z * 0.5 ** 0.5)
    a = z * cdf
    return a, cdf + z * torch.exp(-0.5 * z * z) * 0.3989422804014327, 1.13 * ez + 4 * F * (z.abs() + a.abs()), 0.8 * ez + 2 * grow


def product64(x, w, b):
    size = x.abs() @ w.abs().t()
    z = x @ w.t()
    if b is not None:
        z, size = z + b, size + b.abs()
    return z, (x.shape[1] + 4) * F * size


def check_layer(dtype, x, w, v, b, c, r, dy, act, slope, y, grads):
    """Output and gradients of either layer (v: the up weight, or None).  dZ / dG / dU are rounded to the type once, from what f32 makes of
    activation inputs kept in f32; the bias gradients are sums from before that."""
    u, gated = U[dtype], v is not None
    up = lambda t: None if t is None else t.detach().double()
    x, w, v, b, c, r, dy = map(up, (x, w, v, b, c, r, dy))
    z, ez = product64(x, w, b)
    a, d, ea, ed = act64(z, ez, act, slope)
    if gated:
        g, eg = product64(x, v, c)
        ref = a * g
        e = ea * (g.abs() + eg) + a.abs() * eg + F * ref.abs()
        dz, du = dy * g * d, dy * a
        es = dy.abs() * (ed * (g.abs() + eg) + d.abs() * eg) + 3 * F * dz.abs()
        esu = dy.abs() * ea + 2 * F * du.abs()
    else:
        ref, e = (a, ea) if r is None else (a + r, ea + F * (a + r).abs())
        dz = dy * d
        es = dy.abs() * ed + (F * dz.abs() if act else 0)
    final = lambda want, err: (want, err + u * (want.abs() + err))
    close(y, *final(ref, e), "y")
    (M, K), N = x.shape, w.shape[0]
    zr, ezr = entered(dz, es, dtype)
    want, err = zr @ w, ezr @ w.abs() + (N + 4) * F * ((zr.abs() + ezr) @ w.abs())
    parts = [("w", zr, ezr), ("b", dz, es)]
    if gated:
        ur, eur = entered(du, esu, dtype)
        more = ur.abs() + eur
        want = want + ur @ v
        err = err + eur @ v.abs() + (2 * N + 68) * F * ((zr.abs() + ezr) @ w.abs() + more @ v.abs())
        parts += [("v", ur, eur), ("c", du, esu)]
    close(grads["x"], *final(want, err), "dx")
    for name, t, et in parts:
        if name in "wv":
            close(grads[name], *final(t.t() @ x, et.t() @ x.abs() + (M + 4) * F * ((t.abs() + et).t() @ x.abs())), "d" + name)
        elif name in grads:
            close(grads[name], *final(t.sum(0), et.sum(0) + (M + 4) * F * (t.abs() + et).sum(0)), "d" + name)


def run_layer(gen, dtype, M, K, N, gated, act, bias=True, residual=True, slope=0.2):
    """-> a call that runs the layer with its backward pass and gives check_layer's arguments"""
    x = rnd(gen, M, K, dtype=dtype)
    w, v = (rnd(gen, N, K, dtype=dtype, std=K ** -0.5) for _ in range(2))
    b, c = (rnd(gen, N, dtype=dtype) if bias else None for _ in range(2))
    r, dy = rnd(gen, M, N, dtype=dtype) if residual and not gated else None, rnd(gen, M, N, dtype=dtype)
    leaves = {"x": x, "w": w, "b": b, **({"v": v, "c": c} if gated else {"r": r})}
    leaves = {n: t.requires_grad_() for n, t in leaves.items() if t is not None}

    def call():
        y = B().gated_linear(x, w, v, b, c, act=act, slope=slope) if gated else B().linear_residual(x, w, b, r, act=act, slope=slope)
        grads = dict(zip(leaves, torch.autograd.grad(y, list(leaves.values()), dy)))
        return dtype, x, w, v if gated else None, b, c if gated else None, r, dy, act, slope, y.detach(), grads

    return call


F32, BF16 = TYPES
TILES = [  # type, gated, rows x inputs x outputs, (tile, split) of the forward product, of dX and of dW: every one that the plan chooses
    (F32, 0, (3209, 2246, 7039), (128, False), (256, True), (256, False)), (F32, 0, (3381, 6752, 2136), (256, True), (128, False), (256, False)),
    (F32, 0, (6584, 3333, 2143), (256, False), (128, False), (256, True)), (F32, 0, (3343, 3993, 251), (64, False), (256, False), (64, False)),
    (F32, 0, (3331, 1396, 336), (64, True), (64, False), (128, True)), (F32, 0, (1391, 3118, 326), (128, True), (64, False), (64, True)),
    (F32, 0, (324, 1356, 2826), (64, True), (128, True), (128, False)), (F32, 0, (253, 257, 333), (64, False), (64, True), (64, False)),
    (F32, 1, (2155, 6876, 1665), (256, True), (256, False), (128, False)), (F32, 1, (6587, 2450, 1481), (128, False), (64, False), (256, True)),
    (F32, 1, (917, 1867, 8504), (64, False), (256, True), (128, False)), (F32, 1, (261, 3157, 2116), (64, True), (64, False), (256, False)),
    (F32, 1, (2251, 251, 2952), (256, False), (64, True), (64, True)), (F32, 1, (6353, 408, 417), (64, False), (64, False), (128, True)),
    (F32, 1, (424, 6121, 419), (128, True), (64, False), (64, False)), (F32, 1, (1291, 2311, 259), (64, False), (128, False), (64, True)),
    (F32, 1, (337, 1384, 1667), (64, True), (128, True), (64, False)), (BF16, 0, (5669, 1861, 2214), (256, False), (256, False), (256, True)),
    (BF16, 0, (1989, 2057, 5616), (256, False), (256, True), (256, False)), (BF16, 0, (2329, 5565, 1742), (256, True), (256, False), (256, False)),
    (BF16, 0, (3771, 647, 343), (64, False), (128, False), (128, True)), (BF16, 0, (646, 330, 3827), (128, False), (128, True), (64, False)),
    (BF16, 0, (273, 3580, 769), (128, True), (64, False), (128, False)), (BF16, 0, (252, 1585, 300), (64, True), (64, False), (64, False)),
    (BF16, 0, (1679, 258, 266), (64, False), (64, False), (64, True)), (BF16, 0, (259, 253, 1513), (64, False), (64, True), (64, False)),
    (BF16, 1, (5557, 1801, 1146), (256, False), (256, False), (256, True)), (BF16, 1, (1166, 5569, 1718), (256, True), (128, False), (128, False)),
    (BF16, 1, (775, 1222, 6958), (256, False), (256, True), (128, False)), (BF16, 1, (272, 1288, 2977), (64, False), (64, True), (256, False)),
    (BF16, 1, (267, 3824, 390), (128, True), (64, False), (128, False)), (BF16, 1, (3689, 264, 393), (128, False), (64, False), (128, True)),
    (BF16, 1, (801, 261, 1830), (128, False), (128, True), (64, False)), (BF16, 1, (270, 1857, 251), (64, True), (64, False), (64, False)),
    (BF16, 1, (1844, 251, 255), (64, False), (64, False), (64, True))]


@pytest.mark.parametrize("dtype,gated,sizes,fwd,dx,dw", TILES)
def test_every_product_kernel(dtype, gated, sizes, fwd, dx, dw):
    """All tiles, whole and split over k, of the forward product and of both products of the backward pass, with ragged edges."""
    waves = {256: (2, 4), 128: (2, 2), 64: (4, 1)}
    gen = torch.Generator().manual_seed(sum(sizes))
    result, names = launched(run_layer(gen, dtype, *sizes, gated, (4 if gated else 5) if sum(sizes) % 2 else 1))
    for epi, (tile, split), columns in ((gated, fwd, (False, False)), (0, dx, (False, True)), (0, dw, (True, True))):
        assert ran(names, "blk_gemm_kernel", dtype, tile, tile, *waves[tile], epi, split, *columns), (tile, split, columns, names)
    check_layer(*result)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("gated,M,K,N", [(0, 16, 40, 16400), (1, 7, 65, 9000), (0, 1, 24, 33), (1, 16, 129, 100)])
def test_every_kernel_for_a_few_rows(gated, M, K, N, dtype):
    result, names = launched(run_layer(torch.Generator().manual_seed(N), dtype, M, K, N, gated, 4))
    assert ran(names, "blk_few_rows_kernel", dtype, gated, 4 if -(-N // 16) * (1 + gated) >= 1024 else 8)
    check_layer(*result)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("act", [0, 1, 2, 4, 5])
@pytest.mark.parametrize("gated,M,K,N", [(0, 300, 96, 520), (1, 200, 72, 264), (0, 70, 159, 127), (1, 33, 40, 159)])
def test_layers_keep_in_f32_what_is_not_an_operand(gated, M, K, N, act, dtype):
    """Activation inputs are kept in f32 and bias gradients summed before dZ's rounding: bounds without a rounding of either."""
    check_layer(*run_layer(torch.Generator().manual_seed(M + act), dtype, M, K, N, gated, act, residual=act != 2)())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("D", [32, 64, 128])
def test_attention_keeps_the_output_in_f32_for_the_backward_pass(D, dtype):
    """Rows that weigh 64 keys equally (q = 0) have weights that bf16 holds exactly, and values of 1 or 1 + 2^-7 have means that it does not:
    sum(dO O) of a rounded output would be off by up to 2^-8 of itself, many times the scores' gradients, which are differences of 2^-7 at most.
    Without a rounding of P the output before its own is good to f32, so the bounds have none in sum(dO O)."""
    gen = torch.Generator().manual_seed(D)
    n, H, S = 64, 2, 3
    N, scenes = n * S, [(i * n, i * n + n) for i in range(S)]
    q, k = torch.zeros(N, H, D, dtype=dtype, device="cuda"), 1 + rnd(gen, N, H, D, dtype=dtype, std=0.1)
    v = (1 + (torch.rand(N, H, D, generator=gen) < 0.3).float() * 2.0 ** -7).to(dtype).cuda()
    dout = rnd(gen, N, H, D, dtype=dtype).abs()
    got, _ = run(q, k, v, dout, scenes)
    u, up = U[dtype], lambda t: t.double().view(S, n, H, D).transpose(1, 2)
    K, V, dO = up(k), up(v), up(dout)
    O = V.mean(2, keepdim=True)
    dP, delta = dO @ V.transpose(2, 3), (dO * O).sum(-1, keepdim=True)
    e = ((D + 4) * F * (dO.abs() @ V.transpose(2, 3).abs()) + (D + n + 24) * F * (dO.abs() * O.abs()).sum(-1, keepdim=True)) / n
    dS, eS = entered((dP - delta) / n, e + 40 * F * (dP - delta).abs() / n, dtype)
    want, err = dS @ K, eS @ K.abs() + (n + 4) * F * (dS.abs() @ K.abs())
    want, err = (t.transpose(1, 2).reshape(N, H, D) * D ** -0.5 for t in (want, err))
    close(got["dq"], want, err + u * (want.abs() + err), "dq")
    rounded = O.to(torch.float32).to(dtype).double()  # (that the inputs tell the two apart)
    if dtype == torch.bfloat16:
        off = ((dO * (rounded - O)).sum(-1, keepdim=True) / n * K.sum(2, keepdim=True)).transpose(1, 2).reshape(N, H, D) * D ** -0.5
        assert ((off.abs() > 4 * (err + u * (want.abs() + err))).float().mean()) > 0.5


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("cap", [0.0, 20.0])
@pytest.mark.parametrize("D,axes", [(32, 2), (128, 1)])
def test_slopes_gradient_of_a_small_scene(D, axes, cap, dtype):
    """Of so few pairs that the bound is many times below a rounding of the scores' gradients or of the output to bf16."""
    for seed in range(6):
        gen = torch.Generator().manual_seed(seed)
        N, H = 8, 4
        q, k, v, dout = (rnd(gen, N, H, D, dtype=dtype) for _ in range(4))
        xy, slopes = (torch.rand(N, axes, generator=gen) * 9).cuda(), (torch.rand(H, generator=gen) * 0.4).cuda()
        got, alone = run(q, k, v, dout, [(0, N)], causal=True, cap=cap, xy=xy, slopes=slopes)
        check(got, alone, attention64(q, k, v, visible(N, N, [(0, N)], [(0, N)], True, None), dout, D ** -0.5, cap, xy, xy, slopes))


@pytest.mark.parametrize("gated", [0, 1])
def test_layers_beyond_32_bit_offsets(gated):
    """2^21 rows of 1,032 inputs and 1,040 outputs: inputs, outputs, kept values and gradients of more than 2^31 elements each.  The output's
    gradient is zero but in rows at both ends, which the weights' gradients then are sums over."""
    gen = torch.Generator(device="cuda").manual_seed(gated)
    M, K, N, dtype, act = 1 << 21, 1032, 1040, torch.bfloat16, 4
    x = torch.empty(M, K, dtype=dtype, device="cuda").normal_(generator=gen)
    w, v = (torch.empty(N, K, dtype=dtype, device="cuda").normal_(std=K ** -0.5, generator=gen) for _ in range(2))
    b = torch.empty(N, dtype=dtype, device="cuda").normal_(generator=gen)
    some = torch.cat([torch.arange(50), torch.arange(M - 70, M)]).cuda()
    dy = torch.zeros(M, N, dtype=dtype, device="cuda")
    dy[some] = torch.randn(len(some), N, generator=gen, device="cuda").to(dtype)
    leaves = {"x": x, "w": w, "b": b, **({"v": v} if gated else {})}
    for t in leaves.values():
        t.requires_grad_()
    y = B().gated_linear(x, w, v, b, None, act=act) if gated else B().linear_residual(x, w, b, act=act)
    grads = dict(zip(leaves, torch.autograd.grad(y, list(leaves.values()), dy)))
    assert not grads["x"][50:M - 70].any()
    grads["x"] = grads["x"][some]
    check_layer(dtype, x[some], w, v if gated else None, b, None, None, dy[some], act, 0.0, y.detach()[some], grads)
    with torch.no_grad():
        y0 = B().gated_linear(x, w, v, b, None, act=act) if gated else B().linear_residual(x, w, b, act=act)
        assert torch.equal(y0, y)


def test_attention_beyond_32_bit_offsets():
    """1,100,000 rows of 16 heads of 128: more than 2^31 elements of every operand, output and gradient (and of the f32 output)."""
    gen = torch.Generator(device="cuda").manual_seed(1)
    n, S, H, D, dtype = 50, 22_000, 16, 128, torch.bfloat16
    N = n * S
    q, k, v, dout = (torch.empty(N, H, D, dtype=dtype, device="cuda").normal_(generator=gen) for _ in range(4))
    xy, slopes = torch.rand(N, 1, generator=gen, device="cuda") * 9, torch.rand(H, generator=gen, device="cuda") * 0.3
    scenes = (torch.arange(S + 1, dtype=torch.int32, device="cuda") * n).unfold(0, 2, 1).contiguous()
    some = [0, S // 2, S - 1]
    keep = torch.zeros(S, 1, dtype=torch.bool, device="cuda")
    keep[some] = True
    dout.mul_(keep.expand(S, n).reshape(N, 1, 1))
    got, alone = run(q, k, v, dout, scenes, causal=True, xy=xy, slopes=slopes)
    see, slope, err = visible(n, n, [(0, n)], [(0, n)], True, None), 0.0, 0.0
    for s in some:
        at = slice(s * n, s * n + n)
        want = attention64(q[at], k[at], v[at], see, dout[at], D ** -0.5, 0.0, xy[at], xy[at], slopes)
        close(alone[at], *want["out"], "out without gradients")
        for name in ("out", "dq", "dk", "dv"):
            close(got[name][at], *want[name], name)
        slope, err = slope + want["dslopes"][0], err + want["dslopes"][1]
    close(got["dslopes"], slope, err, "dslopes")
