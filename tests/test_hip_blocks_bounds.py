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
