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
