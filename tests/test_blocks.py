"""CPU: what the transformer-block operators (mggan/hip/blocks.py) refuse, and that their C structures match."""
import os
import re
import subprocess
import sys

import numpy as np
import pytest
import torch

from mggan.hip import HipError, blocks as B, lib as L

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def x(*shape, dtype=torch.float32):
    return torch.zeros(*shape, dtype=dtype)


@pytest.mark.parametrize("args,kw", [
    ((x(3, 4), x(5, 3)), {}),                                              # widths differ
    ((x(3, 4), x(5, 4, 1)), {}),
    ((x(3, 4), x(0, 4)), {}),
    ((x(3, 0), x(5, 0)), {}),
    ((x(3, 4), x(5, 4), x(4)), {}),                                        # bias
    ((x(3, 4), x(5, 4), x(1, 5)), {}),
    ((x(3, 4), x(5, 4), None, x(5)), {}),                                  # a residual is not broadcast
    ((x(3, 4), x(5, 4), None, x(1, 5)), {}),
    ((x(3, 4), x(5, 4, dtype=torch.bfloat16)), {}),                        # types
    ((x(3, 4, dtype=torch.float16), x(5, 4, dtype=torch.float16)), {}),
    ((x(3, 4, dtype=torch.float64), x(5, 4, dtype=torch.float64)), {}),
    ((x(3, 4), x(5, 4)), {"act": 3}),
    ((x(3, 4), x(5, 4)), {"act": "gelu"}),
    ((x(3, 4), x(5, 4)), {}),                                              # (all fits, but for the device)
])
def test_linear_refuses(args, kw):
    with pytest.raises(ValueError, match="linear_residual"):
        B.linear_residual(*args, **kw)


@pytest.mark.parametrize("args,kw", [
    ((x(3, 4), x(5, 4), x(6, 4)), {}),
    ((x(3, 4), x(5, 4), x(5, 3)), {}),
    ((x(3, 4), x(5, 4), x(5, 4), x(4)), {}),
    ((x(3, 4), x(5, 4), x(5, 4), None, x(6)), {}),
    ((x(3, 4), x(5, 4), x(5, 4, dtype=torch.bfloat16)), {}),
    ((x(3, 4), x(5, 4), x(5, 4)), {"act": 17}),
    ((x(3, 4), x(5, 4), x(5, 4)), {}),
])
def test_gated_refuses(args, kw):
    with pytest.raises(ValueError, match="gated_linear"):
        B.gated_linear(*args, **kw)


QKV = (x(6, 4, 16), x(6, 2, 16), x(6, 2, 16))
S = [(0, 6)]


@pytest.mark.parametrize("args,kw", [
    ((x(6, 4), x(6, 4), x(6, 4), S), {}),
    ((x(6, 4, 16), x(6, 3, 16), x(6, 3, 16), S), {}),                      # heads
    ((x(6, 4, 16), x(6, 2, 16), x(6, 4, 16), S), {}),
    ((x(6, 4, 12), x(6, 2, 12), x(6, 2, 12), S), {}),                      # widths
    ((x(6, 4, 136), x(6, 2, 136), x(6, 2, 136), S), {}),
    ((x(6, 4, 16), x(6, 2, 8), x(6, 2, 8), S), {}),
    ((x(6, 4, 16), x(5, 2, 16), x(5, 2, 16), S), {}),                      # fewer keys without kv_scenes
    ((x(6, 4, 16, dtype=torch.bfloat16), x(6, 2, 16), x(6, 2, 16), S), {}),
    (QKV + (S,), {"scale": 0.0}),
    (QKV + (S,), {"scale": -1.0}),
    (QKV + (S,), {"scale": float("nan")}),
    (QKV + (S,), {"cap": -1.0}),
    (QKV + (S,), {"cap": float("inf")}),
    (QKV + (S,), {"prefix": [1]}),                                         # without causal
    (QKV + (S,), {"xy": x(6, 2)}),                                         # positions without slopes
    (QKV + (S,), {"slopes": x(4)}),
    (QKV + (S,), {"kv_xy": x(6, 2)}),
    (QKV + (S,), {"xy": x(6, 3), "slopes": x(4)}),
    (QKV + (S,), {"xy": x(5, 2), "slopes": x(4)}),
    (QKV + (S,), {"xy": x(6, 2), "kv_xy": x(6, 1), "slopes": x(4)}),
    (QKV + (S,), {"xy": x(6, 2, dtype=torch.float64), "slopes": x(4)}),
    (QKV + (S,), {"xy": x(6, 2), "slopes": x(3)}),
    (QKV + (S,), {"xy": x(6, 2).requires_grad_(), "slopes": x(4)}),
    (QKV + (S,), {}),
])
def test_attention_refuses(args, kw):
    with pytest.raises(ValueError, match="attention"):
        B.attention(*args, **kw)


@pytest.mark.parametrize("rows,width", [([(0, 7)], 2), ([(-1, 3)], 2), ([(4, 3)], 2), ([(0, 1, 2)], 2), (["ab"], 2), (5, 2), ([1 << 31], 1),
                                        ([(0, 1)], 1)])
def test_tables_refuse(rows, width):
    with pytest.raises(ValueError, match="attention"):
        B._table("scenes", rows, torch.device("cpu"), 6, width)


def test_c_structures_and_the_packed_arguments_agree():
    """Field by field: the order and types of the C structures are those of the packing formats."""
    sizes = {"long": "q", "int": "i", "float": "f"}
    for path, name, fmt in (("blk_gemm.hip", "BlkLayerArgs", B._LAYER), ("blk_attn.h", "BlkAttnArgs", B._ATTN)):
        src = open(os.path.join(ROOT, "mg-gan_amd", "csrc", path)).read()
        body = re.search(r"struct %s \{(.*?)\n\};" % name, src, re.S).group(1)
        body = re.sub(r"//[^\n]*", "", body)
        got = ""
        for decl in filter(None, (" ".join(d.split()) for d in body.split(";"))):
            kind, names = re.match(r"(?:const )?(\w+) ?(.*)", decl).groups()
            for field in names.split(","):
                got += "Q" if "*" in field else sizes[kind]
        want = "".join(c * int(n or 1) for n, c in re.findall(r"(\d*)([Qqif])", fmt.format))
        assert got == want, (name, got, want)


def test_c_entries_refuse_before_anything_runs():
    lib = L
    ok = dict(x=256, w=512, w2=0, b=0, b2=0, res=0, dy=0, z=0, z2=0, y=768, dx=0, dw=0, db=0, ws=0, ws_bytes=0, ldx=64, M=4, K=64, N=64, act=0,
              dtype=0, slope=0.0)
    for change in (dict(dtype=2), dict(M=0), dict(N=(1 << 20) + 1), dict(x=0), dict(act=3), dict(act=9), dict(ldx=63), dict(ldx=66), dict(x=260),
                   dict(y=772), dict(y=0), dict(M=40, K=8192, N=64, ldx=8192), dict(w2=1024, z=2048)):
        with pytest.raises(HipError):
            lib.mggan_block_layer_fwd(B._LAYER.pack(*{**ok, **change}.values()), 0)
    with pytest.raises(HipError):
        lib.mggan_block_layer_bwd(B._LAYER.pack(*ok.values()), 0)
    attn = dict(q=256, k=256, v=256, dout=0, out=256, dq=0, dk=0, dv=0, dslopes=0, scenes=256, kv_scenes=256, prefix=0, xy=0, kv_xy=0, slopes=0, lse=0,
                out32=0, spans=256, ws=0, ws_bytes=0, q_row=64, q_head=16, k_row=32, k_head=16, v_row=32, v_head=16, N=8, M=8, H=4, Hkv=2, D=16, S=1,
                causal=0, axes=0, dtype=0, scale=1.0, cap=0.0)
    for change in (dict(dtype=5), dict(N=0), dict(M=0), dict(H=3), dict(D=12), dict(D=136), dict(axes=3), dict(axes=1), dict(scale=0.0), dict(cap=-1.0),
                   dict(q=0), dict(k=264), dict(q_row=66), dict(spans=0), dict(spans=260), dict(out=0), dict(scenes=0), dict(S=-1),
                   dict(N=1, M=4096, S=1)):
        with pytest.raises(HipError):
            lib.mggan_block_attention_fwd(B._ATTN.pack(*{**attn, **change}.values()), 0)
    with pytest.raises(HipError):
        lib.mggan_block_attention_bwd(B._ATTN.pack(*attn.values()), 0)
    with pytest.raises(HipError):
        lib.mggan_block_attention_fwd(0, 0)


@pytest.mark.parametrize("kw", [{"scale": 1e-30}, {"scale": 1e39}, {"cap": 1e-30}, {"cap": 1e30}])
def test_scale_and_cap_stay_in_f32s_range(kw):
    """Their quotient and products are f32 factors: outside 2^-60 .. 2^60 the call is refused instead of giving NaN."""
    with pytest.raises(ValueError, match="2\\^60"):
        B.attention(*QKV, S, **kw)


def test_tables_are_told_apart_by_contents(monkeypatch):
    """Kept by value: the same list with other numbers, another limit or other element types is never taken for the one before."""
    monkeypatch.setattr(B, "_s", lambda: 0)
    monkeypatch.setattr(B, "_TABLES", B.BoundedCache(64))
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    cpu, rows = torch.device("cpu"), [[0, 2], [2, 5]]
    first = B._table("scenes", rows, cpu, 6, 2)
    assert first.tolist() == rows and B._table("scenes", [(0, 2), (2, 5)], cpu, 6, 2) is first
    rows[1][1] = 6
    assert B._table("scenes", rows, cpu, 6, 2).tolist() == [[0, 2], [2, 6]]
    with pytest.raises(ValueError, match="of 5"):
        B._table("scenes", rows, cpu, 5, 2)
    t = torch.tensor(rows)
    assert B._table("scenes", t, cpu, 6, 2).tolist() == [[0, 2], [2, 6]]
    t[0, 1] = 1
    assert B._table("scenes", t, cpu, 6, 2).tolist() == [[0, 1], [2, 6]]
    assert B._table("prefix", [3, 4], cpu, 0, 1).tolist() == [3, 4]
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    assert B._table("prefix", [3, 4], cpu, 0, 1).tolist() == [3, 4] and len(B._TABLES.pinned) == 1
    with pytest.raises(ValueError, match="capture"):
        B._table("prefix", [3, 5], cpu, 0, 1)


def stubbed(monkeypatch):
    """The layers and attention without their launches, on the CPU: outputs of the right shapes that carry no derivative."""
    monkeypatch.setattr(B, "_on_current", lambda name, t: True)
    monkeypatch.setattr(B, "_layer_fwd", lambda t, w, w2, b, b2, res, act, slope, keep: (torch.zeros(len(t), len(w)), None, t, w, w2))
    monkeypatch.setattr(B, "_attn_fwd", lambda q, k, v, slopes, rest, keep: (torch.zeros(q.shape), None, None, q, k, v))
    monkeypatch.setattr(B, "_table", lambda name, rows, device, limit, width: torch.tensor(rows, dtype=torch.int32))


FORWARD_MODE = [  # the call of one operand, its shape
    (lambda t: B.linear_residual(t, x(5, 4)), (3, 4)), (lambda t: B.linear_residual(x(3, 4), t), (5, 4)),
    (lambda t: B.linear_residual(x(3, 4), x(5, 4), t), (5,)), (lambda t: B.linear_residual(x(3, 4), x(5, 4), None, t), (3, 5)),
    (lambda t: B.gated_linear(t, x(5, 4), x(5, 4)), (2, 3, 4)), (lambda t: B.gated_linear(x(3, 4), x(5, 4), t), (5, 4)),
    (lambda t: B.gated_linear(x(3, 4), x(5, 4), x(5, 4), x(5), t), (5,)),
    (lambda t: B.attention(t, x(6, 2, 16), x(6, 2, 16), S), (6, 4, 16)), (lambda t: B.attention(x(6, 4, 16), t, x(6, 2, 16), S), (6, 2, 16)),
    (lambda t: B.attention(x(6, 4, 16), x(6, 2, 16), t, S), (6, 2, 16)), (lambda t: B.attention(*QKV, S, xy=x(6, 2), slopes=t), (4,))]


@pytest.mark.parametrize("grad", [True, False])
@pytest.mark.parametrize("call,shape", FORWARD_MODE)
def test_forward_mode_is_refused(call, shape, grad, monkeypatch):
    """A tangent on any operand raises, whether or not a gradient is recorded: the output would silently have none."""
    stubbed(monkeypatch)
    fw = torch.autograd.forward_ad
    with torch.set_grad_enabled(grad):
        call(x(*shape))
        with fw.dual_level():
            call(x(*shape))  # (an open level alone is nothing to refuse)
            with pytest.raises(NotImplementedError):
                call(fw.make_dual(x(*shape), x(*shape)))
        with pytest.raises(Exception):
            torch.func.jvp(call, (x(*shape),), (x(*shape),))


@pytest.mark.parametrize("name", ["xy", "kv_xy"])
def test_positions_with_a_tangent_are_refused(name, monkeypatch):
    stubbed(monkeypatch)
    fw = torch.autograd.forward_ad
    with fw.dual_level(), pytest.raises(ValueError, match="positions have no gradient"):
        B.attention(*QKV, S, slopes=x(4), **{"xy": x(6, 2), "kv_xy": x(6, 2), name: fw.make_dual(x(6, 2), x(6, 2))})


@pytest.mark.parametrize("keys", [64, 5000, 16384, 131008, 131072, 1 << 20])
@pytest.mark.parametrize("H,Hkv,D", [(8, 1, 128), (64, 1, 128), (1024, 1, 128), (1024, 2, 64), (13, 1, 8), (48, 16, 96), (32, 32, 128)])
def test_the_backward_passs_workspace_does_not_grow_with_the_heads(H, Hkv, D, keys):
    """Partial dK and dV stay within 1 GiB (8 bytes a key, head and column they were, 137 GB at 131,008 keys of 1,024 heads)."""
    rows = 1000
    got = L.mggan_block_attention_bwd_workspace(rows, keys, H, Hkv, D)
    rest = 4 * H * rows + 4 * H * -(-rows // 64) + 8 * -(-keys // 64)  # sum(dO O), the slopes' partial sums, the ranges of rows
    assert rest <= got <= rest + 3 * 256 + (1 << 30)
    if H > Hkv and keys * Hkv <= 64 * 2000 and 8 * H * keys * D <= 1 << 30:
        assert got >= rest + 8 * H * keys * D  # (one part a head where they fit)


def test_workspace_queries_of_sizes_that_no_call_takes():
    """They say 0 -- in a process of its own: heads that key heads do not divide ended it by a division by zero."""
    big = (1 << 31) - 1
    calls = ["mggan_block_attention_fwd_workspace(1, 1000, 1, 2, 64, 1)", "mggan_block_attention_fwd_workspace(1, 0, 1, 1, 64, 1)",
             "mggan_block_attention_bwd_workspace(1, 1000, 1, 2, 64)", "mggan_block_attention_bwd_workspace(1, 1000, 8, 2, %d)" % big,
             "mggan_block_layer_workspace(100, %d, %d, 0, 0, 0, 0)" % (big, big), "mggan_block_layer_workspace(%d, 8, 8, 1, 1, 4, 1)" % big]
    code = "from mggan.hip import lib\nfor n in (%s,):\n    assert n == 0, n\nprint('all 0')" % ", ".join("lib." + c for c in calls)
    run = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, cwd=os.path.join(ROOT, "mg-gan_amd"))
    assert run.returncode == 0 and run.stdout.strip() == "all 0", (run.returncode, run.stderr[-500:])


@pytest.mark.parametrize("slope", [1e39, -1e39, float("nan"), float("inf"), "a", None, torch.tensor(0.2, requires_grad=True), torch.zeros(2)])
def test_slopes_that_are_no_f32_number(slope, monkeypatch):
    """Refused as every argument is (ValueError), and a tensor that a gradient is wanted of, which none would go to."""
    stubbed(monkeypatch)
    with pytest.raises(ValueError, match="linear_residual: slope"):
        B.linear_residual(x(3, 4), x(5, 4), act=B.ACT_LEAKY, slope=slope)
    with pytest.raises(ValueError, match="gated_linear: slope"):
        B.gated_linear(x(3, 4), x(5, 4), x(5, 4), act=B.ACT_LEAKY, slope=slope)


def test_numbers_of_any_kind_are_taken(monkeypatch):
    got = []
    stubbed(monkeypatch)
    monkeypatch.setattr(B, "_layer_fwd", lambda t, w, w2, b, b2, res, act, slope, keep: (got.append(slope), (x(3, 5), None, t, w, w2))[1])
    with torch.no_grad():
        for slope in (0, 1, -0.25, True, np.float32(0.5), torch.tensor(2.0, requires_grad=True), 1e38):
            B.linear_residual(x(3, 4), x(5, 4), act=B.ACT_LEAKY, slope=slope)
    assert got == [0.0, 1.0, -0.25, 1.0, 0.5, 2.0, 1e38] and {type(s) for s in got} == {float}


@pytest.mark.parametrize("act", [1.0, "silu", None, 4.5])
def test_activations_are_codes(act):
    with pytest.raises(ValueError, match="activation"):
        B.linear_residual(x(3, 4), x(5, 4), act=act)


@pytest.mark.parametrize("kw", [{"scale": torch.tensor(0.5, requires_grad=True)}, {"cap": torch.tensor(5.0, requires_grad=True)}, {"scale": "a"},
                                {"cap": [1.0]}])
def test_scale_and_cap_are_numbers(kw):
    with pytest.raises(ValueError, match="attention: (scale|cap)"):
        B.attention(*QKV, S, **kw)


@pytest.mark.parametrize("rows,width", [([(0, 2.7)], 2), (torch.tensor([[0.0, 2.5]]), 2), ([("0", "3")], 2), (np.array([[0.0, 3.0]]), 2), ([1.5], 1)])
def test_tables_of_numbers_that_are_not_whole(rows, width):
    """They were cut off: rows [0, 2.7) became [0, 2)."""
    with pytest.raises(ValueError, match="whole numbers"):
        B._table("scenes", rows, torch.device("cpu"), 6, width)


@pytest.mark.parametrize("rows", [np.array([[0, 2], [2, 6]]), torch.tensor([[0, 2], [2, 6]]), [np.array([0, 2]), (np.int32(2), 6)]])
def test_tables_of_whole_numbers_of_any_kind(rows, monkeypatch):
    monkeypatch.setattr(B, "_s", lambda: 0)
    monkeypatch.setattr(B, "_TABLES", B.BoundedCache(64))
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    assert B._table("scenes", rows, torch.device("cpu"), 6, 2).tolist() == [[0, 2], [2, 6]]


@pytest.mark.parametrize("gated,M,K,N", [(0, 300, 96, 520), (1, 200, 72, 264), (0, 70, 159, 127), (1, 33, 40, 159)])
@pytest.mark.parametrize("act", [2, 4, 5])
@pytest.mark.parametrize("mistake,where", [(None, None), ("activation inputs", "dx|dw"), ("bias gradients", "db")])
def test_the_layers_bounds_tell_a_rounding_of_what_is_kept_in_f32(mistake, where, act, gated, M, K, N):
    """The GPU tests' bounds on a layer that is computed here, in 64 bits: it passes, and with activation inputs rounded to bf16 or bias
    gradients summed from the rounded dZ it does not."""
    import test_hip_blocks_bounds as T

    gen, bf16 = torch.Generator().manual_seed(M + act), torch.bfloat16
    rand = lambda *shape, std=1.0: (torch.randn(*shape, generator=gen) * std).to(bf16)
    round_ = lambda t: t.float().to(bf16)
    t, w, v, b, c, dy = rand(M, K), rand(N, K, std=K ** -0.5), rand(N, K, std=K ** -0.5), rand(N), rand(N), rand(M, N)
    X, W, V, DY = (u.double() for u in (t, w, v, dy))
    z, u = X @ W.t() + b.double(), X @ V.t() + c.double() if gated else 1.0
    y = round_(T.act64(z, 0 * z, act, 0.2)[0] * u)
    if mistake == "activation inputs":
        z, u = round_(z).double(), round_(u).double() if gated else 1.0
    a, d = T.act64(z, 0 * z, act, 0.2)[:2]
    dz, du = DY * d * u, DY * a
    zr, ur = round_(dz).double(), round_(du).double()
    if mistake == "bias gradients":
        dz, du = zr, ur
    grads = {"x": zr @ W + (ur @ V if gated else 0), "w": zr.t() @ X, "b": dz.sum(0)}
    if gated:
        grads.update(v=ur.t() @ X, c=du.sum(0))
    check = lambda: T.check_layer(bf16, t, w, v if gated else None, b, c if gated else None, None, dy, act, 0.2, y,
                                  {n: round_(g) for n, g in grads.items()})
    if mistake is None:
        return check()
    with pytest.raises(AssertionError, match=where):
        check()


def test_the_slopes_bound_tells_a_rounding_of_the_scores_gradients():
    import test_hip_blocks_bounds as T

    gen, (N, H, D) = torch.Generator().manual_seed(2), (8, 3, 32)  # (few rows: the bound adds up what roundings do not)
    q, k, v, dout = (torch.randn(N, H, D, generator=gen).to(torch.bfloat16) for _ in range(4))
    xy, slopes = torch.rand(N, 1, generator=gen) * 9, torch.tensor([0.1, 0.3, 0.5])
    see = torch.ones(N, N).tril().bool()
    want, bound = T.attention64(q, k, v, see, dout, D ** -0.5, 0.0, xy, xy, slopes)["dslopes"]
    Q, K, V, dO = (t.double().transpose(0, 1) for t in (q, k, v, dout))
    dist = (xy - xy.t()).abs().double()
    P = torch.softmax((D ** -0.5 * Q @ K.transpose(1, 2) - slopes.double()[:, None, None] * dist).masked_fill(~see, -torch.inf), -1)
    dP = dO @ V.transpose(1, 2)
    dL = P * (dP - (P * dP).sum(-1, keepdim=True))
    assert ((-(dL * dist).sum((1, 2)) - want).abs() <= bound).all()
    rounded = P * (dP - (dO * (P @ V).to(torch.float32).to(torch.bfloat16).double()).sum(-1, keepdim=True))  # (sum(dO O) of a rounded output)
    for wrong in (dL.to(torch.float32).to(torch.bfloat16).double(), rounded):
        assert ((-(wrong * dist).sum((1, 2)) - want).abs() > 2 * bound).all()


def test_the_c_entry_refuses_an_unaligned_f32_output():
    """It is written 16 bytes at a time, as the output is."""
    attn = dict(q=256, k=256, v=256, dout=0, out=256, dq=0, dk=0, dv=0, dslopes=0, scenes=256, kv_scenes=256, prefix=0, xy=0, kv_xy=0, slopes=0, lse=256,
                out32=260, spans=256, ws=0, ws_bytes=0, q_row=64, q_head=16, k_row=32, k_head=16, v_row=32, v_head=16, N=8, M=8, H=4, Hkv=2, D=16, S=1,
                causal=0, axes=0, dtype=1, scale=1.0, cap=0.0)
    with pytest.raises(HipError, match="unaligned"):
        L.mggan_block_attention_fwd(B._ATTN.pack(*attn.values()), 0)
