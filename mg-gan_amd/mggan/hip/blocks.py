"""Operators of a transformer block over the rows of scenes, f32 or bf16, with their backward passes:

    attention(q, k, v, scenes, ...)                   softmax(cap tanh(scale q k / cap) - slope |xy - kv_xy|) v within each scene
    linear_residual(x, weight, bias, residual, act)   act(x W^T + b) + residual
    gated_linear(x, w_gate, w_up, b_gate, b_up, act)  act(x Wg^T + bg) * (x Wu^T + bu)

All operands of a call have one type and live on one device; sums, activations and softmax statistics are held in f32 and
rounded once.  Work goes to torch's current stream, outputs and workspaces come from torch's allocator (so a call can be captured
into a HIP graph), gradients are returned through autograd and are the same bits in every run.  Arguments that do not fit raise
ValueError, a failing launch raises HipError; there is no CPU path."""
import ctypes
import math

import torch
from torch.autograd import Function
from torch.autograd.function import once_differentiable

from .functions import ACT_LEAKY, ACT_NONE, ACT_SIGMOID, BoundedCache, _p, _s
from .lib import lib

ACT_SILU, ACT_GELU = 4, 5
_ACTS = (ACT_NONE, ACT_LEAKY, ACT_SIGMOID, ACT_SILU, ACT_GELU)
_DTYPES = {torch.float32: 0, torch.bfloat16: 1}


def _check(ok, text, *args):
    if not ok:
        raise ValueError(text.format(*args))


def _same(name, x, **others):
    """Every operand has x's type and device, and a device this process can launch on."""
    _check(isinstance(x, torch.Tensor) and x.dtype in _DTYPES, "{}: f32 or bf16 tensors, got {}", name, getattr(x, "dtype", type(x)))
    for n, t in others.items():
        if t is not None:
            _check(isinstance(t, torch.Tensor) and t.dtype == x.dtype, "{}: {} is {}, the first operand is {}", name, n,
                   getattr(t, "dtype", type(t)), x.dtype)
            _check(t.device == x.device, "{}: {} is on {}, the first operand on {}", name, n, t.device, x.device)


def _on_gpu(name, x):
    _check(x.is_cuda, "{}: the operands are on {}; there is no CPU path", name, x.device)


def _aligned(t):
    """Contiguous and 16-byte aligned (a copy where it is not)."""
    if t is None:
        return None
    t = t.contiguous()
    return t.clone() if t.data_ptr() % 16 else t


def _rows(x):
    """(rows, K) view of x with unit inner stride, and its row stride."""
    x = x.reshape(-1, x.shape[-1])
    if x.stride(1) != 1 or (x.shape[0] > 1 and x.stride(0) < x.shape[1]):
        x = x.contiguous()
    return x, (x.stride(0) if x.shape[0] > 1 else x.shape[1])


def _workspace(x, rows, K, N, gated, backward):
    n = lib.mggan_block_layer_workspace(rows, K, N, gated, backward, _DTYPES[x.dtype])
    return torch.empty(n, dtype=torch.uint8, device=x.device), n


def _check_layer(name, x, weight, act, bias, residual=None):
    _check(x.dim() >= 1 and weight.dim() == 2 and x.shape[-1] == weight.shape[1], "{}: rows of {} and a weight of {}", name,
           tuple(x.shape), tuple(weight.shape))
    _check(weight.shape[0] > 0 and weight.shape[1] > 0, "{}: an empty weight {}", name, tuple(weight.shape))
    _check(x.numel() // weight.shape[1] <= 1 << 21 and max(weight.shape) <= 1 << 20, "{}: sizes {} x {} over 2^21 rows, 2^20 columns", name,
           tuple(x.shape), tuple(weight.shape))
    _check(act in _ACTS, "{}: unknown activation {}", name, act)
    _check(bias is None or tuple(bias.shape) == (weight.shape[0],), "{}: a bias of {} for {} outputs", name,
           None if bias is None else tuple(bias.shape), weight.shape[0])
    _check(residual is None or tuple(residual.shape) == tuple(x.shape[:-1]) + (weight.shape[0],),
           "{}: a residual of {} for outputs of {} (it is not broadcast)", name, None if residual is None else tuple(residual.shape),
           tuple(x.shape[:-1]) + (weight.shape[0],))


def _linear_fwd(x, weight, bias, residual, act, slope, keep):
    (x, ldx), weight, bias, residual = _rows(x), weight.contiguous(), _aligned(bias), _aligned(residual)
    (M, K), N = x.shape, weight.shape[0]
    y = torch.empty(M, N, dtype=x.dtype, device=x.device)
    z = torch.empty(M, N, dtype=torch.float32, device=x.device) if keep and act != ACT_NONE else None
    if M:
        ws, n = _workspace(x, M, K, N, 0, 0)
        lib.mggan_block_linear_fwd(_p(x), ldx, _p(weight), _p(bias), _p(residual), _p(y), _p(z), M, K, N, act, float(slope),
                                   _DTYPES[x.dtype], _p(ws), n, _s())
    return y, z, x, weight


class LinearResidualFn(Function):
    @staticmethod
    def forward(ctx, x, weight, bias, residual, act, slope):
        y, z, x, weight = _linear_fwd(x, weight, bias, residual, act, slope, True)
        ctx.act, ctx.slope = act, slope
        ctx.save_for_backward(x, weight, z)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, weight, z = ctx.saved_tensors
        x, ldx = _rows(x)
        (M, K), N = x.shape, weight.shape[0]
        need = ctx.needs_input_grad
        like = dict(dtype=x.dtype, device=x.device)
        make = torch.empty if M else torch.zeros
        dx = make(M, K, **like) if need[0] else None
        dw = make(N, K, **like) if need[1] else None
        db = make(N, **like) if need[2] else None
        if M and any(need[:3]):
            g = _aligned(dy)
            ws, n = _workspace(x, M, K, N, 0, 1)
            lib.mggan_block_linear_bwd(_p(g), _p(z), _p(x), ldx, _p(weight), _p(dx), _p(dw), _p(db), M, K, N, ctx.act, float(ctx.slope),
                                       _DTYPES[x.dtype], _p(ws), n, _s())
        return dx, dw, db, (dy if need[3] else None), None, None


def linear_residual(x, weight, bias=None, residual=None, act=ACT_NONE, slope=0.0):
    """act(x W^T + bias) + residual: x (..., K), weight (N, K), bias (N) or None, residual (..., N) or None -> (..., N).
    act: ACT_NONE, ACT_LEAKY (with `slope`; 0 is ReLU), ACT_SIGMOID, ACT_SILU or ACT_GELU.  x may be a view with any row stride."""
    _same("linear_residual", x, weight=weight, bias=bias, residual=residual)
    _check_layer("linear_residual", x, weight, act, bias, residual)
    _on_gpu("linear_residual", x)
    lead, N = x.shape[:-1], weight.shape[0]
    x, r = x.reshape(-1, x.shape[-1]), None if residual is None else residual.reshape(-1, N)
    with torch.cuda.device(x.device):
        if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, weight, bias, r)):
            y = LinearResidualFn.apply(x, weight, bias, r, act, slope)
        else:
            y = _linear_fwd(x, weight, bias, r, act, slope, False)[0]
    return y.reshape(*lead, N)


def _gated_fwd(x, w_gate, w_up, b_gate, b_up, act, slope, keep):
    (x, ldx), w_gate, w_up, b_gate, b_up = _rows(x), w_gate.contiguous(), w_up.contiguous(), _aligned(b_gate), _aligned(b_up)
    (M, K), N = x.shape, w_gate.shape[0]
    y = torch.empty(M, N, dtype=x.dtype, device=x.device)
    z, u = (torch.empty(M, N, dtype=torch.float32, device=x.device) for _ in range(2)) if keep else (None, None)
    if M:
        ws, n = _workspace(x, M, K, N, 1, 0)
        lib.mggan_block_gated_fwd(_p(x), ldx, _p(w_gate), _p(w_up), _p(b_gate), _p(b_up), _p(y), _p(z), _p(u), M, K, N, act, float(slope),
                                  _DTYPES[x.dtype], _p(ws), n, _s())
    return y, z, u, x, w_gate, w_up


class GatedLinearFn(Function):
    @staticmethod
    def forward(ctx, x, w_gate, w_up, b_gate, b_up, act, slope):
        y, z, u, x, w_gate, w_up = _gated_fwd(x, w_gate, w_up, b_gate, b_up, act, slope, True)
        ctx.act, ctx.slope = act, slope
        ctx.save_for_backward(x, w_gate, w_up, z, u)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, w_gate, w_up, z, u = ctx.saved_tensors
        x, ldx = _rows(x)
        (M, K), N = x.shape, w_gate.shape[0]
        need = ctx.needs_input_grad
        like = dict(dtype=x.dtype, device=x.device)
        make = torch.empty if M else torch.zeros
        dx = make(M, K, **like) if need[0] else None
        dw = make(2 * N, K, **like) if need[1] or need[2] else None
        db = make(2 * N, **like) if need[3] or need[4] else None
        if M:
            g = _aligned(dy)
            ws, n = _workspace(x, M, K, N, 1, 1)
            lib.mggan_block_gated_bwd(_p(g), _p(z), _p(u), _p(x), ldx, _p(w_gate), _p(w_up), _p(dx), _p(dw), _p(db), M, K, N, ctx.act,
                                      float(ctx.slope), _DTYPES[x.dtype], _p(ws), n, _s())
        return (dx, dw[:N] if need[1] else None, dw[N:] if need[2] else None, db[:N] if need[3] else None, db[N:] if need[4] else None,
                None, None)


def gated_linear(x, w_gate, w_up, b_gate=None, b_up=None, act=ACT_SILU, slope=0.0):
    """act(x Wg^T + bg) * (x Wu^T + bu): x (..., K), w_gate and w_up (N, K), biases (N) or None -> (..., N); activations as in
    linear_residual."""
    _same("gated_linear", x, w_gate=w_gate, w_up=w_up, b_gate=b_gate, b_up=b_up)
    _check_layer("gated_linear", x, w_gate, act, b_gate)
    _check_layer("gated_linear", x, w_up, act, b_up)
    _check(w_gate.shape == w_up.shape, "gated_linear: weights of {} and {}", tuple(w_gate.shape), tuple(w_up.shape))
    _on_gpu("gated_linear", x)
    lead, N = x.shape[:-1], w_gate.shape[0]
    x = x.reshape(-1, x.shape[-1])
    with torch.cuda.device(x.device):
        if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, w_gate, w_up, b_gate, b_up)):
            y = GatedLinearFn.apply(x, w_gate, w_up, b_gate, b_up, act, slope)
        else:
            y = _gated_fwd(x, w_gate, w_up, b_gate, b_up, act, slope, False)[0]
    return y.reshape(*lead, N)


# ---- attention ---------------------------------------------------------------------------------------------------------------

class _AttnArgs(ctypes.Structure):  # mirrors csrc/blk_attn.h: BlkAttnArgs
    _fields_ = ([(n, ctypes.c_void_p) for n in ("q", "k", "v", "dout", "out", "dq", "dk", "dv", "dslopes", "scenes", "kv_scenes", "prefix",
                                                "xy", "kv_xy", "slopes", "lse", "out32", "spans", "ws")]
                + [(n, ctypes.c_long) for n in ("ws_bytes", "q_row", "q_head", "k_row", "k_head", "v_row", "v_head")]
                + [(n, ctypes.c_int) for n in ("N", "M", "H", "Hkv", "D", "S", "causal", "axes", "dtype")]
                + [("scale", ctypes.c_float), ("cap", ctypes.c_float)])


_TABLES = BoundedCache(64)


def _table(name, rows, device, limit, width):
    """int32 device tensor of a scene list (width 2) or of per-scene numbers (width 1): checked and kept by its contents when it is a
    host list, taken as it is when it is a device tensor."""
    if isinstance(rows, torch.Tensor) and rows.is_cuda:
        _check(rows.dtype == torch.int32 and rows.device == device and rows.dim() == width and (width == 1 or rows.shape[1] == 2),
               "attention: {} has to be an int32 tensor of (scenes{}) on {}", name, ", 2" if width == 2 else "", device)
        return rows.contiguous()
    try:
        key = tuple((int(a), int(b)) for a, b in rows) if width == 2 else tuple(int(a) for a in rows)
    except (TypeError, ValueError):
        raise ValueError("attention: {} has to be a list or an int32 device tensor".format(name)) from None
    if width == 2:
        for a, b in key:
            _check(0 <= a <= b <= limit, "attention: {} names rows [{}, {}) of {}", name, a, b, limit)
    else:
        _check(all(abs(a) < 2 ** 31 for a in key), "attention: {} out of range", name)
    hit = _TABLES.get((key, device))
    if hit is None:
        hit = torch.tensor(key, dtype=torch.int32).reshape((-1, 2) if width == 2 else (-1,)).to(device)
        _TABLES.put((key, device), hit)
    return hit


def _heads(t):
    """An operand whose rows and heads start at multiples of 16 bytes and whose width is contiguous (a copy where they do not)."""
    ch = 16 // t.element_size()
    ok = t.stride(2) == 1 and t.data_ptr() % 16 == 0 and all(t.shape[i] == 1 or (t.stride(i) % ch == 0 and t.stride(i) >= 0) for i in (0, 1))
    if not ok:
        t = t.contiguous()
        t = t.clone() if t.data_ptr() % 16 else t
    return t, tuple(t.stride(i) if t.shape[i] > 1 else 0 for i in (0, 1))


def _attn_args(q, k, v, scenes, kv_scenes, prefix, xy, kv_xy, slopes, causal, scale, cap):
    a = _AttnArgs()
    (q, (a.q_row, a.q_head)), (k, (a.k_row, a.k_head)), (v, (a.v_row, a.v_head)) = _heads(q), _heads(k), _heads(v)
    a.q, a.k, a.v = _p(q), _p(k), _p(v)
    a.scenes, a.kv_scenes, a.prefix, a.xy, a.kv_xy, a.slopes = _p(scenes), _p(kv_scenes), _p(prefix), _p(xy), _p(kv_xy), _p(slopes)
    (a.N, a.H, a.D), a.M, a.Hkv = q.shape, k.shape[0], k.shape[1]
    a.S, a.causal, a.axes, a.dtype = scenes.shape[0], int(causal), 0 if xy is None else xy.shape[1], _DTYPES[q.dtype]
    a.scale, a.cap = scale, cap
    return a, (q, k, v)


def _attn_fwd(a, q, keep):
    out = torch.empty(a.N, a.H, a.D, dtype=q.dtype, device=q.device)
    lse = torch.empty(2, a.H, a.N, dtype=torch.float32, device=q.device) if keep else None
    out32 = None if not keep else out if q.dtype == torch.float32 else torch.empty(out.shape, dtype=torch.float32, device=q.device)
    spans = torch.empty(lib.mggan_block_attention_span_ints(a.N), dtype=torch.int32, device=q.device)
    ws = None
    if not keep:
        a.ws_bytes = lib.mggan_block_attention_fwd_workspace(a.N, a.M, a.H, a.Hkv, a.D, a.S)
        ws = torch.empty(a.ws_bytes // 4, dtype=torch.float32, device=q.device) if a.ws_bytes else None
        a.ws = _p(ws)
    a.out, a.lse, a.out32, a.spans = _p(out), _p(lse), _p(out32), _p(spans)
    lib.mggan_block_attention_fwd(ctypes.addressof(a), _s())
    return out, lse, out32, spans


class AttentionFn(Function):
    @staticmethod
    def forward(ctx, q, k, v, slopes, rest):
        scenes, kv_scenes, prefix, xy, kv_xy, causal, scale, cap = rest
        ctx.rest = rest
        if q.shape[0] == 0 or k.shape[0] == 0:
            ctx.save_for_backward(q, k, v, slopes)
            ctx.empty = True
            return torch.zeros(q.shape, dtype=q.dtype, device=q.device)
        ctx.empty = False
        a, (q, k, v) = _attn_args(q, k, v, scenes, kv_scenes, prefix, xy, kv_xy, slopes, causal, scale, cap)
        out, lse, out32, spans = _attn_fwd(a, q, True)
        ctx.save_for_backward(q, k, v, slopes, out32, lse, spans)
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, dout):
        scenes, kv_scenes, prefix, xy, kv_xy, causal, scale, cap = ctx.rest
        if ctx.empty:
            return tuple(None if t is None else torch.zeros_like(t) for t in ctx.saved_tensors) + (None,)
        q, k, v, slopes, out32, lse, spans = ctx.saved_tensors
        a, _ = _attn_args(q, k, v, scenes, kv_scenes, prefix, xy, kv_xy, slopes, causal, scale, cap)
        dout = _aligned(dout)
        dq = torch.empty(q.shape, dtype=q.dtype, device=q.device)
        dk, dv = (torch.empty(k.shape, dtype=q.dtype, device=q.device) for _ in range(2))
        dslopes = torch.empty_like(slopes) if slopes is not None and ctx.needs_input_grad[3] else None
        a.ws_bytes = lib.mggan_block_attention_bwd_workspace(a.N, a.H)
        ws = torch.empty(a.ws_bytes // 4, dtype=torch.float32, device=q.device)
        a.dout, a.out32, a.lse, a.spans, a.ws = _p(dout), _p(out32), _p(lse), _p(spans), _p(ws)
        a.dq, a.dk, a.dv, a.dslopes = _p(dq), _p(dk), _p(dv), _p(dslopes)
        lib.mggan_block_attention_bwd(ctypes.addressof(a), _s())
        return dq, dk, dv, dslopes, None


def attention(q, k, v, scenes, kv_scenes=None, *, causal=False, prefix=None, scale=None, cap=0.0, xy=None, kv_xy=None, slopes=None):
    """Attention of every row of a scene over the keys of the same scene: q (N, H, D), k and v (M, Hkv, D) -> (N, H, D); H a multiple
    of Hkv (head h reads key head h // (H // Hkv)), D a multiple of 8 up to 128.

        out_i = sum_j P_ij v_j,    P_i = softmax over the visible j of   s_ij - slopes[h] |xy_i - kv_xy_j|,    s = cap tanh(scale q k / cap)

    scenes, kv_scenes: rows [start, end) of q and of k / v that belong to each scene, as a list of pairs (the framework's
    seq_start_end) or as an int32 device tensor (scenes, 2), which is read when the kernel runs (and clamped to the operands' rows);
    kv_scenes defaults to scenes.  In any order; scenes may share keys; of a row that several scenes name the last one counts.  Rows of
    no scene and rows that see no key give zeros.  What lies outside a row's visible keys is never mixed in, infinities and NaN included.
    causal: row i of a scene of Lq rows and Lk keys sees keys j <= i + Lk - Lq, and in any case those before prefix[scene] (list or int32
    device tensor).  One new row over a long cache is Lq = 1.  scale: > 0, D ** -0.5 by default; cap: 0 for none.
    xy (N, axes) and kv_xy (M, axes; by default xy), f32 with one or two axes, and slopes (H), f32: the bias by distance.  Gradients go to q,
    k, v and slopes, not to positions."""
    name = "attention"
    _same(name, q, k=k, v=v)
    _check(q.dim() == 3 and k.dim() == 3 and k.shape == v.shape and q.shape[2] == k.shape[2], "{}: q {}, k {}, v {}", name, tuple(q.shape),
           tuple(k.shape), tuple(v.shape))
    (N, H, D), (M, Hkv, _) = q.shape, k.shape
    _check(0 < H <= 1024 and Hkv > 0 and H % Hkv == 0, "{}: {} heads over {} key heads", name, H, Hkv)
    _check(D % 8 == 0 and 0 < D <= 128, "{}: a width of {} (a multiple of 8 up to 128)", name, D)
    _check(N <= 1 << 24 and M <= 1 << 30, "{}: {} rows, {} keys", name, N, M)
    scale = D ** -0.5 if scale is None else float(scale)
    cap = 0.0 if cap is None else float(cap)
    _check(scale > 0 and math.isfinite(scale), "{}: scale {} (it has to be positive)", name, scale)
    _check(cap >= 0 and math.isfinite(cap), "{}: cap {}", name, cap)
    _check(prefix is None or causal, "{}: a prefix without causal", name)
    _check((xy is None) == (slopes is None) and (xy is not None or kv_xy is None), "{}: positions and slopes come together", name)
    if xy is not None:
        kv_xy = xy if kv_xy is None else kv_xy
        for n, t, rows in (("xy", xy, N), ("kv_xy", kv_xy, M)):
            _check(t.dtype == torch.float32 and t.dim() == 2 and t.shape[0] == rows and t.shape[1] in (1, 2) and t.shape[1] == xy.shape[1],
                   "{}: {} {} {} for {} rows and one or two axes, f32", name, n, t.dtype, tuple(t.shape), rows)
            _check(t.device == q.device, "{}: {} is on {}", name, n, t.device)
            _check(not (t.requires_grad and torch.is_grad_enabled()), "{}: {} requires a gradient, positions have none: detach it", name, n)
        _check(slopes.dtype == torch.float32 and tuple(slopes.shape) == (H,) and slopes.device == q.device, "{}: slopes {} {} on {}", name,
               slopes.dtype, tuple(slopes.shape), slopes.device)
    _on_gpu(name, q)
    with torch.cuda.device(q.device):
        table = _table("scenes", scenes, q.device, N, 2)
        kv_table = table if kv_scenes is None else _table("kv_scenes", kv_scenes, q.device, M, 2)
        if kv_scenes is None:
            _check(M >= N, "{}: {} rows over {} keys need kv_scenes", name, N, M)
        _check(table.shape == kv_table.shape, "{}: {} scenes of rows, {} of keys", name, table.shape[0], kv_table.shape[0])
        if prefix is not None:
            prefix = _table("prefix", prefix, q.device, 0, 1)
            _check(prefix.shape[0] == table.shape[0], "{}: {} prefixes for {} scenes", name, prefix.shape[0], table.shape[0])
        if xy is not None:
            same = kv_xy is xy
            xy, slopes = xy.detach().contiguous(), slopes.contiguous()
            kv_xy = xy if same else kv_xy.detach().contiguous()
        if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (q, k, v, slopes)):
            return AttentionFn.apply(q, k, v, slopes, (table, kv_table, prefix, xy, kv_xy, causal, scale, cap))
        if N == 0 or M == 0:
            return torch.zeros(q.shape, dtype=q.dtype, device=q.device)
        a, ops = _attn_args(q, k, v, table, kv_table, prefix, xy, kv_xy, slopes, causal, scale, cap)
        return _attn_fwd(a, ops[0], False)[0]
