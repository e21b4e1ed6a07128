"""Operators of a transformer block over the rows of scenes, f32 or bf16, with their backward passes:

    linear_residual(x, weight, bias, residual, act)   act(x W^T + b) + residual
    gated_linear(x, w_gate, w_up, b_gate, b_up, act)  act(x Wg^T + bg) * (x Wu^T + bu)

All operands of a call have one type and live on one device; sums, activations and softmax statistics are held in f32 and
rounded once.  Work goes to torch's current stream, outputs and workspaces come from torch's allocator (so a call can be captured
into a HIP graph), gradients are returned through autograd and are the same bits in every run.  Arguments that do not fit raise
ValueError, a failing launch raises HipError; there is no CPU path."""
import torch
from torch.autograd import Function
from torch.autograd.function import once_differentiable

from .functions import ACT_LEAKY, ACT_NONE, ACT_SIGMOID, _p, _s
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
    z = torch.empty_like(y) if keep and act != ACT_NONE else None
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
    z, u = (torch.empty_like(y), torch.empty_like(y)) if keep else (None, None)
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
