"""Operators of a transformer block over the rows of scenes, f32 or bf16, with their backward passes:

    attention(q, k, v, scenes, ...)                   softmax(cap tanh(scale q k / cap) - slope |xy - kv_xy|) v within each scene
    linear_residual(x, weight, bias, residual, act)   act(x W^T + b) + residual
    gated_linear(x, w_gate, w_up, b_gate, b_up, act)  act(x Wg^T + bg) * (x Wu^T + bu)

All operands of a call have one type and live on one device; sums, activations and softmax statistics are held in f32, outputs and
gradients rounded once.  With bf16 operands the matrix instructions take bf16: the softmax's weights P, the scores' gradients and the
gradients dZ before the activation are rounded to bf16 as well where they enter a product (against 64 bits 0.0024 instead of 0.0017, the
final rounding alone); with f32 operands nothing is.  Work goes to torch's current stream, outputs and workspaces come from torch's allocator (so a call can be captured
into a HIP graph), gradients are returned through autograd and are the same bits in every run.  Arguments that do not fit raise
ValueError, a failing launch raises HipError, forward-mode tangents raise NotImplementedError; there is no CPU path."""
import functools
import operator
import struct
from itertools import chain

import torch
from torch.autograd import Function, forward_ad
from torch.autograd.function import once_differentiable

from .functions import _GET_DEVICE, ACT_LEAKY, ACT_NONE, ACT_SIGMOID, BoundedCache, _p, _s
from .lib import lib

ACT_SILU, ACT_GELU = 4, 5
_ACTS = (ACT_NONE, ACT_LEAKY, ACT_SIGMOID, ACT_SILU, ACT_GELU)
_DTYPES = {torch.float32: 0, torch.bfloat16: 1}
_F32, _F32_MAX = torch.float32, torch.finfo(torch.float32).max

# The calls' arguments as the C structures of csrc/blk_gemm.hip and csrc/blk_attn.h lay them out, packed in one go (a small call is
# bound by the host: filling a ctypes structure field by field took 6 us of a 36 us forward call).
_LAYER = struct.Struct("=14Q2q5if")
_ATTN = struct.Struct("=19Q7q9i2f4x")


@functools.lru_cache(maxsize=1024)
def _layer_workspace(M, K, N, gated, backward, act, dtype):
    return lib.mggan_block_layer_workspace(M, K, N, gated, backward, act, dtype)


@functools.lru_cache(maxsize=1024)
def _attn_sizes(N, M, H, Hkv, D, S):
    """(int32 of the row intervals, bytes for splitting the keys of single rows, bytes of the backward pass)"""
    return (lib.mggan_block_attention_span_ints(N), lib.mggan_block_attention_fwd_workspace(N, M, H, Hkv, D, S),
            lib.mggan_block_attention_bwd_workspace(N, M, H, Hkv, D))


def _bytes(n, like):
    return torch.empty(n, dtype=torch.uint8, device=like.device) if n else None


_current_device = _GET_DEVICE or torch.cuda.current_device


def _same(name, x, *others):
    """Every operand has x's type and device."""
    dtype, device = x.dtype, x.device
    if dtype not in _DTYPES:
        raise ValueError("{}: f32 or bf16 tensors, got {}".format(name, dtype))
    for t in others:
        if t is not None and (t.dtype != dtype or t.device != device):
            raise ValueError("{}: one operand is {} on {}, the first one {} on {}".format(name, t.dtype, t.device, dtype, device))


def _on_current(name, x):
    """Whether x lives on the current device (the call is repeated under its own otherwise)."""
    at = x.get_device()
    if at < 0:
        raise ValueError("{}: the operands are on {}; there is no CPU path".format(name, x.device))
    return at == _current_device()


def _aligned(t):
    """Contiguous and 16-byte aligned (a copy where it is not)."""
    if t is None:
        return None
    if not t.is_contiguous():
        t = t.contiguous()
    return t.clone() if t.data_ptr() % 16 else t


def _any_dual(*tensors):
    """Whether one of them carries a forward-mode tangent (torch.autograd.forward_ad); without an open level none does."""
    if getattr(forward_ad, "_current_level", 0) < 0:
        return False
    return any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors)


def _needs_grad(*tensors):
    """Whether the call goes through its autograd function: for a gradient, or for an operand with a forward-mode tangent, which the
    function refuses (NotImplementedError) where the kernel alone would drop it."""
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                return True
    return _any_dual(*tensors)


def _number(name, what, value):
    """A factor of the call as a float (an f32 one in the kernels): no tensor that a gradient is wanted of."""
    if isinstance(value, torch.Tensor) and (value.requires_grad and torch.is_grad_enabled() or _any_dual(value)):
        raise ValueError("{}: {} has no gradient: detach it".format(name, what))
    try:
        return float(value)
    except (TypeError, ValueError, RuntimeError, OverflowError):
        raise ValueError("{}: {} is not a number: {!r}".format(name, what, value)) from None


# ---- layers ------------------------------------------------------------------------------------------------------------------

def _rows(x, K):
    """x as (rows, K) with unit inner stride, rows that start at multiples of 16 bytes (unless K does not), and its row stride."""
    if x.dim() != 2:
        x = x.reshape(-1, K)
    M, ch = x.shape[0], 16 // x.element_size()
    ld = x.stride(0) if M > 1 else K
    if (x.stride(1) != 1 and K > 1) or ld < K:
        x, ld = x.contiguous(), K
    if K % ch == 0:
        if ld % ch:
            x, ld = x.contiguous(), K
        if x.data_ptr() % 16:
            x, ld = x.clone(memory_format=torch.contiguous_format), K
    return x, ld


def _check_layer(name, x, weight, bias, act, slope):
    """-> the slope as a float"""
    rows, shape = x.shape, weight.shape
    if len(shape) != 2 or not rows or rows[-1] != shape[1] or not shape[0] or not shape[1]:
        raise ValueError("{}: rows of {} and a weight of {}".format(name, tuple(rows), tuple(shape)))
    N, K = shape
    if x.numel() > K << 21 or N > 1 << 20 or K > 1 << 20:
        raise ValueError("{}: sizes {} x {} over 2^21 rows, 2^20 columns".format(name, tuple(x.shape), tuple(weight.shape)))
    if not isinstance(act, int) or act not in _ACTS:
        raise ValueError("{}: unknown activation {}".format(name, act))
    if bias is not None and (bias.dim() != 1 or bias.shape[0] != N):
        raise ValueError("{}: a bias of {} for {} outputs".format(name, tuple(bias.shape), N))
    if type(slope) is not float:
        slope = _number(name, "slope", slope)
    if not -_F32_MAX <= slope <= _F32_MAX:
        raise ValueError("{}: slope {} is not a finite f32 number".format(name, slope))
    return slope


def _layer_fwd(x, w, w2, b, b2, res, act, slope, keep):
    """-> y, kept inputs of the activation, operands as the kernels read them"""
    N, K = w.shape
    (x, ldx), w, b = _rows(x, K), _aligned(w), _aligned(b)
    gated = w2 is not None
    if gated:
        w2, b2 = _aligned(w2), _aligned(b2)
    M, dev, code = x.shape[0], x.device, _DTYPES[x.dtype]
    y = torch.empty(M, N, dtype=x.dtype, device=dev)
    z = torch.empty((1 + gated, M, N), dtype=_F32, device=dev) if keep and (gated or act != ACT_NONE) else None
    if M:
        res = _aligned(res)
        n = _layer_workspace(M, K, N, gated, 0, act, code)
        ws = _bytes(n, x)
        pz = _p(z)
        # (z2 lies M N f32 behind z: 16-byte aligned as the workspace of a call has to be only where M N is a multiple of four)
        z2 = None
        if gated and z is not None:
            z2 = pz + 4 * M * N
            if z2 % 16:
                z = torch.empty((2, M * N + (-M * N) % 4), dtype=_F32, device=dev)
                pz = _p(z)
                z2 = pz + 4 * z.stride(0)
        lib.mggan_block_layer_fwd(_LAYER.pack(_p(x), _p(w), _p(w2), _p(b), _p(b2), _p(res), 0, pz, z2 or 0, _p(y), 0, 0, 0, _p(ws), n, ldx,
                                              M, K, N, act, code, slope), _s())
    return y, z, x, w, w2


def _layer_bwd(ctx, dy):
    x, w, w2, z = ctx.saved_tensors
    gated, need = w2 is not None, ctx.needs_input_grad
    (x, ldx), (N, K) = _rows(x, w.shape[1]), w.shape
    M, dev, dt = x.shape[0], x.device, x.dtype
    code = _DTYPES[dt]
    off = -(-N // (64 // x.element_size())) * (64 // x.element_size()) if gated else 0  # where the up weight's gradient starts
    make = torch.empty if M else torch.zeros
    dx = make(M, K, dtype=dt, device=dev) if need[0] else None
    dw = make(off + N, K, dtype=dt, device=dev) if need[1] or need[2] else None
    db = make((1 + gated) * N, dtype=dt, device=dev) if need[3] or need[4] else None
    if M and (dx is not None or dw is not None or db is not None):
        g = _aligned(dy)
        n = _layer_workspace(M, K, N, gated, 1, ctx.act, code)
        ws = _bytes(n, x)
        lib.mggan_block_layer_bwd(_LAYER.pack(_p(x), _p(w), _p(w2), 0, 0, 0, _p(g), _p(z), _p(z) + 4 * z.stride(0) if gated else 0, 0, _p(dx),
                                              _p(dw), _p(db), _p(ws), n, ldx, M, K, N, ctx.act, code, ctx.slope), _s())
    if not gated:
        return dx, dw, None, db, None, (dy if need[5] else None), None, None
    return (dx, dw[:N] if need[1] else None, dw[off:] if need[2] else None, db[:N] if need[3] else None, db[N:] if need[4] else None, None, None,
            None)


_layer_bwd_once = once_differentiable(_layer_bwd)


class LayerFn(Function):
    """Both layers: a linear one has no second weight and may have a residual."""

    @staticmethod
    def forward(ctx, x, w, w2, b, b2, res, act, slope):
        y, z, x, w, w2 = _layer_fwd(x, w, w2, b, b2, res, act, slope, True)
        ctx.act, ctx.slope = act, slope
        ctx.save_for_backward(x, w, w2, z)
        return y

    @staticmethod
    def backward(ctx, dy):
        return _layer_bwd_once(ctx, dy) if torch.is_grad_enabled() else _layer_bwd(ctx, dy)


def linear_residual(x, weight, bias=None, residual=None, act=ACT_NONE, slope=0.0):
    """act(x W^T + b) + residual: x (..., K), weight (N, K), bias (N) or None, residual (..., N) or None -> (..., N).
    act: ACT_NONE, ACT_LEAKY (with `slope`; 0 is ReLU), ACT_SIGMOID, ACT_SILU or ACT_GELU; the slope is a
    number, without a gradient.  x may be a view with any row stride."""
    _same("linear_residual", x, weight, bias, residual)
    slope = _check_layer("linear_residual", x, weight, bias, act, slope)
    N, two = weight.shape[0], x.dim() == 2
    if residual is not None and residual.shape != x.shape[:-1] + (N,):
        raise ValueError("linear_residual: a residual of {} for outputs of {} (it is not broadcast)".format(
            tuple(residual.shape), tuple(x.shape[:-1]) + (N,)))
    if not _on_current("linear_residual", x):
        with torch.cuda.device(x.device):
            return linear_residual(x, weight, bias, residual, act, slope)
    if not two:
        lead = x.shape[:-1]
        x, residual = x.reshape(-1, x.shape[-1]), None if residual is None else residual.reshape(-1, N)
    if _needs_grad(x, weight, bias, residual):
        y = LayerFn.apply(x, weight, None, bias, None, residual, act, slope)
    else:
        y = _layer_fwd(x, weight, None, bias, None, residual, act, slope, False)[0]
    return y if two else y.reshape(*lead, N)


def gated_linear(x, w_gate, w_up, b_gate=None, b_up=None, act=ACT_SILU, slope=0.0):
    """act(x Wg^T + bg) * (x Wu^T + bu): x (..., K), w_gate and w_up (N, K), biases (N) or None -> (..., N); activations as in
    linear_residual."""
    _same("gated_linear", x, w_gate, w_up, b_gate, b_up)
    slope = _check_layer("gated_linear", x, w_gate, b_gate, act, slope)
    _check_layer("gated_linear", x, w_up, b_up, act, slope)
    if w_gate.shape != w_up.shape:
        raise ValueError("gated_linear: weights of {} and {}".format(tuple(w_gate.shape), tuple(w_up.shape)))
    if not _on_current("gated_linear", x):
        with torch.cuda.device(x.device):
            return gated_linear(x, w_gate, w_up, b_gate, b_up, act, slope)
    two = x.dim() == 2
    if not two:
        lead, x = x.shape[:-1], x.reshape(-1, x.shape[-1])
    if _needs_grad(x, w_gate, w_up, b_gate, b_up):
        y = LayerFn.apply(x, w_gate, w_up, b_gate, b_up, None, act, slope)
    else:
        y = _layer_fwd(x, w_gate, w_up, b_gate, b_up, None, act, slope, False)[0]
    return y if two else y.reshape(*lead, w_gate.shape[0])


# ---- attention ---------------------------------------------------------------------------------------------------------------

_TABLES = BoundedCache(64)
_LEAST = 2.0 ** -60  # of scale and cap: their quotient and their products with log2 e stay normal f32 numbers


def _table(name, rows, device, limit, width):
    """int32 device tensor of a scene list (width 2) or of per-scene numbers (width 1): checked and kept by its contents when it is a
    host list, taken as it is when it is a device tensor."""
    if isinstance(rows, torch.Tensor) and rows.is_cuda:
        shape = rows.shape
        if rows.dtype != torch.int32 or rows.device != device or len(shape) != width or (width == 2 and shape[1] != 2):
            raise ValueError("attention: {} has to be an int32 tensor of (scenes{}) on {}".format(name, ", 2" if width == 2 else "", device))
        return rows if rows.is_contiguous() else rows.contiguous()
    try:
        key = tuple(map(tuple, rows)) if width == 2 else tuple(rows)
        if not {int}.issuperset(map(type, chain.from_iterable(key) if width == 2 else key)) or width == 2 and not {2}.issuperset(map(len, key)):
            key = tuple((operator.index(a), operator.index(b)) for a, b in key) if width == 2 else tuple(map(operator.index, key))
    except (TypeError, ValueError):
        raise ValueError("attention: {} has to be a list of whole numbers or an int32 device tensor".format(name)) from None
    key = (key, limit, device)
    hit = _TABLES.get(key)
    if hit is None:
        for k in key[0]:
            if width == 2 and not 0 <= k[0] <= k[1] <= limit:
                raise ValueError("attention: {} names rows [{}, {}) of {}".format(name, k[0], k[1], limit))
            if width == 1 and abs(k) >= 1 << 31:
                raise ValueError("attention: {} out of range".format(name))
        if torch.cuda.is_current_stream_capturing():
            raise ValueError("attention: {} is a list that no call before the capture had: a capture cannot copy it to the device".format(name))
        table = torch.tensor(key[0], dtype=torch.int32).reshape((-1, 2) if width == 2 else (-1,)).to(device)  # (a copy that is waited for)
        _TABLES.put(key, (table, _s()))
        return table
    if torch.cuda.is_current_stream_capturing():
        _TABLES.pinned.add(key)  # (the graph reads it at every replay: it is never dropped)
    elif hit[1] != _s():
        hit[0].record_stream(torch.cuda.current_stream())  # (dropped from the table, its memory waits for this stream too)
    return hit[0]


def _heads(t):
    """An operand whose rows and heads start at multiples of 16 bytes and whose width is contiguous (a copy where they do not), and its
    two strides."""
    rows, heads, width = t.stride()
    n, h, _ = t.shape
    ch = 16 // t.element_size()
    if width != 1 or t.data_ptr() % 16 or (n > 1 and (rows % ch or rows < 0)) or (h > 1 and (heads % ch or heads < 0)):
        t = t.contiguous()
        t = t.clone() if t.data_ptr() % 16 else t
        rows, heads, _ = t.stride()
    return t, (rows if n > 1 else 0), (heads if h > 1 else 0)


def _attn_fwd(q, k, v, slopes, rest, keep):
    """-> out, the output in f32, row statistics, the operands as the kernels read them"""
    scenes, kv_scenes, prefix, xy, kv_xy, causal, scale, cap = rest
    (q, q_row, q_head), (k, k_row, k_head), (v, v_row, v_head) = _heads(q), _heads(k), _heads(v)
    (N, H, D), (M, Hkv, _), S, dev = q.shape, k.shape, scenes.shape[0], q.device
    ints, n, _ = _attn_sizes(N, M, H, Hkv, D, S)
    out = torch.empty((N, H, D), dtype=q.dtype, device=dev)
    at = 3 * H * N + (-3 * H * N) % 4 if keep else 0  # the row intervals lie behind the softmax statistics
    stats = torch.empty(at + ints, dtype=_F32, device=dev)
    out32 = ws = None
    if keep:
        out32, n = out if q.dtype == _F32 else torch.empty((N, H, D), dtype=_F32, device=dev), 0
    else:
        ws = _bytes(n, q)
    ps = _p(stats)
    lib.mggan_block_attention_fwd(_ATTN.pack(
        _p(q), _p(k), _p(v), 0, _p(out), 0, 0, 0, 0, _p(scenes), _p(kv_scenes), _p(prefix), _p(xy), _p(kv_xy), _p(slopes), ps if keep else 0,
        _p(out32), ps + 4 * at, _p(ws), n, q_row, q_head, k_row, k_head, v_row, v_head, N, M, H, Hkv, D, S, causal,
        0 if xy is None else xy.shape[1], _DTYPES[q.dtype], scale, cap), _s())
    return out, out32, stats, q, k, v


def _attn_bwd(ctx, dout):
    q, k, v, slopes, out32, stats, xy, kv_xy = ctx.saved_tensors
    if stats is None:
        return tuple(None if t is None else torch.zeros_like(t) for t in (q, k, v, slopes)) + (None,)
    scenes, kv_scenes, prefix, _, _, causal, scale, cap = ctx.rest
    (q, q_row, q_head), (k, k_row, k_head), (v, v_row, v_head) = _heads(q), _heads(k), _heads(v)
    (N, H, D), (M, Hkv, _), S, dev, dt = q.shape, k.shape, scenes.shape[0], q.device, q.dtype
    dout = _aligned(dout)
    dq = torch.empty((N, H, D), dtype=dt, device=dev)
    dk = torch.empty((M, Hkv, D), dtype=dt, device=dev)
    dv = torch.empty((M, Hkv, D), dtype=dt, device=dev)
    dslopes = torch.empty(H, dtype=_F32, device=dev) if slopes is not None and ctx.needs_input_grad[3] else None
    n = _attn_sizes(N, M, H, Hkv, D, S)[2]
    ws = _bytes(n, q)
    ps = _p(stats)
    at = 3 * H * N + (-3 * H * N) % 4
    lib.mggan_block_attention_bwd(_ATTN.pack(
        _p(q), _p(k), _p(v), _p(dout), 0, _p(dq), _p(dk), _p(dv), _p(dslopes), _p(scenes), _p(kv_scenes), _p(prefix), _p(xy), _p(kv_xy),
        _p(slopes), ps, _p(out32), ps + 4 * at, _p(ws), n, q_row, q_head, k_row, k_head, v_row, v_head, N, M, H,
        Hkv, D, S, causal, 0 if xy is None else xy.shape[1], _DTYPES[dt], scale, cap), _s())
    return dq, dk, dv, dslopes, None


_attn_bwd_once = once_differentiable(_attn_bwd)


class AttentionFn(Function):
    @staticmethod
    def forward(ctx, q, k, v, slopes, rest):
        # (what the backward pass reads is saved, the positions too: an operand that is written in between raises there.  The scene tables
        # are not read again: the intervals lie behind the statistics)
        ctx.rest = rest[:3] + (None, None) + rest[5:]
        if q.shape[0] == 0 or k.shape[0] == 0:
            ctx.save_for_backward(q, k, v, slopes, None, None, None, None)
            return torch.zeros(q.shape, dtype=q.dtype, device=q.device)
        out, out32, stats, q, k, v = _attn_fwd(q, k, v, slopes, rest, True)
        ctx.save_for_backward(q, k, v, slopes, out32, stats, rest[3], rest[4])
        return out

    @staticmethod
    def backward(ctx, dout):
        return _attn_bwd_once(ctx, dout) if torch.is_grad_enabled() else _attn_bwd(ctx, dout)


def attention(q, k, v, scenes, kv_scenes=None, *, causal=False, prefix=None, scale=None, cap=0.0, xy=None, kv_xy=None, slopes=None):
    """Attention of every row of a scene over the keys of the same scene: q (N, H, D), k and v (M, Hkv, D) -> (N, H, D); H a multiple
    of Hkv (head h reads key head h // (H // Hkv)), D a multiple of 8 up to 128.

        out_i = sum_j P_ij v_j,    P_i = softmax over the visible j of   s_ij - slopes[h] |xy_i - kv_xy_j|,    s = cap tanh(scale q k / cap)

    scenes, kv_scenes: rows [start, end) of q and of k / v that belong to each scene, as a list of pairs (the framework's
    seq_start_end) or as an int32 device tensor (scenes, 2), which is read when the kernel runs (and clamped to the operands' rows);
    kv_scenes defaults to scenes.  A list is copied to the device once for its contents, so inside a capture it has to be one that a call
    before the capture had; a device tensor is read at every replay.  In any order; scenes may share keys; of a row that several scenes name the last one counts.  Rows of
    no scene and rows that see no key give zeros.  What lies outside a row's visible keys is never mixed in, infinities and NaN included.
    causal: row i of a scene of Lq rows and Lk keys sees keys j <= i + Lk - Lq, and in any case those before prefix[scene] (list or int32
    device tensor).  One new row over a long cache is Lq = 1.  scale: > 0, D ** -0.5 by default; cap: 0 for none;
    both numbers between 2^-60 and 2^60, without a gradient.
    xy (N, axes) and kv_xy (M, axes; by default xy), f32 with one or two axes, and slopes (H), f32: the bias by distance.  Gradients go to q,
    k, v and slopes, not to positions."""
    _same("attention", q, k, v)
    rows, keys = q.shape, k.shape
    if len(rows) != 3 or len(keys) != 3 or keys != v.shape or rows[2] != keys[2]:
        raise ValueError("attention: q {}, k {}, v {}".format(tuple(rows), tuple(keys), tuple(v.shape)))
    (N, H, D), (M, Hkv, _) = rows, keys
    if not 0 < H <= 1024 or not Hkv or H % Hkv:
        raise ValueError("attention: {} heads over {} key heads".format(H, Hkv))
    if D % 8 or not 0 < D <= 128:
        raise ValueError("attention: a width of {} (a multiple of 8 up to 128)".format(D))
    if N > 1 << 24 or M > 1 << 30 or N * H > 1 << 29:
        raise ValueError("attention: {} rows of {} heads, {} keys (at most 2^24 rows, 2^29 rows times heads, 2^30 keys)".format(N, H, M))
    scale = D ** -0.5 if scale is None else _number("attention", "scale", scale)
    cap = 0.0 if cap is None else _number("attention", "cap", cap)
    if not _LEAST <= scale <= 1 / _LEAST or not (cap == 0 or _LEAST <= cap <= 1 / _LEAST):
        raise ValueError("attention: scale {} (has to be positive), cap {} (0 or positive), both within 2^-60 and 2^60".format(scale, cap))
    if prefix is not None and not causal:
        raise ValueError("attention: a prefix without causal")
    if (xy is None) != (slopes is None) or (xy is None and kv_xy is not None):
        raise ValueError("attention: positions and slopes come together")
    if kv_scenes is None and M < N:
        raise ValueError("attention: {} rows over {} keys need kv_scenes".format(N, M))
    if xy is not None:
        kv_xy = xy if kv_xy is None else kv_xy
        for t, n in ((xy, N), (kv_xy, M)):
            if t.dtype != _F32 or t.dim() != 2 or t.shape[0] != n or t.shape[1] not in (1, 2) or t.shape[1] != xy.shape[1] or t.device != q.device:
                raise ValueError("attention: positions {} {} on {} for {} rows: f32, one or two axes".format(t.dtype, tuple(t.shape), t.device, n))
            if t.requires_grad and torch.is_grad_enabled() or _any_dual(t):
                raise ValueError("attention: positions have no gradient: detach them")
        if slopes.dtype != _F32 or slopes.dim() != 1 or slopes.shape[0] != H or slopes.device != q.device:
            raise ValueError("attention: slopes {} {} on {} for {} heads".format(slopes.dtype, tuple(slopes.shape), slopes.device, H))
    if not _on_current("attention", q):
        with torch.cuda.device(q.device):
            return attention(q, k, v, scenes, kv_scenes, causal=causal, prefix=prefix, scale=scale, cap=cap, xy=xy, kv_xy=kv_xy, slopes=slopes)
    dev = q.device
    table = _table("scenes", scenes, dev, N, 2)
    kv_table = table if kv_scenes is None else _table("kv_scenes", kv_scenes, dev, M, 2)
    if table.shape[0] != kv_table.shape[0]:
        raise ValueError("attention: {} scenes of rows, {} of keys".format(table.shape[0], kv_table.shape[0]))
    if prefix is not None:
        prefix = _table("prefix", prefix, dev, 0, 1)
        if prefix.shape[0] != table.shape[0]:
            raise ValueError("attention: {} prefixes for {} scenes".format(prefix.shape[0], table.shape[0]))
    if xy is not None:
        same = kv_xy is xy
        xy, slopes = xy.contiguous(), slopes.contiguous()
        kv_xy = xy if same else kv_xy.contiguous()
    rest = (table, kv_table, prefix, xy, kv_xy, bool(causal), scale, cap)
    if _needs_grad(q, k, v, slopes):
        if M * H > 1 << 29:
            raise ValueError("attention: gradients of {} keys for {} heads (at most 2^29 keys times heads)".format(M, H))
        return AttentionFn.apply(q, k, v, slopes, rest)
    if N == 0 or M == 0:
        return torch.zeros(q.shape, dtype=q.dtype, device=q.device)
    return _attn_fwd(q, k, v, slopes, rest, False)[0]
