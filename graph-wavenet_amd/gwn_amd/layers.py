"""Position-wise layers on libgwn: the product with its epilogue, layer norm, and dropout without a
stored mask, with hand-written backward passes.

They extend the reference's position-wise pieces -- ``linear`` (model.py:24-30), the BatchNorm
(model.py:152, 236) and the dropout (model.py:54) -- to channels-last tensors ``[..., C]`` of float32,
float16 or bfloat16, for feed-forward and attention-style blocks around a ``gwnet``.  Sums and
statistics are fp32 whatever the type, and every result is rounded once.

``linear_act``, ``layer_norm`` and ``dropout`` are functions; ``LinearAct``, ``LayerNorm``, ``Dropout``
and ``FeedForward`` hold parameters.  Masks come from a counter: ``seed`` is an int64 device tensor of
one element that the program advances once a step (``seed.add_(1)``, also inside a captured graph),
``salt`` numbers the mask within the step.  A seed that was advanced between a forward and its
backward is refused by autograd's version check, since the backward rebuilds the forward's mask.

The tensors of one call share a device and a type (layer norm's parameters may stay float32); work
is queued on that device's current stream.  Inputs may be strided over their leading axes; where
the last axis is not contiguous or the leading axes do not fold into rows, a copy is made.
"""
import ctypes

import torch
import torch.nn as nn
from torch.autograd.function import once_differentiable

from . import _lib

ACTS = {"none": 0, "relu": 1, "gelu": 2, "gelu_tanh": 3, "silu": 4}
_ELEM = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
F32 = torch.float32


def _check(what, x, *others):
    """x is a device tensor of a known type; the others (None skipped) share its device and type."""
    if not x.is_cuda:
        raise RuntimeError("%s: the HIP path needs tensors on a GPU device (there is no CPU fallback)" % what)
    if x.dtype not in _ELEM:
        raise RuntimeError("%s: float32, float16 or bfloat16 tensors are needed, got %s" % (what, x.dtype))
    for t in others:
        if t is not None and (t.device != x.device or t.dtype != x.dtype):
            raise RuntimeError("%s: tensors of one device and type are needed, got %s %s beside %s %s"
                               % (what, t.dtype, t.device, x.dtype, x.device))


def _check_seed(what, x, p, seed, salt):
    if not 0.0 <= p <= 1.0:
        raise ValueError("%s: the dropout rate must be between 0 and 1, got %s" % (what, p))
    if not 0 <= salt < 2 ** 64:
        raise ValueError("%s: salt must be a 64-bit unsigned number, got %s" % (what, salt))
    if p > 0.0 and (not isinstance(seed, torch.Tensor) or seed.dtype != torch.int64 or seed.numel() != 1
                    or seed.device != x.device):
        raise RuntimeError("%s: dropout needs a seed, an int64 tensor of one element on %s" % (what, x.device))


def _rows(t, c):
    """t [..., c] as rows [m, c] with a row stride >= c and a contiguous last axis (a copy where the
    strides do not allow it) and that row stride."""
    if t.is_contiguous():
        return t, c
    t = t.reshape(-1, c)
    m = t.shape[0]
    if (c > 1 and t.stride(1) != 1) or (m > 1 and t.stride(0) < c):
        t = t.contiguous()
    return t, (t.stride(0) if m > 1 else c)


def _ws(floats, device):
    return torch.empty(floats, device=device, dtype=F32) if floats > 0 else None


class _on:
    """The tensors' device as the current one during a call (nothing to do where it is already)."""

    def __init__(self, t):
        self.guard = None if t.device.index == torch.cuda.current_device() else torch.cuda.device(t.device)

    def __enter__(self):
        if self.guard is not None:
            self.guard.__enter__()

    def __exit__(self, *exc):
        if self.guard is not None:
            self.guard.__exit__(*exc)


# ---- the product with its epilogue ----------------------------------------------------------

def _linear_fwd(x, weight, bias, act, residual, p, seed, salt, keep_z):
    n, k = weight.shape
    y = torch.empty(x.shape[:-1] + (n,), device=x.device, dtype=x.dtype)
    m = y.numel() // n
    z = None
    if keep_z and act:
        z = torch.empty(m, n, device=x.device, dtype=F32 if x.dtype == F32 else torch.float16)
    if m == 0:
        return y, z
    x, ldx = _rows(x, k)
    w, ldw = _rows(weight, k)
    a = _lib.LinearArgs()
    a.x, a.ldx, a.w, a.ldw = x.data_ptr(), ldx, w.data_ptr(), ldw
    if bias is not None:
        bias = bias.contiguous()
        a.bias = bias.data_ptr()
    if residual is not None:
        residual, a.ld_res = _rows(residual, n)
        a.residual = residual.data_ptr()
    a.y, a.ldy = y.data_ptr(), n
    if z is not None:
        a.z, a.ldz = z.data_ptr(), n
    a.M, a.N, a.K, a.elem, a.act = m, n, k, _ELEM[x.dtype], act
    if p > 0.0:
        a.seed_ptr, a.salt, a.drop_p = seed.data_ptr(), salt, p
    with _on(x):
        ws = _ws(_lib.load().gwn_linear_fwd_workspace_floats(ctypes.byref(a)), x.device)
        a.workspace = _lib.ptr(ws)
        _lib.call("gwn_linear_fwd", ctypes.byref(a), _lib.stream())
    return y, z


class _LinearActFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, residual, act, p, seed, salt):
        needs = ctx.needs_input_grad[:3]
        y, z = _linear_fwd(x, weight, bias, act, residual, p, seed, salt, any(needs))
        ctx.save_for_backward(x if needs[1] else None, weight if needs[0] else None, z, seed if p > 0.0 else None)
        ctx.shape, ctx.wshape = x.shape, weight.shape
        ctx.act, ctx.p, ctx.salt = act, p, salt
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, weight, z, seed = ctx.saved_tensors
        n, k = ctx.wshape
        dev, dt = dy.device, dy.dtype
        needs = ctx.needs_input_grad
        dres = dy if needs[3] else None
        dx = torch.empty(ctx.shape, device=dev, dtype=dt) if needs[0] else None
        dw = torch.empty(n, k, device=dev, dtype=dt) if needs[1] else None
        db = torch.empty(n, device=dev, dtype=dt) if needs[2] else None
        if not any(needs[:3]):
            return None, None, None, dres, None, None, None, None
        m = dy.numel() // n
        dy2, ld = _rows(dy, n)
        a = _lib.LinearBwdArgs()
        a.dy, a.ld_dy = dy2.data_ptr(), ld
        if x is not None:
            x, a.ldx = _rows(x, k)
            a.x = x.data_ptr()
        if weight is not None:
            weight, a.ldw = _rows(weight, k)
            a.w = weight.data_ptr()
        if z is not None:
            a.z, a.ldz = z.data_ptr(), n
        a.dx, a.ld_dx, a.dw, a.ld_dw, a.dbias = _lib.ptr(dx), k, _lib.ptr(dw), k, _lib.ptr(db)
        a.M, a.N, a.K, a.elem, a.act = m, n, k, _ELEM[dt], ctx.act
        if seed is not None:
            a.seed_ptr, a.salt, a.drop_p = seed.data_ptr(), ctx.salt, ctx.p
        with _on(dy):
            ws = _ws(_lib.load().gwn_linear_bwd_workspace_floats(ctypes.byref(a)), dev)
            a.workspace = _lib.ptr(ws)
            _lib.call("gwn_linear_bwd", ctypes.byref(a), _lib.stream())
        return dx, dw, db, dres, None, None, None, None


def linear_act(x, weight, bias=None, act="none", residual=None, p=0.0, seed=None, salt=0):
    """``residual + dropout(act(x @ weight.T + bias), p)`` in one launch.

    x ``[..., K]``, weight ``[N, K]``, bias ``[N]``, residual ``[..., N]``; ``act`` one of ``none``,
    ``relu``, ``gelu`` (by erf), ``gelu_tanh``, ``silu``; with ``p`` > 0 the mask of (``seed``, ``salt``) as
    in :func:`dropout`.  Differentiable in x, weight, bias and residual."""
    _check("linear_act", x, weight, bias, residual)
    if act not in ACTS:
        raise ValueError("linear_act: act must be one of %s, got %r" % (", ".join(ACTS), act))
    _check_seed("linear_act", x, p, seed, salt)
    if x.dim() < 1 or weight.dim() != 2 or x.shape[-1] != weight.shape[1] or weight.numel() == 0:
        raise RuntimeError("linear_act: x [..., K] and weight [N, K] do not fit: %s, %s"
                           % (tuple(x.shape), tuple(weight.shape)))
    n = weight.shape[0]
    if bias is not None and bias.shape != (n,):
        raise RuntimeError("linear_act: bias must be [%d], got %s" % (n, tuple(bias.shape)))
    if residual is not None and residual.shape != x.shape[:-1] + (n,):
        raise RuntimeError("linear_act: residual must be %s, got %s"
                           % (tuple(x.shape[:-1]) + (n,), tuple(residual.shape)))
    if torch.is_grad_enabled() and (x.requires_grad or weight.requires_grad
                                    or (bias is not None and bias.requires_grad)
                                    or (residual is not None and residual.requires_grad)):
        return _LinearActFn.apply(x, weight, bias, residual, ACTS[act], float(p), seed, salt)
    return _linear_fwd(x, weight, bias, ACTS[act], residual, float(p), seed, salt, False)[0]


# ---- layer norm -----------------------------------------------------------------------------

def _norm_fwd(x, weight, bias, eps, keep):
    c = x.shape[-1]
    y = torch.empty(x.shape, device=x.device, dtype=x.dtype)
    m = x.numel() // c
    stats = torch.empty(2, m, device=x.device, dtype=F32) if keep else None
    if m == 0:
        return y, stats
    x, ldx = _rows(x, c)
    weight = weight.contiguous() if weight is not None else None
    bias = bias.contiguous() if bias is not None else None
    params = weight if weight is not None else bias
    wide = int(params is not None and params.dtype == F32)
    with _on(x):
        mean = stats.data_ptr() if keep else None
        _lib.call("gwn_layernorm_fwd", x.data_ptr(), ldx, m, c, _ELEM[x.dtype], _lib.ptr(weight), _lib.ptr(bias),
                  wide, eps, y.data_ptr(), c, mean, mean + 4 * m if keep else None, _lib.stream())
    return y, stats


class _LayerNormFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps):
        y, stats = _norm_fwd(x, weight, bias, eps, True)
        ctx.save_for_backward(x, weight, stats)
        ctx.bias_dtype = None if bias is None else bias.dtype
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, weight, stats = ctx.saved_tensors
        c = x.shape[-1]
        m = x.numel() // c
        needs = ctx.needs_input_grad
        pt = weight.dtype if weight is not None else ctx.bias_dtype
        dx = torch.empty(x.shape, device=x.device, dtype=x.dtype) if needs[0] else None
        dw = torch.empty(c, device=x.device, dtype=pt) if needs[1] else None
        db = torch.empty(c, device=x.device, dtype=pt) if needs[2] else None
        x2, ldx = _rows(x, c)
        dy2, ldy = _rows(dy, c)
        weight = weight.contiguous() if weight is not None else None
        elem = _ELEM[x.dtype]
        with _on(x):
            ws = None
            if dw is not None or db is not None:
                ws = _ws(_lib.load().gwn_layernorm_bwd_workspace_floats(m, c, elem), x.device)
            mean = stats.data_ptr()
            _lib.call("gwn_layernorm_bwd", dy2.data_ptr(), ldy, x2.data_ptr(), ldx, m, c, elem, _lib.ptr(weight),
                      int(pt == F32), mean, mean + 4 * m, _lib.ptr(dx), c, _lib.ptr(dw), _lib.ptr(db), _lib.ptr(ws),
                      _lib.stream())
        return dx, dw, db, None


def layer_norm(x, weight=None, bias=None, eps=1e-5):
    """``(x - mean) / sqrt(var + eps) * weight + bias`` over the last axis of x ``[..., C]``.

    weight and bias ``[C]`` (either may be None) have x's type, or are both float32.  Differentiable in
    x, weight and bias."""
    _check("layer_norm", x)
    if x.dim() < 1 or x.shape[-1] == 0:
        raise RuntimeError("layer_norm: x must be [..., C] with C > 0, got %s" % (tuple(x.shape),))
    if not eps >= 0.0:
        raise ValueError("layer_norm: eps must not be negative, got %s" % eps)
    params = [t for t in (weight, bias) if t is not None]
    for t in params:
        if t.shape != x.shape[-1:]:
            raise RuntimeError("layer_norm: weight and bias must be [%d], got %s" % (x.shape[-1], tuple(t.shape)))
        if t.device != x.device or t.dtype not in (x.dtype, F32) or t.dtype != params[0].dtype:
            raise RuntimeError("layer_norm: weight and bias must both be %s or both float32, on %s"
                               % (x.dtype, x.device))
    if torch.is_grad_enabled() and (x.requires_grad or any(t.requires_grad for t in params)):
        return _LayerNormFn.apply(x, weight, bias, eps)
    return _norm_fwd(x, weight, bias, eps, False)[0]


# ---- dropout --------------------------------------------------------------------------------

def _drop(x, residual, p, seed, salt):
    y = torch.empty(x.shape, device=x.device, dtype=x.dtype)
    x = x.contiguous()
    residual = residual.contiguous() if residual is not None else None
    with _on(x):
        _lib.call("gwn_dropout", x.data_ptr(), _lib.ptr(residual), y.data_ptr(), y.numel(), _ELEM[x.dtype],
                  seed.data_ptr(), salt, p, _lib.stream())
    return y


class _DropoutFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, p, seed, salt):
        ctx.save_for_backward(seed)
        ctx.p, ctx.salt = p, salt
        return _drop(x, residual, p, seed, salt)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        dx = _drop(dy, None, ctx.p, ctx.saved_tensors[0], ctx.salt) if ctx.needs_input_grad[0] else None
        return dx, (dy if ctx.needs_input_grad[1] else None), None, None, None


def dropout(x, p, seed, salt=0, residual=None):
    """x with a share ``p`` of its elements set to 0 and the others scaled by 1 / (1 - p), plus
    ``residual`` (x's shape) if given.

    Element i, counted in x's logical order, is kept by the mask of (``seed``, ``salt``): the same one in
    every call with these values, whatever the type or strides, and the one that the backward
    rebuilds.  ``include/gwn.h`` (gwn_dropout) defines the generator.  ``p`` = 0 copies, ``p`` = 1 gives
    the residual (or zeros)."""
    _check("dropout", x, residual)
    _check_seed("dropout", x, p, seed, salt)
    if residual is not None and residual.shape != x.shape:
        raise RuntimeError("dropout: residual must be %s, got %s" % (tuple(x.shape), tuple(residual.shape)))
    if p == 0.0:
        return x.clone() if residual is None else x + residual
    if torch.is_grad_enabled() and (x.requires_grad or (residual is not None and residual.requires_grad)):
        return _DropoutFn.apply(x, residual, float(p), seed, salt)
    return _drop(x, residual, float(p), seed, salt)


# ---- modules --------------------------------------------------------------------------------

class LinearAct(nn.Module):
    """:func:`linear_act` with its weight ``[c_out, c_in]`` and bias (initialised as ``nn.Linear``'s); in
    training with dropout ``p`` after the activation."""

    def __init__(self, c_in, c_out, act="none", p=0.0, bias=True, salt=0):
        super().__init__()
        if act not in ACTS:
            raise ValueError("LinearAct: act must be one of %s, got %r" % (", ".join(ACTS), act))
        proto = nn.Linear(c_in, c_out, bias=bias)
        self.weight, self.bias = proto.weight, proto.bias
        self.act, self.p, self.salt = act, p, salt

    def forward(self, x, residual=None, seed=None):
        p = self.p if self.training else 0.0
        return linear_act(x, self.weight, self.bias, self.act, residual, p, seed, self.salt)


class LayerNorm(nn.Module):
    """:func:`layer_norm` over ``c`` channels with its weight (ones) and bias (zeros)."""

    def __init__(self, c, eps=1e-5):
        super().__init__()
        self.weight = nn.Parameter(torch.ones(c))
        self.bias = nn.Parameter(torch.zeros(c))
        self.eps = eps

    def forward(self, x):
        return layer_norm(x, self.weight, self.bias, self.eps)


class Dropout(nn.Module):
    """:func:`dropout` in training; in evaluation x (plus the residual) as it is."""

    def __init__(self, p, salt=0):
        super().__init__()
        self.p, self.salt = p, salt

    def forward(self, x, seed=None, residual=None):
        if self.training and self.p > 0.0:
            return dropout(x, self.p, seed, self.salt, residual)
        return x if residual is None else x + residual


class FeedForward(nn.Module):
    """``x + dropout(W2 dropout(act(W1 norm(x) + b1)) + b2)`` over the channels of ``[..., c]``: the norm and
    two products, three launches forward.  The masks' salts are ``salt`` and ``salt + 1``."""

    def __init__(self, c, hidden, act="gelu", p=0.0, salt=0):
        super().__init__()
        self.norm = LayerNorm(c)
        self.up = LinearAct(c, hidden, act, p, salt=salt)
        self.down = LinearAct(hidden, c, "none", p, salt=salt + 1)

    def forward(self, x, seed=None):
        return self.down(self.up(self.norm(x), seed=seed), residual=x, seed=seed)
