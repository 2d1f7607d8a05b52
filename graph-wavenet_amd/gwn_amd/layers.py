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

Forward and backward may be captured into a graph (with autograd's own rule: while one is captured, no
eager graph that reaches the same leaves may be alive); replays read ``seed`` anew.

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


def _ws(floats, like):
    return like.new_empty(floats, dtype=F32) if floats > 0 else None


# The raw stream handle and the current device without the Python objects around them: building a
# Stream for its handle costs up to 15 us in a step, as much as a small kernel's whole launch.
_raw_stream = torch._C._cuda_getCurrentRawStream
_device = torch._C._cuda_getDevice


def _here(t):
    """Whether t's device is the current one (in autograd's threads it always is)."""
    return t.device.index == _device()


def _elsewhere(fn):
    """``fn`` (its first argument a tensor) on that tensor's device."""
    def run(t, *args):
        if _here(t):
            return fn(t, *args)
        with torch.cuda.device(t.device):
            return fn(t, *args)
    return run


def _backward(impl):
    """A backward that cannot be differentiated again.  The wrapper that makes it say so is only
    needed where the backward itself is recorded (create_graph)."""
    recorded = once_differentiable(impl)
    return staticmethod(lambda ctx, dy: recorded(ctx, dy) if torch.is_grad_enabled() else impl(ctx, dy))


# ---- the product with its epilogue ----------------------------------------------------------

@_elsewhere
def _linear_fwd(x, weight, bias, act, residual, p, seed, salt, keep_z):
    n, k = weight.shape
    y = x.new_empty(x.shape[:-1] + (n,))
    m = y.numel() // n
    z = None
    if keep_z and act:
        z = x.new_empty((m, n), dtype=F32 if x.dtype == F32 else torch.float16)
    if m == 0:
        return y, z
    x, ldx = _rows(x, k)
    weight, ldw = _rows(weight, k)
    bias = bias if bias is None else bias.contiguous()
    residual, ldr = (None, 0) if residual is None else _rows(residual, n)
    ptr = _lib.ptr
    a = _lib.LinearArgs(x.data_ptr(), ldx, weight.data_ptr(), ldw, ptr(bias), ptr(residual), ldr, y.data_ptr(), n, ptr(z), n,
                        m, n, k, _ELEM[x.dtype], act, seed.data_ptr() if p > 0.0 else None, salt, p, None)
    at = ctypes.byref(a)
    ws = _ws(_lib.load().gwn_linear_fwd_workspace_floats(at), x)
    if ws is not None:
        a.workspace = ws.data_ptr()
    _lib.call("gwn_linear_fwd", at, _raw_stream(x.device.index))
    return y, z


def _linear_bwd(ctx, dy):
    x, weight, z, seed = ctx.saved_tensors
    n, k = ctx.wshape
    needs = ctx.needs_input_grad
    dres = dy if needs[3] else None
    if not (needs[0] or needs[1] or needs[2]):
        return None, None, None, dres, None
    dx = dy.new_empty(ctx.shape) if needs[0] else None
    dw = dy.new_empty((n, k)) if needs[1] else None
    db = dy.new_empty(n) if needs[2] else None
    m = dy.numel() // n
    dy, ldy = _rows(dy, n)
    x, ldx = (None, 0) if x is None else _rows(x, k)
    weight, ldw = (None, 0) if weight is None else _rows(weight, k)
    ptr = _lib.ptr
    a = _lib.LinearBwdArgs(dy.data_ptr(), ldy, ptr(x), ldx, ptr(weight), ldw, ptr(z), n, ptr(dx), k, ptr(dw), k, ptr(db), m,
                           n, k, _ELEM[dy.dtype], ctx.act, ptr(seed), ctx.salt, ctx.p, None)
    at = ctypes.byref(a)
    ws = _ws(_lib.load().gwn_linear_bwd_workspace_floats(at), dy)
    a.workspace = ptr(ws)
    _lib.call("gwn_linear_bwd", at, _raw_stream(dy.device.index))
    return dx, dw, db, dres, None


class _LinearActFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, residual, how):
        act, p, seed, salt = how
        needs = ctx.needs_input_grad
        y, z = _linear_fwd(x, weight, bias, act, residual, p, seed, salt, needs[0] or needs[1] or needs[2])
        ctx.save_for_backward(x if needs[1] else None, weight if needs[0] else None, z, seed if p > 0.0 else None)
        ctx.shape, ctx.wshape = x.shape, weight.shape
        ctx.act, ctx.p, ctx.salt = act, p, salt
        return y

    backward = _backward(_linear_bwd)


def linear_act(x, weight, bias=None, act="none", residual=None, p=0.0, seed=None, salt=0):
    """``residual + dropout(act(x @ weight.T + bias), p)`` in one launch.

    x ``[..., K]``, weight ``[N, K]``, bias ``[N]``, residual ``[..., N]``; ``act`` one of ``none``,
    ``relu``, ``gelu`` (by erf), ``gelu_tanh``, ``silu``; with ``p`` > 0 the mask of (``seed``, ``salt``) as
    in :func:`dropout`.  Differentiable in x, weight, bias and residual."""
    _check("linear_act", x, weight, bias, residual)
    if act not in ACTS:
        raise ValueError("linear_act: act must be one of %s, got %r" % (", ".join(ACTS), act))
    if p != 0.0:
        _check_seed("linear_act", x, p, seed, salt)
    if x.dim() < 1 or weight.dim() != 2 or x.shape[-1] != weight.shape[1] or weight.numel() == 0:
        raise RuntimeError("linear_act: x [..., K] and weight [N, K] do not fit: %s, %s"
                           % (tuple(x.shape), tuple(weight.shape)))
    n, k = weight.shape
    if max(n, k) > 2 ** 20 or x.numel() > k * 2 ** 30:
        raise RuntimeError("linear_act: at most 2^30 rows and 2^20 channels, got %s, %s"
                           % (tuple(x.shape), tuple(weight.shape)))
    if bias is not None and bias.shape != (n,):
        raise RuntimeError("linear_act: bias must be [%d], got %s" % (n, tuple(bias.shape)))
    if residual is not None and residual.shape != x.shape[:-1] + (n,):
        raise RuntimeError("linear_act: residual must be %s, got %s"
                           % (tuple(x.shape[:-1]) + (n,), tuple(residual.shape)))
    if torch.is_grad_enabled() and (x.requires_grad or weight.requires_grad
                                    or (bias is not None and bias.requires_grad)
                                    or (residual is not None and residual.requires_grad)):
        return _LinearActFn.apply(x, weight, bias, residual, (ACTS[act], float(p), seed, salt))
    return _linear_fwd(x, weight, bias, ACTS[act], residual, float(p), seed, salt, False)[0]


# ---- layer norm -----------------------------------------------------------------------------

@_elsewhere
def _norm_fwd(x, weight, bias, eps, keep):
    """y, the rows' statistics if they are to be kept, and the backward's workspace floats."""
    c, elem = x.shape[-1], _ELEM[x.dtype]
    y = x.new_empty(x.shape)
    m = x.numel() // c
    stats = x.new_empty((2, m), dtype=F32) if keep else None
    x, ldx = _rows(x, c)
    weight = weight.contiguous() if weight is not None else None
    bias = bias.contiguous() if bias is not None else None
    params = weight if weight is not None else bias
    wide = int(params is not None and params.dtype == F32)
    mean = stats.data_ptr() if keep else None
    if m:
        _lib.call("gwn_layernorm_fwd", x.data_ptr(), ldx, m, c, elem, _lib.ptr(weight), _lib.ptr(bias), wide, eps,
                  y.data_ptr(), c, mean, mean + 4 * m if keep else None, _raw_stream(x.device.index))
    floats = _lib.load().gwn_layernorm_bwd_workspace_floats(m, c, elem) if keep else 0
    return y, stats, floats


def _norm_bwd(ctx, dy):
    # the thread that runs this starts cold: what the forward can prepare is in ctx.plan
    x, weight, stats = ctx.saved_tensors
    m, c, elem, params, floats = ctx.plan
    needs = ctx.needs_input_grad
    dx = x.new_empty(x.shape) if needs[0] else None
    dw = x.new_empty(c, dtype=params) if needs[1] else None
    db = x.new_empty(c, dtype=params) if needs[2] else None
    ws = x.new_empty(floats, dtype=F32) if needs[1] or needs[2] else None
    x, ldx = _rows(x, c)
    dy, ldy = _rows(dy, c)
    weight = weight.contiguous() if weight is not None else None
    mean, ptr = stats.data_ptr(), _lib.ptr
    _lib.call("gwn_layernorm_bwd", dy.data_ptr(), ldy, x.data_ptr(), ldx, m, c, elem, ptr(weight), int(params == F32), mean,
              mean + 4 * m, ptr(dx), c, ptr(dw), ptr(db), ptr(ws), _raw_stream(x.device.index))
    return dx, dw, db, None


class _LayerNormFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps):
        y, stats, floats = _norm_fwd(x, weight, bias, eps, True)
        ctx.save_for_backward(x, weight, stats)
        params = weight if weight is not None else bias
        ctx.plan = stats.shape[1], x.shape[-1], _ELEM[x.dtype], None if params is None else params.dtype, floats
        return y

    backward = _backward(_norm_bwd)


def layer_norm(x, weight=None, bias=None, eps=1e-5):
    """``(x - mean) / sqrt(var + eps) * weight + bias`` over the last axis of x ``[..., C]``.

    weight and bias ``[C]`` (either may be None) have x's type, or are both float32.  Differentiable in
    x, weight and bias."""
    _check("layer_norm", x)
    if x.dim() < 1 or not 0 < x.shape[-1] <= 2 ** 30:
        raise RuntimeError("layer_norm: x must be [..., C] with 0 < C <= 2^30, got %s" % (tuple(x.shape),))
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
    y = x.new_empty(x.shape)
    x = x.contiguous()
    residual = residual.contiguous() if residual is not None else None
    _lib.call("gwn_dropout", x.data_ptr(), _lib.ptr(residual), y.data_ptr(), y.numel(), _ELEM[x.dtype], seed.data_ptr(),
              salt, p, _raw_stream(x.device.index))
    return y


_drop_fwd = _elsewhere(_drop)


def _drop_bwd(ctx, dy):
    needs = ctx.needs_input_grad
    dx = _drop(dy, None, ctx.p, ctx.saved_tensors[0], ctx.salt) if needs[0] else None
    return dx, (dy if needs[1] else None), None


class _DropoutFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, how):
        p, seed, salt = how
        ctx.save_for_backward(seed)
        ctx.p, ctx.salt = p, salt
        return _drop_fwd(x, residual, p, seed, salt)

    backward = _backward(_drop_bwd)


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
        return _DropoutFn.apply(x, residual, (float(p), seed, salt))
    return _drop_fwd(x, residual, float(p), seed, salt)


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
