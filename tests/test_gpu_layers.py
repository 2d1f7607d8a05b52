"""Position-wise layers (``gwn_amd.layers``) on the HIP path: the product with its epilogue, layer norm
and dropout, forward and backward, against their formulas in 64 bits.

Tolerances are error bounds, element by element.  With u = half a step of the element type, e = 2^-24
half a step of fp32:
  * a sum of n fp32 terms t_i, in any order, is off by at most n e sum|t_i|; products of 16-bit
    values are exact in fp32, products of fp32 values cost another e each;
  * an activation's slope is at most 1.13, its second derivative at most 0.85 (gelu: 0.80, silu: 0.5,
    gelu_tanh: 0.80), and it is evaluated to within ACT = 2e-6 of max(1, |z|);
  * the pre-activation kept for the backward is rounded to f16 (16-bit elements; 2^-11 |z|);
  * dz and every result are rounded once to the element type, u times their size, or to its smallest
    step where they are that small.
"""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
F64 = torch.float64
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
E32 = 2.0 ** -24
ACT = 2e-6
TINY = {"f32": 2.0 ** -126, "f16": 2.0 ** -24, "bf16": 2.0 ** -126}


def half_step(t):
    return torch.finfo(TYPES[t]).eps / 2


# ---- oracles --------------------------------------------------------------------------------

def mask(seed, salt, shape, p, first=0):
    """Kept elements first .. first + prod(shape) of the mask of (seed, salt)."""
    full = (1 << 64) - 1

    def mix(v):
        v = ((v ^ (v >> 30)) * 0xBF58476D1CE4E5B9) & full
        v = ((v ^ (v >> 27)) * 0x94D049BB133111EB) & full
        return v ^ (v >> 31)

    base = mix((seed + 0x9E3779B97F4A7C15 * (salt + 1)) & full)
    i = np.arange(first, first + int(np.prod(shape)), dtype=np.uint64)
    out = np.empty(len(i), dtype=bool)
    for high in np.unique(i >> np.uint64(32)):
        at = (i >> np.uint64(32)) == high
        k = mix((base + int(high)) & full)
        h = (i[at] & np.uint64(0xFFFFFFFF)).astype(np.uint32)
        h = h * np.uint32(0x9E3779B1) + np.uint32(k & 0xFFFFFFFF)
        h ^= h >> np.uint32(16)
        h *= np.uint32(0x7FEB352D)
        h ^= h >> np.uint32(15)
        h += np.uint32(k >> 32)
        h *= np.uint32(0x846CA68B)
        h ^= h >> np.uint32(16)
        out[at] = (h >> np.uint32(8)) >= math.ceil(p * 2 ** 24)
    return torch.from_numpy(out.reshape(shape))


def act64(z, act):
    if act == "relu":
        return torch.where(z > 0, z, torch.zeros_like(z)), (z > 0).to(F64)
    if act == "gelu":
        phi = 0.5 * torch.special.erfc(-z / math.sqrt(2))
        return z * phi, phi + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    if act == "gelu_tanh":
        a = 2 * math.sqrt(2 / math.pi)
        s = torch.special.expit(a * (z + 0.044715 * z ** 3))
        return z * s, s + z * s * (1 - s) * a * (1 + 3 * 0.044715 * z * z)
    if act == "silu":
        s = torch.special.expit(z)
        return z * s, s * (1 + z * (1 - s))
    return z, torch.ones_like(z)


def on_grid(t, step):
    return torch.round(t / step) * step


class LinearCase:
    """Inputs on the host, the formula's results in 64 bits and each result's bound."""

    def __init__(self, m, k, n, t, act, bias, residual, p, seed=3):
        g = torch.Generator().manual_seed(seed * 1000003 + m * 31 + k * 7 + n)
        self.m, self.k, self.n, self.t, self.act, self.p = m, k, n, t, act, p
        self.seed, self.salt = 0x123456789ABCDEF + seed, 7
        dt = TYPES[t]
        x = torch.randn(m, k, generator=g)
        w = torch.randn(n, k, generator=g) * k ** -0.5
        b = torch.randn(n, generator=g) * 0.3
        if act == "relu":  # exact sums: no pre-activation lies on the other side of the border
            step = 2.0 ** (-6 - math.ceil(math.log2(k) / 2))
            x, w, b = on_grid(x, 2.0 ** -6), on_grid(w, step), on_grid(b, step / 2)
        self.x, self.w = x.to(dt), w.to(dt)
        self.b = b.to(dt) if bias else None
        self.r = torch.randn(m, n, generator=g).to(dt) if residual else None
        self.dy = torch.randn(m, n, generator=g).to(dt)
        self._solve()

    def _solve(self):
        x, w, dy = self.x.to(F64), self.w.to(F64), self.dy.to(F64)
        u, tiny = half_step(self.t), TINY[self.t]
        z = x @ w.T
        size = x.abs() @ w.abs().T
        if self.b is not None:
            z = z + self.b.to(F64)
            size = size + self.b.to(F64).abs()
        ez = (self.k + 2) * E32 * size
        a, slope = act64(z, self.act)
        keep = (mask(self.seed, self.salt, (self.m, self.n), self.p).to(F64) / (1 - self.p) if 0 < self.p < 1
                else torch.full((self.m, self.n), float(self.p == 0), dtype=F64))
        y = a * keep
        ea = 1.13 * ez
        if self.act not in ("none", "relu"):
            ea = ea + ACT * z.abs().clamp(min=1)
        ey = (ea + 3 * E32 * a.abs()) * keep
        if self.r is not None:
            y = y + self.r.to(F64)
            ey = ey + E32 * y.abs()
        self.y, self.ey = y, ey + u * y.abs() * (1 + 2.0 ** -8) + tiny
        # backward
        dyk = dy * keep
        dz = dyk * slope
        ezs = ez + (2.0 ** -11 * z.abs() + 2.0 ** -25 if self.t != "f32" else E32 * z.abs())
        es = 0.0 if self.act in ("none", "relu") else 0.85 * ezs + ACT * z.abs().clamp(min=1)
        edz32 = dyk.abs() * es + 3 * E32 * dz.abs()
        edz = edz32 + (u * dz.abs() + tiny if self.act != "none" or self.p > 0 else 0)
        adz = dz.abs() + edz

        def product(e, a, b, be, count):
            return e @ b.abs() + count * E32 * (a @ b.abs()) + be

        self.dx = dz @ w
        self.edx = product(edz, adz, w, 0, self.n + 2) + u * self.dx.abs() * (1 + 2.0 ** -8) + tiny
        self.dw = dz.T @ x
        self.edw = product(edz.T, adz.T, x, 0, self.m + 2) + u * self.dw.abs() * (1 + 2.0 ** -8) + tiny
        self.db = dz.sum(0)
        self.edb = edz32.sum(0) + (self.m + 2) * E32 * adz.sum(0) + u * self.db.abs() * (1 + 2.0 ** -8) + tiny

    def on(self, dev):
        """The leaves (x, w, b, r), dy and the seed on the device."""
        leaves = [None if t is None else t.to(dev).requires_grad_() for t in (self.x, self.w, self.b, self.r)]
        return leaves, self.dy.to(dev), torch.tensor([self.seed], device=dev)

    def check(self, y=None, dx=None, dw=None, db=None, dr=None):
        for name, got, want, err in (("y", y, self.y, self.ey), ("dx", dx, self.dx, self.edx),
                                     ("dw", dw, self.dw, self.edw), ("db", db, self.db, self.edb)):
            if got is not None:
                within(name, got, want, err)
        if dr is not None:
            assert torch.equal(dr.cpu(), self.dy)


def within(name, got, want, err):
    got = got.detach().cpu().to(F64).reshape(want.shape)
    off = (got - want).abs()
    bad = ~(off <= err)
    assert not bad.any(), "%s: %d of %d outside, worst %.3g times the bound at %s: %g, not %g" % (
        name, int(bad.sum()), bad.numel(), float((off / err).nan_to_num(math.inf).max()),
        tuple(int(v) for v in bad.nonzero()[0]), float(got[bad][0]), float(want[bad][0]))


def run_linear(c, dev):
    from gwn_amd.layers import linear_act
    (x, w, b, r), dy, seed = c.on(dev)
    y = linear_act(x, w, b, act=c.act, residual=r, p=c.p, seed=seed, salt=c.salt)
    leaves = [t for t in (x, w, b, r) if t is not None]
    got = dict(zip([q for q, t in (("dx", x), ("dw", w), ("db", b), ("dr", r)) if t is not None],
                   torch.autograd.grad(y, leaves, dy)))
    torch.cuda.synchronize()
    return y, got


# ---- the product with its epilogue ------------------------------------------------------------

LINEAR_SIZES = [(1, 1, 1), (1, 64, 64), (1, 1000, 257), (2, 4097, 33), (3, 7, 5), (5, 129, 2050), (12, 1999, 103),
                (17, 8, 16), (33, 130, 65), (64, 256, 128), (65, 64, 512), (100, 31, 300), (128, 72, 8), (257, 300, 129),
                (300, 520, 40), (511, 96, 272), (1030, 48, 31), (2100, 224, 32), (5000, 33, 12)]


@pytest.mark.parametrize("t", sorted(TYPES))
@pytest.mark.parametrize("i", range(len(LINEAR_SIZES)), ids=["%dx%dx%d" % s for s in LINEAR_SIZES])
def test_linear_act_sizes(gpu, i, t):
    """Every output and gradient at every size, the epilogue's parts in turn."""
    act = ("none", "gelu", "relu", "silu", "gelu_tanh")[i % 5]
    c = LinearCase(*LINEAR_SIZES[i], t, act, bias=i % 3 != 0, residual=i % 2 == 0, p=(0.0, 0.3, 0.1)[i % 3])
    y, got = run_linear(c, gpu)
    c.check(y=y, **got)


@pytest.mark.parametrize("t", sorted(TYPES))
@pytest.mark.parametrize("act", ["none", "relu", "gelu", "gelu_tanh", "silu"])
@pytest.mark.parametrize("p", [0.0, 0.5, 1.0])
@pytest.mark.parametrize("bias,residual", [(False, False), (True, True)])
def test_linear_act_epilogues(gpu, t, act, p, bias, residual):
    c = LinearCase(70, 40, 72, t, act, bias, residual, p)
    y, got = run_linear(c, gpu)
    c.check(y=y, **got)


@pytest.mark.parametrize("t", sorted(TYPES))
@pytest.mark.parametrize("m,k,n", [(3000, 1024, 768), (520, 640, 1100)])
def test_linear_act_larger(gpu, t, m, k, n):
    c = LinearCase(m, k, n, t, "gelu", True, True, 0.1)
    y, got = run_linear(c, gpu)
    c.check(y=y, **got)


@pytest.mark.parametrize("t", sorted(TYPES))
@pytest.mark.parametrize("m,k,n", [(9000, 64, 96), (9000, 65, 63), (20000, 24, 40), (12000, 32, 224), (1300, 64, 600),
                                   (200, 31, 33), (64, 300, 200), (33, 200, 520), (12000, 1, 1)])
def test_linear_act_short_contractions(gpu, t, m, k, n):
    """Contractions of one step of the tiles (64 values, 32 in f32), just under and just over it, each
    tile's width, forward and both gradients."""
    c = LinearCase(m, k, n, t, "silu", True, True, 0.1)
    y, got = run_linear(c, gpu)
    c.check(y=y, **got)


@pytest.mark.parametrize("t", sorted(TYPES))
def test_linear_act_strides_and_offsets(gpu, t):
    """x as a column slice that starts off a 16-byte border, a transposed weight, x with swapped
    leading axes, an expanded output gradient."""
    from gwn_amd.layers import linear_act
    c = LinearCase(66, 72, 40, t, "silu", True, True, 0.0)
    wide = torch.zeros(66, 85, dtype=TYPES[t], device=gpu)
    wide[:, 3:75] = c.x.to(gpu)
    x = wide[:, 3:75].detach().requires_grad_()
    w = c.w.to(gpu).t().contiguous().t().requires_grad_()
    r = torch.zeros(66, 41, dtype=TYPES[t], device=gpu)
    r[:, 1:] = c.r.to(gpu)
    y = linear_act(x, w, c.b.to(gpu), act="silu", residual=r[:, 1:])
    c.check(y=y, **dict(zip(("dx", "dw"), torch.autograd.grad(y, (x, w), c.dy.to(gpu)))))
    x3 = c.x.to(gpu).view(6, 11, 72).transpose(0, 1)  # [11, 6, 72], rows not in order
    y3 = linear_act(x3, w, c.b.to(gpu), act="silu", residual=c.r.to(gpu).view(6, 11, 40).transpose(0, 1))
    assert y3.shape == (11, 6, 40)
    c.check(y=y3.transpose(0, 1).reshape(66, 40))
    c.dy = torch.ones_like(c.dy)
    c._solve()
    x = c.x.to(gpu).requires_grad_()
    linear_act(x, w, c.b.to(gpu), act="silu", residual=c.r.to(gpu)).sum().backward()
    c.check(dx=x.grad)


def test_linear_act_each_gradient_alone(gpu):
    from gwn_amd.layers import linear_act
    c = LinearCase(90, 50, 60, "f32", "gelu", True, True, 0.3)
    (x, w, b, r), dy, seed = c.on(gpu)
    for name, want in (("x", "dx"), ("w", "dw"), ("b", "db"), ("r", "dr")):
        t = dict(x=x.detach(), w=w.detach(), b=b.detach(), r=r.detach())
        t[name].requires_grad_()
        y = linear_act(t["x"], t["w"], t["b"], act="gelu", residual=t["r"], p=0.3, seed=seed, salt=c.salt)
        y.backward(dy)
        c.check(y=y, **{want: t[name].grad})


@pytest.mark.parametrize("t", sorted(TYPES))
def test_linear_act_no_rows(gpu, t):
    from gwn_amd.layers import linear_act
    x = torch.zeros(0, 5, 24, dtype=TYPES[t], device=gpu, requires_grad=True)
    w = torch.randn(40, 24, device=gpu).to(TYPES[t]).requires_grad_()
    b = torch.randn(40, device=gpu).to(TYPES[t]).requires_grad_()
    y = linear_act(x, w, b, act="gelu")
    assert y.shape == (0, 5, 40)
    y.sum().backward()
    assert x.grad.shape == x.shape and not w.grad.any() and not b.grad.any()


@pytest.mark.parametrize("t", sorted(TYPES))
def test_linear_act_infinities(gpu, t):
    """A NaN or infinity in one row stays in that row; where dropout drops it, it is gone; a
    pre-activation past the type's range has its limits as value and slope."""
    from gwn_amd.layers import linear_act
    dt = TYPES[t]
    x = torch.randn(40, 64, device=gpu).to(dt)
    w = (torch.rand(96, 64, device=gpu) + 0.5).to(dt)
    clean = linear_act(x, w, act="gelu")
    for v in (math.nan, math.inf):
        bad = x.clone()
        bad[7, 3] = v
        y = linear_act(bad, w, act="gelu")
        assert not torch.isfinite(y[7]).any()
        keep = torch.arange(40, device=gpu) != 7
        assert torch.equal(y[keep], clean[keep])
        seed = torch.tensor([11], device=gpu)
        y = linear_act(bad, w, act="gelu", p=0.5, seed=seed)
        kept = mask(11, 0, (40, 96), 0.5).to(gpu)
        assert (y[~kept] == 0).all() and not torch.isfinite(y[7][kept[7]]).any()
    big = torch.full((2, 64), 2000.0, device=gpu, dtype=dt)
    big[1] = -2000.0
    for act in ("relu", "gelu", "gelu_tanh", "silu"):
        b = big.clone().requires_grad_()
        y = linear_act(b, w, act=act)
        dx, = torch.autograd.grad(y, b, torch.ones_like(y) / 64)
        assert (y[1] == 0).all() and (dx[1] == 0).all()
        assert torch.isfinite(dx).all() and (dx[0] > 0).all()


def test_relu_slope_of_tiny_values(gpu):
    """A positive pre-activation below f16's smallest step has slope 1, zero and a negative one 0."""
    from gwn_amd.layers import linear_act
    x = torch.tensor([[2.0 ** -14], [-2.0 ** -14], [0.0]], device=gpu, dtype=torch.float16, requires_grad=True)
    w = torch.full((8, 1), 2.0 ** -14, device=gpu, dtype=torch.float16)  # z = +-2^-28, 0
    b = torch.zeros(8, device=gpu, dtype=torch.float16, requires_grad=True)
    y = linear_act(x, w, b, act="relu")
    db, = torch.autograd.grad(y, b, torch.tensor([[1.0], [10.0], [100.0]], device=gpu).half().expand(3, 8).contiguous())
    assert (db == 1.0).all()


@pytest.mark.parametrize("act", ["none", "gelu", "gelu_tanh", "silu"])
def test_linear_act_gradients_against_differences(gpu, act):
    """Along a direction d, (f(+h) - f(-h)) / 2h of f = sum(y dy): off by h^2 / 6 times the third derivative
    (|act'''| <= 2, 1 / 0.7 from the mask), by the two outputs' bounds over 2h (1.5 times theirs at h = 0:
    the sizes at +-h), and by the fp32 inputs' own steps."""
    from gwn_amd.layers import linear_act
    c = LinearCase(24, 40, 28, "f32", act, True, True, 0.3)
    (x, w, b, r), dy, seed = c.on(gpu)
    y, got = run_linear(c, gpu)
    h = 2.0 ** -6

    def f(x, w, b, r):
        with torch.no_grad():
            return (linear_act(x, w, b, act=act, residual=r, p=0.3, seed=seed, salt=c.salt).double() * dy.double()).sum()

    rounding = 1.5 * float((c.ey * c.dy.to(F64).abs()).sum()) / h
    for k, name in enumerate(("dx", "dw", "db", "dr")):
        leaves = [t.detach() for t in (x, w, b, r)]
        g = torch.Generator(device=gpu).manual_seed(k)
        d = torch.randn(leaves[k].shape, device=gpu, generator=g)
        up, down = list(leaves), list(leaves)
        up[k], down[k] = leaves[k] + h * d, leaves[k] - h * d
        step = (up[k].double() - down[k].double()) / (2 * h)  # the direction as the fp32 inputs have it
        slope = float(f(*up) - f(*down)) / (2 * h)
        want = float((got[name].double() * step).sum())
        at = step.cpu().double()
        dzd = {"dx": lambda: at @ c.w.double().T, "dw": lambda: c.x.double() @ at.T,
               "db": lambda: at.expand(24, 28), "dr": lambda: torch.zeros(24, 28, dtype=F64)}[name]()
        third = float((dzd.abs() ** 3 * c.dy.double().abs()).sum()) * 2 / 0.7 * h * h / 6
        inexact = 2 * E32 * float((step.abs() * got[name].abs().double()).sum()) / h
        assert abs(slope - want) <= rounding + third + inexact, name


# ---- layer norm -------------------------------------------------------------------------------

def norm_inputs(m, c, t, wide, seed=1):
    g = torch.Generator().manual_seed(seed * 7919 + m * 13 + c)
    dt = TYPES[t]
    wt = torch.float32 if wide else dt
    x = (torch.randn(m, c, generator=g) * (0.5 + torch.rand(m, 1, generator=g)) + torch.randn(m, 1, generator=g)).to(dt)
    return (x, (1 + 0.2 * torch.randn(c, generator=g)).to(wt), (0.2 * torch.randn(c, generator=g)).to(wt),
            torch.randn(m, c, generator=g).to(dt))


def norm_check(t, x, w, b, dy, eps, y=None, dx=None, dw=None, db=None):
    """Bounds: a row's mean is a sum of c fp32 terms in chains of at most `chain` additions, so it is
    off by chain e mean|x|; rstd by (2 chain + 8) e relatively beside the mean's part; everything
    after is a handful of roundings."""
    wt = t if w is None or w.dtype == TYPES[t] else "f32"
    x, dy = x.to(F64), dy.to(F64)
    m, c = x.shape
    w_ = torch.ones(c, dtype=F64) if w is None else w.to(F64)
    b_ = torch.zeros(c, dtype=F64) if b is None else b.to(F64)
    u, tiny = half_step(t), TINY[t]
    chain = 8 * max(8, math.ceil(c / 2048)) + 16
    mean = x.mean(1, keepdim=True)
    var = ((x - mean) ** 2).mean(1, keepdim=True)
    rs = (var + eps) ** -0.5
    xh = (x - mean) * rs
    emean = chain * E32 * x.abs().mean(1, keepdim=True) + 2 * E32 * mean.abs()
    ed = emean + E32 * (x - mean).abs()
    # var: each centred value off by ed
    evar = 2 * ((x - mean).abs() * ed).mean(1, keepdim=True) + (ed ** 2).mean(1, keepdim=True) + chain * E32 * var
    ers = 0.5 * evar / (var + eps) * 1.1 + 4 * E32  # relative
    exh = ed * rs + xh.abs() * (ers + 2 * E32)
    if y is not None:
        want = xh * w_ + b_
        within("y", y, want, exh * w_.abs() + 3 * E32 * (xh * w_).abs() + 2 * E32 * want.abs()
               + u * want.abs() * (1 + 2.0 ** -8) + tiny)
    h = dy * w_
    eh = E32 * h.abs()
    s1, s2 = h.mean(1, keepdim=True), (h * xh).mean(1, keepdim=True)
    es1 = eh.mean(1, keepdim=True) + chain * E32 * h.abs().mean(1, keepdim=True)
    es2 = (eh * xh.abs() + h.abs() * exh).mean(1, keepdim=True) + (chain + 2) * E32 * (h * xh).abs().mean(1, keepdim=True)
    inner = h - s1 - xh * s2
    if dx is not None:
        want = rs * inner
        e = rs * (eh + es1 + exh * s2.abs() + xh.abs() * es2 + 4 * E32 * (h.abs() + s1.abs() + (xh * s2).abs()))
        within("dx", dx, want, e + want.abs() * (ers + 2 * E32) + u * want.abs() * (1 + 2.0 ** -8) + tiny)
    uw, tw = half_step(wt), TINY[wt]
    if dw is not None:
        want = (dy * xh).sum(0)
        e = (dy.abs() * exh).sum(0) + (m + 2) * E32 * (dy * xh).abs().sum(0)
        within("dw", dw, want, e + uw * want.abs() * (1 + 2.0 ** -8) + tw)
    if db is not None:
        want = dy.sum(0)
        within("db", db, want, (m + 2) * E32 * dy.abs().sum(0) + uw * want.abs() * (1 + 2.0 ** -8) + tw)


NORM_SIZES = [(1, 1), (1, 8), (3, 2), (5, 7), (130, 9), (1000, 16), (700, 32), (257, 33), (300, 64), (64, 100), (90, 128),
              (40, 207), (33, 256), (70, 511), (12, 512), (21, 513), (50, 1024), (31, 1111), (9, 2048), (17, 2049),
              (5, 4096), (7, 5000), (3, 8192), (4, 9001), (2, 16384), (3, 20001), (1100, 2500)]


@pytest.mark.parametrize("t,wide", [("f32", False), ("f16", False), ("bf16", False), ("f16", True), ("bf16", True)])
@pytest.mark.parametrize("m,c", NORM_SIZES)
def test_layer_norm_sizes(gpu, m, c, t, wide):
    from gwn_amd.layers import layer_norm
    x, w, b, dy = norm_inputs(m, c, t, wide)
    xd, wd, bd = (v.to(gpu).requires_grad_() for v in (x, w, b))
    y = layer_norm(xd, wd, bd)
    dx, dw, db = torch.autograd.grad(y, (xd, wd, bd), dy.to(gpu))
    torch.cuda.synchronize()
    norm_check(t, x, w, b, dy, 1e-5, y, dx, dw, db)


@pytest.mark.parametrize("t", sorted(TYPES))
@pytest.mark.parametrize("c", [32, 100, 700, 4100, 20000])
def test_layer_norm_parts(gpu, c, t):
    """Without weight or bias, single gradients, strided rows off a 16-byte border, 4-D inputs."""
    from gwn_amd.layers import layer_norm
    x, w, b, dy = norm_inputs(24, c, t, False)
    wide = torch.zeros(24, c + 9, dtype=TYPES[t], device=gpu)
    wide[:, 3:c + 3] = x.to(gpu)
    xs = wide[:, 3:c + 3]
    for has_w, has_b in ((False, False), (True, False), (False, True)):
        wd = w.to(gpu).requires_grad_() if has_w else None
        bd = b.to(gpu).requires_grad_() if has_b else None
        xd = xs.detach().requires_grad_()
        y = layer_norm(xd, wd, bd, eps=1e-3)
        leaves = [v for v in (xd, wd, bd) if v is not None]
        got = dict(zip(["dx"] + ["dw"] * has_w + ["db"] * has_b, torch.autograd.grad(y, leaves, dy.to(gpu))))
        norm_check(t, x, w if has_w else None, b if has_b else None, dy, 1e-3, y, **got)
    wd, bd = w.to(gpu).requires_grad_(), b.to(gpu).requires_grad_()
    y = layer_norm(xs, wd, bd)
    norm_check(t, x, w, b, dy, 1e-5, y, None, *torch.autograd.grad(y, (wd, bd), dy.to(gpu)))
    x4 = x.to(gpu).view(2, 3, 4, c).permute(2, 0, 1, 3)
    assert torch.equal(layer_norm(x4, wd, bd), y.view(2, 3, 4, c).permute(2, 0, 1, 3))
    norm_check(t, x, w, b, torch.ones_like(dy), 1e-5, None, None,
               *torch.autograd.grad(layer_norm(xs, wd, bd).sum(), (wd, bd)))


@pytest.mark.parametrize("c", [32, 600, 20000])
def test_layer_norm_rows_stand_alone(gpu, c):
    """Constant rows give the bias; a NaN row and a row of infinities leave the others as they are; no
    rows give zero gradients."""
    from gwn_amd.layers import layer_norm
    x, w, b, dy = norm_inputs(9, c, "f32", False)
    w, b = w.to(gpu).requires_grad_(), b.to(gpu).requires_grad_()
    x = x.to(gpu)
    x[2] = 3.25
    y = layer_norm(x, w, b)
    assert torch.equal(y[2], b)
    x[4, 5], x[6, 1] = math.nan, math.inf
    y2 = layer_norm(x, w, b)
    assert torch.isnan(y2[4]).all() and torch.isnan(y2[6]).all()
    keep = [0, 1, 2, 3, 5, 7, 8]
    assert torch.equal(y2[keep], y[keep])
    y = layer_norm(torch.zeros(0, c, device=gpu), w, b)
    y.sum().backward()
    assert y.shape == (0, c) and not w.grad.any() and not b.grad.any()


@pytest.mark.parametrize("c", [5, 48])
def test_layer_norm_gradients_against_differences(gpu, c):
    """Central differences of the 64-bit formula (h = 2^-10, off by h^2 / 6 of the third derivative
    along a unit direction, which rstd <= 4 and |xh| <= sqrt(c) keep below 1e3 |dy|) against the
    kernel's gradients of the same fp32 inputs."""
    from gwn_amd.layers import layer_norm
    x, w, b, dy = norm_inputs(6, c, "f32", False)
    leaves = [v.to(gpu).requires_grad_() for v in (x, w, b)]
    got = torch.autograd.grad(layer_norm(*leaves), leaves, dy.to(gpu))
    h = 2.0 ** -10

    def f(x, w, b):
        mu = x.mean(1, keepdim=True)
        return (((x - mu) / (((x - mu) ** 2).mean(1, keepdim=True) + 1e-5).sqrt() * w + b) * dy.double()).sum()

    for k in range(3):
        at = [v.double() for v in (x, w, b)]
        d = torch.randn(at[k].shape, dtype=F64, generator=torch.Generator().manual_seed(k))
        d /= d.norm()
        up, down = list(at), list(at)
        up[k], down[k] = at[k] + h * d, at[k] - h * d
        slope = float(f(*up) - f(*down)) / (2 * h)
        want = float((got[k].cpu().double() * d).sum())
        assert abs(slope - want) <= 1e3 * h * h / 6 * float(dy.abs().sum()) + 1e-5 * float(got[k].abs().sum())


# ---- dropout ----------------------------------------------------------------------------------

@pytest.mark.parametrize("t", sorted(TYPES))
@pytest.mark.parametrize("shape", [(1,), (7,), (8,), (3, 5, 11), (1000, 33), (512, 1024)])
@pytest.mark.parametrize("p", [0.0, 2.0 ** -24, 0.1, 0.5, 0.999, 1.0])
def test_dropout_mask_and_values(gpu, shape, t, p):
    from gwn_amd.layers import dropout
    g = torch.Generator().manual_seed(5)
    x = (torch.rand(shape, generator=g) + 0.5).to(TYPES[t])
    r = torch.randn(shape, generator=g).to(TYPES[t])
    seed = torch.tensor([987654321987], device=gpu)
    keep = mask(987654321987, 3, shape, p)
    scale = np.float32(1.0 / (1.0 - p)) if p < 1 else np.float32(0)
    want = torch.where(keep, x.float() * float(scale), torch.zeros(()))  # one fp32 product, rounded once
    xd, rd = x.to(gpu).requires_grad_(), r.to(gpu).requires_grad_()
    y = dropout(xd, p, seed, salt=3)
    assert torch.equal(y.cpu(), want.to(TYPES[t]))
    y.backward(xd.detach())
    assert torch.equal(xd.grad, y)
    y = dropout(xd, p, seed, salt=3, residual=rd)
    assert torch.equal(y.cpu(), (want + r.float()).to(TYPES[t]))
    dx, dr = torch.autograd.grad(y, (xd, rd), r.to(gpu))
    assert torch.equal(dx.cpu(), torch.where(keep, r.float() * float(scale), torch.zeros(())).to(TYPES[t]))
    assert torch.equal(dr.cpu(), r)


def test_dropout_drops_infinities_and_takes_strides(gpu):
    from gwn_amd.layers import dropout
    seed = torch.tensor([-5], device=gpu)
    x = torch.full((64, 64), math.nan, device=gpu)
    keep = mask(-5, 0, (64, 64), 0.4).to(gpu)
    y = dropout(x, 0.4, seed)
    assert (y[~keep] == 0).all() and torch.isnan(y[keep]).all()
    x = torch.randn(64, 130, device=gpu).t()[1:65]  # columns of a transposed matrix
    y = dropout(x, 0.4, seed)
    assert torch.equal(y != 0, keep[:64, :64].new_tensor(mask(-5, 0, (64, 64), 0.4).numpy()))
    off = torch.randn(64 * 64 + 1, device=gpu)[1:].view(64, 64)  # off a 16-byte border
    assert torch.equal(dropout(off, 0.4, seed), dropout(off.clone(), 0.4, seed))


def test_dropout_is_random(gpu):
    """Keep rate, and no dependence between neighbours, seeds, salts and shifted streams: each share
    within 5 standard deviations of independent draws."""
    from gwn_amd.layers import dropout
    n = 1 << 22
    one = torch.ones(n, device=gpu)

    def draw(seed, salt, p=0.5):
        return (dropout(one, p, torch.tensor([seed], device=gpu), salt=salt) != 0).float()

    sd = 0.5 / math.sqrt(n)
    a = draw(1, 0)
    for p in (0.1, 0.5, 0.9):
        assert abs(float(draw(1, 0, p).mean()) - (1 - p)) <= 5 * math.sqrt(p * (1 - p) / n)
    for b in (draw(2, 0), draw(1, 1), draw(1 << 32, 0), draw(-1, 0), draw(1, 2 ** 63)):
        assert abs(float((a == b).float().mean()) - 0.5) <= 5 * sd
    for k in (1, 2, 3, 8, 31, 32, 64, 207, 4096, 65536):
        assert abs(float((a[k:] == a[:-k]).float().mean()) - 0.5) <= 5 * 0.5 / math.sqrt(n - k)
    rows = a.view(2048, 2048)
    assert float((rows.mean(0) - 0.5).abs().max()) <= 6 * 0.5 / math.sqrt(2048)
    assert float((rows.mean(1) - 0.5).abs().max()) <= 6 * 0.5 / math.sqrt(2048)


def test_dropout_past_32_bits(gpu):
    """Elements on both sides of position 2^32 follow the 64-bit counter."""
    from gwn_amd.layers import dropout
    n = 2 ** 32 + 4104
    x = torch.ones(n, device=gpu, dtype=torch.bfloat16)
    y = dropout(x, 0.5, torch.tensor([77], device=gpu), salt=1)
    del x
    for first in (0, 2 ** 31 - 512, 2 ** 32 - 4096, n - 4100):
        got = y[first:first + 4100].cpu() != 0
        assert torch.equal(got, mask(77, 1, (4100,), 0.5, first)), first


def test_rows_past_32_bits(gpu):
    """Rows more than 2^31 elements apart, for the product and the norm."""
    from gwn_amd.layers import layer_norm, linear_act
    big = torch.empty(2 * 2 ** 31 + 256, device=gpu, dtype=torch.bfloat16)
    far = big.as_strided((3, 256), (2 ** 31, 1))
    far.copy_(torch.randn(3, 256, device=gpu))
    near = far.contiguous()
    w = torch.randn(64, 256, device=gpu).to(torch.bfloat16)
    assert torch.equal(linear_act(far, w), linear_act(near, w))
    assert torch.equal(layer_norm(far), layer_norm(near))
    dy = torch.randn(3, 256, device=gpu).to(torch.bfloat16)
    got = []
    for v in (far, near):
        v = v.detach().requires_grad_()
        ws = w.detach().requires_grad_()
        got.append(torch.autograd.grad(layer_norm(v), v, dy)
                   + torch.autograd.grad(linear_act(v, ws), (v, ws), dy[:, :64].contiguous()))
    for a, b in zip(*got):
        assert torch.equal(a, b)


def test_outputs_past_32_bits(gpu):
    """More than 2^32 outputs: the last rows' values, mask and gradients are those of a small call (whose
    mask the oracle moves to the same elements)."""
    from gwn_amd.layers import linear_act
    m, k, n = 4200000, 32, 1032
    c = LinearCase(40, k, n, "bf16", "relu", True, False, 0.5)
    x = torch.zeros(m, k, device=gpu, dtype=torch.bfloat16)
    x[-40:] = c.x.to(gpu)
    x.requires_grad_()
    w, b = c.w.to(gpu), c.b.to(gpu)
    seed = torch.tensor([c.seed], device=gpu)
    y = linear_act(x, w, b, act="relu", p=0.5, seed=seed, salt=c.salt)
    assert y.numel() > 2 ** 32
    keep = mask(c.seed, c.salt, (40, n), 0.5, (m - 40) * n)
    z = c.x.double() @ c.w.double().T + c.b.double()  # exact: on grids
    want = torch.where(keep, z.clamp(min=0) * 2, torch.zeros((), dtype=F64))
    assert torch.equal(y[-40:].cpu(), want.to(torch.bfloat16))
    dy = torch.zeros_like(y)
    dy[-40:] = c.dy.to(gpu)
    dx, = torch.autograd.grad(y, x, dy)
    dz = torch.where(keep & (z > 0), c.dy.double() * 2, torch.zeros((), dtype=F64))
    want = dz @ c.w.double()
    within("dx", dx[-40:], want, (n + 2) * E32 * (dz.abs() @ c.w.double().abs())
           + half_step("bf16") * want.abs() * (1 + 2.0 ** -8) + TINY["bf16"])
    assert not dx[:-40].any()


def test_norm_past_32_bits(gpu):
    from gwn_amd.layers import layer_norm
    m, c = 1050000, 4096
    x, w, b, dy = norm_inputs(8, c, "bf16", True)
    big = torch.empty(m, c, device=gpu, dtype=torch.bfloat16)
    big[:] = x[0].to(gpu)
    big[-8:] = x.to(gpu)
    big.requires_grad_()
    y = layer_norm(big, w.to(gpu), b.to(gpu))
    g = torch.zeros_like(y)
    g[-8:] = dy.to(gpu)
    dx, = torch.autograd.grad(y, big, g)
    norm_check("bf16", x, w, b, dy, 1e-5, y[-8:], dx[-8:])
    assert not dx[:-8].any() and torch.equal(y[0], y[m // 2])


# ---- the C entries ----------------------------------------------------------------------------

def fenced(rows, cols, ld, t, dev, fill):
    """A [rows][ld] buffer of ``fill`` whose first cols columns are a matrix."""
    return torch.full((rows, ld), fill, device=dev, dtype=t)


@pytest.mark.parametrize("t", sorted(TYPES))
@pytest.mark.parametrize("m,k,n", [(5, 40, 36), (70, 41, 67), (300, 128, 200)])
def test_linear_entries_leave_the_rest(gpu, t, m, k, n):
    """Every leading dimension longer than its row: what lies behind the rows stays as it was, also
    with the debugging checks of ranges on."""
    import ctypes
    from gwn_amd import _lib
    lib, dt, elem = _lib.load(), TYPES[t], {"f32": 0, "f16": 1, "bf16": 2}[t]
    zt = torch.float32 if t == "f32" else torch.float16
    c = LinearCase(m, k, n, t, "silu", True, True, 0.3)
    x, w, r = (fenced(a, b_, b_ + 5, dt, gpu, math.nan) for a, b_ in ((m, k), (n, k), (m, n)))
    x[:, :k], w[:, :k], r[:, :n] = c.x.to(gpu), c.w.to(gpu), c.r.to(gpu)
    dyb = fenced(m, n, n + 3, dt, gpu, math.nan)
    dyb[:, :n] = c.dy.to(gpu)
    b, seed = c.b.to(gpu), torch.tensor([c.seed], device=gpu)
    y, z = fenced(m, n, n + 7, dt, gpu, 7.0), fenced(m, n, n + 1, zt, gpu, 7.0)
    dx, dw, db = fenced(m, k, k + 2, dt, gpu, 7.0), fenced(n, k, k + 9, dt, gpu, 7.0), torch.empty(n, device=gpu, dtype=dt)
    st = torch.cuda.current_stream().cuda_stream
    f = _lib.LinearArgs(x.data_ptr(), k + 5, w.data_ptr(), k + 5, b.data_ptr(), r.data_ptr(), n + 5, y.data_ptr(), n + 7,
                        z.data_ptr(), n + 1, m, n, k, elem, 4, seed.data_ptr(), c.salt, 0.3, None)
    g = _lib.LinearBwdArgs(dyb.data_ptr(), n + 3, x.data_ptr(), k + 5, w.data_ptr(), k + 5, z.data_ptr(), n + 1,
                           dx.data_ptr(), k + 2, dw.data_ptr(), k + 9, db.data_ptr(), m, n, k, elem, 4, seed.data_ptr(),
                           c.salt, 0.3, None)
    ws = [torch.full((max(1, v),), math.nan, device=gpu) for v in
          (lib.gwn_linear_fwd_workspace_floats(ctypes.byref(f)), lib.gwn_linear_bwd_workspace_floats(ctypes.byref(g)))]
    f.workspace, g.workspace = ws[0].data_ptr(), ws[1].data_ptr()
    lib.gwn_set_sync_check(1)
    try:
        _lib.check(lib.gwn_linear_fwd(ctypes.byref(f), st))
        _lib.check(lib.gwn_linear_bwd(ctypes.byref(g), st))
    finally:
        lib.gwn_set_sync_check(0)
    c.check(y=y[:, :n], dx=dx[:, :k], dw=dw[:, :k], db=db)
    for v, cols in ((y, n), (z, n), (dx, k), (dw, k)):
        assert (v[:, cols:] == 7.0).all()


@pytest.mark.parametrize("t", sorted(TYPES))
@pytest.mark.parametrize("m,k,n", [(7, 50, 36), (40, 2000, 24), (500, 40, 300), (999, 300, 67), (4070, 512, 4050)])
def test_linear_entry_in_place(gpu, t, m, k, n):
    """y in the residual's memory, with few rows, with the contraction split, and over whole and cut tiles."""
    import ctypes
    from gwn_amd import _lib
    lib, elem = _lib.load(), {"f32": 0, "f16": 1, "bf16": 2}[t]
    c = LinearCase(m, k, n, t, "silu", True, True, 0.3)
    x, w, b, y = (v.to(gpu) for v in (c.x, c.w, c.b, c.r))
    seed = torch.tensor([c.seed], device=gpu)
    f = _lib.LinearArgs(x.data_ptr(), k, w.data_ptr(), k, b.data_ptr(), y.data_ptr(), n, y.data_ptr(), n, None, n, m, n, k,
                        elem, 4, seed.data_ptr(), c.salt, 0.3, None)
    ws = torch.full((max(1, lib.gwn_linear_fwd_workspace_floats(ctypes.byref(f))),), math.nan, device=gpu)
    f.workspace = ws.data_ptr()
    _lib.check(lib.gwn_linear_fwd(ctypes.byref(f), torch.cuda.current_stream().cuda_stream))
    torch.cuda.synchronize()
    c.check(y=y)


@pytest.mark.parametrize("t", sorted(TYPES))
@pytest.mark.parametrize("c", [6, 33, 600, 9000, 40000])
def test_norm_entries_in_place(gpu, t, c):
    """y over x and dx over dy, rows apart, what lies between them as it was."""
    from gwn_amd import _lib
    lib, elem, m = _lib.load(), {"f32": 0, "f16": 1, "bf16": 2}[t], 11
    x, w, b, dy = norm_inputs(m, c, t, False)
    xd, yd, gd = (fenced(m, c, c + 3, TYPES[t], gpu, 7.0) for _ in range(3))
    xd[:, :c], yd[:, :c], gd[:, :c] = x.to(gpu), x.to(gpu), dy.to(gpu)
    wd, bd, stats = w.to(gpu), b.to(gpu), torch.empty(2, m, device=gpu)
    dw, db = torch.empty_like(wd), torch.empty_like(bd)
    ws = torch.full((lib.gwn_layernorm_bwd_workspace_floats(m, c, elem),), math.nan, device=gpu)
    st, mean = torch.cuda.current_stream().cuda_stream, stats.data_ptr()
    lib.gwn_set_sync_check(1)
    try:
        _lib.check(lib.gwn_layernorm_fwd(yd.data_ptr(), c + 3, m, c, elem, wd.data_ptr(), bd.data_ptr(), int(t == "f32"), 1e-5,
                                         yd.data_ptr(), c + 3, mean, mean + 4 * m, st))
        _lib.check(lib.gwn_layernorm_bwd(gd.data_ptr(), c + 3, xd.data_ptr(), c + 3, m, c, elem, wd.data_ptr(),
                                         int(t == "f32"), mean, mean + 4 * m, gd.data_ptr(), c + 3, dw.data_ptr(),
                                         db.data_ptr(), ws.data_ptr(), st))
    finally:
        lib.gwn_set_sync_check(0)
    norm_check(t, x, w, b, dy, 1e-5, yd[:, :c], gd[:, :c], dw, db)
    assert (yd[:, c:] == 7.0).all() and (gd[:, c:] == 7.0).all()


@pytest.mark.parametrize("t", sorted(TYPES))
def test_dropout_entry_in_place(gpu, t):
    from gwn_amd import _lib
    from gwn_amd.layers import dropout
    elem = {"f32": 0, "f16": 1, "bf16": 2}[t]
    x, r = torch.randn(5003, device=gpu).to(TYPES[t]), torch.randn(5003, device=gpu).to(TYPES[t])
    seed = torch.tensor([8], device=gpu)
    want = dropout(x, 0.3, seed, salt=2, residual=r)
    st = torch.cuda.current_stream().cuda_stream
    for into in (0, 1):
        a, b = torch.cat([x, x[:9]]), torch.cat([r, r[:9]])
        y = (a, b)[into]
        _lib.call("gwn_dropout", a.data_ptr(), b.data_ptr(), y.data_ptr(), 5003, elem, seed.data_ptr(), 2, 0.3, st)
        assert torch.equal(y[:5003], want) and torch.equal(y[5003:], (x, r)[into][:9])


# ---- together ---------------------------------------------------------------------------------

def test_one_tensor_twice(gpu):
    """The input as its own residual and weight: the gradients add up."""
    from gwn_amd.layers import linear_act
    x = torch.randn(48, 48, device=gpu, requires_grad=True)
    dy = torch.randn(48, 48, device=gpu)
    gx, = torch.autograd.grad(linear_act(x, x, act="gelu", residual=x), x, dy)
    parts = [x.detach().clone().requires_grad_() for _ in range(3)]
    apart = torch.autograd.grad(linear_act(parts[0], parts[1], act="gelu", residual=parts[2]), parts, dy)
    want = sum(v.double() for v in apart)
    assert float((gx.double() - want).abs().max()) <= 4 * E32 * float(sum(v.abs() for v in apart).max())


def test_dropped_places_hide_nan_backward(gpu):
    """Where dropout dropped, neither a NaN pre-activation nor a NaN gradient gets through."""
    from gwn_amd.layers import dropout, linear_act
    seed = torch.tensor([13], device=gpu)
    x = torch.randn(64, 32, device=gpu)
    w = torch.randn(80, 32, device=gpu)
    b = torch.zeros(80, device=gpu)
    keep = mask(13, 0, (64, 80), 0.5).to(gpu)
    clean = []
    for bad in (False, True):
        xs = x.clone().requires_grad_()
        res = torch.zeros(64, 80, device=gpu)
        y = linear_act(xs, w, b, act="gelu", p=0.5, seed=seed, residual=res)
        dy = torch.ones(64, 80, device=gpu)
        if bad:
            dy[~keep] = math.nan
        clean.append(torch.autograd.grad(y, xs, dy)[0])
    assert torch.isfinite(clean[1]).all() and torch.equal(clean[0], clean[1])
    # a bias of NaN in one column: only rows that keep it see it
    b[3] = math.nan
    xs = x.clone().requires_grad_()
    dx, = torch.autograd.grad(linear_act(xs, w, b, act="gelu", p=0.5, seed=seed), xs, torch.ones(64, 80, device=gpu))
    assert torch.equal(torch.isfinite(dx).all(1), ~keep[:, 3])
    xs = x.clone().requires_grad_()
    y = dropout(xs, 0.5, seed)
    dy = torch.ones_like(y)
    dy[y == 0] = math.inf
    assert torch.isfinite(torch.autograd.grad(y, xs, dy)[0]).all()


def test_two_streams_at_once(gpu):
    from gwn_amd.layers import layer_norm
    c = LinearCase(3000, 256, 512, "bf16", "gelu", True, False, 0.2)
    (x, w, b, _), dy, seed = c.on(gpu)
    from gwn_amd.layers import linear_act
    g = torch.ones(512, device=gpu, dtype=torch.bfloat16, requires_grad=True)

    def work():
        y = layer_norm(linear_act(x, w, b, act="gelu", p=0.2, seed=seed, salt=c.salt), g)
        return [y] + list(torch.autograd.grad(y, (x, w, b, g), dy))

    want = work()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    got = []
    for _ in range(4):
        for s in streams:
            with torch.cuda.stream(s):
                got.append(work())
    torch.cuda.synchronize()
    for r in got:
        for p, q in zip(want, r):
            assert torch.equal(p, q)

@pytest.mark.parametrize("t", sorted(TYPES))
def test_epilogue_mask_is_dropouts(gpu, t):
    from gwn_amd.layers import dropout, linear_act
    x = torch.randn(50, 64, device=gpu).to(TYPES[t])
    w = torch.randn(40, 64, device=gpu).to(TYPES[t])
    seed = torch.tensor([4], device=gpu)
    y = linear_act(x, w, p=0.25, seed=seed, salt=9)
    kept = dropout(torch.ones_like(y), 0.25, seed, salt=9) != 0
    assert torch.equal(y != 0, kept)


def feed_forward(t, gpu, p):
    from gwn_amd.layers import FeedForward
    torch.manual_seed(3)
    m = FeedForward(48, 200, "gelu", p, salt=2).to(gpu)
    with torch.no_grad():
        m.norm.weight.add_(torch.randn(48, device=gpu) * 0.1)
        m.norm.bias.add_(torch.randn(48, device=gpu) * 0.1)
    return m.to(TYPES[t])


@pytest.mark.parametrize("t,tol", [("f32", 2e-6), ("f16", 3e-3), ("bf16", 2.4e-2)])
@pytest.mark.parametrize("p", [0.0, 0.2])
def test_feed_forward_block(gpu, t, tol, p):
    """The norm, both products, both masks and the residual in a row, and all gradients, against 64-bit
    autograd of the formulas: a norm-wise error of at most 6 roundings of u = half a step in a row
    (norm, up, down and their gradients), or for fp32 of 32 e."""
    m = feed_forward(t, gpu, p)
    g = torch.Generator().manual_seed(1)
    x = torch.randn(2, 31, 48, generator=g).to(TYPES[t])
    dy = torch.randn(2, 31, 48, generator=g).to(TYPES[t])
    seed = torch.tensor([21], device=gpu)
    xd = x.to(gpu).requires_grad_()
    y = m(xd, seed=seed)
    y.backward(dy.to(gpu))
    v = {k: q.detach().cpu().to(F64).requires_grad_() for k, q in m.named_parameters()}
    x64 = x.to(F64).requires_grad_()
    mu = x64.mean(-1, keepdim=True)
    n = (x64 - mu) / (((x64 - mu) ** 2).mean(-1, keepdim=True) + 1e-5).sqrt() * v["norm.weight"] + v["norm.bias"]
    z = n @ v["up.weight"].T + v["up.bias"]
    a = z * 0.5 * torch.special.erfc(-z / math.sqrt(2)) * mask(21, 2, (2, 31, 200), p) / (1 - p)
    want = x64 + (a @ v["down.weight"].T + v["down.bias"]) * mask(21, 3, (2, 31, 48), p) / (1 - p)
    want.backward(dy.to(F64))

    def near(a, b):
        assert float((a.detach().cpu().to(F64) - b).norm() / b.norm()) <= tol

    near(y, want.detach())
    near(xd.grad, x64.grad)
    for k, q in m.named_parameters():
        near(q.grad, v[k].grad)
    m.eval()
    with torch.no_grad():
        assert torch.equal(m(xd), m(xd, seed=seed))


def test_modules(gpu):
    from gwn_amd.layers import Dropout, LayerNorm, LinearAct, dropout, layer_norm, linear_act
    x, r = torch.randn(9, 24, device=gpu), torch.randn(9, 24, device=gpu)
    seed = torch.tensor([6], device=gpu)
    d = Dropout(0.4, salt=3)
    assert torch.equal(d(x, seed), dropout(x, 0.4, seed, salt=3))
    assert torch.equal(d(x, seed, residual=r), dropout(x, 0.4, seed, salt=3, residual=r))
    with pytest.raises(RuntimeError):
        d(x)
    d.eval()
    assert torch.equal(d(x), x) and torch.equal(d(x, residual=r), x + r)
    m = LinearAct(24, 24, "silu", 0.4, salt=5).to(gpu)
    assert torch.equal(m(x, r, seed), linear_act(x, m.weight, m.bias, "silu", r, 0.4, seed, 5))
    m.eval()
    assert torch.equal(m(x), linear_act(x, m.weight, m.bias, "silu"))
    n = LayerNorm(24, eps=1e-3).to(gpu)
    assert torch.equal(n(x), layer_norm(x, n.weight, n.bias, 1e-3))


def test_checkpointed_block(gpu):
    """Recomputed in the backward, the block draws the same masks: the gradients are the same."""
    from torch.utils.checkpoint import checkpoint
    m = feed_forward("f32", gpu, 0.3)
    x = torch.randn(20, 48, device=gpu, requires_grad=True)
    seed, dy = torch.tensor([2], device=gpu), torch.randn(20, 48, device=gpu)
    leaves = [x] + list(m.parameters())
    want = torch.autograd.grad(m(x, seed=seed), leaves, dy)
    got = torch.autograd.grad(checkpoint(lambda v: m(v, seed=seed), x, use_reentrant=False), leaves, dy)
    for a, b in zip(want, got):
        assert torch.equal(a, b)


def step(m, x, dy, seed):
    y = m(x, seed=seed)
    return [y] + list(torch.autograd.grad(y, [x] + list(m.parameters()), dy))


@pytest.mark.parametrize("t", sorted(TYPES))
def test_block_on_a_stream_and_in_graphs(gpu, t):
    """Forward and backward on a side stream, and captured: two graphs of the same block replayed in
    turn with eager work between, inputs and the seed changing, equal the eager results each time."""
    m = feed_forward(t, gpu, 0.2)
    x = torch.randn(64, 48, device=gpu).to(TYPES[t])
    dy = torch.randn(64, 48, device=gpu).to(TYPES[t])
    seed = torch.tensor([1], device=gpu)

    def eager():
        return [v.detach().clone() for v in step(m, x.detach().clone().requires_grad_(), dy, seed)]

    want = eager()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = eager()
    side.synchronize()
    for a, b in zip(want, got):
        assert torch.equal(a, b)
    import copy
    graphs = []
    for _ in range(2):
        mg = copy.deepcopy(m)  # leaves of its own: no eager graph of them is alive
        xs, ds, ss = x.clone().requires_grad_(), dy.clone(), seed.clone()
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            for _ in range(2):
                step(mg, xs, ds, ss)
        torch.cuda.current_stream().wait_stream(s)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step(mg, xs, ds, ss)
        graphs.append((graph, xs, ds, ss, out))
    for k in range(4):
        graph, xs, ds, ss, out = graphs[k % 2]
        x.copy_(torch.randn(64, 48, device=gpu))
        dy.copy_(torch.randn(64, 48, device=gpu))
        seed.add_(1)
        with torch.no_grad():
            xs.copy_(x)
            ds.copy_(dy)
            ss.copy_(seed)
        want = eager()
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(want, out):
            assert torch.equal(a, b), k


def test_runs_repeat_bitwise(gpu):
    from gwn_amd.layers import layer_norm
    c = LinearCase(2000, 300, 260, "bf16", "gelu", True, True, 0.2)
    x, w, b, dy = norm_inputs(3000, 500, "bf16", True)
    leaves = [v.to(gpu).requires_grad_() for v in (x, w, b)]
    first = None
    for _ in range(3):
        y, got = run_linear(c, gpu)
        now = [y] + list(got.values()) + list(torch.autograd.grad(layer_norm(*leaves), leaves, dy.to(gpu)))
        if first is not None:
            for a, b_ in zip(first, now):
                assert torch.equal(a, b_)
        first = now


def test_training_refuses_a_seed_that_moved(gpu):
    from gwn_amd.layers import dropout, linear_act
    seed = torch.tensor([1], device=gpu)
    x = torch.randn(8, 16, device=gpu, requires_grad=True)
    w = torch.randn(4, 16, device=gpu)
    for y in (dropout(x, 0.5, seed), linear_act(x, w, p=0.5, seed=seed)):
        seed.add_(1)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            y.sum().backward()


def test_layers_refuse(gpu):
    from gwn_amd.layers import LinearAct, dropout, layer_norm, linear_act
    x = torch.randn(4, 16, device=gpu)
    w = torch.randn(8, 16, device=gpu)
    seed = torch.tensor([1], device=gpu)
    for call in (lambda: linear_act(x.cpu(), w.cpu()), lambda: linear_act(x, w.cpu()), lambda: linear_act(x, w.half()),
                 lambda: linear_act(x.double(), w.double()), lambda: linear_act(x, w[:, :15]),
                 lambda: linear_act(x, w[0]), lambda: linear_act(x, w[:0]), lambda: linear_act(x, w, w[:7, 0]),
                 lambda: linear_act(x, w, residual=x), lambda: linear_act(x, w, residual=x[:3, :8]),
                 lambda: linear_act(x, w, p=0.5), lambda: linear_act(x, w, p=0.5, seed=seed.int()),
                 lambda: linear_act(x, w, p=0.5, seed=seed.cpu()), lambda: linear_act(x, w, p=0.5, seed=3),
                 lambda: linear_act(x, w, p=0.5, seed=torch.zeros(2, dtype=torch.int64, device=gpu)),
                 lambda: layer_norm(x, w[0, :8]), lambda: layer_norm(x, w[0].half()), lambda: layer_norm(x[:, :0]),
                 lambda: layer_norm(x.half(), w[0].half(), w[0]), lambda: layer_norm(x, w[0].cpu()),
                 lambda: layer_norm(x.int()), lambda: dropout(x, 0.5, None), lambda: dropout(x, 0.5, seed, residual=x[:3]),
                 lambda: dropout(x, 0.5, seed, residual=x.half())):
        with pytest.raises(RuntimeError):
            call()
    many = torch.zeros(1, 16, device=gpu).expand(2 ** 30 + 1, 16)  # no memory behind them
    wide = torch.zeros(1, device=gpu).expand(2 ** 32 + 16)
    for call in (lambda: linear_act(many, w), lambda: linear_act(x[:, :1], w[:1, :1].expand(2 ** 20 + 1, 1)),
                 lambda: layer_norm(wide)):
        with pytest.raises(RuntimeError, match="2.30"):
            call()
    for call in (lambda: linear_act(x, w, act="sin"), lambda: linear_act(x, w, p=1.5, seed=seed),
                 lambda: linear_act(x, w, p=-0.1, seed=seed), lambda: linear_act(x, w, p=math.nan, seed=seed),
                 lambda: linear_act(x, w, p=0.5, seed=seed, salt=-1), lambda: dropout(x, 0.5, seed, salt=2 ** 64), lambda: linear_act(x, w, p=0.5, seed=seed, salt=2 ** 64),
                 lambda: layer_norm(x, eps=-1.0), lambda: layer_norm(x, eps=math.nan), lambda: dropout(x, 2.0, seed),
                 lambda: LinearAct(4, 4, "sin")):
        with pytest.raises(ValueError):
            call()
    y = linear_act(x.requires_grad_(), w).sum()
    g, = torch.autograd.grad(y, x, create_graph=True)
    with pytest.raises(RuntimeError):  # once differentiable
        g.sum().backward()
