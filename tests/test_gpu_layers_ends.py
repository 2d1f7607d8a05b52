"""Position-wise layers (``gwn_amd.layers``) at the ends of their ranges: the most rows and channels,
values near the types' ends, an activation's tail, long sums.  Oracles and bounds are those of
``test_gpu_layers``."""
import pytest
import torch

from test_gpu_layers import E32, F64, LinearCase, TINY, TYPES, act64, half_step, mask, run_linear, within

pytestmark = pytest.mark.gpu


def test_linear_act_most_rows(gpu):
    """More rows than one launch's tiles cover (2^22 of at most 128 rows where the result is narrow): values, mask
    and gradients on both sides of row 2^29 and at the ends are those of the formula at these rows."""
    from gwn_amd.layers import linear_act
    m, k, n = 2 ** 29 + 5000, 8, 8
    c = LinearCase(120, k, n, "bf16", "relu", True, False, 0.5)
    at = torch.cat([torch.arange(40), torch.arange(2 ** 29 - 20, 2 ** 29 + 20), torch.arange(m - 40, m)]).to(gpu)
    x = torch.zeros(m, k, device=gpu, dtype=torch.bfloat16)
    x[at] = c.x.to(gpu)
    x.requires_grad_()
    w, b = c.w.to(gpu).requires_grad_(), c.b.to(gpu).requires_grad_()
    seed = torch.tensor([c.seed], device=gpu)
    y = linear_act(x, w, b, act="relu", p=0.5, seed=seed, salt=c.salt)
    keep = torch.cat([mask(c.seed, c.salt, (40, n), 0.5, int(r) * n) for r in (0, 2 ** 29 - 20, m - 40)])
    z = c.x.double() @ c.w.double().T + c.b.double()  # exact: on grids
    want = torch.where(keep, z.clamp(min=0) * 2, torch.zeros((), dtype=F64))
    assert torch.equal(y[at].cpu(), want.to(torch.bfloat16))
    dy = torch.zeros_like(y)
    dy[at] = c.dy.to(gpu)
    dx, dw, db = torch.autograd.grad(y, (x, w, b), dy)
    del y, dy
    dz = torch.where(keep & (z > 0), c.dy.double() * 2, torch.zeros((), dtype=F64))  # exact in bfloat16
    u, tiny = half_step("bf16"), TINY["bf16"]
    for name, got, want, size in (("dx", dx[at], dz @ c.w.double(), dz.abs() @ c.w.double().abs()),
                                  ("dw", dw, dz.T @ c.x.double(), dz.T.abs() @ c.x.double().abs()),
                                  ("db", db, dz.sum(0), dz.abs().sum(0))):  # 120 terms, the others are zeros
        within(name, got, want, 122 * E32 * size + u * want.abs() * (1 + 2.0 ** -8) + tiny)
    dx[at] = 0
    assert not dx.any()


def test_linear_act_row_limit(gpu):
    """2^30 rows, the most, of one channel: values at the ends; the weight's and the bias's gradients are sums of 2^30
    products, zeros but for 64 of them."""
    from gwn_amd.layers import linear_act
    m, n = 2 ** 30, 32
    x = torch.zeros(m, 1, device=gpu, dtype=torch.float16)
    at = torch.cat([torch.arange(n), torch.arange(m - n, m)]).to(gpu)
    g = torch.Generator().manual_seed(4)
    xs = torch.randint(-8, 9, (2 * n, 1), generator=g).double() / 4
    ds = torch.randint(-8, 9, (2 * n, 1), generator=g).double() / 8
    x[at] = xs.to(gpu).half()
    w = torch.full((1, 1), 1.5, device=gpu, dtype=torch.float16)
    b = torch.full((1,), 0.25, device=gpu, dtype=torch.float16)
    for v in (x, w, b):
        v.requires_grad_()
    y = linear_act(x, w, b, act="relu")
    z = xs * 1.5 + 0.25  # exact, as all that follows: small multiples of 1/64
    assert torch.equal(y[at].double().cpu(), z.clamp(min=0)) and bool((y[n:m - n] == 0.25).all())
    dy = torch.zeros_like(y)
    dy[at] = ds.to(gpu).half()
    dx, dw, db = torch.autograd.grad(y, (x, w, b), dy)
    dz = ds * (z > 0)
    assert torch.equal(dx[at].double().cpu(), dz * 1.5) and not dx[n:m - n].any()
    assert dw.item() == float((dz * xs).sum()) and db.item() == float(dz.sum())


@pytest.mark.parametrize("t", sorted(TYPES))
@pytest.mark.parametrize("m,k,n", [(3, 2 ** 20, 40), (40, 2 ** 20 - 1, 3), (3, 40, 2 ** 20), (33, 9, 2 ** 20 - 7)])
def test_linear_act_most_channels(gpu, t, m, k, n):
    c = LinearCase(m, k, n, t, "silu", True, True, 0.3)
    y, got = run_linear(c, gpu)
    c.check(y=y, **got)


@pytest.mark.parametrize("c", [2 ** 26 + 40, 2 ** 30])
def test_layer_norm_many_channels(gpu, c):
    """A row of more than 2^26 channels, up to the most: its parameters' gradients are one term each.  Its values are
    +-1 in turn, so its statistics are exact but for 8 roundings of fp32."""
    from gwn_amd.layers import layer_norm
    t = torch.bfloat16
    x = torch.ones(1, c, device=gpu, dtype=t)
    x[:, 1::2] = -1
    w, b = torch.ones(c, device=gpu, dtype=t), torch.full((c,), 0.25, device=gpu, dtype=t)
    w[c // 3:] = 0.5
    dy = torch.randn(1, c, device=gpu, generator=torch.Generator(device=gpu).manual_seed(2)).to(t)
    for v in (x, w, b):
        v.requires_grad_()
    y = layer_norm(x, w, b)
    dw, db = torch.autograd.grad(y, (w, b), dy, retain_graph=True)
    xh = x.detach().double() * (1 + 1e-5) ** -0.5
    off = 8 * E32 + half_step("bf16") * (1 + 2.0 ** -8)
    for at in (slice(0, 4096), slice(c // 3 - 100, c // 3 + 100), slice(2 ** 25 - 64, 2 ** 25 + 64), slice(c - 4096, c)):
        want = xh[0, at] * w[at].double() + b[at].double()
        within("y", y[0, at], want.detach().cpu(), (off * want.abs()).detach().cpu())
        want = dy[0, at].double() * xh[0, at]
        within("dw", dw[at], want.cpu(), (off * want.abs()).cpu() + TINY["bf16"])
        assert torch.equal(db[at], dy[0, at])


@pytest.mark.parametrize("t", ["f32", "bf16"])
@pytest.mark.parametrize("c", [3, 5, 33, 100, 700, 2052, 20000])
def test_layer_norm_backward_of_large_constant_rows(gpu, c, t):
    """Rows of one large value each (a power of two: their sums are exact), a small eps: mean rstd passes fp32's range,
    but xh = 0 and dx = rstd (h - mean(h)).  A mean of h is off by `chain` additions' roundings."""
    from gwn_amd.layers import layer_norm
    eps, dt = 2.0 ** -40, TYPES[t]
    x = (torch.ones(6, c) * 2.0 ** torch.tensor([110.0, 0.0, -3.0, 108.0, 111.0, 112.0])[:, None]).to(dt)
    x[2] = -x[4]
    g = torch.Generator().manual_seed(c)
    w, b, dy = (1 + 0.2 * torch.randn(c, generator=g)).to(dt), torch.randn(c, generator=g).to(dt), torch.randn(6, c, generator=g).to(dt)
    leaves = [v.to(gpu).requires_grad_() for v in (x, w, b)]
    y = layer_norm(*leaves, eps=eps)
    dx, dw, db = torch.autograd.grad(y, leaves, dy.to(gpu))
    assert torch.equal(y.cpu(), b.expand(6, c)) and not dw.any()
    h = dy.to(F64) * w.to(F64)
    chain = 8 * max(8, -(-c // 2048)) + 16
    rs, mean = 2.0 ** 20, h.mean(1, keepdim=True)
    want = rs * (h - mean)
    e = rs * (4 * E32 * (h.abs() + mean.abs()) + (chain + 2) * E32 * h.abs().mean(1, keepdim=True))
    within("dx", dx, want, e + 8 * E32 * want.abs() + half_step(t) * want.abs() * (1 + 2.0 ** -8) + TINY[t])
    within("db", db, dy.to(F64).sum(0), 8 * E32 * dy.to(F64).abs().sum(0) + half_step(t) * dy.to(F64).sum(0).abs() * 1.01 + TINY[t])


@pytest.mark.parametrize("t,last", [("f32", 200), ("bf16", 200), ("f16", 86)])
def test_gelu_tail(gpu, t, last):
    """gelu and its slope from z = -1/16 to -12.5 (f16: -5.4) keep the type's relative precision: Phi's formula is off
    by 1.3e-5 relatively, exp(-z^2 / 2) by its argument's three roundings (3 x 78 x 2^-24 = 1.4e-5), together
    at most 4e-5 with the products'; then one rounding, or two that are the same (dz and dx = dz 1)."""
    from gwn_amd.layers import linear_act
    z = (-torch.arange(1, last + 1) / 16).to(TYPES[t])[:, None]
    w = torch.ones(1, 1, device=gpu, dtype=TYPES[t])
    phi = torch.exp(-z.to(F64) ** 2 / 2) / (2 * torch.pi) ** 0.5
    cdf = 0.5 * torch.special.erfc(-z.to(F64) / 2 ** 0.5)
    value, slope = z.to(F64) * cdf, cdf + z.to(F64) * phi
    u, off = half_step(t) * (1 + 2.0 ** -8), 4e-5
    for rows in (slice(0, last), slice(last - 20, last)):  # of tiles, and of few rows
        x = z[rows].to(gpu).requires_grad_()
        y = linear_act(x, w, act="gelu")
        dx, = torch.autograd.grad(y, x, torch.ones_like(y))
        within("y", y, value[rows], (u + off) * value[rows].abs() + TINY[t])
        within("dx", dx, slope[rows], u * slope[rows].abs() + off * (cdf + z.to(F64).abs() * phi)[rows] + TINY[t])


def test_sums_of_many_rows_have_short_chains(gpu):
    """The gradients of a bias and a norm's bias in fp32: one term is 1, the others so small that 31 of 32 equal sums
    each fall under half a step of 1 if added to it one by one, which would lose 31 e.  A chain of n additions
    loses n e at most: the norm's rows are added in chains of 6 (a group's rows), 3 (a wave's groups), 3 (waves),
    7 and 5 (partial rows), the product's in chains of 4, 4, 7 and 5."""
    from gwn_amd.layers import layer_norm, linear_act
    for m, c, share, chain in ((172224, 32, 5440, 24), (16384, 512, 512, 20)):
        dy = torch.full((m, c), 2.0 ** -24 * (1 - 2.0 ** -6) / share, device=gpu)
        dy[0] = 1
        b = torch.zeros(c, device=gpu, requires_grad=True)
        if c == 32:
            y = layer_norm(torch.randn(m, c, device=gpu), None, b)
        else:
            y = linear_act(torch.randn(m, 8, device=gpu), torch.zeros(c, 8, device=gpu), b)
        db, = torch.autograd.grad(y, b, dy)
        want = dy.double().sum(0).cpu()
        within("db", db, want, (chain + 1) * E32 * want)


@pytest.mark.parametrize("t,last", [("f32", 200), ("bf16", 200), ("f16", 86)])
@pytest.mark.parametrize("act", ["gelu_tanh", "silu"])
def test_sigmoid_tails(gpu, act, t, last):
    """The same for the activations z s(u), s = 1 / (1 + exp(-u)): exp is off by its argument's roundings, u's among
    them (4 x |u| 2^-24, and |u| is at most 88 where the value is above fp32's smallest), together under
    4e-5 of each term of the slope s + z s (1 - s) u'; an s under fp32's smallest normal number may be 0."""
    from gwn_amd.layers import linear_act
    z = (-torch.arange(1, last + 1) / 16).to(TYPES[t])[:, None]
    w = torch.ones(1, 1, device=gpu, dtype=TYPES[t])
    value, slope = act64(z.to(F64), act)
    s = value / z.to(F64)
    u, off = half_step(t) * (1 + 2.0 ** -8), 4e-5
    x = z.to(gpu).requires_grad_()
    y = linear_act(x, w, act=act)
    dx, = torch.autograd.grad(y, x, torch.ones_like(y))
    within("y", y, value, (u + off) * value.abs() + z.to(F64).abs() * 2.0 ** -126 + TINY[t])
    within("dx", dx, slope, u * slope.abs() + off * (s.abs() + (slope - s).abs()) + (1 + (slope / s).abs()) * 2.0 ** -126 + TINY[t])
