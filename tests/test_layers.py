"""The position-wise layers' host side without a GPU: the C entries refuse bad arguments before any
launch, workspace sizes hold, the modules' state dicts, and the dropout generator's constants."""
import ctypes

import pytest
import torch

PTR = 1 << 20  # never dereferenced: every call below is refused, or has nothing to do


def linear_args(lib_mod, cls, **kw):
    a = cls()
    base = dict(M=4, N=8, K=16, elem=2, act=0)
    for name, _ in cls._fields_:
        if name.startswith("ld"):
            base[name] = 16
    base.update({n: PTR for n in ("x", "w", "y", "dy", "z", "dx", "dw", "dbias", "workspace") if hasattr(a, n)})
    for k, v in {**base, **kw}.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("kw", [dict(M=-1), dict(N=0), dict(K=0), dict(K=-3), dict(elem=3), dict(elem=-1), dict(act=5),
                                dict(act=-1), dict(drop_p=0.5), dict(drop_p=1.5, seed_ptr=PTR), dict(drop_p=-0.5, seed_ptr=PTR),
                                dict(drop_p=float("nan"), seed_ptr=PTR), dict(drop_p=0.5, seed_ptr=PTR + 4), dict(x=None),
                                dict(w=None), dict(y=None), dict(ldx=15), dict(ldw=15), dict(ldy=7), dict(x=PTR + 1),
                                dict(w=PTR + 1), dict(y=PTR + 1), dict(residual=PTR, ld_res=7), dict(z=PTR, ldz=7),
                                dict(residual=PTR + 1, ld_res=8), dict(M=(1 << 30) + 1), dict(N=(1 << 20) + 1)])
def test_linear_fwd_refuses(kw):
    from gwn_amd import _lib
    with pytest.raises(_lib.GwnError, match="linear"):
        _lib.call("gwn_linear_fwd", ctypes.byref(linear_args(_lib, _lib.LinearArgs, **kw)), None)


@pytest.mark.parametrize("kw", [dict(M=-1), dict(N=0), dict(K=0), dict(elem=7), dict(act=9), dict(drop_p=0.5), dict(dy=None),
                                dict(x=None), dict(w=None), dict(act=2, z=None), dict(act=1, workspace=None),
                                dict(act=1, workspace=PTR + 4), dict(ld_dy=7), dict(ldx=15), dict(ldw=15), dict(act=2, ldz=7),
                                dict(ld_dx=15), dict(ld_dw=15), dict(dy=PTR + 1), dict(dw=PTR + 1)])
def test_linear_bwd_refuses(kw):
    from gwn_amd import _lib
    with pytest.raises(_lib.GwnError, match="linear_bwd|linear"):
        _lib.call("gwn_linear_bwd", ctypes.byref(linear_args(_lib, _lib.LinearBwdArgs, **kw)), None)


def norm_fwd(**kw):
    a = dict(x=PTR, ldx=32, rows=4, c=32, elem=1, gamma=PTR, beta=PTR, wide=0, eps=1e-5, y=PTR, ldy=32, mean=PTR, rstd=PTR)
    a.update(kw)
    return list(a.values()) + [None]


def norm_bwd(**kw):
    a = dict(dy=PTR, ld_dy=32, x=PTR, ldx=32, rows=4, c=32, elem=1, gamma=PTR, wide=0, mean=PTR, rstd=PTR, dx=PTR, ld_dx=32,
             dgamma=PTR, dbeta=PTR, ws=PTR)
    a.update(kw)
    return list(a.values()) + [None]


@pytest.mark.parametrize("kw", [dict(rows=-1), dict(c=0), dict(c=-4), dict(elem=3), dict(x=None), dict(y=None), dict(ldx=31),
                                dict(ldy=31), dict(x=PTR + 1), dict(y=PTR + 1), dict(gamma=PTR + 1), dict(wide=1, beta=PTR + 2),
                                dict(eps=-1.0), dict(eps=float("nan")), dict(mean=None), dict(rstd=None), dict(mean=PTR + 2)])
def test_layernorm_fwd_refuses(kw):
    from gwn_amd import _lib
    with pytest.raises(_lib.GwnError, match="layernorm"):
        _lib.call("gwn_layernorm_fwd", *norm_fwd(**kw))


@pytest.mark.parametrize("kw", [dict(rows=-1), dict(c=0), dict(elem=-1), dict(dy=None), dict(x=None), dict(mean=None),
                                dict(rstd=None), dict(ws=None), dict(ld_dy=31), dict(ldx=31), dict(ld_dx=31), dict(dy=PTR + 1),
                                dict(dx=PTR + 1), dict(dgamma=PTR + 1), dict(wide=1, dbeta=PTR + 2), dict(ws=PTR + 2)])
def test_layernorm_bwd_refuses(kw):
    from gwn_amd import _lib
    with pytest.raises(_lib.GwnError, match="layernorm"):
        _lib.call("gwn_layernorm_bwd", *norm_bwd(**kw))


@pytest.mark.parametrize("args", [(None, None, PTR, 8, 0, PTR, 0, 0.5), (PTR, None, None, 8, 0, PTR, 0, 0.5),
                                  (PTR, None, PTR, -1, 0, PTR, 0, 0.5), (PTR, None, PTR, 8, 3, PTR, 0, 0.5),
                                  (PTR, None, PTR, 8, 0, None, 0, 0.5), (PTR, None, PTR, 8, 0, PTR, 0, 1.25),
                                  (PTR, None, PTR, 8, 0, PTR, 0, -0.25), (PTR, None, PTR, 8, 0, PTR, 0, float("nan")),
                                  (PTR + 2, None, PTR, 8, 0, PTR, 0, 0.5), (PTR, PTR + 1, PTR, 8, 2, PTR, 0, 0.5),
                                  (PTR, None, PTR, 8, 0, PTR + 4, 0, 0.5)])
def test_dropout_refuses(args):
    from gwn_amd import _lib
    with pytest.raises(_lib.GwnError, match="dropout"):
        _lib.call("gwn_dropout", *args, None)


def test_nothing_to_do_is_no_error():
    from gwn_amd import _lib
    _lib.call("gwn_dropout", None, None, None, 0, 0, None, 0, 0.5, None)
    _lib.call("gwn_layernorm_fwd", *norm_fwd(rows=0, x=None, y=None))
    _lib.call("gwn_layernorm_bwd", *norm_bwd(rows=0, dgamma=None, dbeta=None))
    _lib.call("gwn_layernorm_bwd", *norm_bwd(dx=None, dgamma=None, dbeta=None))
    _lib.call("gwn_linear_fwd", ctypes.byref(linear_args(_lib, _lib.LinearArgs, M=0)), None)
    _lib.call("gwn_linear_bwd", ctypes.byref(linear_args(_lib, _lib.LinearBwdArgs, dx=None, dw=None, dbias=None)), None)


def test_workspace_sizes():
    """A workspace covers what a call writes into it: at least one partial row of the parameters'
    gradients, dz, and where rows are many two partial rows of the bias's."""
    from gwn_amd import _lib
    lib = _lib.load()
    for rows in (0, 1, 7, 5000, 1 << 33):
        for c in (1, 32, 1111, 4096, 20000):
            assert lib.gwn_layernorm_bwd_workspace_floats(rows, c, 2) >= 2 * c
    for m in (0, 1, 300, 20000, 1 << 29):
        for n, k in ((1, 1), (33, 70), (8192, 2048)):
            for elem, size in ((0, 4), (1, 2), (2, 2)):
                kw = dict(M=m, N=n, K=k, elem=elem, act=2, ldw=k, ldx=k, ld_dx=k, ld_dw=k)
                b = linear_args(_lib, _lib.LinearBwdArgs, ld_dy=n, ldz=n, **kw)
                assert lib.gwn_linear_bwd_workspace_floats(ctypes.byref(b)) * 4 >= m * n * size + (8 * n if m > 2000 else 0)
                f = linear_args(_lib, _lib.LinearArgs, ldy=n, ldz=n, **{q: v for q, v in kw.items() if q[:4] != "ld_d"})
                floats = lib.gwn_linear_fwd_workspace_floats(ctypes.byref(f))
                assert floats >= 0
                f.x += size  # off a 16-byte border: x is copied (a few rows are read where they lie)
                assert m <= 32 or lib.gwn_linear_fwd_workspace_floats(ctypes.byref(f)) * 4 >= m * k * size


def test_modules_hold_their_parameters():
    from gwn_amd.layers import FeedForward, LinearAct
    m = FeedForward(16, 64, "silu", 0.1, salt=4)
    assert {k: tuple(v.shape) for k, v in m.state_dict().items()} == {
        "norm.weight": (16,), "norm.bias": (16,), "up.weight": (64, 16), "up.bias": (64,), "down.weight": (16, 64),
        "down.bias": (16,)}
    assert (m.up.salt, m.down.salt) == (4, 5)
    assert LinearAct(3, 5, bias=False).bias is None
    torch.manual_seed(0)
    a = LinearAct(7, 9)
    torch.manual_seed(0)
    b = torch.nn.Linear(7, 9)
    assert torch.equal(a.weight, b.weight) and torch.equal(a.bias, b.bias)


def test_layers_refuse_host_tensors():
    from gwn_amd.layers import dropout, layer_norm, linear_act
    x, w = torch.randn(4, 16), torch.randn(8, 16)
    for call in (lambda: linear_act(x, w), lambda: layer_norm(x), lambda: dropout(x, 0.5, torch.tensor([1]))):
        with pytest.raises(RuntimeError, match="GPU device"):
            call()
