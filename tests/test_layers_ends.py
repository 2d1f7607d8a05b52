"""The position-wise layers' host side at the ends of their ranges, without a GPU."""
import ctypes

import pytest

from test_layers import PTR, linear_args, norm_bwd, norm_fwd


@pytest.mark.parametrize("n,k", [(1, 1), (8, 8), (40, 1000)])
@pytest.mark.parametrize("elem,size", [(0, 4), (1, 2), (2, 2)])
def test_linear_row_limit(n, k, elem, size):
    """2^30 rows have a workspace (for x off a 16-byte border its copy, and dz), one more have none and are refused
    before anything else."""
    from gwn_amd import _lib
    lib, most = _lib.load(), 1 << 30
    for m in (most, most + 1):
        kw = dict(M=m, N=n, K=k, elem=elem, act=2, ldw=k, ldx=k)
        f = linear_args(_lib, _lib.LinearArgs, ldy=n, ldz=n, x=PTR + size, **kw)
        b = linear_args(_lib, _lib.LinearBwdArgs, ld_dy=n, ldz=n, ld_dx=k, ld_dw=k, **kw)
        fw, bw = lib.gwn_linear_fwd_workspace_floats(ctypes.byref(f)), lib.gwn_linear_bwd_workspace_floats(ctypes.byref(b))
        if m == most:
            assert fw * 4 >= m * k * size and bw * 4 >= m * n * size
        else:
            assert fw == 0 and bw == 0
            for name, a in (("gwn_linear_fwd", f), ("gwn_linear_bwd", b)):
                with pytest.raises(_lib.GwnError, match="2.30"):
                    _lib.call(name, ctypes.byref(a), None)


def test_norm_channel_limit():
    from gwn_amd import _lib
    lib, most = _lib.load(), 1 << 30
    assert lib.gwn_layernorm_bwd_workspace_floats(1, most, 2) >= 2 * most
    for name, args in (("gwn_layernorm_fwd", norm_fwd(c=most + 1, ldx=1 << 31, ldy=1 << 31)),
                       ("gwn_layernorm_bwd", norm_bwd(c=most + 1, ldx=1 << 31, ld_dy=1 << 31, ld_dx=1 << 31))):
        with pytest.raises(_lib.GwnError, match="2.30"):
            _lib.call(name, *args)
