"""Entries whose outputs are cleared in part, captured into a graph: every replay clears them again."""
import ctypes

import pytest
import torch

pytestmark = pytest.mark.gpu


def captured(call):
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        call(s.cuda_stream)
    torch.cuda.current_stream().wait_stream(s)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        call(torch.cuda.current_stream().cuda_stream)
    return g


@pytest.mark.parametrize("c", [16, 32])
def test_gcn_partials_past_the_slices(gpu, c):
    """The BatchNorm partials of fewer slices than compute units: those past the slices are zeros after each replay, the
    others and z the eager call's."""
    from gwn_amd import _lib
    lib = _lib.load()
    torch.manual_seed(c)
    n, slices, ld = 24, 5, 32
    rows, width = n * slices, 3 * c
    sup = torch.zeros(ld, ld, device=gpu)
    sup[:n, :n] = torch.rand(n, n, device=gpu) / n
    arr = (ctypes.c_void_p * 1)(sup.data_ptr())
    wm = torch.randn(c, width, device=gpu) * 0.1
    wmt, bm, res = wm.t().contiguous(), torch.randn(c, device=gpu), torch.randn(rows, c, device=gpu)
    h, z = torch.zeros(rows, width, device=gpu), torch.empty(rows, c, device=gpu)
    h[:, :c] = torch.randn(rows, c, device=gpu)
    seed = torch.zeros(1, device=gpu, dtype=torch.int64)
    slots = lib.gwn_gcn_bn_partial_count(rows, n, c, 1, ld)
    assert slots > slices
    part = torch.empty(slots, 3 * c, device=gpu)
    a = _lib.GcnArgs(rows=rows, n=n, c=c, nsup=1, sup=ctypes.cast(arr, ctypes.POINTER(ctypes.c_void_p)), ld_sup=ld,
                     h=h.data_ptr(), ld_h=width, w_mlp=wm.data_ptr(), b_mlp=bm.data_ptr(), residual=res.data_ptr(),
                     z=z.data_ptr(), seed_ptr=seed.data_ptr(), salt=0, drop_p=0.0, bn_partials=part.data_ptr(),
                     w_mlp_t=wmt.data_ptr())

    def call(stream):
        _lib.call("gwn_gcn_fwd", ctypes.byref(a), stream)

    part.fill_(float("nan"))
    call(_lib.stream())
    want, zw = part.clone(), z.clone()
    assert not want[slices:].any()
    g = captured(call)
    for k in range(4):
        part.fill_(float("nan"))
        z.fill_(float(k))
        torch.ones(1000, device=gpu).sum().item()  # the program's own work between the replays
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(part, want) and torch.equal(z, zw)
