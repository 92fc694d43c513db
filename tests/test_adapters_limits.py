"""The largest sizes: row calls past 2^32 work items, and what the adapter calls refuse (CPU: before any launch)."""
import ctypes
import importlib

import pytest
import torch

_lib = importlib.import_module("a-nerf_amd._lib")
E_SHAPE = -2
P = lambda k: ctypes.c_void_p(0x7F0000000000 + 0x1000 * k)          # never read: every call returns before its launch


def _io(**kw):
    io = _lib.AnerfAdapterIO()
    base = dict(dtype=2, n_adapters=3, rank=8, scale=1.0, n_rows=10, n_in=64, n_out=32, x_stride=64, x=P(1).value, weight=P(2).value, down=P(3).value,
                up=P(4).value, offsets=P(5).value, y=P(6).value, h=P(7).value)
    for k, v in {**base, **kw}.items():
        setattr(io, k, v)
    return io


def test_launches_of_too_many_work_items_are_refused():
    lib = _lib.load()
    size = lambda f, **kw: f(ctypes.byref(_io(**kw)))
    every = (lib.anerf_adapter_h_size, lib.anerf_adapter_workspace_size, lib.anerf_adapter_backward_workspace_size)
    for f in every:
        assert size(f, n_rows=2 ** 28 - 1) >= 0 and size(f, n_rows=2 ** 28) == E_SHAPE
        # 2^18 x 2^6 tiles of 64 x 64: 2^24 workgroups of 256
        assert size(f, n_rows=2 ** 24, n_out=2 ** 12 - 64, n_in=64) >= 0
        assert size(f, n_rows=2 ** 24, n_out=2 ** 12) == E_SHAPE and size(f, n_rows=2 ** 24, n_in=2 ** 12) == E_SHAPE
    big = [dict(n_out=2 ** 18, n_in=2 ** 18), dict(n_adapters=1024, rank=1, n_in=2 ** 20, n_out=1), dict(n_adapters=1024, rank=65, n_out=2 ** 19, n_in=1)]
    g = _lib.AnerfAdapterGradIO(P(8).value, 32, P(9).value, P(10).value, P(11).value)
    for kw in big:
        assert size(lib.anerf_adapter_h_size, **kw) > 0                # (the forward transposes nothing)
        assert size(lib.anerf_adapter_backward_workspace_size, **kw) == E_SHAPE
        assert lib.anerf_adapter_backward(ctypes.byref(_io(**kw)), ctypes.byref(g), P(16), 1 << 62, None) == E_SHAPE
    assert size(lib.anerf_adapter_backward_workspace_size, n_adapters=1024, rank=1, n_in=2 ** 19, n_out=1) > 0
    io = _io(n_rows=2 ** 28)
    assert lib.anerf_adapter_linear(ctypes.byref(io), P(9), 1 << 62, None) == E_SHAPE


@pytest.mark.gpu
def test_more_rows_than_work_items_along_one_axis():
    """2^26 + 3 rows: 64 work items a row are more than 2^32"""
    ad = importlib.import_module("a-nerf_amd.adapters")
    T, D, G = 2 ** 26 + 3, 3, 5
    i = torch.arange(T, device="cuda", dtype=torch.int32)
    idx = (i % 7).to(torch.int32)                                       # 5 and 6: no group
    x = torch.stack([(i % 1000), (i // 1000 % 1000), i % 13], 1).half()
    w = (i % 5 + 1).float()[:, None]
    plan = ad.route_rows(idx, G)
    kept = (idx < G)[:, None]
    xs = ad.dispatch_rows(x, plan)
    assert torch.equal(xs, torch.where(kept, x, 0.0)[plan.source.long()])
    back = ad.combine_rows(xs, plan, w)
    want = torch.where(kept, (x.float() * w).half(), 0.0)
    assert torch.equal(back, want)
    del back, want
    z, wl = xs.clone().requires_grad_(), w.clone().requires_grad_()
    dz, dw = torch.autograd.grad(ad.combine_rows(z, plan, wl), [z, wl], x)
    assert torch.equal(dz, torch.where(kept, (x.float() * w).half(), 0.0)[plan.source.long()])
    # sums of squares below 2 * 10^6 + 13^2: whole numbers below 2^24, exact in fp32
    assert torch.equal(dw, torch.where(kept, x.float().square().sum(1, keepdim=True), 0.0))
    del xs, z, dz, dw
    torch.cuda.empty_cache()
