"""CPU: the row-routing and adapter entry points refuse bad arguments on the host, before any launch (no pointer is read)."""
import ctypes
import importlib

import pytest
import torch

_lib = importlib.import_module("a-nerf_amd._lib")
ops = importlib.import_module("a-nerf_amd.ops")
E_CONFIG, E_SHAPE, E_NULL, E_WORKSPACE = -1, -2, -3, -4
P = lambda k: ctypes.c_void_p(0x7F0000000000 + 0x1000 * k)          # never read: every call returns before its launch


def test_route_rows_refuses():
    lib = _lib.load()
    assert lib.anerf_route_rows_workspace_size(100, 8) == 0 and lib.anerf_route_rows_workspace_size(100000, 8) > 0
    for n, g in ((-1, 4), (2 ** 31, 4), (10, 0), (10, 1025)):
        assert lib.anerf_route_rows_workspace_size(n, g) == E_SHAPE
        assert lib.anerf_route_rows(P(1), 1, n, g, P(2), P(3), P(4), P(5), 1 << 20, None) == E_SHAPE
    assert lib.anerf_route_rows(None, 1, 10, 4, P(2), P(3), P(4), P(5), 0, None) == E_NULL
    assert lib.anerf_route_rows(P(1), 1, 10, 4, None, P(3), P(4), P(5), 0, None) == E_NULL
    need = lib.anerf_route_rows_workspace_size(100000, 8)
    assert lib.anerf_route_rows(P(1), 1, 100000, 8, P(2), P(3), P(4), P(5), need - 1, None) == E_WORKSPACE
    assert lib.anerf_route_rows(P(1), 1, 100000, 8, P(2), P(3), P(4), None, need, None) == E_WORKSPACE


def test_dispatch_and_combine_refuse():
    lib = _lib.load()
    for f in (lib.anerf_dispatch_rows, lib.anerf_combine_rows):
        call = lambda dt=0, n=8, k=2, d=4, x=P(1), slot=P(2), kept=P(3), out=P(4): f(x, dt, None, slot, kept, n, k, d, out, None)
        assert call(dt=3) == E_CONFIG and call(k=0) == E_SHAPE and call(k=65) == E_SHAPE and call(n=-1) == E_SHAPE and call(d=-1) == E_SHAPE
        assert call(n=2 ** 30) == E_SHAPE and call(x=None) == E_NULL and call(slot=None) == E_NULL and call(kept=None) == E_NULL and call(out=None) == E_NULL
        assert call(n=0) == 0 and call(d=0) == 0
    back = lambda w=P(1), z=P(2), dz=P(3), dw=P(4), n=8: lib.anerf_combine_rows_backward(P(5), z, 0, w, P(6), P(7), n, 2, 4, dz, dw, None)
    assert back(w=None) == E_NULL and back(z=None) == E_NULL and back(dz=None, dw=None) == 0 and back(n=0) == 0


def _io(**kw):
    io = _lib.AnerfAdapterIO()
    base = dict(dtype=1, n_adapters=3, rank=8, scale=1.0, n_rows=10, n_in=64, n_out=32, x_stride=64, x=P(1).value, weight=P(2).value, down=P(3).value,
                up=P(4).value, offsets=P(5).value, y=P(6).value, h=P(7).value)
    for k, v in {**base, **kw}.items():
        setattr(io, k, v)
    return io


def test_adapter_linear_refuses():
    lib = _lib.load()
    call = lambda ws=P(9), n=1 << 30, **kw: lib.anerf_adapter_linear(ctypes.byref(_io(**kw)), ws, n, None)
    for kw in (dict(n_adapters=0), dict(n_adapters=1025), dict(rank=0), dict(rank=1025), dict(n_rows=-1), dict(n_rows=2 ** 31), dict(n_in=0), dict(n_out=0),
               dict(n_in=2 ** 25), dict(n_rows=2 ** 31 - 1, n_out=2 ** 12), dict(h=P(7).value + 4)):
        assert call(**kw) == E_SHAPE, kw
    assert call(dtype=7) == E_CONFIG and lib.anerf_adapter_linear(None, None, 0, None) == E_NULL
    for k in ("x", "weight", "down", "up", "offsets", "y", "h"):
        assert call(**{k: None}) == E_NULL, k
    assert call(n_rows=0) == 0
    few = dict(n_rows=128, n_in=4096, n_out=4096)
    need = lib.anerf_adapter_workspace_size(ctypes.byref(_io(**few)))
    assert need > 0 and lib.anerf_adapter_workspace_size(ctypes.byref(_io(n_rows=100000, n_in=512, n_out=512))) == 0
    assert call(n=need - 1, **few) == E_WORKSPACE and call(ws=None, n=need, **few) == E_WORKSPACE
    assert call(ws=ctypes.c_void_p(P(9).value + 4), **few) == E_SHAPE
    assert lib.anerf_adapter_h_size(ctypes.byref(_io())) >= 10 * 16 * 4 and lib.anerf_adapter_h_size(ctypes.byref(_io(rank=0))) == E_SHAPE


def test_adapter_linear_few_refuses():
    lib = _lib.load()
    call = lambda g=P(8), **kw: lib.anerf_adapter_linear_few(ctypes.byref(_io(**{**dict(offsets=None), **kw})), g, 1, None)
    assert call(n_rows=65) == E_SHAPE and call(rank=0) == E_SHAPE and call(dtype=5) == E_CONFIG and call(h=P(7).value + 4) == E_SHAPE
    assert call(g=None) == E_NULL and call(n_rows=0) == 0 and lib.anerf_adapter_linear_few(None, P(8), 1, None) == E_NULL
    for k in ("x", "weight", "down", "up", "y", "h"):
        assert call(**{k: None}) == E_NULL, k


def test_adapter_backward_refuses():
    lib = _lib.load()
    need = lib.anerf_adapter_backward_workspace_size(ctypes.byref(_io()))
    assert need > 0 and lib.anerf_adapter_backward_workspace_size(ctypes.byref(_io(rank=0))) == E_SHAPE
    g = _lib.AnerfAdapterGradIO(P(1).value, 32, P(2).value, P(3).value, P(4).value)
    assert lib.anerf_adapter_backward_workspace_size(ctypes.byref(_io(n_rows=0))) > 0 and lib.anerf_adapter_workspace_size(ctypes.byref(_io(n_rows=0))) == 0
    call = lambda io, g=g, ws=P(16), n=need: lib.anerf_adapter_backward(ctypes.byref(io), None if g is None else ctypes.byref(g), ws, n, None)
    assert call(_io(), None) == E_NULL and call(_io(), n=need - 1) == E_WORKSPACE and call(_io(), ws=None) == E_WORKSPACE
    assert call(_io(), ws=ctypes.c_void_p(P(16).value + 16)) == E_SHAPE and call(_io(h=None)) == E_NULL and call(_io(x=None)) == E_NULL
    assert call(_io(), _lib.AnerfAdapterGradIO(P(1).value, 32, None, None, None)) == 0


def test_structs_match_the_compiled_header(tmp_path):
    import os
    import subprocess
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    src = tmp_path / "sz.c"
    src.write_text('#include "anerf.h"\n#include <stdio.h>\n#include <stddef.h>\nint main(void){printf("%zu %zu %zu %zu %zu %d %d %d\\n", sizeof(AnerfAdapterIO), '
                   'offsetof(AnerfAdapterIO, n_rows), offsetof(AnerfAdapterIO, scale_of), offsetof(AnerfAdapterIO, h), sizeof(AnerfAdapterGradIO), '
                   'ANERF_F32, ANERF_BF16, ANERF_F16);return 0;}\n')
    exe = tmp_path / "sz"
    subprocess.check_call(["gcc", "-I", os.path.join(root, "include"), str(src), "-o", str(exe)])
    got = [int(v) for v in subprocess.check_output([str(exe)]).split()]
    A, G = _lib.AnerfAdapterIO, _lib.AnerfAdapterGradIO
    assert got == [ctypes.sizeof(A), A.n_rows.offset, A.scale_of.offset, A.h.offset, ctypes.sizeof(G)] + [ops.ROW_DTYPES[t] for t in
                                                                                             (torch.float32, torch.bfloat16, torch.float16)]


def test_cpu_tensors_are_refused():
    ad = importlib.import_module("a-nerf_amd.adapters")
    with pytest.raises(TypeError):
        ad.route_rows(torch.zeros(4, dtype=torch.long), 2)
    with pytest.raises(TypeError):
        ad.adapter_linear(torch.zeros(4, 8), torch.zeros(3, 8), torch.zeros(1, 2, 8), torch.zeros(1, 3, 2), torch.zeros(4, dtype=torch.long))
    with pytest.raises(TypeError):
        ad.dispatch_rows(torch.zeros(4, 8), None)


def test_adapters_leave_the_networks_state_dict_alone():
    ad, networks = importlib.import_module("a-nerf_amd.adapters"), importlib.import_module("a-nerf_amd.networks")
    net = networks.NeRF(input_ch=360, input_ch_bones=72, input_ch_views=648, use_viewdirs=True)
    keys, params = set(net.state_dict()), len(list(net.parameters()))
    a = ad.NetAdapters(net, 3, rank=2)
    net.set_adapters(a)
    assert set(net.state_dict()) == keys and len(list(net.parameters())) == params and len(net.named_path_params()) == 24
    assert len(a.state_dict()) == 24 and a.down("pts_linears.5").shape == (3, 2, 688) and not a.up("rgb_linear").any()
    b = ad.NetAdapters(net, 3, rank=2)
    b.load_state_dict(a.state_dict())
    assert torch.equal(b.down("views_linears.0"), a.down("views_linears.0"))
    with pytest.raises(ValueError):
        networks.NeRF(input_ch=360, input_ch_bones=72, input_ch_views=648, use_viewdirs=True)(torch.zeros(2, 1080), subject_idxs=torch.zeros(2))


def test_negative_row_strides_are_refused():
    lib = _lib.load()
    io = _io(x_stride=-64)
    assert lib.anerf_adapter_workspace_size(ctypes.byref(io)) == E_SHAPE and lib.anerf_adapter_linear(ctypes.byref(io), P(9), 1 << 30, None) == E_SHAPE
    assert lib.anerf_adapter_linear_few(ctypes.byref(io), P(10), 1, None) == E_SHAPE
    g = _lib.AnerfAdapterGradIO()
    g.g, g.g_stride, g.dx = P(11).value, -32, P(12).value
    assert lib.anerf_adapter_backward(ctypes.byref(_io()), ctypes.byref(g), P(9), 1 << 30, None) == E_SHAPE
