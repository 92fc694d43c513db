"""The largest sizes: row calls past 2^32 work items, and what the adapter calls refuse (CPU: before any launch)."""
import ctypes
import gc
import importlib

import pytest
import torch

_lib = importlib.import_module("a-nerf_amd._lib")
E_SHAPE = -2
P = lambda k: ctypes.c_void_p(0x7F0000000000 + 0x1000 * k)          # never read: every call returns before its launch


@pytest.fixture(scope="module", autouse=True)
def give_back_what_the_allocator_cached():
    """other tests account for single allocations: blocks of this module's sizes would serve them instead of fresh ones"""
    yield
    gc.collect()
    if torch.cuda.is_available():
        torch.cuda.empty_cache()


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
def test_the_backward_wants_what_the_forward_returned():
    ops = importlib.import_module("a-nerf_amd.ops")
    x, W, A, B = (torch.zeros(*s, device="cuda") for s in ((80, 32), (24, 32), (3, 4, 32), (3, 24, 4)))
    plan = ops.route_rows(torch.zeros(80, dtype=torch.long, device="cuda"), 3)
    for h in (None, [1.0], torch.zeros(4, device="cuda"), torch.zeros(80, 64)):
        with pytest.raises(ValueError, match="h must be"):
            ops.adapter_backward(torch.zeros(80, 24, device="cuda"), x, W, A, B, plan, h)


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


@pytest.mark.gpu
@pytest.mark.parametrize("form", ["poses", "one pose", "codes"])
def test_a_large_render_holds_a_piece_of_its_points(form, monkeypatch):
    """an adapted render without gradients: the encoded rows of the whole call are never in memory together, and the picture is that of the
    whole call (a row's sums may be taken in another order: the bar of the other pictures)"""
    networks, raycaster = importlib.import_module("a-nerf_amd.networks"), importlib.import_module("a-nerf_amd.raycaster")
    autograd_path, ad, synth = (importlib.import_module("a-nerf_amd." + m) for m in ("autograd_path", "adapters", "synth"))
    n, S, Ni, dev = 600, 64, 16, "cuda"
    codes = form == "codes"
    kw = dict(use_framecode=True, framecode_ch=16, n_framecodes=6) if codes else {}
    ck = dict(cutoff=True, cutoff_dist=0.5, cutoff_inputs=True, cutoff_dim=24)
    nets = []
    for seed in (11, 12):
        nets.append(networks.NeRF(D=8, W=256, input_ch=360, input_ch_bones=72, input_ch_views=648, use_viewdirs=True, **kw))
        nets[-1].load_state_dict({k: torch.tensor(v) for k, v in synth.make_net_params(seed, **(dict(framecode_ch=16, n_codes=6) if codes else {})).items()})
    ev, eb, ed = (networks.get_embedder(7, 0, 24, cutoff_kwargs=dict(ck))[0], networks.get_embedder(0, 0, 72)[0],
                  networks.get_embedder(4, 0, 72, cutoff_kwargs=dict(ck, dist_inputs=True))[0])
    caster = raycaster.RayCaster(nets[0], ev, eb, ed, network_fine=nets[1]).to(dev).requires_grad_(False).eval()
    torch.manual_seed(1)
    ads = [ad.NetAdapters(net, 3, rank=4) for net in nets]
    with torch.no_grad():
        for a in ads:
            for name in ad.LAYERS:
                a.up(name).normal_(0, 0.05)
    caster.set_adapters(*ads)
    ro, rd, kp, skts, bones, cyls, _ = synth.scene_batch(n, [0, 1, 2], H=128, W=128, focal=150.0, ray_seed=3, per_ray_pose=True)
    t = lambda v: torch.tensor(v, dtype=torch.float32, device=dev)
    pipeline = importlib.import_module("a-nerf_amd.pipeline")
    rb = pipeline.make_ray_batch(t(ro), t(rd))
    one = form == "one pose"
    cut = lambda v: t(v)[:1] if one else t(v)
    subjects = torch.arange(n, device=dev) % 4
    cams = (torch.arange(n, device=dev) % 7 - 1).float() if codes else None             # -1: the mean code
    call = lambda: caster(rb, N_samples=S, kp_batch=cut(kp), skts=cut(skts), cyls=cut(cyls), cams=cams, subject_idxs=subjects, N_importance=Ni,
                          preproc_kwargs={"density_scale": 1.0})
    whole = call()
    monkeypatch.setattr(autograd_path, "ENCODE_POINTS", 5000)                            # 78 rays of the first pass, 62 of the second
    call()
    torch.cuda.empty_cache()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    parts = call()
    # one copy of all encoded rows of the second pass alone
    assert torch.cuda.max_memory_allocated() - before < n * (S + Ni) * 1080 * 4
    for k in ("rgb_map", "acc_map", "rgb0"):
        assert float((whole[k] - parts[k]).abs().max()) < 1e-4, k
    assert float(whole["acc_map"].max()) > 0.1
    # as many poses or cameras as a piece of the second pass has rays are not one per ray
    bad = dict(N_samples=S, kp_batch=cut(kp), skts=cut(skts), cyls=cut(cyls), cams=cams, subject_idxs=subjects, N_importance=Ni)
    with pytest.raises(ValueError, match="skts"):
        caster(rb, **{**bad, "skts": t(skts)[:5000 // S]})
    if codes:
        with pytest.raises(ValueError, match="cams"):
            caster(rb, **{**bad, "cams": cams[:5000 // S]})
