"""Adapters in training: gradients over several ranks (CPU, gloo), captured steps whose schedule moves tau, forward
mode."""
import gc
import importlib
import os
import sys
import types

import pytest
import torch
import torch.distributed as dist
import torch.multiprocessing as mp

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
ad = importlib.import_module("a-nerf_amd.adapters")
networks = importlib.import_module("a-nerf_amd.networks")
ops = importlib.import_module("a-nerf_amd.ops")
raycaster = importlib.import_module("a-nerf_amd.raycaster")
trainer = importlib.import_module("a-nerf_amd.trainer")


@pytest.fixture(scope="module", autouse=True)
def give_back_what_the_allocator_cached():
    """other tests account for single allocations: blocks of this module's sizes would serve them instead of fresh ones"""
    yield
    gc.collect()
    if torch.cuda.is_available():
        torch.cuda.empty_cache()


def small_caster(single=False):
    """a caster on the CPU that is never asked to render, and its adapters"""
    mk = lambda: networks.NeRF(D=8, W=256, input_ch=360, input_ch_bones=72, input_ch_views=648, use_viewdirs=True)
    torch.manual_seed(3)
    net = mk()
    c = raycaster.RayCaster(net, None, None, None, network_fine=net if single else mk(), single_net=single).requires_grad_(False)
    ads = [ad.NetAdapters(net, 2, rank=2)] + ([] if single else [ad.NetAdapters(c.network_fine, 2, rank=3)])
    return c, ads


def trainer_of(caster, optimizer):
    args = types.SimpleNamespace(opt_pose_step=1)
    return trainer.Trainer(args, {"hwf": (4, 4, 1.0)}, optimizer, None, {"ray_caster": raycaster.RayParallel(caster)}, {}, device=None)


def _rank(rank, world, port, single, q):
    os.environ["MASTER_ADDR"], os.environ["MASTER_PORT"] = "127.0.0.1", str(port)
    dist.init_process_group("gloo", rank=rank, world_size=world)
    torch.set_num_threads(2)
    caster, ads = small_caster(single)
    par = raycaster.RayParallel(caster)
    assert par.sync_gradients() is None                                    # nothing to train yet
    caster.set_adapters(*ads)
    params = [p for a in ads for p in a.parameters()]
    before = [p.detach().clone() for p in params]
    tr = trainer_of(caster, torch.optim.SGD(params, lr=1.0))
    tr.render_kwargs_train["ray_caster"] = par                             # the wrapper that has synchronised before they were attached
    stats = tr.optimize(sum(((rank + 1.0) * (i + 1) * p).sum() for i, p in enumerate(params)), 0, True)
    # the mean of (rank + 1) (i + 1) over two ranks is 1.5 (i + 1)
    ok = all(torch.allclose(b - p.detach(), torch.full_like(p, 1.5 * (i + 1)), rtol=1e-5, atol=1e-5) for i, (b, p) in enumerate(zip(before, params)))
    want = sum(p.numel() * (1.5 * (i + 1)) ** 2 for i, p in enumerate(params)) ** 0.5
    ok &= abs(float(stats["total_norm"]) - want) < 1e-4 * want
    ok &= abs(float(stats["avg_norm"]) - want / len(params) ** 0.5) < 1e-4 * want
    # detached again: their gradients are no business of the caster's any more
    caster.set_adapters(None)
    (params[0] * (rank + 1.0)).sum().backward()
    par.sync_gradients()
    ok &= bool((params[0].grad == rank + 1.0).all()) and float(trainer.get_gradnorm(par)[0]) == 0.0
    q.put((rank, ok))
    dist.barrier()
    dist.destroy_process_group()


@pytest.mark.parametrize("single", [False, True])
def test_adapter_gradients_are_averaged_over_the_ranks(single):
    """Trainer.optimize with a torch optimiser over attached adapters: both ranks step with the mean of their gradients"""
    import socket
    s = socket.socket()
    s.bind(("127.0.0.1", 0))
    port = s.getsockname()[1]
    s.close()
    ctx = mp.get_context("spawn")
    q = ctx.Queue()
    ps = [ctx.Process(target=_rank, args=(r, 2, port, single, q)) for r in range(2)]
    for p in ps:
        p.start()
    try:
        got = dict(q.get(timeout=100) for _ in ps)
    finally:
        for p in ps:
            p.join(timeout=30)
            if p.is_alive():
                p.terminate()
    assert got == {0: True, 1: True}


def test_the_gradient_norm_counts_attached_adapters():
    caster, ads = small_caster()
    caster.set_adapters(*ads)
    for a in ads:
        for p in a.parameters():
            p.grad = torch.ones_like(p)
    n = [p.numel() for a in ads for p in a.parameters()]
    for c in (caster, raycaster.RayParallel(caster)):
        tot, avg = trainer.get_gradnorm(c)
        assert abs(float(tot) - sum(n) ** 0.5) < 1e-3 and abs(float(avg) - (sum(n) / len(n)) ** 0.5) < 1e-3


def test_a_captured_step_belongs_to_the_adapters_it_was_captured_with(monkeypatch):
    """Trainer.enable_graph: attaching, exchanging and detaching adapters selects another graph"""
    graph_step = importlib.import_module("a-nerf_amd.graph_step")
    caster, ads = small_caster()
    tr = trainer_of(caster, torch.optim.SGD(ads[0].parameters(), lr=1.0))
    tr.args.opt_pose_stop, tr.args.opt_pose = None, False
    keys = []
    tr._fused = types.SimpleNamespace(param_groups=[{}], _due=lambda i, only: [0])
    tr._static = graph_step.StaticBatch("cpu")
    tr._gs = types.SimpleNamespace(step=lambda i, key, due: keys.append(key) or {"loss_dict": {}, "stats": {}, "optim": {}, "alpha": None})
    monkeypatch.setattr(tr, "_finish_iteration", lambda *a: None)
    batch = {"target_s": torch.zeros(4, 3), "subject_idxs": torch.zeros(4, dtype=torch.long)}
    for attached in ([None], ads, ads, [ad.NetAdapters(caster.network, 2), ads[1]], [None]):
        caster.set_adapters(*attached)
        tr._train_batch_graphed(batch, 0, 0)
    assert len(set(keys)) == 3 and keys[0] == keys[4] and keys[1] == keys[2]


@pytest.mark.gpu
@pytest.mark.parametrize("form", ["cast", "stacked", "rows", "weights", "dispatched", "chain"])
def test_the_capture_guard_sees_leaves_behind_other_operations(form, monkeypatch):
    """a captured backward beside a living eager graph is refused also where the leaf is not an argument itself: master weights cast to the
    rows' type, parameters stacked, rows of a trained layer in front.  The capture is only claimed: a real one would end the process without it"""
    r = lambda *s: torch.randn(*s, device="cuda")
    idx, W = torch.arange(8, device="cuda") % 2, r(16, 32)
    A, B, lin, w = r(2, 4, 32).requires_grad_(), r(2, 16, 4).requires_grad_(), r(32, 32).requires_grad_(), r(8, 1).requires_grad_()
    x, plan = r(8, 32), ad.route_rows(idx, 2)
    other = r(2, 4, 32).requires_grad_()

    def call():
        if form == "cast":
            return ad.adapter_linear(x.bfloat16(), W.bfloat16(), A.bfloat16(), B.bfloat16(), idx)
        if form == "stacked":
            return ad.adapter_linear(x, W, torch.stack([A[0] * 2, A[1]]), torch.cat([B[:1], B[1:]]), plan)
        if form == "rows":
            return ad.adapter_linear(torch.relu(x @ lin), W, A.detach(), B.detach(), idx)
        if form == "weights":
            return ad.combine_rows(x, plan, torch.sigmoid(w))
        if form == "dispatched":
            return ad.dispatch_rows((x @ lin) * 2, plan)
        return ad.adapter_linear(ad.adapter_linear(x, r(32, 32), A * 1.0, r(2, 32, 4), idx), W, A.detach(), B.detach(), idx)

    alive = call()
    unrelated = ad.adapter_linear(x, W, other * 1.0, B.detach(), idx)              # lives on, shares no leaf
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        y = call()
        monkeypatch.setattr(ad, "_capturing", lambda: True)
        with pytest.raises(RuntimeError, match="eager graph"):
            y.float().sum().backward()
        del alive
        call().float().sum().backward()
    side.synchronize()
    assert unrelated.requires_grad


@pytest.mark.gpu
@pytest.mark.parametrize("form", ["adapters", "staged", "staged bf16x3", "staged poses"])
def test_the_staged_passes_in_a_captured_step_follow_tau(form):
    """GraphedTrainStep over the passes that are composed one by one -- an adapted render, and the staged route of a plain one (with pose
    gradients too) -- while the schedule moves tau and the learning rate every iteration: bit for bit the eager steps"""
    import test_graph_step as tg
    optim = importlib.import_module("a-nerf_amd.optim")
    graph_step, render_mod = importlib.import_module("a-nerf_amd.graph_step"), importlib.import_module("a-nerf_amd.render")
    dev, n_rays, n_iter = torch.device("cuda"), 96, 7
    runs = []
    for mode in ("eager", "graph"):
        torch.manual_seed(7)
        caster, opt, popt, st = tg._setup(form == "staged poses", n_rays, dev)
        subjects = None
        if form == "adapters":
            opt.detach()
            caster.requires_grad_(False)
            ads = [ad.NetAdapters(net, 3, rank=4) for net in (caster.network, caster.network_fine)]
            with torch.no_grad():
                for a in ads:
                    for name in ad.LAYERS:
                        a.up(name).normal_(0, 0.05)
            caster.set_adapters(*ads)
            opt = optim.FusedAdam([p for a in ads for p in a.parameters()], lr=5e-4)
            opt.materialize()
            subjects = torch.arange(n_rays, device=dev) % 4
        else:
            opt.detach()
            caster.train_route = "staged"
            caster.train_precision = "bf16x3" if form.endswith("bf16x3") else "fp32"

        def iteration(k):
            b, cams = st["batch"], None
            if popt is not None:
                kp, bones, skts, _, _ = popt(st["pidx"])
                b, cams = dict(b, kp_batch=kp, skts=skts, bones=bones), torch.zeros(n_rays, device=dev)
            out = render_mod.render(512, 512, 600.0, chunk=4096, rays=st["rays"], use_viewdirs=True, ray_caster=caster, cams=cams, subject_idxs=subjects,
                                    N_samples=32, N_importance=16, perturb=1.0, raw_noise_std=1.0,
                                    preproc_kwargs={"density_scale": 1.0, "density_fn": torch.nn.functional.relu}, **b)
            loss, _ = optim.fused_nerf_loss(out, st["target"], bgs=1.0, loss_fn="MSE")
            optim.backward(loss)
            opt.step(zero_grad=True, i=k)
            return {"loss": loss, "rgb": out["rgb_map"]}

        gs = graph_step.GraphedTrainStep(iteration, caster, opt, eager_steps=2, enabled=mode == "graph")
        trace = []
        for k in range(1, n_iter + 1):
            tg._schedule(caster, opt, k)
            out = gs.step(k)
            trace.append((out["loss"].detach().clone(), out["rgb"].detach().clone()))
        torch.cuda.synchronize()
        runs.append((trace, opt.flat.clone(), gs))
    (e, ef, _), (g, gf, gs) = runs
    assert gs.replays >= 3 and not gs.eager_only, gs.eager_only
    for k, (a, b) in enumerate(zip(e, g)):
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1]), k + 1
    assert torch.equal(ef, gf)


def test_the_dev_forms_of_the_staged_passes_refuse():
    import ctypes
    lib_mod = importlib.import_module("a-nerf_amd._lib")
    lib, cc, P = lib_mod.load(), ops.PathConfig().c(), ctypes.c_void_p(0x7F0000001000)          # never read: every call returns before its launch
    sv = lib_mod.AnerfSaved(P, P, P, P, P, 128)
    fwd = lambda prec=0, block=P, packed=P, saved=sv, s=16: lib.anerf_mlp_raw_train_dev(ctypes.byref(cc), prec, packed, P, P, 11, P, P, 0, None, None, 0, block, P, P, 4, s,
                                                                                      P, ctypes.byref(saved), None)
    for prec in (0, 1):
        assert fwd(prec, block=None) == -3 and fwd(prec, packed=None) == -3 and fwd(prec, s=4) == -2 and fwd(prec, s=100) == -4
    assert fwd(2) == -1
    bwd = lambda block=P, dx=P, stride=384, n=4: lib.anerf_encode_backward_dev(ctypes.byref(cc), dx, P, P, 11, P, P, stride, block, P, P, n, 16, P, P, P, None)
    assert bwd(block=None) == -3 and bwd(dx=None) == -3 and bwd(stride=0) == -2 and bwd(n=0) == 0


def _plan_stub():
    buf = torch.zeros(64, dtype=torch.int32)
    return ops.RowPlan(buf, 4, 1, 3, (4,))


def test_forward_mode_is_refused_not_dropped(monkeypatch):
    """a dual tensor does not `require grad`: its tangent must not vanish (the launches are stubbed: nothing is computed)"""
    import torch.autograd.forward_ad as fw
    calls = []
    monkeypatch.setattr(ops, "dispatch_rows", lambda x, plan, w=None: calls.append(1) or torch.zeros(4, 8))
    monkeypatch.setattr(ops, "combine_rows", lambda z, plan, w=None: calls.append(1) or torch.zeros(4, 8))
    monkeypatch.setattr(ops, "_adapter_linear", lambda *a, **k: calls.append(1) or (torch.zeros(4, 6), torch.zeros(4, 16)))
    monkeypatch.setattr(ops, "_adapter_linear_few", lambda *a, **k: calls.append(1) or torch.zeros(4, 6))
    monkeypatch.setattr(ops, "_route_rows", lambda *a: _plan_stub())
    monkeypatch.setattr(ad, "_check_tensors", lambda *a: None)                   # (tensors on the CPU are refused there)
    plan, r = _plan_stub(), torch.randn
    x, w, W, A, B, b, s = r(4, 8), r(4, 1), r(6, 8), r(3, 2, 8), r(3, 6, 2), r(6), torch.ones(3)
    idx = torch.zeros(4, dtype=torch.long)
    lin = lambda **k: ad.adapter_linear(**{**dict(x=x, weight=W, down=A, up=B, rows=plan, bias=b, scale=s), **k})
    with fw.dual_level():
        d = lambda t: fw.make_dual(t, torch.ones_like(t))
        cases = [lambda: ad.dispatch_rows(d(x), plan), lambda: ad.combine_rows(d(x), plan), lambda: ad.combine_rows(x, plan, d(w))]
        for rows in (plan, idx):
            cases += [lambda k=k, t=t, rows=rows: lin(rows=rows, **{k: d(t)}) for k, t in (("x", x), ("weight", W), ("down", A), ("up", B), ("bias", b), ("scale", s))]
        for i, f in enumerate(cases):
            for grad in (True, False):                                           # no_grad does not switch forward mode off
                with pytest.raises((NotImplementedError, RuntimeError)), torch.set_grad_enabled(grad):
                    f()
                    pytest.fail(f"case {i} answered without its tangent", pytrace=False)
        # and calls without a tangent run there as anywhere
        n = len(calls)
        ad.dispatch_rows(x, plan), ad.combine_rows(x, plan, w), lin(), lin(rows=idx)
        assert len(calls) == n + 4


@pytest.mark.gpu
def test_adapters_train_through_the_graphed_trainer():
    """Trainer.enable_graph over attached adapters and a FusedAdam of them, tau and the learning rate scheduled by the trainer itself, an exchange
    of the adapters in the middle: bit for bit the eager trainer"""
    import numpy as np
    import test_trajectory as tj
    synth, optim = importlib.import_module("a-nerf_amd.synth"), importlib.import_module("a-nerf_amd.optim")
    case, dev = tj.CASES["surreal"], torch.device("cuda")
    args = tj.ref_args(case["args"])
    args.cutoff_step, args.cutoff_rate = 1, 1.05                                   # tau = 20 * 1.05 ^ (i / 1000): 500 steps of fp32 an iteration
    data_attrs = {"skel_type": tj.Skel, "near": 0.0, "far": 1.0, "n_views": tj.N_POSES, "hwf": (512, 512, 600.0),
                  "joint_coords": np.tile(np.eye(3, dtype=np.float32), (24, 1, 1))}
    runs = []
    for graphed in (False, True):
        torch.manual_seed(5)
        rk_train, rk_test, _, _, _, _ = raycaster.create_raycaster(args, data_attrs, device=dev)
        caster = rk_test["ray_caster"]
        for net, seed in ((caster.network, case["seeds"][0]), (caster.network_fine, case["seeds"][1])):
            net.load_state_dict({k: torch.tensor(v) for k, v in synth.make_net_params(seed, args.multires, args.multires_views, 0, tj.N_POSES).items()})
        caster.train().requires_grad_(False)
        caster._rng = ops.DeviceRng(seed=77, stream_id=1)
        sets = [[ad.NetAdapters(net, 3, rank=4) for net in (caster.network, caster.network_fine)] for _ in range(2)]
        opt = optim.FusedAdam([p for ads in sets for a in ads for p in a.parameters()], lr=1e-3)
        opt.materialize()
        tr = trainer.Trainer(args, data_attrs, opt, None, rk_train, rk_test, popt_kwargs=None, device=dev)
        if graphed:
            tr.enable_graph(eager_steps=1)
        batch = tj._batch(case, dev)
        n = case["n"]
        losses = []
        for i in range(1, 13):
            caster.set_adapters(*sets[0 if i <= 4 or i > 8 else 1])
            batch["subject_idxs"] = (torch.arange(n, device=dev) * i) % 4
            loss, _ = tr.train_batch(batch, i=i, global_step=i)
            losses.append(loss["total_loss"].detach().clone())
        torch.cuda.synchronize()
        runs.append((losses, opt.flat.clone(), tr, caster))
    (e, ef, _, ec), (g, gf, tr, gc_) = runs
    assert not tr._gs.eager_only and tr._gs.captures == 2 and tr._gs.replays >= 8, (tr._gs.eager_only, tr._gs.captures, tr._gs.replays)
    assert all(torch.equal(a, b) for a, b in zip(e, g)) and torch.equal(ef, gf) and len({float(v) for v in e}) == 12
    assert gc_.embed_fn.get_tau() == ec.embed_fn.get_tau() == float(np.float32(20.0 * 1.05 ** 0.012))
