"""Adapters in training: gradients over several ranks (CPU, gloo)."""
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
raycaster = importlib.import_module("a-nerf_amd.raycaster")
trainer = importlib.import_module("a-nerf_amd.trainer")


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
