"""CPU: nothing that outlives an iteration holds its autograd graph (one that lives through the next capture ends the process there)."""
import importlib
import types
import typing
import weakref

import torch

graph_step = importlib.import_module("a-nerf_amd.graph_step")


class _Probe(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, token):
        ctx.token = token
        return x * 1.0

    @staticmethod
    def backward(ctx, g):
        return g, None


class _Token:
    pass


class _Named(typing.NamedTuple):
    y: torch.Tensor
    n: int


def test_results_of_eager_iterations_hold_no_graph():
    w = torch.ones(3, requires_grad=True)
    alive = []

    def step_fn(i):
        token = _Token()
        alive.append(weakref.ref(token))
        y = _Probe.apply(w, token)
        loss = (y * i).sum()
        loss.backward()
        return {"loss": loss, "more": {"maps": [y, (y + 1,)], "n": i, "none": None, "named": _Named(y, i)}}

    emb = types.SimpleNamespace()
    for kw in (dict(enabled=False), dict(eager_steps=5)):
        gs = graph_step.GraphedTrainStep(step_fn, types.SimpleNamespace(embed_fn=emb, embeddirs_fn=emb), types.SimpleNamespace(_due=lambda i: [0], param_groups=[{}]), **kw)
        out = gs.step(2)
        assert alive[-1]() is None                                             # the iteration's graph is gone although its results live
        tensors = [out["loss"], out["more"]["maps"][0], out["more"]["maps"][1][0]]
        assert not any(t.requires_grad for t in tensors) and float(out["loss"]) == 6.0 and torch.equal(tensors[2], torch.full((3,), 2.0))
        assert out["more"]["n"] == 2 and out["more"]["none"] is None and type(out["more"]["named"]) is _Named and not out["more"]["named"].y.requires_grad


def test_the_pose_layer_drops_its_last_graph_before_it_builds_the_next(monkeypatch):
    import numpy as np
    pose_opt = importlib.import_module("a-nerf_amd.pose_opt")
    layer = pose_opt.PoseOptLayer(torch.rand(3, 24, 3), torch.rand(3, 24, 3), torch.rand(1, 24, 3))
    alive, seen = [], []

    def kinematic(bones, pelvis, rest):
        seen.append([r() is not None for r in alive])
        token = _Token()
        alive.append(weakref.ref(token))
        y = _Probe.apply(bones, token)
        return y, y * 2, y * 3, y * 4

    monkeypatch.setattr(pose_opt, "calculate_kinematic", kinematic)
    for _ in range(3):
        sum(t.sum() for t in layer(np.array([0, 2, 2]))).backward()
    assert seen == [[], [False], [False, False]] and layer.last_unique["rots"].shape[0] == 2
