"""CPU: what GraphedTrainStep.step hands out holds no autograd graph (one that lives through a capture ends the process there)."""
import importlib
import types
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


def test_results_of_eager_iterations_hold_no_graph():
    w = torch.ones(3, requires_grad=True)
    alive = []

    def step_fn(i):
        token = _Token()
        alive.append(weakref.ref(token))
        y = _Probe.apply(w, token)
        loss = (y * i).sum()
        loss.backward()
        return {"loss": loss, "more": {"maps": [y, (y + 1,)], "n": i, "none": None}}

    emb = types.SimpleNamespace()
    for kw in (dict(enabled=False), dict(eager_steps=5)):
        gs = graph_step.GraphedTrainStep(step_fn, types.SimpleNamespace(embed_fn=emb, embeddirs_fn=emb), types.SimpleNamespace(_due=lambda i: [0], param_groups=[{}]), **kw)
        out = gs.step(2)
        assert alive[-1]() is None                                             # the iteration's graph is gone although its results live
        tensors = [out["loss"], out["more"]["maps"][0], out["more"]["maps"][1][0]]
        assert not any(t.requires_grad for t in tensors) and float(out["loss"]) == 6.0 and torch.equal(tensors[2], torch.full((3,), 2.0))
        assert out["more"]["n"] == 2 and out["more"]["none"] is None
