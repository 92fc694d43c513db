"""Cases of the row-routing and low-rank-adapter operators: what they cost, and what they have to answer.

A radiance network that serves many subjects keeps ONE set of shared weights and a pair of thin matrices per subject and
layer.  A batch holds the rows of many subjects at once, so the rows are put in order of their subject, go through the layers,
and come back (`route_rows`, `dispatch_rows`, `combine_rows`), and each layer is the shared projection with the row's own
low-rank term beside it (`adapter_linear`).  The same operators are what a mixture of experts and a server of many fine-tuned
copies of one language model run; the cases hold sizes of both.

Kinds of a case
  sort        plan of the rows' groups and the rows in group order            (forward)
  sort_grad   the rows out and back with weights, and the gradients of both   (forward + backward)
  adapter     y = x W^T + b + scale (x A_i^T) B_i^T, i the row's adapter       (forward)
  adapter_grad  the same with the gradients of x, A and B                     (forward + backward; W and b are frozen)
"""
import importlib
import math

import numpy as np
import torch

own = False

DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
BYTES = {"fp32": 4, "bf16": 2, "fp16": 2}

X_COLS, WIDTH = 432, 256      # the radiance network's encoded input and its layers


# ---------------------------------------------------------------------------------------------------------------- cases
def listed():
    return [
        # one decoding step of a small mixture: 33 tokens, two experts each; all of it is launch latency
        dict(name="sort_step", kind="sort", rows=33, k=2, groups=8, width=256, dtype="fp32", none=0.0),
        # the encoded sample points of 819 rays, 80 samples each, by subject
        dict(name="sort_points", kind="sort", rows=65520, k=1, groups=16, width=1080, dtype="fp32", none=0.02),
        # a wide mixture's prefill: 8 of 128 experts a token
        dict(name="sort_wide", kind="sort", rows=8192, k=8, groups=128, width=2048, dtype="bf16", none=0.0),
        # a training step's rows at odd sizes, some pairs dropped
        dict(name="sort_grad_odd", kind="sort_grad", rows=6001, k=3, groups=24, width=1001, dtype="fp16", none=0.05),
        # a training step of a mixture: 4 of 64 experts a token
        dict(name="sort_grad", kind="sort_grad", rows=16384, k=4, groups=64, width=1024, dtype="bf16", none=0.0),
        # one token of one request: the shared weight is read once and nothing else counts
        dict(name="adapter_one", kind="adapter", rows=1, cin=4096, cout=4096, adapters=32, rank=16, dtype="bf16", none=0.0, bias=False),
        # one decoding step of 48 requests, hardly two with the same adapter, some with none
        dict(name="adapter_step", kind="adapter", rows=48, cin=4096, cout=8192, adapters=64, rank=16, dtype="bf16", none=0.1, bias=False),
        # a prefill of many requests
        dict(name="adapter_prefill", kind="adapter", rows=8192, cin=4096, cout=4096, adapters=24, rank=32, dtype="bf16", none=0.05, bias=False),
        # odd sizes throughout
        dict(name="adapter_odd", kind="adapter", rows=1021, cin=1111, cout=777, adapters=5, rank=12, dtype="fp16", none=0.2, bias=True),
        # the skip layer of the radiance network over the points of 819 rays of 16 subjects
        dict(name="adapter_points", kind="adapter", rows=65520, cin=X_COLS + WIDTH, cout=WIDTH, adapters=16, rank=8, dtype="fp32", none=0.0, bias=True),
        # a training step of 12 adapters at once
        dict(name="adapter_grad", kind="adapter_grad", rows=4096, cin=2048, cout=2048, adapters=12, rank=16, dtype="bf16", none=0.0, bias=False),
        # fine-tuning 8 subjects together: the network's skip layer over the points of 300 rays, 80 samples each
        dict(name="adapter_grad_points", kind="adapter_grad", rows=24000, cin=X_COLS + WIDTH, cout=WIDTH, adapters=8, rank=8, dtype="fp32", none=0.0, bias=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["sort", "sort_grad", "adapter", "adapter_grad"])
    dtype = rng.choice(["fp32", "bf16", "fp16"])
    none = rng.choice([0.0, 0.0, 0.03, 0.3])
    if kind in ("sort", "sort_grad"):
        k, width = rng.randint(1, 8), _log(rng, 3, 2048)
        most = (120 << 20 if kind == "sort" else 64 << 20) // (width * k * BYTES[dtype])
        return dict(kind=kind, rows=_log(rng, 1, max(1, min(65536, most))), k=k, groups=_log(rng, 1, 256), width=width, dtype=dtype, none=none)
    cin, cout = _log(rng, 16, 4096), _log(rng, 1 if kind == "adapter" else 16, 4096)
    adapters = _log(rng, 1, 64)
    rank = min(_log(rng, 1, 64), 1024 // adapters)
    most = int((10e9 if dtype == "fp32" else 40e9) / (2 * cin * cout))
    return dict(kind=kind, rows=_log(rng, 1, max(1, min(65536, most, (128 << 20) // (4 * (cin + cout))))), cin=cin, cout=cout, adapters=adapters,
                rank=rank, dtype=dtype, none=none, bias=rng.random() < 0.5)


def work(case):
    c, kind = case, case["kind"]
    if kind in ("sort", "sort_grad"):
        es, pairs = BYTES[c["dtype"]], c["rows"] * c["k"]
        plan = 8 * pairs + 4 * (2 * pairs + c["groups"] + 1)
        one, many = c["rows"] * c["width"] * es, pairs * c["width"] * es
        if kind == "sort":
            return {"bytes": plan + one + many, "flops": 0}
        # x, z, gxs, gy, w in; xs, y, dx, dz, dw out
        return {"bytes": plan + 4 * one + 4 * many + 8 * pairs, "flops": 8 * pairs * c["width"]}
    es, m, ci, co, r = BYTES[c["dtype"]], c["rows"], c["cin"], c["cout"], c["rank"]
    used = min(c["adapters"], m)
    thin = used * r * (ci + co)
    if kind == "adapter":
        return {"bytes": es * (m * (ci + co) + ci * co + thin) + 8 * m, "flops": 2 * m * ci * co + 2 * m * r * (ci + co)}
    return {"bytes": es * (2 * m * (ci + co) + ci * co + thin + c["adapters"] * r * (ci + co)) + 8 * m,
            "flops": 4 * m * ci * co + 6 * m * r * (ci + co)}


# --------------------------------------------------------------------------------------------------------------- inputs
def _groups(gen, shape, n, none, dev):
    """group of every row: popular groups and rare ones, as requests and subjects come; `none` of them in no group"""
    u = torch.rand(shape, generator=gen, device=dev)
    idx = (u * u * n).long().clamp_(max=n - 1)
    order = torch.randperm(n, generator=gen, device=dev)
    idx = order[idx]
    if none:
        idx = torch.where(torch.rand(shape, generator=gen, device=dev) < none, torch.full_like(idx, -1), idx)
    return idx


def _inputs(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed * 7919 + 17)
    dt = DTYPES[case["dtype"]]
    normal = lambda *shape, s=1.0, t=None: (torch.randn(*shape, generator=gen, device=dev) * s).to(dt if t is None else t)
    c, s = case, {}
    if c["kind"] in ("sort", "sort_grad"):
        s["idx"] = _groups(gen, (c["rows"], c["k"]), c["groups"], c["none"], dev)
        s["x"] = normal(c["rows"], c["width"])
        if c["kind"] == "sort_grad":
            pairs = c["rows"] * c["k"]
            s["z"], s["gxs"] = normal(pairs, c["width"]), normal(pairs, c["width"])
            s["gy"] = normal(c["rows"], c["width"])
            s["w"] = torch.softmax(torch.randn(c["rows"], c["k"], generator=gen, device=dev), -1)
        return s
    m, ci, co, n, r = c["rows"], c["cin"], c["cout"], c["adapters"], c["rank"]
    s["idx"] = _groups(gen, (m,), n, c["none"], dev)
    s["x"], s["weight"] = normal(m, ci), normal(co, ci, s=1 / math.sqrt(ci))
    s["bias"] = normal(co, s=0.2) if c["bias"] else None
    s["down"], s["up"] = normal(n, r, ci, s=1 / math.sqrt(ci)), normal(n, co, r, s=0.5 / math.sqrt(r))
    if c["kind"] == "adapter_grad":
        s["g"] = normal(m, co)
    return s


SCALE = 1.5


def prepare(case, seed):
    s = _inputs(case, seed)
    s["case"] = case
    if own:
        s["lib"] = importlib.import_module("a-nerf_amd.adapters")
        if case["kind"] == "sort_grad":
            s["x"].requires_grad_()
            s["z"].requires_grad_()
            s["w"].requires_grad_()
        if case["kind"] == "adapter_grad":
            for k in ("x", "down", "up"):
                s[k].requires_grad_()
    return s


# ------------------------------------------------------------------------------------------------------------- plain form
def _plain_plan(idx, n):
    g = idx.reshape(-1)
    g = torch.where((g >= 0) & (g < n), g, torch.full_like(g, n))
    count = (torch.arange(n + 1, device=g.device)[:, None] == g).to(torch.int32).cumsum(1, dtype=torch.int32)
    start = torch.cat([torch.zeros(1, dtype=torch.int32, device=g.device), count[:, -1].cumsum(0, dtype=torch.int32)])
    slot = start[g] + count.gather(0, g[None])[0] - 1
    pairs = torch.arange(g.numel(), dtype=torch.int32, device=g.device)
    source = torch.empty_like(slot).scatter_(0, slot.long(), pairs)
    return start[:n + 1], source, slot.view(idx.shape)


def _plain_dispatch(x, offsets, source, k):
    kept = torch.arange(source.numel(), device=x.device) < offsets[-1]
    return torch.where(kept[:, None], x[(source // k).long()], torch.zeros((), dtype=x.dtype, device=x.device))


def _plain_combine(z, offsets, slot, w):
    kept = slot < offsets[-1]
    rows = torch.where(kept[..., None], z[slot.long()].float(), torch.zeros((), device=z.device))
    return rows if w is None else rows * torch.where(kept, w, torch.zeros_like(w))[..., None]


def _plain_pick(idx, n):
    """[rows, n] of 0 and 1: the row's adapter"""
    return (idx[:, None] == torch.arange(n, device=idx.device)).float()


def _plain_linear(x, weight, bias, down, up, pick):
    """the sum in 32 bits: every adapter's thin product, the row's own one picked, spread, and multiplied up"""
    n, r, ci = down.shape
    h = ((x @ down.reshape(n * r, ci).t()).view(-1, n, r) * pick[..., None]).reshape(-1, n * r)
    y = x @ weight.t() + SCALE * (h @ up.permute(0, 2, 1).reshape(n * r, -1))
    return y if bias is None else y + bias


def _run_plain(s):
    c = s["case"]
    if c["kind"] == "sort":
        offsets, source, slot = _plain_plan(s["idx"], c["groups"])
        return {"offsets": offsets, "source": source, "slot": slot, "rows": _plain_dispatch(s["x"], offsets, source, c["k"])}
    if c["kind"] == "sort_grad":
        offsets, source, slot = _plain_plan(s["idx"], c["groups"])
        dt = s["x"].dtype
        kept = slot < offsets[-1]
        rows = _plain_dispatch(s["x"], offsets, source, c["k"])
        y = _plain_combine(s["z"], offsets, slot, s["w"]).sum(1).to(dt)
        dx = _plain_combine(s["gxs"], offsets, slot, None).sum(1).to(dt)
        dw = (_plain_combine(s["z"], offsets, slot, None) * s["gy"].float()[:, None]).sum(-1)
        wk = torch.where(kept, s["w"], torch.zeros_like(s["w"])).reshape(-1)[source.long()]
        dz = (s["gy"][(source // c["k"]).long()].float() * wk[:, None]).to(dt)
        return {"rows": rows, "y": y, "dx": dx, "dz": dz, "dw": dw}
    dt = s["x"].dtype
    n, r, ci = s["down"].shape
    pick = _plain_pick(s["idx"], n)
    x, weight, down, up = s["x"].float(), s["weight"].float(), s["down"].float(), s["up"].float()
    y = _plain_linear(x, weight, None if s["bias"] is None else s["bias"].float(), down, up, pick).to(dt)
    if c["kind"] == "adapter":
        return {"y": y}
    g = s["g"].float()
    co = g.shape[1]
    spread = lambda t: (t.view(-1, n, r) * pick[..., None]).reshape(-1, n * r)
    h = spread(x @ down.reshape(n * r, ci).t())
    u = SCALE * spread(g @ up.permute(1, 0, 2).reshape(co, n * r))
    dx = g @ weight + u @ down.reshape(n * r, ci)
    return {"y": y, "dx": dx.to(dt), "ddown": (u.t() @ x).view(n, r, ci).to(dt),
            "dup": (SCALE * (h.t() @ g)).view(n, r, co).permute(0, 2, 1).contiguous().to(dt)}



# ------------------------------------------------------------------------------------------------- the framework's kernels
def _run_own(s):
    c, lib = s["case"], s["lib"]
    if c["kind"] == "sort":
        with torch.no_grad():
            plan = lib.route_rows(s["idx"], c["groups"])
            return {"offsets": plan.offsets, "source": plan.source, "slot": plan.slot, "rows": lib.dispatch_rows(s["x"], plan)}
    if c["kind"] == "sort_grad":
        plan = lib.route_rows(s["idx"], c["groups"])
        rows = lib.dispatch_rows(s["x"], plan)
        y = lib.combine_rows(s["z"], plan, s["w"])
        dx, dz, dw = torch.autograd.grad([rows, y], [s["x"], s["z"], s["w"]], [s["gxs"], s["gy"]])
        return {"rows": rows.detach(), "y": y.detach(), "dx": dx, "dz": dz, "dw": dw}
    if c["kind"] == "adapter":
        with torch.no_grad():
            return {"y": lib.adapter_linear(s["x"], s["weight"], s["down"], s["up"], s["idx"], bias=s["bias"], scale=SCALE)}
    y = lib.adapter_linear(s["x"], s["weight"], s["down"], s["up"], s["idx"], bias=s["bias"], scale=SCALE)
    dx, dd, du = torch.autograd.grad(y, [s["x"], s["down"], s["up"]], s["g"])
    return {"y": y.detach(), "dx": dx, "ddown": dd, "dup": du}


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ----------------------------------------------------------------------------------------------------------------- exact
def _exact_plan(idx, n):
    g = idx.reshape(-1).cpu().numpy()
    g = np.where((g < 0) | (g >= n), n, g)
    source = np.argsort(g, kind="stable")
    slot = np.empty_like(source)
    slot[source] = np.arange(len(g))
    offsets = np.searchsorted(g[source], np.arange(n + 1), side="left")
    return offsets, source, slot


def _exact_rows(s, n):
    """adapter -> its rows"""
    idx = s.cpu().numpy()
    return [torch.from_numpy(np.nonzero(idx == i)[0]).to(s.device) for i in range(n)]


def exact(case, seed):
    c, s = case, _inputs(case, seed)
    dev = s["x"].device
    put = lambda a: torch.from_numpy(np.ascontiguousarray(a)).to(dev)
    if c["kind"] in ("sort", "sort_grad"):
        offsets, source, slot = _exact_plan(s["idx"], c["groups"])
        kept, k = int(offsets[-1]), c["k"]
        token = put(source[:kept] // k)
        rows = torch.zeros(len(source), c["width"], dtype=torch.float64, device=dev)
        rows[:kept] = s["x"][token].double()
        if c["kind"] == "sort":
            ints = lambda a: put(a.astype(np.int32))
            return {"offsets": ints(offsets), "source": ints(source), "slot": ints(slot).view(s["idx"].shape), "rows": rows}
        w = s["w"].reshape(-1)[put(source[:kept])].double()[:, None]
        y = torch.zeros(c["rows"], c["width"], dtype=torch.float64, device=dev).index_add_(0, token, s["z"][:kept].double() * w)
        dx = torch.zeros_like(y).index_add_(0, token, s["gxs"][:kept].double())
        gy = s["gy"].double()[token]
        dz = torch.zeros_like(rows)
        dz[:kept] = gy * w
        dw = torch.zeros(len(source), dtype=torch.float64, device=dev)
        dw[put(source[:kept])] = (gy * s["z"][:kept].double()).sum(1)
        return {"rows": rows, "y": y, "dx": dx, "dz": dz, "dw": dw.view(s["idx"].shape)}
    n = c["adapters"]
    x, weight = s["x"].double(), s["weight"].double()
    y = x @ weight.t()
    if s["bias"] is not None:
        y += s["bias"].double()
    grad = c["kind"] == "adapter_grad"
    if grad:
        g = s["g"].double()
        dx = g @ weight
        ddown, dup = torch.zeros(s["down"].shape, dtype=torch.float64, device=dev), torch.zeros(s["up"].shape, dtype=torch.float64, device=dev)
    for i, rows in enumerate(_exact_rows(s["idx"], n)):
        if not len(rows):
            continue
        a, b = s["down"][i].double(), s["up"][i].double()
        xi = x[rows]
        y[rows] += SCALE * (xi @ a.t()) @ b.t()
        if grad:
            gi = g[rows]
            u = SCALE * gi @ b
            dx[rows] += u @ a
            ddown[i], dup[i] = u.t() @ xi, SCALE * gi.t() @ (xi @ a.t())
    return {"y": y, "dx": dx, "ddown": ddown, "dup": dup} if grad else {"y": y}
