"""One set of shared weights for many subjects: rows put in order of their subject and back, and projections with a low-rank adapter
of its own for every row.

The reference fine-tunes a whole network per subject (its *_finetune configurations).  Here a subject is a pair of thin matrices
beside every shared layer, and a batch may hold rows of many subjects:

    plan = route_rows(subject_idxs, n_subjects)           # stable sort of the rows by subject, on the device
    xs   = dispatch_rows(x, plan)                         # the rows in that order
    ys   = adapter_linear(xs, W, A, B, plan.sorted(), b)  # x W^T + b + scale (x A_i^T) B_i^T, layer after layer
    y    = combine_rows(ys, plan, weights)                # back, the k groups of a row added with their weights

`adapter_linear` also takes rows in any order, with the adapter index of each.  All calls are differentiable (rows, weights, A and B),
enqueue HIP kernels on torch's current stream, and neither allocate outside torch nor wait for the device, so they can be captured.
Row types: float32, bfloat16, float16; sums are held in float32 and rounded once.  The shared projection is frozen: asking for its
gradient is refused.
"""
import math
import threading
import weakref

import torch
import torch.nn as nn
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from . import ops
from .ops import RowPlan, SortedRows, route_rows  # noqa: F401


# A leaf's gradient node belongs to the stream it was first used on, and lives as long as any graph that reaches the leaf.  While an
# EAGER graph of a leaf is alive, a backward that is being captured makes autograd order the capturing stream against that other
# stream -- which a capture does not allow, and the exception ends the process.  The calls below therefore know which of their graphs are
# alive, and refuse such a backward with an exception that can be handled.  (Graphs that hold none of these calls they do not know.)
class _Graph:
    """one call's graph: the leaves among its arguments, the nodes behind the others, and the stream it was built on (alive while autograd
    holds the call's node)"""
    __slots__ = ("leaves", "nodes", "stream", "__weakref__")

    def __init__(self, asking):
        self.leaves, self.nodes = [t for t in asking if t.is_leaf], [t.grad_fn for t in asking if not t.is_leaf]
        self.stream = torch._C._cuda_getCurrentRawStream(torch._C._cuda_getDevice())

    def reach(self):
        """ids of all leaves that the graph gives gradients to (walked where a capture asks for it only)"""
        ids, seen, todo = {id(t) for t in self.leaves}, {}, list(self.nodes)
        while todo:
            node = todo.pop()
            if node is None or node in seen:
                continue
            seen[node] = True
            leaf = getattr(node, "variable", None)
            if leaf is not None:
                ids.add(id(leaf))
            todo += [n for n, _ in node.next_functions]
        return ids


_alive, _alive_lock = weakref.WeakSet(), threading.Lock()


def _graph_of(*tensors):
    asking = [t for t in tensors if t is not None and t.requires_grad]
    if not asking:
        return None
    graph = _Graph(asking)
    with _alive_lock:
        _alive.add(graph)
    return graph


def _capturing():
    return torch.cuda.is_current_stream_capturing()


def _check_capture(graph):
    if graph is None or not _capturing():
        return
    with _alive_lock:
        others = [other for other in _alive if other is not graph and other.stream != graph.stream]
    mine = graph.reach() if others else ()
    if any(not mine.isdisjoint(other.reach()) for other in others):
        raise RuntimeError("this backward is being captured while an eager graph of the same leaf tensor is alive (an output of an eager call that "
                           "is still referenced): drop it before the capture")


def _once(backward):
    """once_differentiable, at its price (10 us of a small step) only where a graph of the backward is asked for"""
    checked = once_differentiable(backward)

    def run(ctx, *grads):
        return checked(ctx, *grads) if torch.is_grad_enabled() else backward(ctx, *grads)
    return run


class _DispatchFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, plan, graph):
        ctx.plan, ctx.graph = plan, graph
        return ops.dispatch_rows(x, plan)

    @staticmethod
    @_once
    def backward(ctx, g):
        _check_capture(ctx.graph)
        return ops.combine_rows(g, ctx.plan), None, None


class _CombineFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, z, weights, plan, graph):
        ctx.plan, ctx.graph = plan, graph
        ctx.save_for_backward(z if weights is not None and ctx.needs_input_grad[1] else None, weights)
        return ops.combine_rows(z, plan, weights)

    @staticmethod
    @_once
    def backward(ctx, g):
        _check_capture(ctx.graph)
        z, weights = ctx.saved_tensors
        if weights is None:
            return ops.dispatch_rows(g, ctx.plan), None, None, None
        dz, dw = ops.combine_rows_backward(g, z, ctx.plan, weights, ctx.needs_input_grad[0], ctx.needs_input_grad[1])
        return dz, dw, None, None


def dispatch_rows(x, plan):
    """x [T, ...] -> [T * k, ...]: row t at the positions plan.slot[t] of its groups; the rows behind the kept ones are zero."""
    _check_plan(plan, "dispatch_rows")
    if not _needs_grad(x):
        return ops.dispatch_rows(x, plan)
    return _DispatchFn.apply(x, plan, _graph_of(x))


def combine_rows(z, plan, weights=None):
    """z [T * k, ...] in group order -> [T, ...]: y[t] = sum_j weights[t, j] * z[plan.slot[t, j]] over the kept pairs (weights None: 1).
    A row whose pairs are all dropped gets zeros; what z or weights hold for a dropped pair is not read."""
    _check_plan(plan, "combine_rows")
    if not _needs_grad(z, weights):
        return ops.combine_rows(z, plan, weights)
    return _CombineFn.apply(z, weights, plan, _graph_of(z, weights))


def _needs_grad(t, w=None):
    return _forward_mode() or torch.is_grad_enabled() and (torch.is_tensor(t) and t.requires_grad or torch.is_tensor(w) and w.requires_grad)


def _forward_mode():
    """inside a level of forward-mode differentiation, whose dual tensors need not require a gradient (and which no_grad does not switch
    off): a call goes through its autograd function there, which refuses tangents instead of losing them"""
    return forward_ad._current_level >= 0


def _check_plan(plan, name):
    if not isinstance(plan, RowPlan):
        raise TypeError(f"{name}: expected the RowPlan of route_rows, got {type(plan).__name__}")


class _AdapterFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, down, up, weight, bias, rows, scale, scale_of, graph):
        y, h = ops._adapter_linear(x, weight, down, up, rows, bias, scale, scale_of)
        ctx.save_for_backward(x, down, up, weight, scale_of, h)
        ctx.rows, ctx.scale, ctx.graph = rows, scale, graph
        return y

    @staticmethod
    @_once
    def backward(ctx, g):
        _check_capture(ctx.graph)
        x, down, up, weight, scale_of, h = ctx.saved_tensors
        if g.stride(-1) != 1 or g.stride(0) < g.shape[1]:
            g = g.contiguous()
        want = ctx.needs_input_grad
        dx, ddown, dup = ops._adapter_backward(g, x, weight, down, up, ctx.rows, h, ctx.scale, scale_of, want[0], want[1], want[2])
        return dx, ddown, dup, None, None, None, None, None, None


def _check_tensors(x, weight, down, up, bias):
    """raises what is wrong with them (asked for after the one-line test of adapter_linear failed)"""
    ops._rows_like(x, "adapter_linear: x")
    for t, name, dim in ((weight, "weight", 2), (down, "down", 3), (up, "up", 3), (bias, "bias", 1)):
        if t is None and name == "bias":
            continue
        ops._rows_like(t, f"adapter_linear: {name}", x.device, x.dtype)
        if t.dim() != dim:
            raise ValueError(f"adapter_linear: {name} must have {dim} dimensions, got {tuple(t.shape)}")


def _like(t, dtype, dev, dim):
    return torch.is_tensor(t) and t.dtype is dtype and t.device == dev and t.ndim == dim


def adapter_linear(x, weight, down, up, rows, bias=None, scale=1.0):
    """y = x W^T + bias + scale_i (x A_i^T) B_i^T for every row of x, i the row's adapter.

    x [..., K]; weight [N, K]; bias [N] or None; down [L, R, K] (A); up [L, N, R] (B), all of one type and on one device.
    rows: the adapter of every row -- an int32 / int64 tensor of x's leading shape (a value outside 0 .. L-1: no adapter, the shared
    projection alone), the RowPlan of such indices (k = 1; worth keeping where several layers see the same rows), or plan.sorted()
    for dispatched rows.  scale: a number, or a float32 tensor [L].
    Gradients: x, A and B; weight and bias are frozen."""
    dtype, dev = getattr(x, "dtype", None), getattr(x, "device", None)
    if not (dtype in ops.ROW_DTYPES and x.is_cuda and _like(weight, dtype, dev, 2) and _like(down, dtype, dev, 3) and _like(up, dtype, dev, 3) and
            (bias is None or _like(bias, dtype, dev, 1))):
        _check_tensors(x, weight, down, up, bias)
    (N, K), (L, R, down_in), grads, lead = weight.shape, down.shape, torch.is_grad_enabled(), x.shape[:-1]
    if x.ndim < 1 or x.shape[-1] != K or down_in != K or up.shape != (L, N, R) or (bias is not None and bias.shape[0] != N):
        raise ValueError(f"adapter_linear: x {tuple(x.shape)}, weight {tuple(weight.shape)}, down {tuple(down.shape)}, up {tuple(up.shape)}" +
                         ("" if bias is None else f", bias {tuple(bias.shape)}") + " do not fit together")
    if N < 1 or K < 1 or L < 1 or R < 1 or L > ops._lib.MAX_GROUPS or R > ops._lib.MAX_RANK:
        raise ValueError(f"adapter_linear: 1 .. {ops._lib.MAX_GROUPS} adapters of rank 1 .. {ops._lib.MAX_RANK} and no empty side, got {tuple(down.shape)}")
    if grads and (weight.requires_grad or (bias is not None and bias.requires_grad)):
        raise ValueError("adapter_linear: weight and bias are frozen beside adapters (requires_grad_(False) them, or detach)")
    grads = grads and (x.requires_grad or down.requires_grad or up.requires_grad) or _forward_mode()
    scale_of = None
    if torch.is_tensor(scale):
        if scale.dtype != torch.float32 or scale.device != dev or tuple(scale.shape) != (L,):
            raise ValueError(f"adapter_linear: scale must be a number or a float32 tensor [{L}] on {dev}")
        if torch.is_grad_enabled() and scale.requires_grad:
            raise ValueError("adapter_linear: scale has no gradient")
        scale, scale_of = 1.0, scale.contiguous()
    flat = x if x.ndim == 2 else x.reshape(-1, K)
    M = flat.shape[0]
    if torch.is_tensor(rows):
        if rows.shape != lead and rows.shape != (M,):
            raise ValueError(f"adapter_linear: {tuple(rows.shape)} adapter indices for rows {tuple(lead)}")
        if rows.device != dev:
            raise ValueError(f"adapter_linear: indices on {rows.device}, rows on {dev}")
        if rows.dtype is not torch.int64 and rows.dtype is not torch.int32:
            raise TypeError(f"adapter_linear: adapter indices must be int32 / int64, got {rows.dtype}")
        few = M <= ops._lib.FEW_ROWS and not grads      # a decoding step: no plan, W streams through once
        rows = rows if rows.ndim == 1 else rows.reshape(-1)
        rows = rows.contiguous() if few else ops._route_rows(rows, M, 1, L)
    elif not isinstance(rows, (RowPlan, SortedRows)):
        raise TypeError(f"adapter_linear: rows must be indices, a RowPlan or its sorted(), got {type(rows).__name__}")
    if flat.stride(1) != 1 or flat.stride(0) < K:
        flat = flat.contiguous()
    weight, down_, up_, bias = weight.contiguous(), down.contiguous(), up.contiguous(), None if bias is None else bias.contiguous()
    scale = float(scale)
    if torch.is_tensor(rows):
        y = ops._adapter_linear_few(flat, weight, down_, up_, rows, bias, scale, scale_of)
        return y if x.ndim == 2 else y.reshape(lead + (N,))
    if rows.n_rows != M or rows.device != dev or rows.k != 1:
        raise ValueError(f"adapter_linear: a plan of {rows.n_rows} rows with {rows.k} group(s) each on {rows.device} for {M} rows on {dev}")
    if rows.n_groups < L:
        raise ValueError(f"adapter_linear: a plan of {rows.n_groups} groups for {L} adapters")
    if grads:
        y = _AdapterFn.apply(flat, down_, up_, weight, bias, rows, scale, scale_of, _graph_of(x, down, up))
    else:
        y = ops._adapter_linear(flat, weight, down_, up_, rows, bias, scale, scale_of, keep_h=False)[0]
    return y if x.ndim == 2 else y.reshape(lead + (N,))


LAYERS = [f"pts_linears.{i}" for i in range(8)] + ["alpha_linear", "feature_linear", "views_linears.0", "rgb_linear"]


class NetAdapters(nn.Module):
    """Low-rank adapters of `n_subjects` subjects beside all twelve layers of a NeRF: A ~ U(+-1/sqrt(in)) and B = 0, so that every subject
    starts as the shared network.  `net.set_adapters(adapters)` attaches them: net(x, subject_idxs=...) then evaluates every row with its
    subject's adapter.  The parameters are this module's own (its state_dict, its optimiser group); the network's are untouched, and
    its checkpoint keeps the reference's keys."""

    def __init__(self, net, n_subjects, rank=8, scale=1.0):
        super().__init__()
        if not 1 <= int(n_subjects) < ops._lib.MAX_GROUPS or not 1 <= int(rank) <= ops._lib.MAX_RANK:
            raise ValueError(f"NetAdapters: 1 .. {ops._lib.MAX_GROUPS - 1} subjects of rank 1 .. {ops._lib.MAX_RANK}, got {n_subjects} and {rank}")
        self.n_subjects, self.rank, self.scale = int(n_subjects), int(rank), float(scale)
        mods = dict(net.named_modules())
        p = net.alpha_linear.weight
        for name in LAYERS:
            out, inp = mods[name].weight.shape
            down = torch.empty(self.n_subjects, self.rank, inp, dtype=p.dtype, device=p.device).uniform_(-1 / math.sqrt(inp), 1 / math.sqrt(inp))
            self.register_parameter("down_" + name.replace(".", "_"), nn.Parameter(down))
            self.register_parameter("up_" + name.replace(".", "_"), nn.Parameter(torch.zeros(self.n_subjects, out, self.rank, dtype=p.dtype, device=p.device)))

    def down(self, name):
        return getattr(self, "down_" + name.replace(".", "_"))

    def up(self, name):
        return getattr(self, "up_" + name.replace(".", "_"))

    def plan(self, subject_idxs):
        """RowPlan of subject_idxs [P] or [P, k]; an index outside 0 .. n_subjects-1 is the shared network (a group of its own, behind the
        subjects': such rows are kept and have no adapter)"""
        if not torch.is_tensor(subject_idxs) or subject_idxs.dtype not in (torch.int32, torch.int64):
            raise TypeError("subject_idxs must be an int32 / int64 tensor")
        known = (subject_idxs >= 0) & (subject_idxs < self.n_subjects)
        return route_rows(torch.where(known, subject_idxs, self.n_subjects), self.n_subjects + 1)

    def forward(self, net, x, subject_idxs, subject_weights=None):
        """The adapted NeRF.forward: x [..., input width] encoded rows, subject_idxs [...] or [..., k] -> raw [..., 4].  k subjects a row: their
        raw outputs added with subject_weights [..., k] (None: added)."""
        lead = tuple(x.shape[:-1])
        P = math.prod(lead)
        if not torch.is_tensor(subject_idxs) or tuple(subject_idxs.shape[:len(lead)]) != lead or subject_idxs.dim() > len(lead) + 1:
            raise ValueError(f"subject_idxs must have shape {lead} or {lead + ('k',)}")
        k = subject_idxs.shape[-1] if subject_idxs.dim() > len(lead) else 1
        if subject_weights is not None:
            if subject_weights.shape != subject_idxs.shape:
                raise ValueError(f"subject_weights {tuple(subject_weights.shape)} for subject_idxs {tuple(subject_idxs.shape)}")
            subject_weights = subject_weights.reshape(P, k)
        plan = self.plan(subject_idxs.reshape(P, k))
        rows = plan.sorted()
        mods = dict(net.named_modules())
        lin = lambda name, v: adapter_linear(v, mods[name].weight, self.down(name), self.up(name), rows, mods[name].bias, self.scale)
        dnet, view = net.dnet_input, net.input_ch_views
        xs = dispatch_rows(x.reshape(P, x.shape[-1]), plan)
        pos, u = xs[:, :dnet], [xs[:, dnet:dnet + view]]
        if net.use_framecode:
            table, cam = net.framecodes.table_for(xs[:, -1], net.training)
            u.append(table[cam.long().clamp(0, table.shape[0] - 1)])      # (as the fused kernels take indices)
        h = pos
        for i in range(net.D):
            h = torch.relu(lin(f"pts_linears.{i}", h))
            if i in net.skips:
                h = torch.cat([pos, h], -1)
        sigma = lin("alpha_linear", h)
        g = torch.relu(lin("views_linears.0", torch.cat([lin("feature_linear", h)] + u, -1)))
        raw = torch.cat([lin("rgb_linear", g), sigma], -1)
        return combine_rows(raw, plan, subject_weights).reshape(lead + (4,))
