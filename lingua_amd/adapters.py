"""Low-rank adapters of many requests at once, beside a projection that they share: the projection runs once for all tokens, on whatever
linear serves it (``Fp8Linear``, ``Mxfp4Linear``, ``nn.Linear``), and every token gets its own adapter's product added to it,

    out_t = y_t + scale_i (x_t A_i^T) B_i,   i = index[t]

with a bank of adapters ``a`` [n, rank, in_features] and ``b`` [n, rank, out_features], both with the rank in front: forward and backward pass
then run on the same kernels.  (A checkpoint's second factor, [out_features, rank], is transposed once when it is put into the bank:
``AdaptedLinear.load``.)  ``index`` is on the GPU, one entry a token: tokens of one batch may have different adapters, in any order, or none.

Serving: ``add_lowrank`` on the projection's output.  Training: the same call is differentiable in y, x, a and b, so that several adapters
learn side by side on one batch.  ``add_adapters(model, n, rank)`` puts a bank beside every linear that a filter names; ``Requests`` holds
the index of the running batch, and the order of its tokens, which is made once for all layers.
"""
import re
from typing import Optional, Union

import torch

from . import _lib, ops
from . import float8 as f8
from .swiglu import Fp8FeedForward


class Plan:
    """Tokens by adapter, from ``route``: of use for every call on the same index, number of adapters and shape of tokens."""

    def __init__(self, order, starts, n, shape):
        self.order, self.starts, self.n, self.shape = order, starts, n, tuple(shape)


def route(index: torch.Tensor, n: int) -> Plan:
    """The order of the tokens by adapter for ``index`` (int32 or int64, any shape): 0 .. n - 1, or -1 for a token without an adapter.  Any
    other value makes its token's results NaN (the index lives on the GPU: the host cannot refuse it)."""
    if n < 1:
        raise RuntimeError(f"route: a bank of {n} adapters")
    return Plan(*ops.lowrank_route(index.flatten(), n), n, index.shape)


class LowRankFn(torch.autograd.Function):
    """``add_lowrank`` on 2-D operands."""

    @staticmethod
    def forward(ctx, y, x, a, b, scale, order, starts):
        plan = order, starts
        h = ops.lowrank_shrink(x, a, plan)
        need = ctx.needs_input_grad
        ctx.save_for_backward(x if need[2] else None, a if need[1] else None, b if need[1] or need[2] else None, h if need[3] else None, scale, order, starts)
        ctx.learns = tuple(f8._learns(t) for t in (x, a, b))
        ctx.sizes, ctx.order = (a.shape[0], a.shape[1]), f8._stamp(order)
        return ops.lowrank_expand(y, h, b, scale, plan)

    @staticmethod
    def backward(ctx, gy):
        if gy.dtype != torch.bfloat16:
            raise RuntimeError(f"add_lowrank backward: bf16 gradients required, got {gy.dtype}")
        x, a, b, h, scale, order, starts = ctx.saved_tensors
        f8._unchanged(ctx.order, order, "add_lowrank", "the order of the tokens was")
        plan, (n, r) = (order.contiguous(), starts.contiguous()), ctx.sizes   # (hooks hand them back in any layout)
        need_y, need_x, need_a, need_b = ctx.needs_input_grad[:4]
        gx = ga = gb = None
        varies = f8._learns(gy)
        with torch.no_grad():
            sides = []
            together = need_b and (need_x or need_a) and ops.lowrank_outer_shrink_pays(gy.shape[0], r, gy.shape[1])
            if need_x or need_a:
                if together:
                    gb, gh = ops.lowrank_outer_shrink(h, gy, b, scale, plan)
                else:
                    gh = ops.lowrank_shrink(gy, b, plan)
                if need_x:
                    gx = ops.lowrank_expand(None, gh, a, scale, plan)
                if need_a:
                    sides.append((gh, x))
            if need_b and not together:
                sides.append((h, gy))
            if sides:
                grads = ops.lowrank_outer(sides, scale, n, r, plan)
                gb = grads.pop() if need_b and not together else gb
                ga = grads.pop() if need_a else None
        lx, la, lb = ctx.learns
        gx, ga, gb = f8._once("add_lowrank", (gx, ga, gb), (varies or la or lb, varies or lx or lb, varies or lx or la))
        return (gy if need_y else None), gx, ga, gb, None, None, None


def add_lowrank(y: torch.Tensor, x: torch.Tensor, a: torch.Tensor, b: torch.Tensor, index: Union[torch.Tensor, Plan], scale: Optional[torch.Tensor] = None):
    """``y + scale[i] * (x @ a[i].T) @ b[i]`` for every token, i its entry of ``index``; differentiable in y, x, a and b.

    ``y``      bf16 [..., N], the shared projection's output
    ``x``      bf16 [..., K], its input
    ``a, b``   bf16 [n, r, K] and [n, r, N]; r a multiple of 8 up to 128, K and N multiples of 8
    ``index``  int32 or int64 of the tokens' shape, or the ``Plan`` that ``route`` made of it; a token with -1 has no adapter
    ``scale``  fp32 [n], or None for ones; no gradient flows to it: one that asks for a gradient is an error
    """
    what = "add_lowrank"
    planned = isinstance(index, Plan)
    if f8._native_call(x, 0) and f8._plain_call() and (not planned or (index.n == a.shape[0] and index.shape == x.shape[:-1])):
        at = (None, index.order, index.starts) if planned else (index, None, None)
        out = _lib.native_for(x.get_device()).add_lowrank(y, x, a, b, scale, *at)
        if out is not None:
            return out
    if scale is not None and scale.requires_grad and torch.is_grad_enabled():
        raise RuntimeError(f"{what}: the scale asks for a gradient, and none flows to it")
    if a.dim() != 3 or b.dim() != 3 or a.shape[:2] != b.shape[:2] or x.dim() < 1 or y.dim() < 1 or x.shape[-1] != a.shape[2] or y.shape[-1] != b.shape[2]:
        raise RuntimeError(f"{what}: factors {tuple(a.shape)} and {tuple(b.shape)} do not fit an input {tuple(x.shape)} and an output {tuple(y.shape)}")
    for t in (y, x, a, b):
        if t.dtype != torch.bfloat16:
            raise RuntimeError(f"{what}: bf16 operands required, got {t.dtype}")
        if t.device != x.device:
            raise RuntimeError(f"{what}: operands on {t.device} and {x.device}")
    if a.shape[1] % 8 or not 8 <= a.shape[1] <= 128 or a.shape[2] % 8 or b.shape[2] % 8:
        raise RuntimeError(f"{what}: a rank that is a multiple of 8 up to 128 and features that are multiples of 8 are wanted, got {tuple(a.shape)} and {tuple(b.shape)}")
    if x.shape[:-1] != y.shape[:-1] or tuple(index.shape) != x.shape[:-1]:
        raise RuntimeError(f"{what}: x {tuple(x.shape)}, y {tuple(y.shape)} and the index {tuple(index.shape)} are not of the same tokens")
    if planned:
        if index.n != a.shape[0]:
            raise RuntimeError(f"{what}: the plan is for {index.n} adapters, the bank holds {a.shape[0]}")
    elif index.device != x.device:
        raise RuntimeError(f"{what}: the index is on {index.device}, the operands on {x.device}")
    f8._refuse_captured(y, x, a, what)
    f8._refuse_captured(b, None, None, what)
    if not planned and not (torch.is_grad_enabled() and any(t.requires_grad for t in (y, x, a, b))) and f8._plain_call():
        out = ops.lowrank_add(y.reshape(-1, y.shape[-1]), x.reshape(-1, x.shape[-1]), a, b, index.flatten(), scale)
        return out.view(y.shape)
    plan = index if planned else route(index, a.shape[0])
    if y.dim() == 2:
        return LowRankFn.apply(y, x, a, b, scale, plan.order, plan.starts)
    tokens = y.shape[:-1]
    out = LowRankFn.apply(y.reshape(-1, y.shape[-1]), x.reshape(-1, x.shape[-1]), a, b, scale, plan.order, plan.starts)
    return out.view(*tokens, y.shape[-1])


class Requests:
    """Which adapter each token of the running batch has, shared by the banks of a model: ``set`` it before a forward pass, and not again before
    that pass's backward pass is done (which would be an error, also where ``torch.utils.checkpoint`` computes the forward pass again; with
    ``use_reentrant=True`` nothing is kept of that pass, and what the last one went by has to do).  Without an index (``set(None)``) the adapters are left out.

    The order of the tokens is written to the same memory for every batch of one shape, so that a captured forward pass that is replayed
    after a ``set`` sees it.  That memory is kept for the shapes that a capture asked for and the last 64 others."""

    _read = None   # what the last forward pass went by: a plan and its version

    def __init__(self, n: int):
        self.n, self._plan = n, None
        self._plans = {}        # of each shape of tokens, the latest last
        self._captured = set()  # those that a graph goes on reading

    @property
    def plan(self) -> Optional[Plan]:
        """The running batch's."""
        if not torch.compiler.is_compiling():
            now = self._plan, 0 if self._plan is None else self._plan.order._version
            if not f8._in_backward():
                self._read = now
            elif self._read not in (None, now):
                raise RuntimeError("Requests: set between a forward pass and its recomputation")
        if self._plan is not None and torch.cuda.is_current_stream_capturing():
            self._captured.add((self._plan.shape, self._plan.order.device))
        return self._plan

    def set(self, index: Optional[torch.Tensor]) -> None:
        """``index`` int32 or int64 on the GPU, of the shape of the batch's tokens."""
        if index is None:
            self._plan = None
            return
        key = tuple(index.shape), index.device
        plan = self._plans.get(key)
        if plan is None:
            with torch.inference_mode(False):   # (a training step may be the next to want it)
                plan = route(index, self.n)
            others = [k for k in self._plans if k not in self._captured]
            if len(others) >= 64:
                del self._plans[others[0]]
        else:
            ops.lowrank_route(index.flatten(), self.n, out=(plan.order, plan.starts))
            del self._plans[key]
        self._plans[key] = self._plan = plan
        if torch.cuda.is_current_stream_capturing():
            self._captured.add(key)


class AdaptedLinear(torch.nn.Module):
    """A linear and a bank of adapters beside it: ``linear(x)`` plus every token's own low-rank product, by the index that ``requests`` holds.
    ``a`` starts random and ``b`` at zero, so that a fresh adapter changes nothing."""

    def __init__(self, linear: torch.nn.Module, requests: Requests, rank: int, alpha: Optional[float] = None):
        super().__init__()
        w = linear.weight
        self.linear, self.requests = linear, requests
        self.a = torch.nn.Parameter(torch.empty((requests.n, rank, w.shape[1]), dtype=torch.bfloat16, device=w.device))
        self.b = torch.nn.Parameter(torch.zeros((requests.n, rank, w.shape[0]), dtype=torch.bfloat16, device=w.device))
        self.register_buffer("scale", torch.full((requests.n,), (rank if alpha is None else alpha) / rank, dtype=torch.float32, device=w.device))
        torch.nn.init.normal_(self.a, std=w.shape[1] ** -0.5)

    @torch.no_grad()
    def load(self, i: int, down: torch.Tensor, up: torch.Tensor, scale: float = 1.0) -> None:
        """Adapter i from a checkpoint's factors ``down`` [rank, in_features] and ``up`` [out_features, rank]; a lower rank than the bank's is
        filled up with zeros."""
        rank = down.shape[0]
        if not 0 <= i < self.a.shape[0] or rank > self.a.shape[1] or down.shape[1] != self.a.shape[2] or up.shape != (self.b.shape[2], rank):
            raise RuntimeError(f"AdaptedLinear.load: factors {tuple(down.shape)} and {tuple(up.shape)} do not fit place {i} of a bank {tuple(self.a.shape)}, {tuple(self.b.shape)}")
        self.a[i].zero_()[:rank].copy_(down)
        self.b[i].zero_()[:rank].copy_(up.t())
        self.scale[i] = scale

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        y = self.linear(x)
        plan = self.requests.plan
        return y if plan is None else add_lowrank(y, x, self.a, self.b, plan, self.scale.float())   # (a model's `to` may have rounded it)

    def extra_repr(self):
        return f"adapters={self.a.shape[0]}, rank={self.a.shape[1]}"


def add_adapters(root_module: torch.nn.Module, requests: Requests, rank: int, filter: str, alpha: Optional[float] = None) -> torch.nn.Module:
    """Put a bank of ``requests.n`` adapters beside every ``nn.Linear`` (or ``Fp8Linear``, ``Mxfp4Linear``) whose dotted name matches
    ``filter``; the linears keep their parameters, under ``linear.`` in the state dict.  A linear that stands at several places gets a bank at
    each (one in a shared parent: one bank).  A filter that names no linear is an error.  Fused feed-forwards multiply by their linears' weights
    themselves, so those take no adapters: an error."""
    filter_re = re.compile(filter)
    for name, module in root_module.named_modules(remove_duplicate=False):
        if isinstance(module, Fp8FeedForward):
            for child in ("w1", "w2", "w3"):
                if filter_re.search(f"{name}.{child}" if name else child):
                    raise RuntimeError(f"add_adapters: {name!r} is a fused feed-forward, whose {child} is not called (leave it out of fuse_feed_forward)")
    if not any(isinstance(m, (torch.nn.Linear, AdaptedLinear)) and filter_re.search(name) for name, m in root_module.named_modules(remove_duplicate=False)):
        raise RuntimeError(f"add_adapters: the filter {filter!r} names no linear")

    def walk(module: torch.nn.Module, name: str) -> torch.nn.Module:
        if isinstance(module, AdaptedLinear):   # (the linear inside is not adapted twice)
            return module
        for child_name, child in list(module._modules.items()):
            if child is not None:
                setattr(module, child_name, walk(child, f"{name}.{child_name}" if name else child_name))
        return AdaptedLinear(module, requests, rank, alpha) if isinstance(module, torch.nn.Linear) and filter_re.search(name) else module

    return walk(root_module, "")
