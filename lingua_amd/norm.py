"""RMSNorm whose output arrives at the fp8 linears already quantised.

``Fp8RMSNorm`` is a drop-in for the reference's ``RMSNorm``
(lingua/transformer.py:264-292: ``(x.float() * rsqrt(mean(x^2) + eps) * weight.float()).type_as(x)``).
Its backward is one kernel too (``l8_rmsnorm_bwd``).  Its forward (``l8_rmsnorm_cast_rowwise``) writes the bf16
output and, from the same registers, the row-wise fp8 copy that the linears
fed by the norm (wq / wk / wv, w1 / w3) would otherwise each compute in a pass
of their own (lingua/float8.py:86-87, :43-47).  The quantised copy is handed
over through the memo of ``lingua_amd.float8`` that already lets such linears
share one cast, so nothing changes in the attention / MLP modules.

Opt-in: ``fuse_rmsnorm(model)`` after (or before) ``convert_linears_to_fp8``.

``add_rmsnorm`` is the norm of a residual sum together with the sum, as the
second half of a block computes it (lingua/transformer.py:497-543:
``h = x + attention(...)``, then ``ffn_norm(h)``): one pass over both operands
forward, and one backward that adds the two gradients of the sum.
``fuse_residual_norm(model)`` has the blocks of a model call it.
"""
import re

import torch

from . import _lib, ops
from . import float8 as f8


class Fp8RMSNormFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, eps, training):
        if x.dtype != torch.bfloat16:
            raise RuntimeError(f"Fp8RMSNorm: bf16 activations required, got {x.dtype}")
        x2d = x.flatten(end_dim=-2)
        want_col, res = bool(training and f8.config.fp8_wgrad), None
        if f8._native_call(x2d, 0):
            res = _lib.native_for(x2d.get_device()).rmsnorm_fwd(x2d, weight, eps, want_col)
        if res is None:
            col = torch.empty(x2d.shape[1], dtype=torch.float32, device=x.device) if want_col else None
            res = (*ops.rmsnorm_cast_rowwise(x2d, weight, eps, want_q=True, col_amax=col, want_rstd=True, on_lines=True), col)
        y2d, q, s, rstd, col = res
        if f8.config.share_input_casts:
            f8._fwd_cast.put(y2d, (q, s, col), "rmsnorm")
        ctx.save_for_backward(x2d, weight, rstd)
        ctx.x_shape = x.shape
        return y2d.unflatten(0, x.shape[:-1])

    @staticmethod
    def backward(ctx, gy):
        x2d, weight, rstd = ctx.saved_tensors
        if gy.dtype != torch.bfloat16:
            raise RuntimeError(f"Fp8RMSNorm.backward: bf16 grad_out required, got {gy.dtype}")
        gy2d, res = gy.flatten(end_dim=-2), None
        if f8._native_call(gy2d, 0):
            res = _lib.native_for(gy2d.get_device()).rmsnorm_bwd(gy2d, x2d, weight, rstd)
        gx2d, gw = ops.rmsnorm_bwd(gy2d, x2d, weight, rstd, gw_dtype=weight.dtype) if res is None else res
        gx = gx2d.reshape(ctx.x_shape) if ctx.needs_input_grad[0] else None
        return gx, (gw if ctx.needs_input_grad[1] else None), None, None


class Fp8AddRMSNormFn(torch.autograd.Function):
    """``add_rmsnorm`` on 2-D operands.  (It returns what it made and no views of it: those could not be written in place.)"""

    @staticmethod
    def forward(ctx, x, residual, weight, eps, training):
        if x.dtype != torch.bfloat16 or residual.dtype != torch.bfloat16:
            raise RuntimeError(f"add_rmsnorm: bf16 activations required, got {x.dtype} and {residual.dtype}")
        want_col = bool(training and f8.config.fp8_wgrad)
        col = torch.empty(x.shape[1], dtype=torch.float32, device=x.device) if want_col else None
        h, y, q, s, rstd = ops.add_rmsnorm_cast_rowwise(x, residual, weight, eps, col_amax=col, on_lines=True)
        if f8.config.share_input_casts:   # (the memo keeps its tensor: not the graph behind it)
            f8._fwd_cast.put(y.detach(), (q, s, col), "rmsnorm")
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(h, weight, rstd)
        ctx.sum_learns = x.requires_grad or residual.requires_grad
        return h, y

    @staticmethod
    def backward(ctx, gh, gy):
        h, weight, rstd = ctx.saved_tensors
        need = ctx.needs_input_grad
        for g in (gh, gy):
            if g is not None and g.dtype != torch.bfloat16:
                raise RuntimeError(f"add_rmsnorm backward: bf16 gradients required, got {g.dtype}")
        if gy is None:   # only the sum was used
            return gh if need[0] else None, gh if need[1] else None, None, None, None
        gy_learns = f8._learns(gy)
        gx_varies = ctx.sum_learns or f8._learns(weight) or f8._learns(gh) or gy_learns
        with torch.no_grad():
            if gh is None:
                gx, gw = ops.rmsnorm_bwd(gy, h, weight, rstd, gw_dtype=weight.dtype)
            else:
                gx, gw = ops.add_rmsnorm_bwd(gy, gh, h, weight, rstd, gw_dtype=weight.dtype)
        grads = gx if need[0] else None, gx if need[1] else None, gw if need[2] else None
        return (*f8._once("add_rmsnorm", grads, (gx_varies, gx_varies, ctx.sum_learns or gy_learns)), None, None)


def add_rmsnorm(x: torch.Tensor, residual: torch.Tensor, weight: torch.Tensor, eps: float):
    """``h = x + residual`` (rounded to bf16) and ``y = rmsnorm(h) * weight``: returns ``(h, y)``, shaped like x [..., C].  The fp8
    linears that are called on ``y`` find it quantised, as behind an ``Fp8RMSNorm``."""
    if x.dim() < 2:
        raise RuntimeError(f"add_rmsnorm: expected [..., C] with at least one leading dimension, got {tuple(x.shape)}")
    training = torch.is_grad_enabled()
    if f8._native_call(x, 0) and f8._plain_call():
        res = _lib.native_for(x.get_device()).add_rmsnorm(x, residual, weight, eps, bool(training and f8.config.fp8_wgrad))
        if res is not None:
            h, y, q, s, col = res
            if f8.config.share_input_casts:   # (the memo keeps its tensor: not the graph behind it)
                f8._fwd_cast.put(y.detach().flatten(end_dim=-2), (q, s, col), "rmsnorm")
            return h, y
    f8._refuse_captured(x, residual, weight, "add_rmsnorm")
    if x.shape != residual.shape:
        raise RuntimeError(f"add_rmsnorm: x and residual must have the same shape, got {tuple(x.shape)} and {tuple(residual.shape)}")
    if x.dim() == 2:
        return Fp8AddRMSNormFn.apply(x, residual, weight, eps, training)
    h, y = Fp8AddRMSNormFn.apply(x.flatten(end_dim=-2), residual.flatten(end_dim=-2), weight, eps, training)
    return h.unflatten(0, x.shape[:-1]), y.unflatten(0, x.shape[:-1])


class Fp8RMSNorm(torch.nn.Module):
    """Same parameters and state-dict keys as the reference's RMSNorm (``weight``; ``eps`` attribute)."""

    def __init__(self, dim: int, eps: float = 1e-6, weight: torch.nn.Parameter = None):
        super().__init__()
        self.eps = eps
        self.weight = weight if weight is not None else torch.nn.Parameter(torch.ones(dim))

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        # grad mode is read here: inside an autograd Function's forward it is always off
        return Fp8RMSNormFn.apply(x, self.weight, self.eps, torch.is_grad_enabled())

    def add(self, x: torch.Tensor, residual: torch.Tensor):
        """``(x + residual, this norm of it)`` in one pass."""
        return add_rmsnorm(x, residual, self.weight, self.eps)

    def reset_parameters(self):
        torch.nn.init.ones_(self.weight)


def fuse_rmsnorm(root_module: torch.nn.Module, filter: str = r"(attention_norm|ffn_norm)$") -> torch.nn.Module:
    """Swap every module whose dotted name matches ``filter`` and that looks like the reference's RMSNorm
    (class name ``RMSNorm``, a 1-D ``weight`` and an ``eps``) for an ``Fp8RMSNorm`` over the same Parameter.
    The default filter takes the two norms of a block, whose outputs feed fp8 linears, and leaves the final
    norm in front of the bf16 output head alone."""
    filter_re = re.compile(filter)

    def replace(module: torch.nn.Module, name: str) -> torch.nn.Module:
        if isinstance(module, Fp8RMSNorm) or not filter_re.search(name):
            return module
        w = getattr(module, "weight", None)
        if type(module).__name__ != "RMSNorm" or not isinstance(w, torch.nn.Parameter) or w.dim() != 1 or not hasattr(module, "eps"):
            raise RuntimeError(f"fuse_rmsnorm: {name!r} ({type(module).__name__}) is not an RMSNorm with weight and eps")
        return Fp8RMSNorm(w.numel(), float(module.eps), weight=w)

    return f8.named_replace(replace, root_module)


class _ResidualNormForward:
    """``forward`` of a block whose second norm takes the residual sum with it (lingua/transformer.py:497-543: ``h = x +
    attention(attention_norm(x), ...)``, ``h + feed_forward(ffn_norm(h))``)."""

    def forward(self, x, *args, **kwargs):
        h, y = self.ffn_norm.add(x, self.attention(self.attention_norm(x), *args, **kwargs))
        return h + self.feed_forward(y)

    def __reduce_ex__(self, protocol):   # pickled by the class that it was fused from
        return _fused_like, (type(self).__mro__[2],), self.__dict__


_fused_classes = {}


def _fused_class(cls):
    if cls not in _fused_classes:
        _fused_classes[cls] = type(cls.__name__, (_ResidualNormForward, cls), {"__module__": cls.__module__})
    return _fused_classes[cls]


def _fused_like(cls):
    return cls.__new__(_fused_class(cls))


def fuse_residual_norm(root_module: torch.nn.Module, filter: str = r"layers\.[0-9]+$") -> torch.nn.Module:
    """In every module whose dotted name matches ``filter`` and whose children are exactly ``attention``, ``feed_forward``,
    ``attention_norm`` and an ``Fp8RMSNorm`` ``ffn_norm`` (the reference's TransformerBlock, lingua/transformer.py:497-543, after
    ``fuse_rmsnorm``), the residual sum in front of ``ffn_norm`` becomes part of it.  The caller vouches that the module computes
    ``h = x + attention(attention_norm(x), ...)``, ``h + feed_forward(ffn_norm(h))``; modules, parameters and state-dict keys stay."""
    filter_re = re.compile(filter)
    for name, module in root_module.named_modules():
        if not filter_re.search(name) or isinstance(module, _ResidualNormForward):
            continue
        children = dict(module.named_children())
        if (set(children) != {"attention", "feed_forward", "attention_norm", "ffn_norm"} or not isinstance(children["ffn_norm"], Fp8RMSNorm) or
                list(module.parameters(recurse=False))):
            raise RuntimeError(f"fuse_residual_norm: {name!r} ({type(module).__name__}) is not a block of attention, feed_forward, "
                               "attention_norm and an Fp8RMSNorm ffn_norm (run fuse_rmsnorm first)")
        module.__class__ = _fused_class(type(module))
    return root_module
