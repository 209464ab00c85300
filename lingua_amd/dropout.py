"""Dropout from a counter-based generator: which elements stay follows from a seed, a step, a call site and the element's place, so no
mask is stored -- forward and backward compute the same bits, and so does a forward pass that activation checkpointing runs again.

``numbers(seed, device)`` makes the two numbers {seed, step} that a program keeps on the GPU; it adds one to the step between two training
steps (``n[1] += 1``, which a captured graph may do by itself: its replays then drop other elements).  Changed between a forward pass and its
backward pass they are an error, as every saved tensor's in-place change is, also where ``torch.utils.checkpoint`` (``use_reentrant=False``) computes
the forward pass again; the replay of a graph that changes them is not seen by the host.  Ranks that hold other tokens take other seeds.
``Drop(p, numbers, site)`` says what a call drops; calls of one step that are to drop independently have sites of their own.  The norms of ``lingua_amd.norm`` take a ``Drop`` for the operand that they
add to the residual.  ``Dropout`` stands in for ``nn.Dropout``; ``convert_dropouts(model, numbers)`` swaps the modules and numbers their sites.

The share that is dropped is the multiple of 2^-16 next to ``p``, and what stays is scaled by that share.  A dropped element is zero whatever
it held: an infinity or NaN that is dropped is gone.
"""
import re
from typing import NamedTuple

import torch

from . import _lib, ops
from . import float8 as f8


class Drop(NamedTuple):
    p: float                # 0 .. 1
    numbers: torch.Tensor   # int64 {seed, step} on the GPU
    site: int = 0           # 0 .. 2^32 - 1


def numbers(seed: int, device="cuda") -> torch.Tensor:
    """int64 ``{seed, 0}``: the seed, any 64 bits, and the first step."""
    seed &= (1 << 64) - 1
    return torch.tensor([seed - (1 << 64) if seed >> 63 else seed, 0], dtype=torch.int64, device=device)


class DropoutFn(torch.autograd.Function):
    """``dropout`` and, with a residual, ``dropout_add``."""

    @staticmethod
    def forward(ctx, x, residual, numbers, p, site):
        ctx.save_for_backward(numbers)
        ctx.p, ctx.site, ctx.added, ctx.numbers = p, site, residual is not None, f8._stamp(numbers)
        return ops.dropout(x, Drop(p, numbers, site), residual)

    @staticmethod
    def backward(ctx, g):
        if g.dtype != torch.bfloat16:
            raise RuntimeError(f"dropout backward: bf16 gradients required, got {g.dtype}")
        numbers, = ctx.saved_tensors
        f8._unchanged(ctx.numbers, numbers, "dropout_add" if ctx.added else "dropout", "the seed and step were")
        gx = None
        if ctx.needs_input_grad[0]:
            varies = f8._learns(g)
            with torch.no_grad():
                gx = ops.dropout(g, Drop(ctx.p, numbers.contiguous(), ctx.site))   # (hooks hand it back in any layout)
            gx, = f8._once("dropout", (gx,), (varies,))
        return gx, (g if ctx.needs_input_grad[1] else None), None, None, None


def _dropout(x, residual, drop, what):
    threshold = ops._drop_args(drop, x.device, what)[2]
    if f8._native_call(x, 0) and f8._plain_call():
        y = _lib.native_for(x.get_device()).dropout(x, residual, drop.numbers, drop.site, threshold)
        if y is not None:
            return y
    f8._refuse_captured(x, residual, None, what)
    return DropoutFn.apply(x, residual, drop.numbers, drop.p, drop.site)


def dropout(x: torch.Tensor, drop: Drop) -> torch.Tensor:
    """x, bf16 of any shape, with a share of its elements dropped and the others scaled up; differentiable."""
    return _dropout(x, None, drop, "dropout")


def dropout_add(x: torch.Tensor, residual: torch.Tensor, drop: Drop) -> torch.Tensor:
    """``residual + dropout(x, drop)`` in one pass, rounded once; differentiable."""
    return _dropout(x, residual, drop, "dropout_add")


class Dropout(torch.nn.Module):
    """``nn.Dropout`` by the generator.  ``numbers`` is shared by the modules of a model and no buffer of theirs: it stays where it was made
    when a module moves."""

    def __init__(self, p: float, numbers: torch.Tensor, site: int = 0):
        super().__init__()
        self.p, self.numbers, self.site = p, numbers, site

    def drop(self):
        """What a fused sum takes: the ``Drop`` of this module in training, else None."""
        return Drop(self.p, self.numbers, self.site) if self.training else None

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        return dropout(x, self.drop()) if self.training else x

    def extra_repr(self):
        return f"p={self.p}, site={self.site}"


def convert_dropouts(root_module: torch.nn.Module, numbers: torch.Tensor, filter: str = "") -> torch.nn.Module:
    """Swap every ``nn.Dropout`` whose dotted name matches ``filter`` for a ``Dropout`` on ``numbers``, with sites 0, 1, ... in the order of
    the module tree; sites that the model's ``Dropout`` modules have already are passed over.  A module that stands at several places
    becomes one at each, with sites of their own."""
    filter_re = re.compile(filter)
    taken = {m.site for m in root_module.modules() if isinstance(m, Dropout)}
    site = iter(i for i in range(1 << 32) if i not in taken)

    def of(module):
        return Dropout(module.p, numbers, next(site)).train(module.training)

    if type(root_module) is torch.nn.Dropout and filter_re.search(""):
        return of(root_module)
    for name, parent in list(root_module.named_modules(remove_duplicate=False)):
        for child_name, child in parent._modules.items():
            if type(child) is torch.nn.Dropout and filter_re.search(f"{name}.{child_name}" if name else child_name):
                setattr(parent, child_name, of(child))
    return root_module
