"""Dropout from a counter-based generator: which elements stay follows from a seed, a step, a call site and the element's place, so no
mask is stored -- forward and backward compute the same bits, and so does a forward pass that activation checkpointing runs again.

``numbers(seed, device)`` makes the two numbers {seed, step} that a program keeps on the GPU; it adds one to the step (``n[1] += 1``) behind every
backward pass, also those of the micro-batches of one training step, which would else drop the same elements.  A captured graph may do so by
itself: its replays then drop other elements.  Changed between a forward pass and its
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


_SITES, _CALLS = 1 << 20, 1 << 12   # sites that modules number, and calls of each: call k of a module drops as site + k * 2^20


class _Pass:
    """One forward pass of a model, in which the calls of each of its dropouts are counted: hooks around the model's forward."""

    def __init__(self, dropouts):
        self.dropouts = dropouts
        for m in dropouts:
            m._pass = self
        self.running = False

    def begin(self, model, args):
        for m in self.dropouts:
            m._calls = 0
        self.running = True

    def end(self, model, args, out):
        self.running = False


class Dropout(torch.nn.Module):
    """``nn.Dropout`` by the generator.  ``numbers`` is shared by the modules of a model and no buffer of theirs: it stays where it was made
    when a module moves.

    Each call (of the module or of ``drop``) within a forward pass of the model that ``convert_dropouts`` was given drops other elements: the
    first goes by ``site``, call k by ``site + k * 2^20``.  Outside such a pass -- a module made by hand, a model whose parts are called one by
    one -- nothing says where a pass begins, and every call of a step drops by ``site``: the same places of equal shapes.  A pass that
    activation checkpointing computes again has to call the module once: of several calls nothing says which one is repeated, an error; and
    ``numbers`` that changed since the last forward pass are one too."""

    _pass, _calls, _several, _version = None, 0, False, None   # (here, so that a module that was pickled without them has them)

    def __init__(self, p: float, numbers: torch.Tensor, site: int = 0):
        super().__init__()
        self.p, self.numbers, self.site = p, numbers, site

    def drop(self):
        """What a fused sum takes: the ``Drop`` of this module in training, else None."""
        if not self.training:
            return None
        call = 0
        if torch.compiler.is_compiling() or not f8._in_backward():
            if self._pass is not None and self._pass.running:
                call = self._calls
                self._calls += 1
                if call:
                    self._several = True
            if not torch.compiler.is_compiling():
                self._version = f8._stamp(self.numbers)
        elif self._several:
            raise RuntimeError("Dropout: called several times in a forward pass, of which one is computed again: use a module for each call")
        elif self._version not in (None, f8._stamp(self.numbers)):   # (others in their place as well)
            raise RuntimeError("Dropout: the seed and step were modified by an inplace operation between the forward pass and its recomputation, or exchanged")
        if call and (self.site >= _SITES or call >= _CALLS):
            raise RuntimeError(f"Dropout: call {call} of site {self.site} in one forward pass; sites below 2^20 have 4096")
        return Drop(self.p, self.numbers, self.site + call * _SITES)

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        return dropout(x, self.drop()) if self.training else x

    def extra_repr(self):
        return f"p={self.p}, site={self.site}"


def convert_dropouts(root_module: torch.nn.Module, numbers: torch.Tensor, filter: str = "") -> torch.nn.Module:
    """Swap every ``nn.Dropout`` whose dotted name matches ``filter`` for a ``Dropout`` on ``numbers``, with sites 0, 1, ... in the order of
    the module tree; sites that the model's ``Dropout`` modules have already are passed over.  A module that stands at several places
    becomes one at each, with sites of their own; one inside a shared parent stays one, whose calls in a forward pass of ``root_module``
    drop other elements each, as those of any module do that is called several times.  (A container without a forward pass of its own
    cannot tell those calls apart: an error where it holds such a parent.)  Forward passes of one step, as of its micro-batches, drop the
    same elements unless the step's number is advanced between them.  Parts of a model that are converted one by one with the same
    ``numbers`` get the same sites: convert it as a whole."""
    filter_re = re.compile(filter)
    taken = {m.site % _SITES for m in root_module.modules() if isinstance(m, Dropout)}
    site = iter(i for i in range(_SITES) if i not in taken)

    def of(module):
        return Dropout(module.p, numbers, next(site)).train(module.training)

    if type(root_module) is torch.nn.Dropout and filter_re.search(""):
        return of(root_module)
    places, seen, shared = {}, set(), None
    for name, parent in root_module.named_modules(remove_duplicate=False):
        for child_name, child in parent._modules.items():
            if type(child) is not torch.nn.Dropout:
                continue
            if filter_re.search(f"{name}.{child_name}" if name else child_name):
                places[id(parent), child_name] = parent, child_name, child
            if (parent, child_name) in seen:
                shared = parent, child_name, name
            seen.add((parent, child_name))
    if shared and type(root_module).forward is torch.nn.Module.forward and (id(shared[0]), shared[1]) in places:
        raise RuntimeError(f"convert_dropouts: {shared[2]!r} stands at several places of a {type(root_module).__name__}, which has no forward pass of its own")
    made = []
    for parent, child_name, child in places.values():
        made.append(of(child))
        setattr(parent, child_name, made[-1])
    if made:
        one = _Pass(made)
        root_module.register_forward_pre_hook(one.begin)
        root_module.register_forward_hook(one.end, always_call=True)
    return root_module
