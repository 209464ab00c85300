"""Rotary positions of queries and keys, the step between the attention projections and the attention.

``apply_rotary_emb`` has the arguments of the reference's function of that name (lingua/transformer.py) and takes its table; ``rotary``
is the general form: either layout of pairs, a part of the head, tokens at positions given as a tensor, tables from ``rotary_tables``
for contexts longer than the trained one.  Forward and backward are one kernel launch each (``l8_rotary``) for queries and keys
together; q and k may be column slices of one product (``lingua_amd.qkv.fuse_qkv``), nothing is copied on the way in.

``rotary_axes`` is the form for images and video: a token stands at a place of up to four axes, and each axis turns its share of the pairs.
"""
import math
from typing import Optional, Sequence

import torch

from . import _lib, ops
from . import float8 as f8

LAYOUTS = ("interleaved", "half")
ORDERS = ("sections", "rounds")


class RotaryFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, xq, xk, cos, sin, positions, in_halves, sections=None, in_rounds=False):
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(cos, sin, positions)
        ctx.in_halves, ctx.axes = in_halves, {} if sections is None else {"sections": sections, "in_rounds": in_rounds}
        return ops.rotary(xq, xk, cos, sin, positions, in_halves, **ctx.axes)

    @staticmethod
    def backward(ctx, gq, gk):
        for g in (gq, gk):
            if g is not None and g.dtype != torch.bfloat16:
                raise RuntimeError(f"rotary backward: bf16 gradients required, got {g.dtype}")
        gq = gq if ctx.needs_input_grad[0] else None
        gk = gk if ctx.needs_input_grad[1] else None
        varies = (f8._learns(gq), f8._learns(gk))
        if gq is not None or gk is not None:
            cos, sin, positions = ctx.saved_tensors
            with torch.no_grad():
                gq, gk = ops.rotary(gq, gk, cos, sin, positions, ctx.in_halves, inverse=True, **ctx.axes)
        return (*f8._once("rotary", (gq, gk), varies), None, None, None, None, None, None)


def rotary(xq: torch.Tensor, xk: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor, positions: Optional[torch.Tensor] = None,
           layout: str = "interleaved"):
    """``(xq, xk)`` [B,S,H,D] bf16 with the first ``rot = 2 * cos.shape[1]`` columns of every head turned by the angles of their
    tokens' positions; the others are copied.

    ``cos``, ``sin``  fp32 [P, rot / 2], position by frequency (``rotary_tables``); no gradient flows to them.
    ``positions``     int32 or int64, broadcastable to [B,S]; None: token s stands at position s.  A position outside [0, P) gives NaN
                      for its token (positions live on the GPU: the host cannot refuse them).
    ``layout``        "interleaved": pairs (2 i, 2 i + 1), the reference's; "half": pairs (i, i + rot / 2).
    """
    if layout not in LAYOUTS:
        raise RuntimeError(f"rotary: unknown layout {layout!r}, one of {LAYOUTS}")
    if f8._native_call(xq, 0) and f8._plain_call():
        res = _lib.native_for(xq.get_device()).rotary_pair(xq, xk, cos, sin, positions, layout == "half")
        if res is not None:
            return res
    f8._refuse_captured(xq, xk, None, "rotary")
    return RotaryFn.apply(xq, xk, cos, sin, positions, layout == "half")


def rotary_axes(xq: torch.Tensor, xk: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor, positions: torch.Tensor, sections: Sequence[int],
                order: str = "sections", layout: str = "interleaved"):
    """``(xq, xk)`` [B,S,H,D] bf16 with pairs of columns turned by the positions of their tokens on several axes: pair i, of axis a, by the
    angle of row ``positions[a,b,s]``, column i of the tables; the columns behind the last pair are copied.

    ``cos``, ``sin``  fp32 [P, pairs]: ``rotary_tables`` (one run of frequencies over all pairs) or ``axes_tables`` (one for each axis); no
                      gradient flows to them: tables that ask for one are an error
    ``positions``     int32 or int64, broadcastable to [axes,B,S].  A token of which any position is outside [0, P) becomes NaN.
    ``sections``      pairs that each of up to four axes turns, their sum cos.shape[1]
    ``order``         "sections": an axis's pairs side by side, the axes in their order; "rounds": a pair to each axis in turn, an axis that
                      has its share being passed over
    ``layout``        as in ``rotary``
    """
    if layout not in LAYOUTS:
        raise RuntimeError(f"rotary_axes: unknown layout {layout!r}, one of {LAYOUTS}")
    if order not in ORDERS:
        raise RuntimeError(f"rotary_axes: unknown order {order!r}, one of {ORDERS}")
    if (cos.requires_grad or sin.requires_grad) and torch.is_grad_enabled():
        raise RuntimeError("rotary_axes: the tables ask for a gradient, and none flows to them")
    sections = tuple(sections)
    if f8._native_call(xq, 0) and f8._plain_call():
        res = _lib.native_for(xq.get_device()).rotary_pair(xq, xk, cos, sin, positions, layout == "half", sections, order == "rounds")
        if res is not None:
            return res
    f8._refuse_captured(xq, xk, None, "rotary_axes")
    return RotaryFn.apply(xq, xk, cos, sin, positions, layout == "half", sections, order == "rounds")


def apply_rotary_emb(xq: torch.Tensor, xk: torch.Tensor, seq_dim: int, freqs_cis: torch.Tensor):
    """The reference's ``apply_rotary_emb``: xq, xk [B,S,H,D] (``seq_dim`` 1) or [B,H,S,D] (2), freqs_cis fp32 [S, D / 2, 2, 2] of
    rotation matrices ((cos, -sin), (sin, cos)), read where it lies."""
    if seq_dim not in (1, 2):
        raise RuntimeError(f"apply_rotary_emb: seq_dim 1 or 2, got {seq_dim}")
    if freqs_cis.dim() != 4 or freqs_cis.shape[2:] != (2, 2) or xq.dim() != 4 or freqs_cis.shape[:2] != (xq.shape[seq_dim], xq.shape[3] // 2):
        raise RuntimeError(f"apply_rotary_emb: freqs_cis {tuple(freqs_cis.shape)} does not fit xq {tuple(xq.shape)}")
    cos, sin = freqs_cis[:, :, 0, 0], freqs_cis[:, :, 1, 0]
    if seq_dim == 1:
        return rotary(xq, xk, cos, sin)
    q, k = rotary(xq.transpose(1, 2), xk.transpose(1, 2), cos, sin)
    return q.transpose(1, 2), k.transpose(1, 2)


def rotary_tables(rot: int, length: int, theta: float = 10000.0, scaling: Optional[str] = None, factor: float = 1.0,
                  trained_length: Optional[int] = None, device=None):
    """``(cos, sin)`` fp32 [length, rot / 2] of the angles p * theta^(-2 i / rot), computed in 64 bits: an angle of position 10^5 has
    lost two of its digits in 32.

    ``scaling``, for contexts ``factor`` times as long as the trained one:
      None      the angles as they are
      "linear"  positions interpolated: p / factor (Chen et al. 2023)
      "ntk"     theta * factor^(rot / (rot - 2)): the lowest frequency is interpolated, the highest stays
      "yarn"    frequencies that turn fewer than once within ``trained_length`` positions are interpolated, those that turn more than 32
                times stay, a ramp in between; cosines and sines are multiplied by 0.1 ln(factor) + 1 (Peng et al. 2023)
    """
    if rot < 2 or rot % 2 or length < 0:
        raise RuntimeError(f"rotary_tables: an even number of columns and a length are wanted, got {rot} and {length}")
    if scaling not in (None, "linear", "ntk", "yarn"):
        raise RuntimeError(f"rotary_tables: unknown scaling {scaling!r}")
    if scaling is not None and factor < 1:
        raise RuntimeError(f"rotary_tables: a factor of at least 1 is wanted, got {factor}")
    i = torch.arange(0, rot, 2, device=device, dtype=torch.float64)
    size = 1.0
    if scaling == "ntk":
        if rot < 4:
            raise RuntimeError("rotary_tables: ntk scaling needs more than one frequency")
        theta = theta * factor ** (rot / (rot - 2))
    freq = float(theta) ** (-i / rot)
    if scaling == "linear":
        freq = freq / factor
    elif scaling == "yarn":
        if not trained_length:
            raise RuntimeError("rotary_tables: yarn scaling needs trained_length")
        # the index at which a frequency turns n times within the trained length
        def index_of(turns):
            return rot * math.log(trained_length / (turns * 2 * math.pi)) / (2 * math.log(theta))
        low, high = max(math.floor(index_of(32)), 0), min(math.ceil(index_of(1)), rot - 1)
        ramp = ((i / 2 - low) / max(high - low, 1e-3)).clamp(0, 1)
        freq = freq * (1 - ramp) + freq / factor * ramp
        size = 0.1 * math.log(factor) + 1.0
    angle = torch.arange(length, device=device, dtype=torch.float64)[:, None] * freq
    return (angle.cos() * size).float(), (angle.sin() * size).float()


def pair_axes(sections: Sequence[int], order: str = "sections"):
    """The axis that each pair of ``rotary_axes`` turns by: a list of sum(sections) numbers."""
    left = list(sections)
    if order not in ORDERS or any(n < 0 for n in left):
        raise RuntimeError(f"pair_axes: shares of pairs and an order of {ORDERS} are wanted, got {left} and {order!r}")
    if order == "sections":
        return [a for a, n in enumerate(left) for _ in range(n)]
    return [a for turn in range(max(left, default=0)) for a, n in enumerate(left) if turn < n]


def axes_tables(sections: Sequence[int], length: int, theta: float = 10000.0, order: str = "sections", device=None):
    """``(cos, sin)`` fp32 [length, sum(sections)] for ``rotary_axes`` with a run of frequencies for each axis, as models of images have
    them: the j-th of an axis's n pairs turns by p * theta^(-j / n)."""
    if length < 0:
        raise RuntimeError(f"axes_tables: a length is wanted, got {length}")
    cos, sin = (torch.empty((length, sum(sections)), dtype=torch.float32, device=device) for _ in range(2))
    of = torch.tensor(pair_axes(sections, order), device=device)
    for a, n in enumerate(sections):
        if n:
            cos[:, of == a], sin[:, of == a] = rotary_tables(2 * n, length, theta, device=device)
    return cos, sin
