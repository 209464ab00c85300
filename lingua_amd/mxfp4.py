"""Linears in MXFP4: e2m1 codes in blocks of 32 along the reduction with a power-of-two scale each (OCP Microscaling formats 1.0),
half the bytes of the fp8 path and twice its matrix rate.

``Mxfp4Linear`` stands in for ``nn.Linear`` as ``lingua_amd.Fp8Linear`` does; ``convert_linears_to_mxfp4(model, filter)`` swaps the
modules.  All three products run on codes:

    y  = Q(x) Q(w)^T + bias        blocks along in_features
    gx = Q(gy) Q(w)                blocks along out_features
    gw = Q(gy)^T Q(x)              blocks along the tokens

with x, w and gy rounded to nearest; gradients pass the rounding unchanged.  Forward reads x and w once each and makes from that read
both copies it and backward multiplies with; backward holds the 17/32 byte per element of the transposed copies instead of x.

Four bits are a coarse rounding of a gradient, and no step here (no random rounding, no rotation) keeps its mean: for training the fp8
path is the safer one, this one serves inference and quantisation-aware fine-tuning first.

``pack`` and ``linear_packed`` are the form for serving: a weight quantised once, activations quantised on the way into the product.
"""
import re
from typing import Optional

import torch

from . import _lib, ops
from . import float8 as f8


def _check_operands(a, w):
    if a.dtype != torch.bfloat16 or w.dtype != torch.bfloat16:
        raise RuntimeError(f"mxfp4_linear: bf16 input and weight required, got {a.dtype} and {w.dtype}")
    if not a.is_cuda or a.device != w.device:
        raise RuntimeError(f"mxfp4_linear: input and weight must be on the same GPU, got {a.device} and {w.device} (there is no CPU path)")
    if a.dim() < 2 or w.dim() != 2 or a.shape[-1] != w.shape[1]:
        raise RuntimeError(f"mxfp4_linear: input {tuple(a.shape)} and weight {tuple(w.shape)} do not fit")
    if w.shape[1] % 16 or w.shape[0] % 16:
        raise RuntimeError(f"mxfp4_linear: in_features ({w.shape[1]}) and out_features ({w.shape[0]}) must be multiples of 16")


class Mxfp4LinearFn(torch.autograd.Function):
    """``a @ w.T + bias`` on 2-D operands with MXFP4 products, forward and backward."""

    @staticmethod
    def forward(ctx, a, w, bias):
        need_a, need_w = ctx.needs_input_grad[0], ctx.needs_input_grad[1]
        (qa, sa), at = ops.cast_mxfp4(a, transposed=need_w, on_lines=True)
        (qw, sw), wt = ops.cast_mxfp4(w, transposed=need_a, on_lines=True)
        ctx.save_for_backward(*(at or (None, None)), *(wt or (None, None)))
        return ops.gemm_mxfp4_nt(qa, qw, sa, sw, bias)

    @staticmethod
    def backward(ctx, gy):
        if gy.dtype != torch.bfloat16:
            raise RuntimeError(f"mxfp4_linear backward: bf16 grad_out required, got {gy.dtype}")
        qat, sat, qwt, swt = ctx.saved_tensors
        need_a, need_w, need_bias = ctx.needs_input_grad
        ga = gw = gbias = None
        with torch.no_grad():
            if need_a or need_w:
                rows, cols = ops.cast_mxfp4(gy, rowwise=need_a, transposed=need_w, on_lines=True)
                if need_a:
                    ga = ops.gemm_mxfp4_nt(rows[0], qwt, rows[1], swt)
                if need_w:
                    gw = ops.gemm_mxfp4_nt(cols[0], qat, cols[1], sat)
            if need_bias:
                gbias = ops.col_sum(gy) if ops.rows_on_16_bytes(gy) else gy.sum(dim=0)
        gy_learns = f8._learns(gy)   # (what was kept of the one operand says that the other learns)
        return f8._once("mxfp4_linear", (ga, gw, gbias), (gy_learns or qat is not None, gy_learns or qwt is not None, gy_learns))


def mxfp4_linear(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``x @ weight.T + bias`` in MXFP4, x [..., K] and weight [N, K] bf16, K and N multiples of 16; differentiable."""
    if f8._native_call(x, 0) and f8._plain_call():
        y = _lib.native_for(x.get_device()).mxfp4_linear(x, weight, bias)
        if y is not None:
            return y
    _check_operands(x, weight)
    f8._refuse_captured(x, weight, bias, "mxfp4_linear")
    if x.dim() == 2:
        return Mxfp4LinearFn.apply(x, weight, bias)
    return Mxfp4LinearFn.apply(x.flatten(end_dim=-2), weight, bias).unflatten(0, x.shape[:-1])


def pack(weight: torch.Tensor):
    """``(codes, scales)`` of a weight [N, K] for ``linear_packed``: [N, 16 * ceil(K / 32)] and [N, ceil(K / 32)]."""
    return ops.cast_mxfp4(weight.detach(), on_lines=True)[0]


def linear_packed(x: torch.Tensor, codes: torch.Tensor, scales: torch.Tensor, bias: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``x @ weight.T + bias`` of a weight kept in MXFP4 (``pack``, or the same bytes as uint8 from a checkpoint), x [..., K] bf16.  No
    gradients: x, bias and weight are taken as they are."""
    if x.dim() < 2:
        raise RuntimeError(f"linear_packed: expected [..., K] with at least one leading dimension, got {tuple(x.shape)}")
    if x.dim() == 2:
        return ops.mxfp4_linear_fwd(x.detach(), codes, scales, bias)
    return ops.mxfp4_linear_fwd(x.detach().flatten(end_dim=-2), codes, scales, bias).unflatten(0, x.shape[:-1])


class Mxfp4Linear(torch.nn.Linear):
    def forward(self, input: torch.Tensor) -> torch.Tensor:
        weight, bias = self.weight, self.bias
        if torch.is_grad_enabled() and (input.requires_grad or weight.requires_grad or (bias is not None and bias.requires_grad)) or not f8._plain_call():
            return mxfp4_linear(input, weight, bias)
        _check_operands(input, weight)
        return linear_packed(input, *_packed_weight(weight), bias)


def _packed_weight(w):
    """The weight's row-wise copy; with ``lingua_amd.config.cache_weight_casts`` kept until the weight changes, as the fp8 path's is."""
    slot = f8._weight_casts._slot(w) if f8.config.cache_weight_casts else None
    if slot is None:
        return pack(w)
    if "mxfp4" not in slot:
        slot["mxfp4"] = pack(w)
    return slot["mxfp4"]


def convert_linears_to_mxfp4(root_module: torch.nn.Module, filter: str) -> torch.nn.Module:
    """Swap every exact ``nn.Linear`` whose dotted name matches ``filter`` for an ``Mxfp4Linear`` that shares the same Parameter objects;
    a matching subclass of ``nn.Linear`` (an already converted layer, say) raises AssertionError, as in ``convert_linears_to_fp8``."""
    filter_re = re.compile(filter)

    def replace(module: torch.nn.Module, name: str) -> torch.nn.Module:
        if not isinstance(module, torch.nn.Linear) or not filter_re.search(name):
            return module
        assert type(module) == torch.nn.Linear, str(type(module))
        new_module = Mxfp4Linear(module.in_features, module.out_features, bias=module.bias is not None, dtype=module.weight.dtype,
                                 device=module.weight.device)
        new_module.weight = module.weight
        new_module.bias = module.bias
        return new_module

    out = f8.named_replace(replace, root_module)
    torch._dynamo.reset_code_caches()   # a model compiled before the swap traces afresh
    return out
