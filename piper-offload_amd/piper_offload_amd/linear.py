"""Linear layers over stored weights: MXFP4 weights and one weight per group of rows, with gradients.

After a merge a packed weight is used as it is stored, without a dense copy:

* :func:`mx_linear` -- ``x @ W.T + bias`` for an :class:`MXWeight` in MXFP4;
* :func:`grouped_linear` -- consecutive groups of rows, each with a weight of
  its own (the experts of a mixture, one adapter per request), dense or MXFP4.

Gradients: to ``x`` for every weight, to the weight where it is dense.  A
packed weight is frozen, as is a bias.  With quantised inputs the gradient
passes straight through the rounding.

The experts of a packed stack lie one below the other in one ``MXWeight`` of
``groups * out`` rows; :func:`expert_view` gives one of them as a weight of its
own, for a LoRA merge in place.
"""

from __future__ import annotations

import torch

from . import kernels as K
from .formats import MXWeight

__all__ = ["expert_view", "grouped_linear", "mx_linear"]

_FP4 = getattr(torch, "float4_e2m1fn_x2", None)


def _packed(label: str, weight: MXWeight) -> tuple[torch.Tensor, torch.Tensor]:
    if weight.elem_dtype is not _FP4 or _FP4 is None:
        raise ValueError(f"{label} supports MXFP4 weights, got elements of {weight.elem_dtype}.")
    if weight.block_size != 32:
        raise ValueError(f"{label} supports block size 32, got {weight.block_size}.")
    return weight.qdata.view(torch.uint8), weight.scale.view(torch.uint8)


def _stacked(label: str, weight: MXWeight, groups: int) -> tuple[torch.Tensor, torch.Tensor]:
    q, s = _packed(label, weight)
    rows = q.shape[0]
    if groups < 1 or rows % groups:
        raise ValueError(f"{label}: {rows} rows do not divide into {groups} weights.")
    if weight.is_swizzled_scales and rows // groups % 128:
        raise ValueError(f"{label}: swizzled scales of stacked weights need rows divisible by 128, got {rows // groups}.")
    if not q.is_contiguous() or not s.is_contiguous():
        raise ValueError(f"{label} requires contiguous MXFP4 storage.")
    return q.view(groups, rows // groups, q.shape[1]), s.view(groups, s.shape[0] // groups, s.shape[1])


def expert_view(weight: MXWeight, index: int, groups: int) -> MXWeight:
    """Weight ``index`` of ``groups`` stacked along the rows of ``weight``, sharing its storage."""
    q, s = _stacked("expert_view", weight, groups)
    if not 0 <= index < groups:
        raise ValueError(f"expert_view: index {index} is not one of {groups}.")
    return MXWeight(q[index].view(weight.qdata.dtype), s[index].view(weight.scale.dtype), weight.elem_dtype,
                    weight.block_size, weight.orig_dtype, weight.is_swizzled_scales, weight.scaling_mode)


class _MxLinear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, qdata, scale, swizzled, bias, activation_dtype):  # noqa: ANN001, ANN205
        ctx.save_for_backward(qdata, scale)
        ctx.swizzled = swizzled
        return K.mx_matmul(x, qdata, scale, swizzled=swizzled, bias=bias, activation_dtype=activation_dtype)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):  # noqa: ANN001, ANN205
        qdata, scale = ctx.saved_tensors
        return K.mx_matmul_input_grad(dy, qdata, scale, swizzled=ctx.swizzled), None, None, None, None, None


class _GroupedMx(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, qdata, scale, ends, swizzled, activation_dtype):  # noqa: ANN001, ANN205
        ctx.save_for_backward(qdata, scale, ends)
        ctx.swizzled = swizzled
        return K.grouped_mx_matmul(x, qdata, scale, ends, swizzled=swizzled, activation_dtype=activation_dtype)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):  # noqa: ANN001, ANN205
        qdata, scale, ends = ctx.saved_tensors
        return K.grouped_mx_matmul_input_grad(dy, qdata, scale, ends, swizzled=ctx.swizzled), None, None, None, None, None


class _GroupedDense(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, ends):  # noqa: ANN001, ANN205
        ctx.save_for_backward(x, weight, ends)
        return K.grouped_matmul(x, weight, ends)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):  # noqa: ANN001, ANN205
        x, weight, ends = ctx.saved_tensors
        dx = K.grouped_matmul_input_grad(dy, weight, ends) if ctx.needs_input_grad[0] else None
        dw = K.grouped_matmul_weight_grad(dy, x, ends) if ctx.needs_input_grad[1] else None
        return dx, dw, None


def mx_linear(x: torch.Tensor, weight: MXWeight, bias: torch.Tensor | None = None, *,
              activation_dtype: torch.dtype | None = None) -> torch.Tensor:
    """``x @ W.T + bias`` over an MXFP4 weight, as :func:`.kernels.mx_matmul`; differentiable in ``x``."""
    q, s = _packed("MX linear", weight)
    if bias is not None and bias.requires_grad and torch.is_grad_enabled():
        raise ValueError("MX linear: the bias is frozen with its packed weight; detach it.")
    return _MxLinear.apply(x, q, s, weight.is_swizzled_scales, bias, activation_dtype)


def grouped_linear(x: torch.Tensor, weight: torch.Tensor, ends: torch.Tensor, *,
                   activation_dtype: torch.dtype | None = None) -> torch.Tensor:
    """Rows ``ends[e-1] : ends[e]`` of ``x`` times weight ``e``; rows past ``ends[-1]`` give zeros.

    ``weight``: dense [groups, out, in], differentiable like ``x``, or an MXFP4 ``MXWeight`` whose rows are the
    groups' weights one below the other.  ``ends``: int32 [groups] on the GPU.
    """
    if isinstance(weight, MXWeight):
        q, s = _stacked("Grouped linear", weight, ends.shape[0] if ends.ndim == 1 else 0)
        return _GroupedMx.apply(x, q, s, ends, weight.is_swizzled_scales, activation_dtype)
    if activation_dtype is not None:
        raise ValueError("Grouped linear quantises its input for MXFP4 weights only.")
    return _GroupedDense.apply(x, weight, ends)
