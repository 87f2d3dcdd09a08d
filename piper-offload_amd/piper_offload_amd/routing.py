"""Mixtures of experts: the choice of experts, and rows to their experts and back, with gradients.

    routing = route_experts(x @ router.t(), top_k)
    h = grouped_linear(dispatch_experts(x, routing), up, routing.ends)
    ...
    y = combine_experts(grouped_linear(h, down, routing.ends), routing)

Everything stays on the GPU: nothing waits for the number of an expert's rows,
so all of it can be captured in a graph.  A padding token whose row of logits
is -inf has no expert; its rows are zeros, and so is its output.
"""

from __future__ import annotations

import torch

from . import kernels as K
from .kernels import Routing

__all__ = ["Routing", "combine_experts", "dispatch_experts", "route_experts"]


class _Route(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, top_k, bias, score, groups, top_groups, group_best, renormalize, scale):  # noqa: ANN001, ANN205
        r = K.route_topk(logits, top_k, bias=bias, score=score, groups=groups, top_groups=top_groups, group_best=group_best,
                         renormalize=renormalize, scale=scale)
        ctx.save_for_backward(logits, r.expert)
        ctx.how = dict(score=score, renormalize=renormalize, scale=scale)
        ctx.mark_non_differentiable(r.expert, r.position, r.ends)
        return tuple(r)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dweight, *_):  # noqa: ANN001, ANN205
        return K.route_topk_grad(dweight, *ctx.saved_tensors, **ctx.how), *(None,) * 8


class _Dispatch(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, position, ends):  # noqa: ANN001, ANN205
        ctx.save_for_backward(position, ends)
        return K.dispatch_rows(x, position, ends)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):  # noqa: ANN001, ANN205
        return K.dispatch_rows_grad(dy, *ctx.saved_tensors), None, None


class _Combine(torch.autograd.Function):
    @staticmethod
    def forward(ctx, h, weight, position, ends):  # noqa: ANN001, ANN205
        ctx.save_for_backward(h, weight, position, ends)
        return K.combine_rows(h, weight, position, ends)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):  # noqa: ANN001, ANN205
        return *K.combine_rows_grad(dy, *ctx.saved_tensors), None, None


def route_experts(logits: torch.Tensor, top_k: int, *, bias: torch.Tensor | None = None, score: str = "softmax",
                  groups: int = 1, top_groups: int = 1, group_best: int = 1, renormalize: bool = True,
                  scale: float = 1.0) -> Routing:
    """The ``top_k`` experts of every token, as :func:`.kernels.route_topk`; ``weight`` is differentiable in ``logits``."""
    if bias is not None and bias.requires_grad and torch.is_grad_enabled():
        raise ValueError("Routing: the bias decides alone and has no gradient; detach it.")
    return Routing(*_Route.apply(logits, top_k, bias, score, groups, top_groups, group_best, renormalize, scale))


def dispatch_experts(x: torch.Tensor, routing: Routing) -> torch.Tensor:
    """The rows of ``x`` [tokens, cols] side by side per expert: [tokens * top_k, cols]; differentiable in ``x``."""
    return _Dispatch.apply(x, routing.position, routing.ends)


def combine_experts(h: torch.Tensor, routing: Routing) -> torch.Tensor:
    """The weighted sums of what the experts return: [tokens, cols]; differentiable in ``h`` and ``routing.weight``."""
    return _Combine.apply(h, routing.weight, routing.position, routing.ends)
