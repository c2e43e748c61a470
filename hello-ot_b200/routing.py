"""An assignment of tokens to experts applied to rows of features.

``route_plan`` sorts the entries of an assignment (a router's choice, or a
transport plan between tokens and experts, see ``assignment_of_plan``) by expert;
``route_dispatch`` brings the tokens' rows into that order for the experts, and
``route_combine`` brings the experts' rows back to their tokens, weighted.  Both are
differentiable; ``route_dispatch_grad`` and ``route_combine_grad`` are their
gradients by themselves, whose results have no history.  Entries without an expert (an index outside
0..num_experts-1) are sorted last, receive zero rows and add nothing.

The calls enqueue work on the current stream and never wait for the device, so the
sorted arrays always have tokens * slots rows; ``plan.offsets[-1]`` of them (on the
device) belong to an expert.
"""
from __future__ import annotations

from typing import NamedTuple

import torch
from torch.autograd.function import once_differentiable

from ._lib import host


class RoutePlan(NamedTuple):
    """Entries t * slots + k of an assignment sorted by expert (int32 device tensors).

    order: the entry of each place.  position [tokens, slots]: the place of each
    entry.  offsets [num_experts + 1]: first place of each expert; the last is the
    number of entries that have one.
    """
    order: torch.Tensor
    position: torch.Tensor
    offsets: torch.Tensor

    @property
    def tokens(self) -> int:
        return self.position.shape[0]

    @property
    def slots(self) -> int:
        return self.position.shape[1]

    @property
    def num_experts(self) -> int:
        return self.offsets.numel() - 1

    @property
    def counts(self) -> torch.Tensor:
        """Entries of each expert."""
        return self.offsets[1:] - self.offsets[:-1]


def route_plan(index, num_experts: int) -> RoutePlan:
    """Stable sort of an assignment ``index`` ([tokens] or [tokens, slots], int32 or int64) by expert."""
    return RoutePlan(*host().route_plan(index, num_experts))


def route_dispatch_grad(dsorted, plan):
    """Gradient of ``route_dispatch`` with respect to x: each token's sorted rows added up."""
    return host().route_combine(dsorted, plan[1], plan[2], None, "route_dispatch_grad")


def route_combine_grad(dy, z, plan, weights=None, *, need_weights: bool = True):
    """Gradients of ``route_combine`` with respect to z and weights, as (dz, dweights); dweights is None
    without weights or with ``need_weights=False``."""
    return host().route_combine_grad(dy, z, plan[1], plan[2], weights, bool(need_weights))


class _Dispatch(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, position, offsets):
        ctx.save_for_backward(position, offsets)
        ctx.save_for_forward(position, offsets)
        return host().route_dispatch(x, position, offsets)

    @staticmethod
    @once_differentiable
    def backward(ctx, dsorted):
        return route_dispatch_grad(dsorted, (None, *ctx.saved_tensors)), None, None

    @staticmethod
    def jvp(ctx, dx, _position, _offsets):
        return route_dispatch(dx, (None, *ctx.saved_tensors))


class _Combine(torch.autograd.Function):
    @staticmethod
    def forward(ctx, z, position, offsets, weights):
        ctx.set_materialize_grads(False)  # a tangent that is not there is None
        ctx.save_for_backward(z, position, offsets, weights)
        ctx.save_for_forward(z, position, offsets, weights)
        return host().route_combine(z, position, offsets, weights, "route_combine")

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        if dy is None:
            return None, None, None, None
        z, position, offsets, weights = ctx.saved_tensors
        dz, dw = route_combine_grad(dy, z, (None, position, offsets), weights, need_weights=ctx.needs_input_grad[3])
        return dz, None, None, dw

    @staticmethod
    def jvp(ctx, dz, _position, _offsets, dw):
        z, position, offsets, weights = ctx.saved_tensors
        plan = None, position, offsets
        if dw is None:
            return route_combine(dz, plan, weights)
        if dz is None:
            return route_combine(z, plan, dw)
        # both sums in fp32, so that theirs is rounded once
        return (route_combine(dz.float(), plan, weights) + route_combine(z.float(), plan, dw)).to(z.dtype)


def route_dispatch(x, plan):
    """x's rows [tokens, width] in the plan's order, [tokens * slots, width]; zero rows for entries without
    an expert.  Differentiable in x, backward and forward."""
    if host().recorded(x):
        return _Dispatch.apply(x, plan[1], plan[2])
    return host().route_dispatch(x, plan[1], plan[2])


def route_combine(z, plan, weights=None):
    """sum_k weights[t, k] z[position[t, k]] over the entries with an expert, [tokens, width]; weights of 1
    when there are none.  Differentiable in z and weights, backward and forward."""
    if host().recorded(z, weights):
        return _Combine.apply(z, plan[1], plan[2], weights)
    return host().route_combine(z, plan[1], plan[2], weights, "route_combine")


def assignment_of_plan(rows, cols, mass, tokens: int, *, tolerance: float = 0.0, device=None):
    """The assignment of a transport plan from tokens to experts: (index int32 [tokens, slots], weights
    float32 [tokens, slots]).  An edge of more than ``tolerance`` mass is an entry; a token's weights are its
    edges' shares of its mass, heaviest expert first (the lower expert first on a tie); tokens with fewer
    edges than the most get -1 and weight 0.  Waits for the device (the number of slots is a shape)."""
    dev = torch.device(device) if device is not None else (rows.device if torch.is_tensor(rows) else torch.device("cuda"))
    r = torch.as_tensor(rows, device=dev).to(torch.int64).view(-1)
    c = torch.as_tensor(cols, device=dev).to(torch.int64).view(-1)
    m = torch.as_tensor(mass, device=dev).to(torch.float64).view(-1)
    if not r.numel() == c.numel() == m.numel():
        raise ValueError("rows, cols and mass must have equal lengths")
    if not bool(torch.isfinite(m).all()):
        raise ValueError("a mass of the plan is not finite")
    live = m > tolerance
    r, c, m = r[live], c[live], m[live]
    if r.numel() and (int(r.min()) < 0 or int(r.max()) >= tokens):
        raise ValueError("a row of the plan is outside the tokens")
    if c.numel() and (int(c.min()) < 0 or int(c.max()) >= 2 ** 31 - 1):
        raise ValueError("a column of the plan is no expert: negative, or 2^31 - 1 and above")
    by = torch.argsort(c, stable=True)
    by = by[torch.argsort(m[by], descending=True, stable=True)]
    by = by[torch.argsort(r[by], stable=True)]
    r, c, m = r[by], c[by], m[by]
    count = torch.bincount(r, minlength=tokens)
    slots = max(1, int(count.max()) if tokens else 1)
    slot = torch.arange(r.numel(), device=dev) - (torch.cumsum(count, 0) - count)[r]
    index = torch.full((tokens, slots), -1, dtype=torch.int32, device=dev)
    weights = torch.zeros((tokens, slots), dtype=torch.float64, device=dev)
    index[r, slot] = c.to(torch.int32)
    weights[r, slot] = m
    total = weights.sum(1, keepdim=True)
    return index, (weights / torch.where(total > 0, total, torch.ones_like(total))).to(torch.float32)
