"""The experts of a routed layer: products of rows sorted by expert with each expert's weight.

``x`` holds the sorted rows (``route_dispatch`` brings them into that order) and
``offsets`` the first row of each expert, as ``plan.offsets`` gives it; rows behind
the last expert's are not read and give zero rows.  Without offsets one expert has
all rows: a dense layer, whose weights may be 2-D.  Weights are [experts, hidden,
width] in x's type; slices of one larger weight are taken as they are.  Sums are fp32
and rounded once to the rows' type.  Calls enqueue work on the current stream and never wait for the
device.
"""
from __future__ import annotations

import torch
from torch.autograd.function import once_differentiable

from ._lib import host


def expert_product_grad(dy, x, weight, offsets=None, *, needs=(True, True)):
    """Gradients of ``expert_product`` with respect to x and weight, as (dx, dweight), None where ``needs`` is
    False: dx = dy W of the row's expert, dweight the sum of dy^T x over each expert's rows.  The results have no
    history."""
    return host().expert_product_grad(dy, x, weight, offsets, bool(needs[0]), bool(needs[1]))


def expert_gated_grad(dh, x, w_gate, w_up, offsets=None, *, activation: str = "silu", needs=(True, True, True)):
    """Gradients of ``expert_gated`` with respect to x, w_gate and w_up, as (dx, dw_gate, dw_up), None where
    ``needs`` is False.  Both projections are computed again from the inputs; their gradients pass to the three
    products in the rows' type.  The results have no history."""
    return host().expert_gated_grad(dh, x, w_gate, w_up, offsets, activation, *map(bool, needs))


class _Product(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, offsets):
        ctx.save_for_backward(x, weight, offsets)
        return host().expert_product(x, weight, offsets)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, weight, offsets = ctx.saved_tensors
        return *expert_product_grad(dy, x, weight, offsets, needs=ctx.needs_input_grad[:2]), None


class _Gated(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w_gate, w_up, offsets, activation):
        ctx.activation = activation
        ctx.save_for_backward(x, w_gate, w_up, offsets)
        return host().expert_gated(x, w_gate, w_up, offsets, activation)

    @staticmethod
    @once_differentiable
    def backward(ctx, dh):
        x, w_gate, w_up, offsets = ctx.saved_tensors
        return *expert_gated_grad(dh, x, w_gate, w_up, offsets, activation=ctx.activation,
                                  needs=ctx.needs_input_grad[:3]), None, None


def expert_product(x, weight, offsets=None):
    """x W^T of each row's expert, [rows, hidden].  Differentiable in x and weight."""
    if host().recorded(x, weight):
        return _Product.apply(x, weight, offsets)
    return host().expert_product(x, weight, offsets)


def expert_gated(x, w_gate, w_up, offsets=None, *, activation: str = "silu"):
    """act(x Wg^T) * (x Wu^T) of each row's expert, [rows, hidden], in one kernel: neither projection reaches
    memory.  activation: "silu", g / (1 + exp(-g)), or "gelu", g (1 + erf(g / sqrt 2)) / 2.  Differentiable in x and
    both weights; nothing but the inputs is saved."""
    if host().recorded(x, w_gate, w_up):
        return _Gated.apply(x, w_gate, w_up, offsets, activation)
    return host().expert_gated(x, w_gate, w_up, offsets, activation)
