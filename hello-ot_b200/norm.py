"""Root-mean-square norm of rows with the residual's addition, its output in 8 bits, and its gradients.

Rows are the last dimension of tensors of any shape.  Sums are fp32, whatever the
type, and results are rounded once; so a row's squares have to sum to an fp32 number
(values of some 1e18 at most, and with eps 0 of some 1e-18 at least).  Calls enqueue
work on the current stream and never wait for the device.
"""
from __future__ import annotations

from typing import NamedTuple, Optional

import torch
from torch.autograd.function import once_differentiable

from ._lib import host


class Rows8(NamedTuple):
    """Rows in 8 bits: values e4m3 [..., width], scales e8m0 (powers of two) [..., ceil(width / 32)], one for each 32
    columns of a row.  A row's numbers are value * scale; a group that holds a value which is not finite reads as NaN."""
    values: torch.Tensor
    scales: torch.Tensor


def rms_norm_grad(dy, x, weight, *, dsum=None, eps: float = 1e-6, needs=(True, True)):
    """Gradients of ``rms_norm`` with respect to the normalised rows and weight, as (dx, dweight), None where
    ``needs`` is False.  ``x`` are the rows that were normalised (the returned sum, where there was a residual; x and
    the residual then have the same gradient dx) and ``dsum`` the gradient that reaches that sum from elsewhere.  The
    results have no history."""
    return host().rms_norm_grad(dy, x, weight, dsum, eps, bool(needs[0]), bool(needs[1]))


class _Norm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, residual, eps):
        ctx.set_materialize_grads(False)
        ctx.eps = eps
        y, _, total = host().rms_norm(x, weight, residual, eps, False)
        ctx.save_for_backward(x if residual is None else total, weight)
        return y if residual is None else (y, total)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, dsum=None):
        x, weight = ctx.saved_tensors
        need_x, need_w, need_residual, _ = ctx.needs_input_grad
        if dy is None:  # the norm itself went nowhere
            dx, dw = dsum, None
        else:
            dx, dw = rms_norm_grad(dy, x, weight, dsum=dsum, eps=ctx.eps, needs=(need_x or need_residual, need_w))
        return dx if need_x else None, dw, dx if need_residual else None, None


def rms_norm(x, weight, residual=None, *, eps: float = 1e-6):
    """x / sqrt(mean(x^2) + eps) * weight over the last dimension.  With ``residual`` (x's shape and type) the rows
    x + residual are normalised, and (y, x + residual) is returned; y is computed from the sum before it is rounded.
    weight: [width] of any of the three types.  Differentiable in all three."""
    if host().recorded(x, weight, residual):
        return _Norm.apply(x, weight, residual, host().number(eps))
    y, _, total = host().rms_norm(x, weight, residual, eps, False)
    return y if residual is None else (y, total)


def rms_norm_8bit(x, weight, residual=None, *, eps: float = 1e-6) -> tuple[Rows8, Optional[torch.Tensor]]:
    """``rms_norm`` with y in 8 bits, as (Rows8, x + residual or None).  The scale of 32 columns is the smallest power of
    two by which their largest magnitude fits e4m3's 448, so nothing saturates.  The results have no history."""
    values, scales, total = host().rms_norm(x, weight, residual, eps, True)
    return Rows8(values, scales), total


def rows_of_8bit(rows, *, dtype=torch.float32):
    """The numbers that ``Rows8`` stand for, in ``dtype`` (exact in float32 and bfloat16, but for subnormal ones)."""
    return host().rows_of_8bit(rows[0], rows[1], dtype)
