"""Rows of a table by index, scaled, and the table's gradient by sorted tokens.

Calls enqueue work on the current stream and never wait for the device.  An id
outside 0..rows-1 (-1 for padding, say) selects no row: a zero row in the lookup,
nothing in the gradient.
"""
from __future__ import annotations

import torch
from torch.autograd.function import once_differentiable

from ._lib import host


def embedding_grad(dy, ids, rows: int, *, scale: float = 1.0, dtype=None, out=None, accumulate: bool = False):
    """Gradient of ``embedding_lookup`` with respect to its table: [rows, width], row v the sum of scale * dy
    over ids == v, summed in fp32 and rounded once to ``dtype`` (dy's, or float32).  ``out`` receives it;
    ``accumulate=True`` adds it to what ``out`` holds and leaves the rows that no id names untouched;
    it shares no memory with dy.  The result has no history."""
    return host().embedding_grad(dy, ids, rows, scale, dtype, out, bool(accumulate))


class _Lookup(torch.autograd.Function):
    @staticmethod
    def forward(ctx, table, ids, scale):
        ctx.rows, ctx.scale = table.shape[0], scale
        ctx.save_for_backward(ids)
        ctx.save_for_forward(ids)
        return host().embedding_lookup(table, ids, scale)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        ids, = ctx.saved_tensors
        if ctx.rows == 0:
            return dy.new_zeros((0, dy.shape[-1])), None, None
        return embedding_grad(dy, ids, ctx.rows, scale=ctx.scale), None, None

    @staticmethod
    def jvp(ctx, dtable, _ids, _scale):
        ids, = ctx.saved_tensors
        return embedding_lookup(dtable, ids, scale=ctx.scale)


def embedding_lookup(table, ids, *, scale: float = 1.0):
    """scale * table[ids], [*ids.shape, width], in fp32 and rounded once to the table's type.  ids: int32 or
    int64 of any shape.  Differentiable in the table, backward (a dense
    gradient) and forward."""
    if host().recorded(table):
        return _Lookup.apply(table, ids, host().number(scale))
    return host().embedding_lookup(table, ids, scale)
