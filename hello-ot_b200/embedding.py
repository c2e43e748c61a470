"""Rows of a table by index, scaled, and the table's gradient by sorted tokens.

Calls enqueue work on the current stream and never wait for the device.  An id
outside 0..rows-1 (-1 for padding, say) selects no row: a zero row in the lookup,
nothing in the gradient.
"""
from __future__ import annotations

import torch
from torch.autograd.function import once_differentiable

from ._lib import FLOAT_TYPES, call, device_of, feature_rows, index_bytes, load_library


def _lookup(table, ids, scale):
    size = index_bytes(ids, "ids")
    table, stride = feature_rows(table, "table")
    device = device_of("embedding_lookup", table, ids)
    ids = ids.contiguous()
    n, (rows, width) = ids.numel(), table.shape
    if n >= 2 ** 31:
        raise ValueError("embedding_lookup: at most 2^31 - 1 ids")
    out = table.new_empty((*ids.shape, width))
    call(device, load_library().hb_embedding_lookup, FLOAT_TYPES[table.dtype], table.data_ptr(), stride, rows, width,
         ids.data_ptr(), size, n, scale, out.data_ptr())
    return out


def embedding_grad(dy, ids, rows: int, *, scale: float = 1.0, dtype=None, out=None, accumulate: bool = False):
    """Gradient of ``embedding_lookup`` with respect to its table: [rows, width], row v the sum of scale * dy
    over ids == v, summed in fp32 and rounded once to ``dtype`` (dy's, or float32).  ``out`` receives it;
    ``accumulate=True`` adds it to what ``out`` holds and leaves the rows that no id names untouched."""
    what = "embedding_grad"
    size = index_bytes(ids, "ids")
    if dy.shape[:-1] != ids.shape or dy.dim() < 1:
        raise ValueError(f"{what}: dy {tuple(dy.shape)} does not fit ids {tuple(ids.shape)}")
    width = dy.shape[-1]
    rows = int(rows)
    if not 1 <= rows < 2 ** 31 - 1:
        raise ValueError(f"{what}: rows must be positive and below 2^31 - 1")
    if ids.numel() >= 2 ** 31:
        raise ValueError(f"{what}: at most 2^31 - 1 ids")
    dy, stride = feature_rows(dy.reshape(ids.numel(), width), "dy")
    if stride * dy.element_size() >= 2 ** 32:
        dy, stride = dy.contiguous(), width
    if dtype is None:
        dtype = dy.dtype if out is None else out.dtype
    if dtype != dy.dtype and dtype != torch.float32:
        raise ValueError(f"{what}: the gradient of {dy.dtype} rows is {dy.dtype} or float32, not {dtype}")
    if out is None:
        if accumulate:
            raise ValueError(f"{what}: accumulate needs out")
        device = device_of(what, dy, ids)
        out = dy.new_empty((rows, width), dtype=dtype)
    else:
        device = device_of(what, dy, ids, out)
        if out.dtype != dtype or out.shape != (rows, width) or not out.is_contiguous():
            raise ValueError(f"{what}: out must be a contiguous {dtype} tensor of shape {(rows, width)}")
    ids = ids.contiguous()
    n = ids.numel()
    L = load_library()
    nbytes = L.hb_embedding_grad_workspace(n, rows, width)
    ws = dy.new_empty(nbytes, dtype=torch.uint8)
    call(device, L.hb_embedding_grad, FLOAT_TYPES[dy.dtype], dy.data_ptr(), stride, ids.data_ptr(), size, n, rows, width,
         scale, FLOAT_TYPES[dtype], out.data_ptr(), bool(accumulate), ws.data_ptr(), nbytes)
    return out


class _Lookup(torch.autograd.Function):
    @staticmethod
    def forward(ctx, table, ids, scale):
        ctx.rows, ctx.scale = table.shape[0], scale
        ctx.save_for_backward(ids)
        return _lookup(table, ids, scale)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        ids, = ctx.saved_tensors
        return embedding_grad(dy, ids, ctx.rows, scale=ctx.scale), None, None


def embedding_lookup(table, ids, *, scale: float = 1.0):
    """scale * table[ids], [*ids.shape, width], in fp32 and rounded once to the table's type.  ids: int32 or
    int64 of any shape.  Differentiable in the table (a dense gradient)."""
    if table.requires_grad and torch.is_grad_enabled():
        return _Lookup.apply(table, ids, scale)
    return _lookup(table, ids, scale)
