"""An assignment of tokens to experts applied to rows of features.

``route_plan`` sorts the entries of an assignment (a router's choice, or a
transport plan between tokens and experts, see ``assignment_of_plan``) by expert;
``route_dispatch`` brings the tokens' rows into that order for the experts, and
``route_combine`` brings the experts' rows back to their tokens, weighted.  Both are
differentiable; ``route_dispatch_grad`` and ``route_combine_grad`` are their
gradients by themselves.  Entries without an expert (an index outside
0..num_experts-1) are sorted last, receive zero rows and add nothing.

The calls enqueue work on the current stream and never wait for the device, so the
sorted arrays always have tokens * slots rows; ``plan.offsets[-1]`` of them (on the
device) belong to an expert.
"""
from __future__ import annotations

from typing import NamedTuple

import torch
from torch.autograd.function import once_differentiable

from ._lib import FLOAT_TYPES, call, device_of, feature_rows, index_bytes, load_library


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
    if index.dim() not in (1, 2) or (index.dim() == 2 and index.shape[1] < 1):
        raise ValueError(f"index must be [tokens] or [tokens, slots], got {tuple(index.shape)}")
    size = index_bytes(index, "index")
    num_experts = int(num_experts)
    if not 1 <= num_experts < 2 ** 31 - 1:
        raise ValueError("num_experts must be positive and below 2^31 - 1")
    n = index.numel()
    if n >= 2 ** 31:
        raise ValueError("an assignment holds at most 2^31 - 1 entries")
    device = device_of("route_plan", index)
    index = index.contiguous()
    L = load_library()
    int32 = torch.int32
    order = index.new_empty(n, dtype=int32)
    position = index.new_empty((index.shape[0], 1 if index.dim() == 1 else index.shape[1]), dtype=int32)
    offsets = index.new_empty(num_experts + 1, dtype=int32)
    nbytes = L.hb_index_sort_workspace(n, num_experts)
    ws = index.new_empty(nbytes, dtype=torch.uint8) if nbytes else None
    call(device, L.hb_index_sort, index.data_ptr(), size, n, num_experts, order.data_ptr(), position.data_ptr(),
         offsets.data_ptr(), None if ws is None else ws.data_ptr(), nbytes)
    return RoutePlan(order, position, offsets)


def _places(plan, what: str):
    """(position, address of the number of entries with an expert) of a checked plan."""
    _, position, offsets = plan
    int32 = torch.int32
    if position.dtype != int32 or offsets.dtype != int32 or position.dim() != 2 or offsets.dim() != 1:
        raise ValueError(f"{what}: a plan holds int32 position [tokens, slots] and offsets [num_experts + 1]")
    ends = offsets.numel()
    if not position.is_contiguous() or not offsets.is_contiguous() or ends < 2 or position.size(1) < 1:
        raise ValueError(f"{what}: a plan's tensors are contiguous, with at least one slot and one expert")
    return position, offsets.data_ptr() + 4 * (ends - 1)


def _weights(weights, position, what: str):
    if weights.dtype not in FLOAT_TYPES:
        raise ValueError(f"{what}: weights must be float32, float16 or bfloat16, got {weights.dtype}")
    if weights.shape != position.shape and (weights.shape != position.shape[:1] or position.size(1) != 1):
        raise ValueError(f"{what}: weights {tuple(weights.shape)} do not fit an assignment {tuple(position.shape)}")
    return weights.contiguous()


def _dispatch(x, plan):
    x, stride = feature_rows(x, "x")
    position, kept = _places(plan, "route_dispatch")
    tokens, slots = position.shape
    if x.shape[0] != tokens:
        raise ValueError(f"route_dispatch: x has {x.shape[0]} rows for {tokens} tokens")
    device = device_of("route_dispatch", x, position, plan.offsets)
    width = x.shape[1]
    out = x.new_empty((tokens * slots, width))
    call(device, load_library().hb_route_dispatch, FLOAT_TYPES[x.dtype], x.data_ptr(), stride, tokens, slots, width,
         position.data_ptr(), kept, out.data_ptr())
    return out


def _combine(z, plan, weights, what="route_combine"):
    z, stride = feature_rows(z, "z")
    position, kept = _places(plan, what)
    tokens, slots = position.shape
    if z.shape[0] != tokens * slots:
        raise ValueError(f"{what}: {z.shape[0]} sorted rows for {tokens} x {slots} entries")
    if weights is None:
        device, wptr, wtype = device_of(what, z, position, plan.offsets), None, 0
    else:
        weights = _weights(weights, position, what)
        device = device_of(what, z, position, plan.offsets, weights)
        wptr, wtype = weights.data_ptr(), FLOAT_TYPES[weights.dtype]
    width = z.shape[1]
    out = z.new_empty((tokens, width))
    call(device, load_library().hb_route_combine, FLOAT_TYPES[z.dtype], z.data_ptr(), stride, tokens, slots, width,
         position.data_ptr(), kept, wptr, wtype, out.data_ptr())
    return out


def route_dispatch_grad(dsorted, plan):
    """Gradient of ``route_dispatch`` with respect to x: each token's sorted rows added up."""
    return _combine(dsorted, plan, None, "route_dispatch_grad")


def route_combine_grad(dy, z, plan, weights=None, *, need_weights: bool = True):
    """Gradients of ``route_combine`` with respect to z and weights, as (dz, dweights); dweights is None
    without weights or with ``need_weights=False``."""
    what = "route_combine_grad"
    dy, dy_stride = feature_rows(dy, "dy")
    z, z_stride = feature_rows(z, "z")
    position, kept = _places(plan, what)
    tokens, slots = position.shape
    if dy.shape != (tokens, z.shape[1]) or z.shape[0] != tokens * slots or dy.dtype != z.dtype:
        raise ValueError(f"{what}: dy {tuple(dy.shape)} {dy.dtype} and z {tuple(z.shape)} {z.dtype} do not fit an "
                         f"assignment {tuple(position.shape)}")
    dw, wptr, wtype = None, None, 0
    if weights is None:
        device = device_of(what, dy, z, position, plan.offsets)
    else:
        weights = _weights(weights, position, what)
        device = device_of(what, dy, z, position, plan.offsets, weights)
        wptr, wtype = weights.data_ptr(), FLOAT_TYPES[weights.dtype]
        if need_weights:
            dw = torch.empty_like(weights)
    dz = z.new_empty((tokens * slots, z.shape[1]))
    call(device, load_library().hb_route_combine_grad, FLOAT_TYPES[z.dtype], dy.data_ptr(), dy_stride, z.data_ptr(),
         z_stride, tokens, slots, z.shape[1], position.data_ptr(), kept, wptr, wtype, dz.data_ptr(),
         None if dw is None else dw.data_ptr())
    return dz, dw


class _Dispatch(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, plan):
        ctx.plan = plan
        return _dispatch(x, plan)

    @staticmethod
    @once_differentiable
    def backward(ctx, dsorted):
        return route_dispatch_grad(dsorted, ctx.plan), None


class _Combine(torch.autograd.Function):
    @staticmethod
    def forward(ctx, z, plan, weights):
        ctx.plan = plan
        ctx.save_for_backward(z, weights)
        return _combine(z, plan, weights)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        z, weights = ctx.saved_tensors
        dz, dw = route_combine_grad(dy, z, ctx.plan, weights, need_weights=ctx.needs_input_grad[2])
        return dz, None, dw


def route_dispatch(x, plan):
    """x's rows [tokens, width] in the plan's order, [tokens * slots, width]; zero rows for entries without
    an expert.  Differentiable in x."""
    if x.requires_grad and torch.is_grad_enabled():
        return _Dispatch.apply(x, plan)
    return _dispatch(x, plan)


def route_combine(z, plan, weights=None):
    """sum_k weights[t, k] z[position[t, k]] over the entries with an expert, [tokens, width]; weights of 1
    when there are none.  Differentiable in z and weights."""
    if torch.is_grad_enabled() and (z.requires_grad or (weights is not None and weights.requires_grad)):
        return _Combine.apply(z, plan, weights)
    return _combine(z, plan, weights)


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
    live = m > tolerance
    r, c, m = r[live], c[live], m[live]
    if r.numel() and (int(r.min()) < 0 or int(r.max()) >= tokens):
        raise ValueError("a row of the plan is outside the tokens")
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
