"""One AdamW step over many tensors at once, with fp32 states or states in 8 bits.

Calls enqueue work on the current stream and never wait for the device: the count of
steps lies on the device, so a captured step counts on in every replay.
"""
from __future__ import annotations

from typing import NamedTuple, Optional

import torch

from ._lib import host


class AdamWState(NamedTuple):
    """What a step keeps for a list of parameters (lists in the parameters' order).

    exp_avg, exp_avg_sq: the moments m and v in float32; or, with scales, e4m3 codes of m and of sqrt(v) in the
    parameters' shapes.  exp_avg_scale, exp_avg_sq_scale: float32, one for each 256 elements in memory order; None in
    32 bits.  master: float32 parameters, None for those without (or for all).  step: steps done, int32 on the device.
    """
    exp_avg: list
    exp_avg_sq: list
    exp_avg_scale: Optional[list]
    exp_avg_sq_scale: Optional[list]
    master: Optional[list]
    step: torch.Tensor


def adamw_state(params, *, bits: int = 32, master: bool = False) -> AdamWState:
    """The state before the first step.  bits: 32 or 8; ``master=True`` keeps 16-bit parameters in float32 beside
    them, so that a step smaller than their spacing is not lost."""
    params = list(params)
    if bits not in (8, 32):
        raise ValueError(f"adamw_state: bits must be 8 or 32, got {bits}")
    if not params:
        raise ValueError("adamw_state: no parameters")
    dtype = torch.float8_e4m3fn if bits == 8 else torch.float32

    def zeros(p):
        return torch.empty_like(p, dtype=torch.uint8 if bits == 8 else dtype, requires_grad=False).zero_().view(dtype)

    def scales(p):
        return torch.zeros(-(-p.numel() // 256), dtype=torch.float32, device=p.device)

    copies = [None if p.dtype == torch.float32 else p.detach().float() for p in params] if master else None
    return AdamWState([zeros(p) for p in params], [zeros(p) for p in params], [scales(p) for p in params] if bits == 8 else None,
                      [scales(p) for p in params] if bits == 8 else None, copies,
                      torch.zeros((), dtype=torch.int32, device=params[0].device))


def adamw_step(params, grads, state, *, lr, betas=(0.9, 0.999), eps: float = 1e-8, weight_decay: float = 0.01,
               norm=None, max_norm=None) -> None:
    """One step in place: m = b1 m + (1 - b1) g, v = b2 v + (1 - b2) g^2, p = p (1 - lr weight_decay) -
    lr / (1 - b1^t) m / (sqrt(v) / sqrt(1 - b2^t) + eps), t = ++state.step.

    grads: of their parameters' types or float32, unchanged.  ``norm`` (float32 on the device, ``grad_norm``'s) with
    ``max_norm`` scales them by min(1, max_norm / (norm + 1e-6)) on the way, which saves ``clip_grad_norm``'s pass.
    lr: a number, or one float32 value on the device that a captured step reads anew.  m and v are rounded to float32 at
    every operation; the change of p is within 2^-19 of itself, and its divisor at least 2^-63; parameters without a
    master are rounded to their own type.  eps: 0 to 1e30.  Tensors that are written share no memory with others of the
    call.  A norm or gradient that is not a number makes what it reaches that, states included: in 8 bits the 256
    elements that share its scale."""
    host().adamw_step(params, grads, *state[:6], lr, *betas, eps, weight_decay, norm, max_norm)


def adamw_moments(state):
    """(m, v) of a state as lists of float32 tensors; of 8-bit states the numbers that their codes stand for."""
    if state[2] is None:
        return [m.clone() for m in state[0]], [v.clone() for v in state[1]]
    return host().adamw_moments(*state[:4])
