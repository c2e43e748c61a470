"""The global norm of many gradients, and the gradients clipped to a limit.

Calls enqueue work on the current stream and never wait for the device: the norm
comes back as a float32 scalar on the device.
"""
from __future__ import annotations

import torch

from ._lib import host


def _list(v):
    return [v] if torch.is_tensor(v) else v if isinstance(v, (list, tuple)) else list(v)


def grad_norm(grads):
    """sqrt of the sum of squares of all elements of a list of tensors (float32 scalar on the device, without
    history)."""
    return host().clip(_list(grads), None, None, "grad_norm")


def clip_grad_norm(grads, max_norm: float, *, out=None):
    """Scales a list of gradients by min(1, max_norm / (norm + 1e-6)), norm their global norm, in place or into
    ``out`` (tensors of the same shapes, of the gradients' types or float32), and returns the norm before
    clipping (float32 scalar on the device).  A norm that is not a number makes every gradient that.  Tensors that
    are written share no memory with one another, nor with a gradient that they are not in place of."""
    if max_norm is None:
        raise ValueError("clip_grad_norm: max_norm must be a number >= 0, got None")
    return host().clip(_list(grads), max_norm, None if out is None else _list(out), "clip_grad_norm")
