"""The global norm of many gradients, and the gradients clipped to a limit.

Calls enqueue work on the current stream and never wait for the device: the norm
comes back as a float32 scalar on the device.
"""
from __future__ import annotations

from array import array

import torch

from ._lib import FLOAT_TYPES, check, current, on_device


def _dense(t) -> bool:
    """Whether t's elements fill one stretch of memory, in any order of its dimensions."""
    if t.is_contiguous():
        return True
    size = 1
    for step, length in sorted((s, n) for s, n in zip(t.stride(), t.shape) if n > 1):
        if step != size:
            return False
        size *= length
    return True


def _addresses(tensors, what: str):
    """Host arrays (addresses, element types) of float tensors, each dense in memory."""
    for t in tensors:
        if t.dtype not in FLOAT_TYPES:
            raise ValueError(f"{what}: gradients are float32, float16 or bfloat16, got {t.dtype}")
        if not _dense(t):
            raise ValueError(f"{what}: gradients must be dense in memory, got strides {t.stride()} for {tuple(t.shape)}")
    addresses = array("Q", [t.data_ptr() for t in tensors])
    if len({a for a in addresses if a}) != sum(1 for a in addresses if a):
        raise ValueError(f"{what}: a tensor is listed twice")
    return addresses, array("i", [FLOAT_TYPES[t.dtype] for t in tensors])


def _address(a):
    return a.buffer_info()[0] if a else None


def _run(grads, limit, out, what):
    grads = [grads] if torch.is_tensor(grads) else list(grads)
    if not grads:
        raise ValueError(f"{what}: no gradients")
    L = on_device(what, *grads)
    pointers, types = _addresses(grads, what)
    sizes = array("q", [g.numel() for g in grads])
    first = grads[0]
    norm = torch.empty((), dtype=torch.float32, device=first.device)
    nbytes = L.hb_clip_workspace(len(grads))
    ws = torch.empty(nbytes, dtype=torch.uint8, device=first.device)
    common = (len(grads), _address(pointers), _address(sizes), _address(types))
    if limit is None:
        with current(first) as stream:
            rc = L.hb_grad_norm(*common, norm.data_ptr(), ws.data_ptr(), nbytes, stream)
    else:
        limit = float(limit)
        if not limit >= 0.0:
            raise ValueError(f"{what}: max_norm must be a number >= 0, got {limit}")
        to_pointers, to_types = pointers, types
        if out is not None:
            out = [out] if torch.is_tensor(out) else list(out)
            if len(out) != len(grads):
                raise ValueError(f"{what}: {len(out)} outputs for {len(grads)} gradients")
            on_device(what, first, *out)
            for g, o in zip(grads, out):
                if o.shape != g.shape or (o.dtype != g.dtype and o.dtype != torch.float32):
                    raise ValueError(f"{what}: an output has its gradient's shape, and its type or float32; got "
                                     f"{tuple(o.shape)} {o.dtype} for {tuple(g.shape)} {g.dtype}")
                if o.stride() != g.stride() and not (o.is_contiguous() and g.is_contiguous()):
                    raise ValueError(f"{what}: an output has its gradient's strides")
                if o.dtype != g.dtype and o.data_ptr() == g.data_ptr() and g.numel():
                    raise ValueError(f"{what}: an output in place has its gradient's type")
            to_pointers, to_types = _addresses(out, what)
        with current(first) as stream:
            rc = L.hb_clip_grad_norm(*common, _address(to_pointers), _address(to_types), limit, norm.data_ptr(),
                                     ws.data_ptr(), nbytes, stream)
    check(rc)
    return norm


def grad_norm(grads):
    """sqrt of the sum of squares of all elements of a list of tensors (float32 scalar on the device)."""
    return _run(grads, None, None, "grad_norm")


def clip_grad_norm(grads, max_norm: float, *, out=None):
    """Scales a list of gradients by min(1, max_norm / (norm + 1e-6)), norm their global norm, in place or into
    ``out`` (tensors of the same shapes, of the gradients' types or float32), and returns the norm before
    clipping (float32 scalar on the device).  A norm that is not a number makes every gradient that."""
    return _run(grads, max_norm, out, "clip_grad_norm")
