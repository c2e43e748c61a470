"""The global norm of many gradients, and the gradients clipped to a limit.

Calls enqueue work on the current stream and never wait for the device: the norm
comes back as a float32 scalar on the device.
"""
from __future__ import annotations

from array import array

import torch

from ._lib import FLOAT_TYPES, call, device_of, load_library


def _dense(t) -> bool:
    """Whether t's elements fill one stretch of memory, in any order of its dimensions."""
    size = 1
    for step, length in sorted((s, n) for s, n in zip(t.stride(), t.shape) if n > 1):
        if step != size:
            return False
        size *= length
    return True


def _addresses(tensors, what: str):
    """Host arrays (addresses, element types) of float tensors, each dense in memory, and whether all are
    contiguous."""
    try:
        types = array("i", [FLOAT_TYPES[t.dtype] for t in tensors])
    except KeyError as e:
        raise ValueError(f"{what}: gradients are float32, float16 or bfloat16, got {e.args[0]}") from None
    contiguous = False not in map(torch.Tensor.is_contiguous, tensors)
    if not contiguous:
        for t in tensors:
            if not t.is_contiguous() and not _dense(t):
                raise ValueError(f"{what}: gradients must be dense in memory, got strides {t.stride()} for "
                                 f"{tuple(t.shape)}")
    addresses = list(map(torch.Tensor.data_ptr, tensors))
    if len(set(addresses)) != len(addresses):  # tensors without elements may share an address
        full = [t.data_ptr() for t in tensors if t.numel()]
        if len(set(full)) != len(full):
            raise ValueError(f"{what}: a tensor is listed twice")
    return array("Q", addresses), types, contiguous


def _tensors(v):
    return [v] if torch.is_tensor(v) else list(v)


def _run(grads, limit, out, what):
    grads = _tensors(grads)
    if not grads:
        raise ValueError(f"{what}: no gradients")
    first = grads[0]
    device = device_of(what, *grads)
    pointers, types, contiguous = _addresses(grads, what)
    sizes = array("q", map(torch.Tensor.numel, grads))
    L = load_library()
    norm = first.new_empty((), dtype=torch.float32)
    nbytes = L.hb_clip_workspace(len(grads))
    ws = first.new_empty(nbytes, dtype=torch.uint8)
    host = [len(grads), pointers.buffer_info()[0], sizes.buffer_info()[0], types.buffer_info()[0]]
    if limit is None:
        call(device, L.hb_grad_norm, *host, norm.data_ptr(), ws.data_ptr(), nbytes)
        return norm
    limit = float(limit)
    if not limit >= 0.0:
        raise ValueError(f"{what}: max_norm must be a number >= 0, got {limit}")
    to_pointers, to_types = pointers, types
    if out is not None:
        out = _tensors(out)
        if [g.shape for g in grads] != [o.shape for o in out]:
            raise ValueError(f"{what}: outputs have their gradients' shapes")
        device_of(what, first, *out)
        to_pointers, to_types, to_contiguous = _addresses(out, what)
        if not (contiguous and to_contiguous) and any(o.stride() != g.stride() for g, o in zip(grads, out)
                                                      if not (g.is_contiguous() and o.is_contiguous())):
            raise ValueError(f"{what}: outputs have their gradients' strides")
        if to_types != types:
            for g, o in zip(grads, out):
                if o.dtype != g.dtype and (o.dtype != torch.float32 or (g.numel() and o.data_ptr() == g.data_ptr())):
                    raise ValueError(f"{what}: an output has its gradient's type, or is float32 and not in place; got "
                                     f"{o.dtype} for {g.dtype}")
    call(device, L.hb_clip_grad_norm, *host, to_pointers.buffer_info()[0], to_types.buffer_info()[0], limit,
         norm.data_ptr(), ws.data_ptr(), nbytes)
    return norm


def grad_norm(grads):
    """sqrt of the sum of squares of all elements of a list of tensors (float32 scalar on the device)."""
    return _run(grads, None, None, "grad_norm")


def clip_grad_norm(grads, max_norm: float, *, out=None):
    """Scales a list of gradients by min(1, max_norm / (norm + 1e-6)), norm their global norm, in place or into
    ``out`` (tensors of the same shapes, of the gradients' types or float32), and returns the norm before
    clipping (float32 scalar on the device).  A norm that is not a number makes every gradient that."""
    return _run(grads, max_norm, out, "clip_grad_norm")
