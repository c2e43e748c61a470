"""Plain 64-bit forms of the routing, lookup and clipping operators, and the error bounds their tests use.

Bounds: ``U`` is a type's unit roundoff (half the spacing at 1), ``FLOOR`` half its
smallest subnormal.  A sum of m products held in fp32 is off by at most about
m 2^-24 times the sum of their magnitudes, whatever its order; rounding the result
adds U of it.
"""
import numpy as np
import torch

U = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
FLOOR = {torch.float32: 2.0 ** -150, torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134}
E32 = 2.0 ** -24
DTYPES = [torch.float32, torch.float16, torch.bfloat16]


def f64(t):
    return t.detach().to(torch.float64).cpu().numpy()


def plan(index, experts):
    """(order, position, offsets) of a stable sort by expert."""
    index = np.asarray(index)
    flat = index.reshape(-1)
    key = np.where((flat >= 0) & (flat < experts), flat, experts)
    order = np.argsort(key, kind="stable")
    position = np.empty_like(order)
    position[order] = np.arange(order.size)
    count = np.bincount(key, minlength=experts + 1)[:experts]
    return order, position.reshape(index.shape[0], -1), np.concatenate([[0], np.cumsum(count)])


def combine(z, position, kept, weights):
    """(sum_k w z, sum_k |w z|) over the places below kept."""
    t, k = position.shape
    out, mag = np.zeros((t, z.shape[1])), np.zeros((t, z.shape[1]))
    for j in range(k):
        live = position[:, j] < kept
        row = z[position[live, j]] * (1.0 if weights is None else weights[live, j][:, None])
        out[live] += row
        mag[live] += np.abs(row)
    return out, mag


def assert_within(got, want, bound, what=""):
    got = f64(got) if torch.is_tensor(got) else np.asarray(got, dtype=np.float64)
    assert got.shape == want.shape, (what, got.shape, want.shape)
    off = np.abs(got - want)
    assert np.all(off <= bound), f"{what}: off by {np.max(off - bound)} more than the bound"
