"""Plain 64-bit forms of the experts' products with bounds of their fp32 sums.

A sum of m products held in fp32 is off by at most about m 2^-23 of the sum of their
magnitudes, whatever its order: 2^-24 a step where it is rounded, 2^-23 where the
tensor cores cut it off.  Rounding the result adds U of it (rows_reference).  The
activations are smooth: |act'| <= 1.13, |act''| <= 0.8; their fast exponential and
quotient are off by at most (4 + 2 |g|) 2^-23 of the value, and the error function's
complement by 2^-23.
"""
import math

import torch

import rows_reference as ref

E23 = 2.0 ** -23


def groups(counts, behind=0):
    """(offsets, rows) of consecutive experts with these counts."""
    offsets = [0]
    for c in counts:
        offsets.append(offsets[-1] + c)
    return offsets, offsets[-1] + behind


def activation(g, name):
    """(act, act') in 64 bits."""
    if name == "silu":
        s = torch.sigmoid(g)
        return g * s, s * (1 + g * (1 - s))
    cdf = torch.special.ndtr(g)
    return g * cdf, cdf + g * torch.exp(-0.5 * g * g) / math.sqrt(2 * math.pi)


def close(got, want, bound, what):
    assert got.shape == want.shape, (what, got.shape, want.shape)
    off = (got.double() - want).abs()
    worst = (off - bound).max() if off.numel() else torch.tensor(0.0)
    assert bool((off <= bound).all()), f"{what}: off by {float(worst)} more than the bound ({int((~(off <= bound)).sum())} places)"


def _sum(a, b):
    """(a b, its error) for 64-bit matrices."""
    return a @ b, a.shape[1] * E23 * (a.abs() @ b.abs())


def product(x, w, offsets, dtype):
    """(y, bound): x [rows, width], w [experts, hidden, width] in 64 bits."""
    y = x.new_zeros((x.shape[0], w.shape[1]))
    bound = torch.zeros_like(y)
    for e, (a, b) in enumerate(zip(offsets, offsets[1:])):
        v, err = _sum(x[a:b], w[e].t())
        y[a:b], bound[a:b] = v, err + ref.U[dtype] * (v.abs() + err) + ref.FLOOR[dtype]
    return y, bound


def product_grad(dy, x, w, offsets, dtype):
    """((dx, bound), (dw, bound))."""
    dx, dw = torch.zeros_like(x), torch.zeros_like(w)
    bx, bw = torch.zeros_like(x), torch.zeros_like(w)
    u, floor = ref.U[dtype], ref.FLOOR[dtype]
    for e, (a, b) in enumerate(zip(offsets, offsets[1:])):
        v, err = _sum(dy[a:b], w[e])
        dx[a:b], bx[a:b] = v, err + u * (v.abs() + err) + floor
        v, err = _sum(dy[a:b].t(), x[a:b])
        dw[e], bw[e] = v, err + u * (v.abs() + err) + floor
    return (dx, bx), (dw, bw)


def _projections(x, gate, up, name):
    g, eg = _sum(x, gate.t())
    u, eu = _sum(x, up.t())
    act, slope = activation(g, name)
    fast = (4 + 2 * g.abs()) * E23
    e_act = 1.13 * eg + fast * act.abs() + g.abs() * E23
    e_slope = 0.8 * eg + fast * (slope.abs() + 1) + (1 + g.abs()) * E23
    return u, eu, act, e_act, slope, e_slope


def gated(x, gate, up, offsets, name, dtype):
    """(h, bound)."""
    h = x.new_zeros((x.shape[0], gate.shape[1]))
    bound = torch.zeros_like(h)
    for e, (a, b) in enumerate(zip(offsets, offsets[1:])):
        u, eu, act, e_act, _, _ = _projections(x[a:b], gate[e], up[e], name)
        v = act * u
        err = (act.abs() + e_act) * eu + e_act * u.abs() + E23 * v.abs()
        h[a:b], bound[a:b] = v, err + ref.U[dtype] * (v.abs() + err) + ref.FLOOR[dtype]
    return h, bound


def gated_grad(dh, x, gate, up, offsets, name, dtype):
    """((dx, bound), (dgate, bound), (dup, bound)): dg and du pass in dtype."""
    dx, bx = torch.zeros_like(x), torch.zeros_like(x)
    dw, bw = [torch.zeros_like(gate) for _ in range(2)], [torch.zeros_like(gate) for _ in range(2)]
    ut, floor = ref.U[dtype], ref.FLOOR[dtype]
    for e, (a, b) in enumerate(zip(offsets, offsets[1:])):
        u, eu, act, e_act, slope, e_slope = _projections(x[a:b], gate[e], up[e], name)
        d = dh[a:b]
        parts = []
        for v, err in ((d * u * slope, d.abs() * ((u.abs() + eu) * e_slope + eu * slope.abs()) + 2 * E23 * (d * u * slope).abs()),
                       (d * act, d.abs() * e_act + E23 * (d * act).abs())):
            parts.append((v, err + ut * (v.abs() + err) + floor))
        total, error = torch.zeros_like(x[a:b]), torch.zeros_like(x[a:b])
        for i, ((v, err), w) in enumerate(zip(parts, (gate[e], up[e]))):
            total += v @ w
            error += err @ w.abs() + 2 * v.shape[1] * E23 * ((v.abs() + err) @ w.abs())
            s = v.t() @ x[a:b]
            se = err.t() @ x[a:b].abs() + v.shape[0] * E23 * ((v.abs() + err).t() @ x[a:b].abs())
            dw[i][e], bw[i][e] = s, se + ut * (s.abs() + se) + floor
        dx[a:b], bx[a:b] = total, error + ut * (total.abs() + error) + floor
    return (dx, bx), (dw[0], bw[0]), (dw[1], bw[1])
