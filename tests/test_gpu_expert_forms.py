"""The experts' products where their forms differ: activations of far values."""
import math

import pytest
import torch

import expert_reference as er
import rows_reference as ref

pytestmark = pytest.mark.gpu


def _alone(cuda, g, dtype, u):
    """Rows whose projections are g and u exactly: (x, w_gate, w_up)."""
    x = torch.stack([g, torch.full_like(g, u)], 1).to(dtype)
    return x, torch.tensor([[1.0, 0.0]], device=cuda).to(dtype), torch.tensor([[0.0, 1.0]], device=cuda).to(dtype)


def _gelu(g):
    """(value, slope, their bell's term) in 64 bits; relative on the left too."""
    g = g.double()
    cdf = 0.5 * torch.special.erfc(-g * math.sqrt(0.5))
    bell = torch.exp(-0.5 * g * g) / math.sqrt(2 * math.pi)
    return g * cdf, cdf + g * bell, cdf, g.abs() * bell


@pytest.mark.parametrize("rows", [16, 40_000])
def test_gelu_of_far_values_in_32_bits(hb, cuda, rows):
    """Relative to the value, however small.  The normal distribution's function is within 5 units of 2^-23, g its own rounding
    of a product; the slope's exponential within 2 units and g^2 / 2 2^-24 of its argument's rounding, and
    two products and a sum are rounded."""
    g = torch.linspace(-12.5, 6.0, rows, device=cuda)
    x, gate, up = _alone(cuda, g, torch.float32, 1.0)
    value, slope, cdf, bell = _gelu(g)
    e23 = er.E23
    bound = 6 * e23 * value.abs() + ref.FLOOR[torch.float32]
    er.close(hb.expert_gated(x, gate, up, activation="gelu")[:, 0], value, bound, "gelu")
    dx, dgate, dup = hb.expert_gated_grad(torch.ones((rows, 1), device=cuda), x, gate, up, activation="gelu")
    er.close(dx[:, 1], value, bound, "du")
    er.close(dx[:, 0], slope, 5 * e23 * cdf + (g.double().square() / 4 + 4) * e23 * bell + e23 * slope.abs(), "dg")
