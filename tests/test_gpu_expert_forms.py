"""The experts' products where their forms differ: activations of far values, rows that lie far apart, tiles past the
first band, parts of sums over pairs of blocks."""
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


@pytest.mark.parametrize("name", ["gelu", "silu"])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("rows", [16, 4000])
def test_activations_of_far_values_in_16_bits(hb, cuda, rows, dtype, name):
    """Relative to the value: the approximations are within 2^-18 and the exponential's argument within 2 g^2 2^-24 (silu:
    2 |g| 2^-23), the result is rounded once.  u lifts what fp16 would hold in fewer bits."""
    left = -9.0 if dtype == torch.float16 else -12.5
    g = torch.linspace(left, -0.001, rows, device=cuda).to(dtype).float()
    lift = 2.0 ** 15
    x, gate, up = _alone(cuda, g, dtype, lift)
    value, slope, cdf, bell = _gelu(g)
    if name == "silu":
        value, slope = er.activation(g.double(), "silu")
        cdf, bell = torch.sigmoid(g.double()), (g.double() * torch.sigmoid(g.double())).abs()
    u, floor = ref.U[dtype], ref.FLOOR[dtype]
    near = 2.0 ** -18 + 2 * g.double().square() * 2.0 ** -24 + 2 * g.double().abs() * er.E23
    bound = lift * value.abs() * (near * (1 + u) + u) + floor
    er.close(hb.expert_gated(x, gate, up, activation=name)[:, 0], lift * value, bound, name)
    x[:, 1] = 1.0
    dx, _, _ = hb.expert_gated_grad(torch.full((rows, 1), lift, device=cuda).to(dtype), x, gate, up, activation=name)
    er.close(dx[:, 1], lift * value, bound, "du")
    # dg passes on in dtype and its product is exact: rounded once
    er.close(dx[:, 0], lift * slope, lift * (near * (cdf + bell) * (1 + u) + u * slope.abs()) + floor, "dg")


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_rows_far_apart(hb, cuda, dtype):
    """Rows more than 2^31 elements apart are taken like any others."""
    gen = torch.Generator(device=cuda).manual_seed(6)
    apart, width = 2 ** 31 + 8, 24
    room = torch.empty(apart + width, dtype=dtype, device=cuda)
    far = room.as_strided((2, width), (apart, 1))
    far.copy_(torch.randn((2, width), generator=gen, device=cuda))
    near = far.contiguous()
    gate, up = (torch.randn((2, width, width), generator=gen, device=cuda).to(dtype) for _ in range(2))
    first = torch.tensor([0, 1, 2], dtype=torch.int32, device=cuda)
    assert torch.equal(hb.expert_product(far, gate, first), hb.expert_product(near, gate, first))
    assert torch.equal(hb.expert_gated(far, gate, up, first), hb.expert_gated(near, gate, up, first))
    for got, want in ((hb.expert_product_grad(far, far, gate, first), hb.expert_product_grad(near, near, gate, first)),
                      (hb.expert_gated_grad(far, far, gate, up, first), hb.expert_gated_grad(near, near, gate, up, first))):
        assert all(torch.equal(a, b) for a, b in zip(got, want))


# counts, rows behind the last, width, hidden.  Tiles of an expert come in bands of 8: several bands and a partial one with several
# tiles of columns, in pairs of blocks and by single ones (few rows an expert on average); sums over rows cut into parts over
# pairs; weights with more than one band of their own.
BANDS = {
    "bands of pairs": ([4500, 2300], 300, 264, 520),
    "bands of single blocks": ([1300] + [0] * 9 + [60, 7], 20, 264, 392),
    "parts over pairs": ([6000], 0, 264, 520),
    "parts over pairs, uneven": ([9000, 17, 0, 3300], 5, 136, 200),
    "bands of weights": ([200, 130], 0, 300, 2600),
    "bands of wide rows": ([150, 300], 9, 2600, 264),
}


@pytest.mark.parametrize("dtype", ref.DTYPES)
@pytest.mark.parametrize("shape", BANDS)
def test_bands_and_parts(hb, cuda, shape, dtype):
    counts, behind, width, hidden = BANDS[shape]
    gen = torch.Generator(device=cuda).manual_seed(len(shape))
    offsets, rows = er.groups(counts, behind)
    first = torch.tensor(offsets, dtype=torch.int32, device=cuda)

    def normal(*size, scale=1.0):
        return (torch.randn(size, generator=gen, device=cuda) * scale).to(dtype)

    x, dy = normal(rows, width), normal(rows, hidden)
    gate, up = (normal(len(counts), hidden, width, scale=width ** -0.5) for _ in range(2))
    x[offsets[-1]:], dy[offsets[-1]:] = float("nan"), float("inf")
    x64, dy64 = x.double(), dy.double()
    x64[offsets[-1]:], dy64[offsets[-1]:] = 0, 0
    y = hb.expert_product(x, gate, first)
    er.close(y, *er.product(x64, gate.double(), offsets, dtype), "product")
    h = hb.expert_gated(x, gate, up, first)
    er.close(h, *er.gated(x64, gate.double(), up.double(), offsets, "silu", dtype), "gated")
    got = [*hb.expert_product_grad(dy, x, gate, first), *hb.expert_gated_grad(dy, x, gate, up, first)]
    wants = [*er.product_grad(dy64, x64, gate.double(), offsets, dtype),
             *er.gated_grad(dy64, x64, gate.double(), up.double(), offsets, "silu", dtype)]
    for name, g, (want, bound) in zip(("dx", "dw", "gated dx", "dgate", "dup"), got, wants):
        er.close(g, want, bound, name)
    again = [*hb.expert_product_grad(dy, x, gate, first), *hb.expert_gated_grad(dy, x, gate, up, first)]
    assert all(torch.equal(a, b) for a, b in zip(got, again)) and torch.equal(y, hb.expert_product(x, gate, first))
