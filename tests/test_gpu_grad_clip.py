"""Global gradient norm and clipping against 64-bit forms.

Bound: squares are added in fp32 over at most 32 values, so the sum is off by at
most 32 2^-24 of itself, the norm by half of that, and it is rounded to fp32: 17
2^-24 relative.  The factor carries that and its own rounding: 19 2^-24.
"""
import math

import numpy as np
import pytest
import torch

import rows_reference as ref

pytestmark = pytest.mark.gpu
NORM = 17 * ref.E32
FACTOR = 19 * ref.E32


def _tensors(rng, cuda, sizes, dtypes, scale=1.0):
    return [torch.as_tensor(rng.normal(size=n) * scale, device=cuda).to(dtypes[i % len(dtypes)])
            for i, n in enumerate(sizes)]


def _norm(tensors):
    return math.sqrt(math.fsum(float((ref.f64(t) ** 2).sum()) for t in tensors))


def _check_clipped(got, grads, limit):
    norm = _norm(grads)
    factor = min(1.0, limit / (norm + 1e-6))
    for g, o in zip(grads, got):
        want = ref.f64(g) * factor
        u = ref.U[o.dtype]
        bound = (FACTOR + ref.E32) * np.abs(want) * (1 + u) + u * np.abs(want) + ref.FLOOR[o.dtype]
        ref.assert_within(o, want, bound)


SIZES = {"one": [1], "tail": [8191, 8192, 8193, 3], "empty among": [0, 5, 0, 70000, 0], "few": [1000 + 37 * i for i in range(14)],
         "most of the short list": [17 + i for i in range(64)], "long list": [1 + i % 9 for i in range(65)],
         "several lists": [1 + i % 40 for i in range(2500)], "large": [20_000_003, 5_000_000], "large in several lists": [8001 - i % 3 for i in range(1100)]}


@pytest.mark.parametrize("sizes", SIZES)
@pytest.mark.parametrize("dtypes", [[torch.float32], [torch.bfloat16], [torch.float16, torch.float32, torch.bfloat16]])
def test_norm_and_clip_match_64_bits(hb, cuda, sizes, dtypes):
    rng = np.random.default_rng(len(sizes))
    grads = _tensors(rng, cuda, SIZES[sizes], dtypes)
    norm = _norm(grads)
    assert abs(float(hb.grad_norm(grads)) - norm) <= NORM * norm
    for limit in (0.37 * norm, 0.0, 3 * norm + 1, math.inf):
        out = [torch.full_like(g, 7.0) for g in grads]
        before = [g.clone() for g in grads]
        got = hb.clip_grad_norm(grads, limit, out=out)
        assert got.shape == () and got.dtype == torch.float32 and abs(float(got) - norm) <= NORM * norm
        assert all(torch.equal(g, b) for g, b in zip(grads, before))
        _check_clipped(out, grads, limit)
        full = [torch.empty_like(g, dtype=torch.float32) for g in grads]
        hb.clip_grad_norm(grads, limit, out=full)
        _check_clipped(full, grads, limit)
        here = [g.clone() for g in grads]
        assert torch.equal(hb.clip_grad_norm(here, limit), got)
        assert all(torch.equal(h, o) for h, o in zip(here, out))


def test_extremes(hb, cuda):
    """Squares beyond and below fp32's range, zeros, infinities and NaN."""
    for value, dtype in ((1e30, torch.float32), (1e-30, torch.float32), (2e38, torch.bfloat16), (1e-35, torch.bfloat16),
                         (6e-8, torch.float16), (6e4, torch.float16)):
        g = [torch.full((5000,), value, dtype=dtype, device=cuda), torch.zeros(100, device=cuda)]
        norm = _norm(g)
        got = float(hb.grad_norm(g))
        assert math.isinf(got) if norm > 3.4e38 else abs(got - norm) <= NORM * norm
    mixed = [torch.full((64,), 1e25, device=cuda), torch.ones(100_000, device=cuda)]
    assert abs(float(hb.grad_norm(mixed)) - _norm(mixed)) <= NORM * _norm(mixed)
    zero = [torch.zeros(77, device=cuda), torch.empty(0, device=cuda)]
    assert float(hb.clip_grad_norm(zero, 1.0)) == 0.0 and not zero[0].any()
    assert float(hb.grad_norm([torch.empty(0, device=cuda)])) == 0.0
    infinite = [torch.ones(10, device=cuda), torch.tensor([math.inf, 1.0], device=cuda)]
    assert math.isinf(float(hb.clip_grad_norm(infinite, 1.0)))
    assert not infinite[0].any() and math.isnan(float(infinite[1][0])) and float(infinite[1][1]) == 0.0
    bad = [torch.ones(10, device=cuda), torch.tensor([math.nan, 1.0], device=cuda)]
    assert math.isnan(float(hb.clip_grad_norm(bad, 1.0))) and bool(torch.isnan(bad[0]).all())


def test_strides_and_addresses(hb, cuda):
    gen = torch.Generator(device=cuda).manual_seed(3)
    base = torch.randn(10_001, generator=gen, device=cuda)
    wide = torch.randn((50, 40), generator=gen, device=cuda)
    grads = [base[1:], wide.t(), torch.randn((3, 4, 5), generator=gen, device=cuda).permute(2, 0, 1), wide.new_ones(())]
    norm = _norm(grads)
    out = [torch.empty_like(g) for g in grads]  # the same strides
    assert abs(float(hb.clip_grad_norm(grads, 1.0, out=out)) - norm) <= NORM * norm
    _check_clipped(out, grads, 1.0)
    copies = [g.clone() for g in grads]
    hb.clip_grad_norm(copies, 1.0)
    _check_clipped(copies, grads, 1.0)
    single = torch.full((9,), 2.0, device=cuda)
    assert float(hb.clip_grad_norm(single, 3.0)) == 6.0 and abs(float(single[0]) - 1.0) < 1e-6


def test_graph_and_stream(hb, cuda):
    gen = torch.Generator(device=cuda).manual_seed(6)
    grads = [torch.randn(n, generator=gen, device=cuda) for n in (3, 50_000, 8192)]
    out = [torch.empty_like(g) for g in grads]
    hb.clip_grad_norm(grads, 0.5, out=out)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        norm = hb.clip_grad_norm(grads, 0.5, out=out)
    for g in grads:
        g.normal_(generator=gen)
    graph.replay()
    torch.cuda.synchronize()
    again = [torch.empty_like(g) for g in grads]
    assert torch.equal(norm, hb.clip_grad_norm(grads, 0.5, out=again))
    assert all(torch.equal(a, b) for a, b in zip(out, again))


def test_clipped_gradients_count_as_changed(hb, cuda):
    g = torch.ones(10, device=cuda)
    before = g._version
    hb.grad_norm([g])
    assert g._version == before
    hb.clip_grad_norm([g], 1.0)
    assert g._version > before


def test_refusals(hb, cuda):
    g = torch.ones((4, 6), device=cuda)
    for call in (lambda: hb.grad_norm([]), lambda: hb.grad_norm([g.double()]), lambda: hb.grad_norm([g.cpu()]),
                 lambda: hb.grad_norm([g[:, ::2]]), lambda: hb.grad_norm([g.expand(3, 4, 6)]), lambda: hb.grad_norm([g, g]),
                 lambda: hb.clip_grad_norm([g], -1.0), lambda: hb.clip_grad_norm([g], math.nan),
                 lambda: hb.clip_grad_norm([g], 1.0, out=[]), lambda: hb.clip_grad_norm([g], 1.0, out=[g[:3]]),
                 lambda: hb.clip_grad_norm([g], 1.0, out=[g.half()]),
                 lambda: hb.clip_grad_norm([g], 1.0, out=[g.t().contiguous().t()]),
                 lambda: hb.clip_grad_norm([g.half(), g.bfloat16()], 1.0, out=[g, g])):
        with pytest.raises(ValueError):
            call()
    assert bool((g == 1).all())
