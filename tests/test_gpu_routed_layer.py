"""The operators together, as examples/routed_layer.py runs them: an exact transport plan as the router of a
trained layer."""
import importlib.util
from pathlib import Path

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
EXAMPLE = Path(__file__).resolve().parents[1] / "examples" / "routed_layer.py"


@pytest.fixture(scope="module")
def example():
    spec = importlib.util.spec_from_file_location("routed_layer", EXAMPLE)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


def test_training_steps(example, cuda):
    history = example.train(steps=6, tokens=256, experts=4, width=32, rows=60)
    losses = [h[0] for h in history]
    assert losses[-1] < losses[0]
    for loss, norm, counts in history:
        assert np.isfinite(loss) and norm > 0
        # masses are equal: an expert has 64 tokens, plus those it shares (a vertex plan shares at most 3 tokens)
        assert all(48 <= c <= 80 for c in counts)


def test_layer_gradients_match_64_bits(example, hb, cuda):
    """Gradients of the whole layer against the same layer written in 64-bit torch operations and its autograd.
    Tolerance: every value passes fewer than 8 sums of at most 64 terms in fp32, so 8 * 64 * 2^-24 of the
    largest gradient."""
    gen = torch.Generator(device=cuda).manual_seed(3)
    tokens, experts, width, rows = 96, 4, 24, 30
    table = torch.randn((rows, width), generator=gen, device=cuda).requires_grad_()
    weight = (torch.randn((experts, width, width), generator=gen, device=cuda) / width ** 0.5).requires_grad_()
    centres = torch.randn((experts, width), generator=gen, device=cuda)
    target = torch.randn((tokens, width), generator=gen, device=cuda)
    ids = torch.randint(0, rows, (tokens,), generator=gen, device=cuda)
    x = hb.embedding_lookup(table, ids, scale=1.5)
    index, weights = example.balanced_assignment(hb, x, centres)
    weights = weights.requires_grad_()
    plan = hb.route_plan(index, experts)
    y = hb.route_combine(example.experts_forward(hb.route_dispatch(x, plan), weight, plan.offsets), plan, weights)
    torch.backends.cuda.matmul.allow_tf32 = False
    (y - target).square().mean().backward()

    t64, w64, r64 = (v.detach().double().requires_grad_() for v in (table, weight, weights))
    x64 = t64[ids] * 1.5
    y64 = torch.zeros((tokens, width), dtype=torch.float64, device=cuda)
    for k in range(index.shape[1]):
        live = (index[:, k] >= 0).nonzero().view(-1)
        z = torch.einsum("td,ted->te", x64[live], w64[index[live, k].long()])
        y64 = y64.index_add(0, live, r64[live, k].unsqueeze(1) * z)
    (y64 - target.double()).square().mean().backward()
    for got, want in ((table.grad, t64.grad), (weight.grad, w64.grad), (weights.grad, r64.grad)):
        assert float((got.double() - want).abs().max()) <= 8 * 64 * 2.0 ** -24 * float(want.abs().max())
