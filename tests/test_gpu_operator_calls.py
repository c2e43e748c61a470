"""What the routing, lookup and clipping calls keep to beside their results on ordinary arguments."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def _plan(hb, cuda, gen, tokens=40, slots=2, experts=5):
    return hb.route_plan(torch.randint(-1, experts, (tokens, slots), generator=gen, device=cuda), experts)


def test_plan_changed_before_backward(hb, cuda):
    """A plan is part of what the gradients need: written to in between, they are refused as for any saved tensor."""
    gen = torch.Generator(device=cuda).manual_seed(1)
    plan = _plan(hb, cuda, gen)
    for call in (lambda: hb.route_dispatch(torch.randn((40, 8), generator=gen, device=cuda).requires_grad_(), plan),
                 lambda: hb.route_combine(torch.randn((80, 8), generator=gen, device=cuda).requires_grad_(), plan)):
        y = call()
        y.sum().backward()
        for part in (plan.position, plan.offsets):
            y = call()
            part.add_(0)
            with pytest.raises(RuntimeError, match="modified by an inplace operation"):
                y.sum().backward()
