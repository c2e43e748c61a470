"""A layer of experts fed by exact balanced transport: every operator of a routed training step together.

    python examples/routed_layer.py [--steps 8] [--tokens 512] [--experts 8] [--width 64]

Each step looks the tokens' features up in a table, solves the transport of the
tokens (mass 1/T each) to the experts' centres (mass 1/E each) exactly, and reads the
plan as an assignment: nearly every token goes to one expert and every expert gets its
share of the mass.  The rows are dispatched by expert, go through each expert's
product, and come back weighted.  The backward pass runs the operators' gradients down
to the table, the global norm of all gradients is clipped, and a plain gradient step
follows.
"""
from __future__ import annotations

import argparse
import sys
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parents[1]))
import __graft_entry__ as entry  # noqa: E402


def balanced_assignment(hb, x, centres, tolerance=1e-6):
    """(index, weights) of the exact transport from the rows of x to the centres, equal masses on both sides."""
    x, centres = x.detach().float().contiguous(), centres.detach().float().contiguous()
    tokens, experts = x.shape[0], centres.shape[0]
    cost = hb.leaf_cost_matrix(x, centres, "l2^2", source_offset=x.double().square().sum(1),
                               target_offset=centres.double().square().sum(1))
    mass = torch.full((tokens,), 1.0 / tokens, dtype=torch.float64, device=x.device)
    share = torch.full((experts,), 1.0 / experts, dtype=torch.float64, device=x.device)
    leaf = hb.solve_leaf_resident(cost / cost.max(), mass, share, tolerance=tolerance)
    # edges of less than a thousandth of a token's mass are the solver's tolerance, not the plan
    return hb.assignment_of_plan(leaf.keys // experts, leaf.keys % experts, leaf.values, tokens,
                                 tolerance=1e-3 / tokens)


def experts_forward(rows, weight, offsets):
    """Each expert's product on its sorted rows; rows without an expert stay zero."""
    ends = offsets.tolist()  # waits for the device: here the experts' rows are sizes of plain products
    out = [rows[a:b] @ w.t() for a, b, w in zip(ends, ends[1:], weight)]
    return torch.cat([*out, rows[ends[-1]:]])


def step(hb, table, ids, weight, centres, target, limit, rate):
    """One training step; returns (loss, gradient norm, tokens of each expert)."""
    x = hb.embedding_lookup(table, ids, scale=float(table.shape[1]) ** 0.5)
    index, weights = balanced_assignment(hb, x, centres)
    plan = hb.route_plan(index, weight.shape[0])
    z = experts_forward(hb.route_dispatch(x, plan), weight, plan.offsets)
    y = hb.route_combine(z, plan, weights)
    loss = (y - target).square().mean()
    loss.backward()
    norm = hb.clip_grad_norm([table.grad, weight.grad], limit)
    with torch.no_grad():
        for p in (table, weight):
            p -= rate * p.grad
            p.grad = None
    return loss.item(), norm.item(), plan.counts.tolist()


def train(steps=8, tokens=512, experts=8, width=64, rows=200, seed=0, limit=0.5, rate=0.5, device="cuda"):
    """Runs the steps on synthetic tokens; returns their (loss, norm, counts)."""
    hb = entry.load_package()
    gen = torch.Generator(device=device).manual_seed(seed)

    def normal(*shape):
        return torch.randn(shape, generator=gen, device=device)

    table = (normal(rows, width) / width ** 0.5).requires_grad_()
    weight = (normal(experts, width, width) / width ** 0.5).requires_grad_()
    centres, target = normal(experts, width), normal(rows, width)
    ids = torch.randint(0, rows, (tokens,), generator=gen, device=device)
    return [step(hb, table, ids, weight, centres, target[ids], limit, rate) for _ in range(steps)]


if __name__ == "__main__":
    parser = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    for name, value in (("steps", 8), ("tokens", 512), ("experts", 8), ("width", 64)):
        parser.add_argument("--" + name, type=int, default=value)
    for i, (loss, norm, counts) in enumerate(train(**vars(parser.parse_args()))):
        print(f"step {i}: loss {loss:.5f}, gradient norm {norm:.4f}, tokens by expert {counts}")
