"""A pre-norm block of gated experts, trained in 16 bits: the whole step between a table and a loss.

    python examples/routed_block.py [--steps 8] [--tokens 512] [--experts 8] [--width 64] [--hidden 128]

Each step looks the tokens up, normalises them, routes them by the exact balanced
transport to the experts' centres, runs each expert's gated feed-forward and the
product back to the tokens' width, and adds the weighted result to the residual
stream under the second norm.  The backward pass runs the operators' gradients; one
AdamW step updates all parameters, clipped by the gradients' global norm on the way.
"""
from __future__ import annotations

import argparse
import sys
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parents[1]))
sys.path.insert(0, str(Path(__file__).resolve().parent))
import __graft_entry__ as entry  # noqa: E402
from routed_layer import balanced_assignment  # noqa: E402

NAMES = ("table", "gain_in", "gate", "up", "down", "gain_out")


def parameters(rows, experts, width, hidden, dtype=torch.bfloat16, seed=0, device="cuda"):
    """The block's parameters by name."""
    gen = torch.Generator(device=device).manual_seed(seed)

    def normal(*shape, scale):
        return (torch.randn(shape, generator=gen, device=device) * scale).to(dtype).requires_grad_()

    ones = [torch.ones(width, dtype=dtype, device=device).requires_grad_() for _ in range(2)]
    return dict(zip(NAMES, (normal(rows, width, scale=1.0), ones[0], normal(experts, hidden, width, scale=width ** -0.5),
                            normal(experts, hidden, width, scale=width ** -0.5), normal(experts, width, hidden, scale=hidden ** -0.5), ones[1])))


def block(hb, p, ids, plan, weights):
    """The block's output: normalised stream of x + experts(norm(x))."""
    x = hb.embedding_lookup(p["table"], ids)
    rows = hb.route_dispatch(hb.rms_norm(x, p["gain_in"]), plan)
    h = hb.expert_gated(rows, p["gate"], p["up"], plan.offsets)
    delta = hb.route_combine(hb.expert_product(h, p["down"], plan.offsets), plan, weights)
    return hb.rms_norm(delta, p["gain_out"], x)[0]


def step(hb, p, state, ids, centres, target, rate, limit):
    """One training step; returns (loss, gradient norm)."""
    with torch.no_grad():
        x = hb.embedding_lookup(p["table"], ids)
        index, weights = balanced_assignment(hb, hb.rms_norm(x, p["gain_in"]), centres)
        plan = hb.route_plan(index, centres.shape[0])
    loss = (block(hb, p, ids, plan, weights).float() - target).square().mean()
    loss.backward()
    params, grads = list(p.values()), [v.grad for v in p.values()]
    norm = hb.grad_norm(grads)
    hb.adamw_step(params, grads, state, lr=rate, weight_decay=0.01, norm=norm, max_norm=limit)
    for v in params:
        v.grad = None
    return loss.item(), norm.item()


def train(steps=8, tokens=512, experts=8, width=64, hidden=128, rows=200, dtype=torch.bfloat16, bits=8, rate=1e-2, limit=1.0, seed=0,
          device="cuda"):
    """Runs the steps on synthetic tokens; returns their (loss, norm)."""
    hb = entry.load_package()
    gen = torch.Generator(device=device).manual_seed(seed + 1)
    p = parameters(rows, experts, width, hidden, dtype, seed, device)
    state = hb.adamw_state(p.values(), bits=bits, master=True)
    centres = torch.randn((experts, width), generator=gen, device=device)
    target = torch.randn((rows, width), generator=gen, device=device)
    ids = torch.randint(0, rows, (tokens,), generator=gen, device=device)
    return [step(hb, p, state, ids, centres, target[ids], rate, limit) for _ in range(steps)]


if __name__ == "__main__":
    parser = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    for name, value in (("steps", 8), ("tokens", 512), ("experts", 8), ("width", 64), ("hidden", 128)):
        parser.add_argument("--" + name, type=int, default=value)
    for i, (loss, norm) in enumerate(train(**vars(parser.parse_args()))):
        print(f"step {i}: loss {loss:.5f}, gradient norm {norm:.4f}")
