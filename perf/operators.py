"""Measured cases of the routing, lookup and clipping operators, with their plain forms.

Three groups that a training or serving step runs around the products of its
experts: entries of an assignment sorted by expert, rows dispatched and combined
back with weights (and the gradients); rows of a table looked up by index with a
scale (and the table's gradient); the global norm of many gradients and the
clipped gradients.  ``run`` makes one pass: in elementary torch operations in 32
bits, or with the framework's own calls when ``own`` is true.
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
MOST_ELEMENTS = 1 << 30  # entries x width of the largest case


def listed():
    return [
        # one token of a decode step, two experts: latency
        {"name": "route_token", "kind": "route", "tokens": 1, "slots": 2, "experts": 16, "width": 2048,
         "dtype": "bf16", "dropped": 0.0, "balanced": False},
        # a ragged serving batch whose router leaves some entries without an expert
        {"name": "route_ragged", "kind": "route", "tokens": 1037, "slots": 3, "experts": 37, "width": 1000,
         "dtype": "f16", "dropped": 0.05, "balanced": False},
        # a cloud split evenly over 1024 groups by an exact assignment: one expert per row, equal counts
        {"name": "route_assignment", "kind": "route", "tokens": 262144, "slots": 1, "experts": 1024, "width": 128,
         "dtype": "f32", "dropped": 0.0, "balanced": True},
        # the prompts of a serving batch
        {"name": "route_prompt", "kind": "route", "tokens": 32768, "slots": 4, "experts": 64, "width": 2048,
         "dtype": "bf16", "dropped": 0.0, "balanced": False},
        # gradients of a small layer in 32 bits, odd sizes
        {"name": "route_grad_odd", "kind": "route_grad", "tokens": 4099, "slots": 2, "experts": 8, "width": 257,
         "dtype": "f32", "dropped": 0.02, "balanced": False},
        # gradients of one layer in a training step
        {"name": "route_grad_train", "kind": "route_grad", "tokens": 65536, "slots": 8, "experts": 128,
         "width": 2048, "dtype": "bf16", "dropped": 0.0, "balanced": False},
        # the tokens of a decode step of a few requests: latency
        {"name": "lookup_token", "kind": "lookup", "tokens": 5, "rows": 32768, "width": 2048, "dtype": "bf16"},
        # the tokens of long prompts
        {"name": "lookup_prompt", "kind": "lookup", "tokens": 32768, "rows": 131072, "width": 2048, "dtype": "bf16"},
        # gradient of a small table in 32 bits, odd sizes
        {"name": "lookup_grad_odd", "kind": "lookup_grad", "tokens": 1000, "rows": 5003, "width": 129,
         "dtype": "f32"},
        # gradient of the token table of a training step; a few rows take much of the batch
        {"name": "lookup_grad_train", "kind": "lookup_grad", "tokens": 131072, "rows": 65536, "width": 2048,
         "dtype": "bf16"},
        # gradients of a small model: matrices with odd sides and vectors
        {"name": "clip_small", "kind": "clip", "tensors": 14, "elements": 200_003, "dtype": "f32", "limit": 1.0},
        # gradients of a large model
        {"name": "clip_train", "kind": "clip", "tensors": 60, "elements": 800_000_000, "dtype": "bf16",
         "limit": 1.0},
    ]


def _log(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    kind = rng.choice(["route", "route", "route_grad", "route_grad", "lookup", "lookup_grad", "lookup_grad", "clip"])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    if kind in ("route", "route_grad"):
        width = _log(rng, 16, 2048)
        if rng.random() < 0.5:
            width = max(16, width // 8 * 8)
        slots = rng.randint(1, 8)
        tokens = _log(rng, 1 if kind == "route" else 16, 65536)
        tokens = min(tokens, MOST_ELEMENTS // (2 * slots * width))
        experts = _log(rng, max(2, slots), 1024)
        dropped = rng.choice([0.0, 0.0, 0.1 * rng.random()])
        return {"kind": kind, "tokens": tokens, "slots": slots, "experts": experts, "width": width, "dtype": dtype,
                "dropped": dropped, "balanced": slots == 1 and rng.random() < 0.5}
    if kind in ("lookup", "lookup_grad"):
        width = _log(rng, 16, 2048)
        if rng.random() < 0.5:
            width = max(16, width // 8 * 8)
        return {"kind": kind, "tokens": _log(rng, 1 if kind == "lookup" else 16, 131072),
                "rows": _log(rng, 16, 131072), "width": width, "dtype": dtype}
    return {"kind": kind, "tensors": rng.randint(1, 60), "elements": _log(rng, 1000, 400_000_000), "dtype": dtype,
            "limit": rng.choice([0.5, 1.0, 1e9])}


def _sizes(case):
    """Element counts of a clip case's tensors: a few large ones, many small ones, odd counts among them."""
    n, total = case["tensors"], case["elements"]
    shares = [1.0 / (1 + i % 5) ** 2 for i in range(n)]
    return [max(1, int(total * s / sum(shares)) - i % 3) for i, s in enumerate(shares)]


def _index(case, gen):
    """An assignment [tokens, slots]: distinct experts a token by skewed scores, or equal counts; -1 where an
    entry has no expert."""
    t, k, e = case["tokens"], case["slots"], case["experts"]
    if case["balanced"]:
        index = (torch.randperm(t, generator=gen, device="cuda") % e).view(t, 1)
        score = torch.ones((t, 1), device="cuda")
    else:
        lean = torch.randn(e, generator=gen, device="cuda") * 0.5
        score, index = (torch.randn((t, e), generator=gen, device="cuda") + lean).topk(k, dim=1)
    weights = torch.softmax(score, dim=1)
    if case["dropped"]:
        gone = torch.rand((t, k), generator=gen, device="cuda") < case["dropped"]
        index = torch.where(gone, torch.full_like(index, -1), index)
    return index, weights


def _plan(index, experts):
    """(order, position, offsets) of an assignment, entries without an expert last."""
    flat = index.reshape(-1)
    key = torch.where((flat >= 0) & (flat < experts), flat, torch.full_like(flat, experts))
    key, order = torch.sort(key, stable=True)
    position = torch.empty_like(order)
    position[order] = torch.arange(order.numel(), device=order.device)
    offsets = torch.searchsorted(key, torch.arange(experts + 1, device=key.device))
    return order.to(torch.int32), position.view(index.shape).to(torch.int32), offsets.to(torch.int32)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    kind, dtype = case["kind"], DTYPES[case["dtype"]]

    def normal(*shape):
        return torch.randn(shape, generator=gen, device="cuda", dtype=dtype)

    state = {"kind": kind}
    if kind in ("route", "route_grad"):
        t, k, d = case["tokens"], case["slots"], case["width"]
        state["experts"] = case["experts"]
        state["index"], state["weights"] = _index(case, gen)
        state["z"] = normal(t * k, d)  # the experts' outputs, in sorted order
        if kind == "route":
            state["x"] = normal(t, d)
        else:
            state["dy"], state["dsorted"] = normal(t, d), normal(t * k, d)
            state["plan"] = _plan(state["index"], case["experts"])
    elif kind in ("lookup", "lookup_grad"):
        n, v, d = case["tokens"], case["rows"], case["width"]
        # a row's chance goes as 1 / (its rank + 3): a few rows are very frequent
        u = torch.rand(n, generator=gen, device="cuda", dtype=torch.float64)
        ids = (3.0 * (1.0 + v / 3.0) ** u - 3.0).long().clamp_(0, v - 1)
        state["ids"] = torch.randperm(v, generator=gen, device="cuda")[ids]
        state["rows"], state["scale"] = v, math.sqrt(d)
        if kind == "lookup":
            state["table"] = normal(v, d)
        else:
            state["dy"] = normal(n, d)
    else:
        state["limit"] = case["limit"]
        state["grads"] = [normal(n).mul_(0.02) for n in _sizes(case)]
        state["out"] = [torch.empty_like(g) for g in state["grads"]]
    return state


def _run_own(s):
    import __graft_entry__ as entry
    hb = entry.load_package()
    kind = s["kind"]
    if kind == "route":
        plan = hb.route_plan(s["index"], s["experts"])
        return {"order": plan.order, "position": plan.position, "offsets": plan.offsets,
                "sorted": hb.route_dispatch(s["x"], plan), "combined": hb.route_combine(s["z"], plan, s["weights"])}
    if kind == "route_grad":
        plan = hb.RoutePlan(*s["plan"])
        dz, dw = hb.route_combine_grad(s["dy"], s["z"], plan, s["weights"])
        return {"dz": dz, "dw": dw, "dx": hb.route_dispatch_grad(s["dsorted"], plan)}
    if kind == "lookup":
        return {"y": hb.embedding_lookup(s["table"], s["ids"], scale=s["scale"])}
    if kind == "lookup_grad":
        return {"dtable": hb.embedding_grad(s["dy"], s["ids"], s["rows"], scale=s["scale"])}
    return {"norm": hb.clip_grad_norm(s["grads"], s["limit"], out=s["out"]), "clipped": s["out"]}


def _combine(z, position, kept, weights):
    """sum_k weights[t, k] z[position[t, k]] over the entries that have an expert, in 32 bits."""
    rows = z.float()[position.reshape(-1).long()].view(*position.shape, z.shape[1])
    there = (position < kept).unsqueeze(-1)
    if weights is not None:
        rows = rows * weights.float().unsqueeze(-1)
    return torch.where(there, rows, torch.zeros((), device=z.device)).sum(1)


def run(state):
    if own:
        return _run_own(state)
    s, kind = state, state["kind"]
    if kind == "route":
        order, position, offsets = _plan(s["index"], s["experts"])
        kept, slots = offsets[-1], s["index"].shape[1]
        there = (torch.arange(order.numel(), device=order.device) < kept).unsqueeze(-1)
        rows = torch.where(there, s["x"].float()[(order // slots).long()], torch.zeros((), device=order.device))
        return {"order": order, "position": position, "offsets": offsets, "sorted": rows.to(s["x"].dtype),
                "combined": _combine(s["z"], position, kept, s["weights"]).to(s["z"].dtype)}
    if kind == "route_grad":
        order, position, offsets = s["plan"]
        kept, slots = offsets[-1], position.shape[1]
        there = torch.arange(order.numel(), device=order.device) < kept
        zero = torch.zeros((), device=order.device)
        dy = s["dy"].float()[(order // slots).long()]
        dz = torch.where(there.unsqueeze(-1), dy * s["weights"].float().reshape(-1)[order.long()].unsqueeze(-1), zero)
        dot = torch.where(there, (dy * s["z"].float()).sum(1), zero)
        return {"dz": dz.to(s["z"].dtype), "dw": dot[position.long()].to(s["weights"].dtype),
                "dx": _combine(s["dsorted"], position, kept, None).to(s["dsorted"].dtype)}
    if kind == "lookup":
        return {"y": (s["table"][s["ids"]].float() * s["scale"]).to(s["table"].dtype)}
    if kind == "lookup_grad":
        total = torch.zeros((s["rows"], s["dy"].shape[1]), device=s["dy"].device)
        return {"dtable": (total.index_add_(0, s["ids"], s["dy"].float()) * s["scale"]).to(s["dy"].dtype)}
    norm = torch.stack([g.float().square().sum() for g in s["grads"]]).sum().sqrt()
    factor = (s["limit"] / (norm + 1e-6)).clamp(max=1.0)
    return {"norm": norm, "clipped": [(g.float() * factor).to(g.dtype) for g in s["grads"]]}


def exact(case, seed):
    s, kind = prepare(case, seed), case["kind"]
    if kind in ("route", "route_grad"):
        # entry by entry: where it goes, counted from the assignment itself
        flat = s["index"].reshape(-1)
        n, k, e = flat.numel(), case["slots"], case["experts"]
        entry = torch.arange(n, device="cuda")
        valid = (flat >= 0) & (flat < e)
        order = torch.argsort(torch.where(valid, flat, e) * n + entry)  # keys are all different
        live = order[:int(valid.sum())]
        token, w = live // k, s["weights"].double().reshape(-1)[live].unsqueeze(-1)
        z = s["z"][:live.numel()].double()

        def back(rows):
            return torch.zeros((case["tokens"], rows.shape[1]), dtype=torch.float64, device="cuda").index_add_(0, token, rows)

        if kind == "route":
            rows = torch.zeros((n, case["width"]), dtype=torch.float64, device="cuda")
            rows[:live.numel()] = s["x"].double()[token]
            return {"order": None, "position": None, "offsets": None, "sorted": rows, "combined": back(w * z)}
        dy = s["dy"].double()[token]
        dw = torch.zeros(n, dtype=torch.float64, device="cuda")
        dw[live] = torch.einsum("nd,nd->n", dy, z)
        del z
        dz = torch.zeros((n, case["width"]), dtype=torch.float64, device="cuda")
        torch.mul(dy, w, out=dz[:live.numel()])
        del dy
        return {"dz": dz, "dw": dw.view(s["weights"].shape), "dx": back(s["dsorted"][:live.numel()].double())}
    if kind == "lookup":
        return {"y": s["table"].double().index_select(0, s["ids"]) * s["scale"]}
    if kind == "lookup_grad":
        total = torch.zeros((s["rows"], case["width"]), dtype=torch.float64, device="cuda")
        return {"dtable": total.index_put_((s["ids"],), s["dy"].double() * s["scale"], accumulate=True)}
    norm = math.sqrt(math.fsum(float(g.double().pow(2).sum()) for g in s["grads"]))
    factor = min(1.0, case["limit"] / (norm + 1e-6))
    return {"norm": torch.tensor(norm, dtype=torch.float64), "clipped": [g.double() * factor for g in s["grads"]]}


def work(case):
    size = DTYPES[case["dtype"]].itemsize
    kind = case["kind"]
    if kind in ("route", "route_grad"):
        t, k, e, d = case["tokens"], case["slots"], case["experts"], case["width"]
        live = t * k * (1.0 - case["dropped"])
        if kind == "route":  # ids and x in, plan and sorted rows out; experts' rows and weights in, tokens out
            return {"bytes": t * k * (8 + 4 + 4 + 4) + (e + 1) * 4 + (t + t * k + live + t) * d * size,
                    "flops": 2 * live * d}
        return {"bytes": t * k * (4 + 4 + 4) + (t + live + t * k + live + t) * d * size, "flops": 4 * live * d}
    if kind == "lookup":  # each row that is named, once
        n, d = case["tokens"], case["width"]
        rank = torch.arange(case["rows"], dtype=torch.float64)
        chance = torch.log1p(1.0 / (rank + 3.0)) / math.log1p(case["rows"] / 3.0)
        named = float((1.0 - (1.0 - chance) ** n).sum())
        return {"bytes": n * 8 + (n + named) * d * size, "flops": n * d}
    if kind == "lookup_grad":
        n, v, d = case["tokens"], case["rows"], case["width"]
        return {"bytes": n * 8 + (n + v) * d * size, "flops": n * d}
    n = sum(_sizes(case))
    return {"bytes": 2 * n * size, "flops": 3 * n}
